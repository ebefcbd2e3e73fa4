"""me_sample_minp where a search's border lies among the entries that cannot be picked, and at the ends of the number range: against the
same 64-bit rules as test_sample_minp_gpu.py."""
import math

import pytest
import torch

from test_sample_minp_gpu import compare, reference, sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [3000, 8192, 32000, 40000])
@pytest.mark.parametrize("masked", [-math.inf, torch.finfo(torch.float32).min])
def test_top_k_ends_among_masked_entries(V, masked):
    """more of top_k than there are entries to pick from: the last bin (32 temperatures below the maximum) holds positive logits next to masked ones,
    so its entries' images span the whole 64-bit range"""
    g = torch.Generator().manual_seed(V)
    temp = torch.tensor([0.1, 0.2, 0.3, 0.1, 0.2, 0.3, 0.15])
    last = torch.tensor([1.5, 1.5, 1.5, 6.0, 6.0, 6.0, 24.0])     # where the last bin begins, about
    x = torch.randn(len(temp), V, generator=g) * 2.5
    x = torch.minimum(x, torch.tensor(8.0))
    x += (last + 32 * temp - x.amax(1))[:, None]
    n = max(300, V // 30)
    for b in range(len(temp)):
        x[b, torch.randperm(V, generator=g)[:n]] = masked
    special = [0, 1, 2]
    for top_k in (V - n + 1, V - 1, V - len(special) + 1, V - n // 2):
        for top_p, min_p in ((0.7, 0.0), (0.98, 0.0), (1.0, 0.0), (0.9, 0.05)):
            compare(x, special, temp, top_k, top_p, min_p, torch.rand(len(temp), generator=g))


@pytest.mark.parametrize("V", [40, 5000, 40000])
def test_logits_of_the_whole_range_at_the_largest_temperatures(V):
    """a bin's upper border in logits, lo / 32 times the temperature, does not fit 32 bits; differences of logits do not either"""
    x = torch.linspace(-3e38, 3e38, V, dtype=torch.float64).float().flip(0).repeat(4, 1)
    x[1] = x[1].roll(V // 3)
    x[2, V // 2:] = torch.finfo(torch.float32).min
    x[3, ::3] = -math.inf
    top = torch.finfo(torch.float32).max
    u = torch.tensor([0.99, 0.7, 0.9999, 0.5])
    for temp in (torch.tensor([top, 3e38, 1e38, top]), torch.full((4,), 2e37)):
        for top_k, top_p, min_p in ((0, 1.0, 0.0), (V - V // 8, 1.0, 0.0), (V - 1, 0.98, 0.1), (0, 0.9, 0.0)):
            compare(x, [], temp, top_k, top_p, min_p, u)


@pytest.mark.parametrize("V", [40, 5000, 40000])
def test_weights_that_are_one_in_64_bits_pass_a_min_p_of_one(V):
    """logits that differ by less than 2^-54 temperatures: exp() of 64 bits is 1, and 1 >= 1 keeps them all"""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(4, V, generator=g)
    x[0] *= 1e-38
    x[1] *= 1e-20
    x[2, V // 2] = -math.inf
    temp = torch.tensor([1.0, 0.5, math.inf, 1e30])
    u = torch.tensor([0.1, 0.4, 0.6, 0.9])
    for top_k, top_p in ((0, 1.0), (V // 2, 1.0), (0, 0.9), (V - 1, 0.5)):
        ids, n = sample(x, [], temp, top_k, top_p, 1.0, u)
        for b in range(4):                                       # an infinite temperature counts as the largest number (-inf / inf is none)
            want, (lo, hi) = reference(x[b].numpy(), [], temp[b].clamp(max=torch.finfo(torch.float32).max), top_k, top_p, 1.0, u[b])
            assert ids[b] in want and lo <= n[b] <= hi, (b, ids[b], want, n[b], (lo, hi))
