"""me_sample_minp / me_sample_minp_step on the GPU against the rules in 64 bits: picks and numbers of choices are whole numbers and have to be
equal, unless the 64-bit value lies nearer to a border than the kernel's weight unit can tell."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, special, temp, top_k, top_p, min_p, u):
    """one row: (set of ids that may be picked, (fewest, most) choices)"""
    x = x.astype(np.float64).copy()
    x[np.isnan(x)] = 0.0
    x[[s for s in special if 0 <= s < len(x)]] = -np.inf
    order = np.argsort(-x, kind="stable")
    y = x[order]
    if y[0] == -np.inf:
        return {0}, (0, 0)
    with np.errstate(invalid="ignore"):
        d = np.where(y == y[0], 0.0, y - y[0])
    w = np.exp(d / float(np.float32(temp)))
    # weights rounded to 2^-45 in the kernel, 64-bit rounding here: what a cumulative weight may be off
    eps = len(w) * 2.0 ** -45 + np.cumsum(w)[-1] * 2.0 ** -48
    n0 = len(w) if top_k <= 0 else min(top_k, len(w))
    lo = hi = n0
    if 0 < top_p < 1:
        cum, limit = np.cumsum(w[:n0]), float(np.float32(top_p)) * w[:n0].sum()
        lo = max(1, int(np.searchsorted(cum, limit - eps, side="right")))
        hi = max(1, int(np.searchsorted(cum, limit + eps, side="right")))
    m = int(np.count_nonzero((w >= float(np.float32(min_p))) & (w > 0)))
    ids = set()
    for n in {min(lo, m), min(hi, m)}:
        cum = np.cumsum(w[:n])
        t = float(np.float32(u)) * cum[-1]
        last = int(np.count_nonzero(w[:n] > 2.0 ** -46)) - 1
        a, b = (min(int(np.searchsorted(cum, t + e, side="right")), last) for e in (-eps, eps))
        ids |= set(order[a:b + 1].tolist())
    return ids, (min(lo, m), min(hi, m))


def sample(x, special, temp, top_k, top_p, min_p, u, ld=0):
    from midiemo import ops
    B, V = x.shape
    buf = torch.full((B, max(ld, V)), 77.0, device="cuda")
    buf[:, :V] = x.cuda()
    ids = torch.full((B,), -5, dtype=torch.int64, device="cuda")
    n = torch.full((B,), -5, dtype=torch.int32, device="cuda")
    sp = torch.tensor(special, dtype=torch.int32, device="cuda") if special else None
    ops.sample_minp(buf, V, sp, temp.cuda(), top_k, top_p, min_p, u.cuda(), ids, n)
    return ids.cpu().tolist(), n.cpu().tolist()


def compare(x, special, temp, top_k, top_p, min_p, u, ld=0):
    ids, n = sample(x, special, temp, top_k, top_p, min_p, u, ld)
    sharp = 0
    for b in range(x.shape[0]):
        want, (lo, hi) = reference(x[b].numpy(), special, temp[b], top_k, top_p, min_p, u[b])
        assert ids[b] in want and lo <= n[b] <= hi, (b, ids[b], want, n[b], (lo, hi))
        sharp += len(want) == 1 and lo == hi
    return sharp


RULES = [(0, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (50, 1.0, 0.0), (1, 0.9, 0.1), (7, 0.6, 0.02), (200, 0.95, 0.3), (0, 0.0001, 0.0), (0, 0.999, 0.0001)]


@pytest.mark.parametrize("V", [1, 2, 5, 64, 257, 1007, 1025, 4096, 4097, 20000, 32512, 32513, 65537, 131071, 262144])
@pytest.mark.parametrize("kind", ["smooth", "16bit", "peaked"])
def test_picks_follow_the_rules(V, kind):
    B = 6 if V <= 65537 else 3
    g = torch.Generator().manual_seed(V + len(kind))
    x = torch.randn(B, V, generator=g) * (20.0 if kind == "peaked" else 2.5)
    if kind == "16bit":
        x = x.bfloat16().float()
    temp = 0.3 + 2 * torch.rand(B, generator=g)
    special = [] if V < 5 else [0, 3, V - 1, V + 9, -4]
    sharp = total = 0
    for top_k, top_p, min_p in RULES:
        u = torch.rand(B, generator=g)
        u[0] = 0.0
        u[1 % B] = 1.0 - 2.0 ** -24
        sharp += compare(x, special, temp, top_k, top_p, min_p, u, ld=V + 3)
        total += B
    assert sharp >= total - 1                                   # the borders hardly ever leave a choice open


def test_every_rank_is_reached():
    """the inverse of the whole distribution: u in the middle of every entry's interval picks that entry, ties by index"""
    V = 300
    x = torch.zeros(V)
    x[::3] = 1.0
    w = torch.exp(x.double())
    order = sorted(range(V), key=lambda j: (-float(x[j]), j))
    cum = torch.cumsum(w[order], 0)
    u = ((cum - w[order] / 2) / cum[-1]).float()
    ids, n = sample(x.expand(V, V), [], torch.ones(V), 0, 1.0, 0.0, u)
    assert ids == order and n == [V] * V


@pytest.mark.parametrize("V", [9, 3000, 30000, 262144])
def test_equal_logits_and_wide_ties(V):
    """one bin holds the whole row: the search has to go down to the index"""
    x = torch.full((4, V), -2.5)
    x[2, ::2] = -2.5 + 1e-6
    x[3] = 0.0
    x[3, 1::2] = -0.0
    u = torch.tensor([0.0, 0.123456, 0.5, 0.999999])
    for top_k, top_p, min_p in [(0, 1.0, 0.0), (max(1, V // 3), 1.0, 0.0), (0, 0.37, 0.0), (max(1, V // 3), 0.61, 1.0)]:
        compare(x, [], torch.tensor([1.0, 50.0, 0.7, 1e-3]), top_k, top_p, min_p, u)


@pytest.mark.parametrize("V", [40, 5000, 40000])
def test_rows_with_values_that_are_not_numbers(V):
    low = torch.finfo(torch.float32).min
    x = torch.randn(8, V, generator=torch.Generator().manual_seed(1))
    x[0] = -math.inf                                            # nothing to choose from
    x[1] = math.nan                                             # NaN counts as 0: all alike
    x[2, 5:9] = math.inf                                        # they share the weight
    x[3] = low                                                  # masked by the lowest value, one entry left
    x[3, 7] = 1.0
    x[4] = low                                                  # masked everywhere
    x[5, ::2] = -math.inf
    x[6, 1::2] = math.nan
    x[7] = torch.linspace(-3e38, 3e38, V)
    u = torch.tensor([0.4, 0.7, 0.6, 0.5, 0.99, 0.2, 0.8, 0.3])
    for rules in [(0, 1.0, 0.0), (0, 0.9, 0.1), (3, 0.8, 0.0), (2, 1.0, 1.0)]:
        compare(x, [1, 2], torch.full((8,), 0.9), *rules, u)
    ids, n = sample(x, list(range(V)), torch.ones(8), 0, 0.9, 0.1, u)            # every id barred
    assert ids == [0] * 8 and n == [0] * 8


def test_uniforms_at_and_beyond_their_ends():
    x = torch.tensor([[0.0, 1.0, -math.inf, 0.5]]).expand(5, -1)
    ids, n = sample(x, [], torch.ones(5), 0, 1.0, 0.0, torch.tensor([-0.5, 0.0, 1.0, 2.0, math.nan]))
    assert ids == [1, 1, 0, 0, 1] and n == [3] * 5


@pytest.mark.parametrize("V", [12, 3000, 9000, 40000])
def test_temperatures_at_and_beyond_their_ends(V):
    """what is not positive counts as 0 (one of the largest, by u), an infinite one makes all entries alike"""
    x = torch.randn(8, V, generator=torch.Generator().manual_seed(5))
    x[:, 7] = x[:, 3] = 9.0
    x[:, 5] = -math.inf
    temp = torch.tensor([0.0, -1.0, math.nan, -math.inf, 1e-42, 1e-30, math.inf, 3e38])
    u = torch.tensor([0.2, 0.7, 0.4, 0.9, 0.6, 0.3, 0.0, 0.5])
    for rules in [(0, 1.0, 0.0), (0, 0.9, 0.1), (50, 1.0, 0.0), (3, 0.9, 0.5)]:
        ids, n = sample(x, [], temp, *rules, u)
        if rules[1] == 1.0:
            assert ids[:6] == [3, 7, 3, 7, 7, 3] and n[:6] == [2] * 6
        else:                                                    # the nucleus drops the second: half and half passes 0.9
            assert ids[:6] == [3] * 6 and n[:6] == [1] * 6
        kept = min(V - 1, rules[0] or V)
        order = sorted(range(V), key=lambda j: (-float(x[6, j]), j))
        if rules[1] == 1.0:
            assert ids[6] == order[0] and n[6:] == [kept] * 2
            order = sorted(range(V), key=lambda j: (-float(x[7, j]), j))
            assert ids[7] == order[int(0.5 * kept)]


def test_frequencies_follow_the_weights():
    V, B = 12, 4096
    x = torch.randn(V, generator=torch.Generator().manual_seed(4))
    u = (torch.arange(B, dtype=torch.float64) + 0.5).div(B).float()              # a stratified sample: counts are off by at most one each
    ids, _ = sample(x.expand(B, V), [], torch.full((B,), 0.8), 0, 1.0, 0.05, u)
    p = torch.softmax(x.double() / float(np.float32(0.8)), 0)
    p = torch.where(p >= 0.05 * p.max(), p, 0.0)
    p = p / p.sum()
    count = torch.bincount(torch.tensor(ids), minlength=V).double()
    assert bool(((count - p * B).abs() <= 1.01).all())


def test_agrees_with_the_narrow_kernel():
    """without min-p the rules are those of me_sample_topk_topp (f32): the same picks wherever u lies away from a border"""
    from midiemo import ops
    V, B = 1018, 64
    g = torch.Generator().manual_seed(9)
    x, u, temp = torch.randn(B, V, generator=g) * 3, torch.rand(B, generator=g), 0.5 + torch.rand(B, generator=g)
    for top_k, top_p in [(0, 0.7), (20, 0.95), (0, 1.0)]:
        a, na = torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
        ops.sample_topk_topp(x.cuda(), V, None, temp.cuda(), top_k, top_p, u.cuda(), a, na)
        b, nb = sample(x, [], temp, top_k, top_p, 0.0, u)
        assert sum(p == q for p, q in zip(a.tolist(), b)) >= B - 1 and sum(p == q for p, q in zip(na.tolist(), nb)) >= B - 1


@pytest.mark.parametrize("V", [1007, 9000])
def test_step_form_is_the_row_form(V):
    """temperature from the token just fed, the uniform from the table, the counter updated (generate.py:138-163, 186-189)"""
    import generate as G
    from midiemo import ops
    B, steps = 5, 6
    g = torch.Generator().manual_seed(V)
    ts = (torch.rand(V, generator=g) < 0.3)
    prev = torch.randint(0, V, (B, 1), generator=g)
    rc = torch.tensor([0.0, 3.0, 9.0, 40.0, 1.0])
    table = torch.rand(steps, B, generator=g)
    pos = torch.tensor([13], dtype=torch.int32, device="cuda")
    x = torch.randn(B, V, generator=g) * 4
    d_rc = rc.cuda()
    ids, n = torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    ops.sample_minp_step(x.cuda(), V, None, prev.cuda(), ts.to(torch.uint8).cuda(), d_rc, 1.2, 0.8, 0.5, 0, 0.9, 0.05, table.cuda(), pos, 10, ids, n)
    temp = G.sampling_temperature(prev[:, 0].cuda(), rc.cuda(), ts.cuda(), 1.2, 0.8, 0.5).cpu()
    want, wn = sample(x, [], temp, 0, 0.9, 0.05, table[3])
    assert ids.tolist() == want and n.tolist() == wn
    assert torch.equal(d_rc.cpu(), G.update_repeat_counts(rc, torch.tensor(wn)))


def test_repeats_and_replays():
    from midiemo import ops
    B, V = 7, 50000
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(B, V, generator=g, device="cuda").bfloat16().float()
    temp, u = torch.ones(B, device="cuda"), torch.rand(B, generator=g, device="cuda")
    ids, n = torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")

    def call():
        ops.sample_minp(x, V, None, temp, 100, 0.9, 0.01, u, ids, n)
    call()
    torch.cuda.synchronize()
    first = ids.clone(), n.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, first[0]) and torch.equal(n, first[1])
        u.copy_(torch.rand(B, generator=g, device="cuda"))
        call()
        first = ids.clone(), n.clone()
        ids.zero_()


def test_tensors_on_the_host_are_refused():
    from midiemo import ops
    x, one, ids = torch.zeros(2, 50).cuda(), torch.ones(2).cuda(), torch.empty(2, dtype=torch.int64).cuda()
    for bad in ((one.cpu(), one, ids), (one, one.cpu(), ids), (one, one, ids.cpu())):
        with pytest.raises(RuntimeError, match="sampling: "):
            ops.sample_minp(x, 50, None, bad[0], 0, 0.9, 0.0, bad[1], bad[2])
    with pytest.raises(RuntimeError, match="sampling: "):
        ops.sample_minp(x, 50, torch.zeros(1, dtype=torch.int32), one, 0, 0.9, 0.0, one, ids)
