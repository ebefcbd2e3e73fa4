"""The quantised cache at ends of its range that test_kvq_gpu.py leaves out: the largest and smallest queries over 8-bit rows, device positions that begin
before the cache."""
import math

import pytest
import torch

import kvq_reference as R
from test_kvq_gpu import DT, cache, expect_rows, rows, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dh", [32, 48, 64])
@pytest.mark.parametrize("T,q_at,k_at", [("bf16", 2.0 ** 117, 2.0 ** -80), ("bf16", "max", 2.0 ** -90), ("f32", 2.0 ** 117, 2.0 ** -80), ("f32", "max", 2.0 ** -90),
                                         ("f32", 2.0 ** -120, 2.0 ** 118), ("bf16", 2.0 ** -120, 2.0 ** 118), ("f16", "max", 1.0)])
def test_queries_at_the_ends_of_the_range(T, q_at, k_at, dh, bits):
    """query times code passes the largest f32 (or falls below the smallest) where query times key does not"""
    T, B, H, n = DT[T], 2, 3, 16
    g = torch.Generator().manual_seed(dh)
    sign = (torch.randint(0, 2, (B, 1, H, dh), generator=g) * 2 - 1).float()
    k = (sign * (1 + torch.arange(n) / 16)[None, :, None, None] * k_at).to(T)       # logit j: (1 + j / 16) dh q_at k_at / sqrt(dh), rounding 2^-7 of it at most
    v = torch.randn(B, n, H, dh, generator=g).to(T)
    q = (sign[:, 0] * (torch.finfo(T).max if q_at == "max" else q_at)).to(T).cuda()
    c = cache(B, H, 32, dh, bits)
    c.write(k.cuda(), v.cuda(), 0)
    kk, vv = [t.cpu().double().transpose(1, 2) for t in c.read(0, n, torch.float32)]
    s = (q.cpu().double()[:, :, None] * kk).sum(-1) / math.sqrt(dh)
    w = torch.softmax(s, -1)
    want = (w[..., None] * vv).sum(2)
    # logits: dh + 16 roundings of 2^-24 and what the parts leave of the query (2^-17 / 2^-19 of it, in f32 2^-25 / 2^-29), as in test_kvq_gpu.check
    left = {4: 2.0 ** (-29 if T == torch.float32 else -19), 8: 2.0 ** (-25 if T == torch.float32 else -17)}[bits]
    d = s.abs().amax(-1) * 2 * ((dh + 16) * 2.0 ** -24 + left)
    big = vv.abs().amax((2, 3))
    if q_at != 2.0 ** -120:
        assert float(w.amax(-1).min()) == 1.0 and float((s[..., 15] - s[..., 14] - 2 * d).min()) > 200      # nothing but key 15 has a weight
        d = torch.zeros_like(d)
    bound = (big * (2 * d + left * 128 + 80 * 2.0 ** -24))[..., None] + want.abs() * torch.finfo(T).eps / 2
    fresh = cache(B, H, 32, dh, bits)
    fresh.write(k[:, :-1].cuda(), v[:, :-1].cuda(), 0)
    outs = [c.attend(q, n - 1), c.attend(q, n - 1, nsplit=3), c.attend(q, n - 1, rel=torch.zeros(32, dh, dtype=T, device="cuda")),
            fresh.append_attend(q, k[:, -1].contiguous().cuda(), v[:, -1].contiguous().cuda(), n - 1)]
    for i, out in enumerate(outs):
        err = (out.cpu().double() - want).abs()
        assert bool((err <= bound).all()), (i, float(err.max()), float(bound.min()))


@pytest.mark.parametrize("bits", [4, 8])
def test_sequences_whose_device_position_lies_outside_are_left_out(bits):
    """as a whole, also where later rows of the call would reach into the cache; nothing of them is written, and they read as zeros"""
    B, H, dh, n, room = 5, 2, 48, 70, 96
    x = rows(B, n, H, dh, torch.bfloat16, 7)
    p = torch.tensor([-1, -33, 96, -2 ** 31, 60], dtype=torch.int32, device="cuda")
    d = x.cuda()
    c = cache(B, H, room, dh, bits)
    for t in (c.k, c.v):
        t.fill_(0x21)
    for t in (c.k_scale, c.v_scale):
        t.fill_(3.0)
    c.write(d[:, :, 1], d[:, :, 2], p)
    for t, held in ((c.k, 0x21), (c.v, 0x21), (c.k_scale, 3.0), (c.v_scale, 3.0)):
        assert bool((t[:4] == held).all()) and bool((t[4].flatten(1) != held).any())
    for part, back in zip((1, 2), c.read(p, n, torch.bfloat16)):
        assert bool((back[:4] == 0).all()) and bool((back[4, 36:] == 0).all())
        assert same(back[4, :36].cpu(), expect_rows(x[4:, :36, part], bits, torch.bfloat16)[2][0])
