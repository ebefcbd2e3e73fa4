"""The quantised cache's format and its attention in 64 bits, written from the definition (shared by test_kvq_cpu.py and test_kvq_gpu.py)."""
import math

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
GRID = {4: E2M1, 8: E4M3}
TOP = {4: 6.0, 8: 448.0}


def scale_of(x, bits):
    """bfloat16-valued scales (float32) of rows x [..., dh]"""
    amax = x.float().abs().amax(-1)
    amax = torch.where(torch.isnan(x.float()).any(-1), torch.full_like(amax, math.nan), amax)
    s = ((amax * torch.tensor(1 / TOP[bits], dtype=torch.float32)).view(torch.int32) & -65536).view(torch.float32)
    s = torch.where(amax >= 2.0 ** -96, s, torch.zeros_like(s))
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, math.nan))


def codes_of(x, bits):
    """codes (uint8, sign in the top bit of the code) and scales of rows x [..., dh]: nearest, ties to the even code"""
    s, grid = scale_of(x, bits), GRID[bits]
    live = torch.isfinite(s) & (s > 0)
    y = torch.where(live[..., None], x.double() / torch.where(live, s, torch.ones_like(s))[..., None].double(), torch.zeros((), dtype=torch.float64))
    border = (grid[1:] + grid[:-1]) / 2
    a = y.abs()
    lo, hi = torch.bucketize(a, border), torch.bucketize(a, border, right=True)
    i = torch.where(lo % 2 == 0, lo, hi)
    neg = torch.signbit(y)
    return (i | (neg.long() << (bits - 1))).to(torch.uint8), s


def values_of(codes, s, bits):
    """what codes and scales stand for, float64"""
    top = 1 << (bits - 1)
    v = GRID[bits][(codes.long() & (top - 1)).clamp(max=len(GRID[bits]) - 1)]
    return torch.where(codes.long() & top > 0, -v, v) * s.double()[..., None]


def position(which, token, d, dh, bits):
    """position of a code in its block of 32 tokens, as include/midiemo.h states it"""
    if which == "v":
        return d * 32 + token if bits == 4 else (token // 16) * 16 * dh + d * 16 + token % 16
    if dh == 64:
        group, i = 2 * (token // 16) + d // 32, d % 32
    elif dh == 32:
        group, i = token // 16, d
    elif d < 32:
        group, i = 2 * (token // 16), d
    else:
        group, i = 1, 16 * (token // 16) + d - 32
    if bits == 4:
        return (group * 16 + token % 16) * 32 + i
    return (i // 16) * 16 * dh + (group * 16 + token % 16) * 16 + i % 16


def unpack(packed, which, dh, bits):
    """packed [B, H, blocks, bytes] (CPU) -> codes uint8 [B, H, blocks * 32, dh]"""
    flat = packed if bits == 8 else torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    at = torch.tensor([[position(which, t, d, dh, bits) for d in range(dh)] for t in range(32)])
    assert sorted(at.flatten().tolist()) == list(range(32 * dh))
    c = flat[..., at.flatten()]
    return c.reshape(*packed.shape[:2], packed.shape[2] * 32, dh)


def attend(q, k, v, pos, rel, key_pad):
    """q [B, H, dh], k / v float64 [B, H, n, dh], pos list -> out float64 and what a bound on a kernel's error is made of: the sum of weights times |v|,
    the largest sum of a logit's magnitudes, the largest |q|_max sum |k|, and the sum over tiles of 128 keys of 128 times the largest weight times |v|_max"""
    B, H, dh = q.shape
    out = torch.zeros(B, H, dh, dtype=torch.float64)
    weight = torch.zeros(B, H, dh, dtype=torch.float64)
    logit = torch.zeros(B, H, dtype=torch.float64)
    digits = torch.zeros(B, H, dtype=torch.float64)
    tiles = torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        n = pos[b] + 1
        keep = [j for j in range(n) if key_pad is None or j >= key_pad.shape[1] or not key_pad[b, j]]
        if not keep:
            continue
        kk, vv = k[b][:, keep], v[b][:, keep]
        qq = q[b].double()
        mag = (qq.abs()[:, None] * kk.abs()).sum(-1)
        s = (qq[:, None] * kk).sum(-1)
        if rel is not None:
            e = rel.double()[[rel.shape[0] - 1 - pos[b] + j for j in keep]]
            s = s + qq @ e.t()
            mag = mag + qq.abs() @ e.abs().t()
        s, mag = s / math.sqrt(dh), mag / math.sqrt(dh)
        w = torch.softmax(s, -1)
        out[b] = (w[..., None] * vv).sum(1)
        weight[b] = (w[..., None] * vv.abs()).sum(1)
        logit[b] = (mag + s.abs()).amax(-1)
        digits[b] = (qq.abs().amax(-1)[:, None] * kk.abs().sum(-1)).amax(-1) / math.sqrt(dh)
        ww, scale = torch.zeros(H, -(-n // 128) * 128, dtype=torch.float64), torch.zeros(H, -(-n // 128) * 128, dtype=torch.float64)
        ww[:, keep], scale[:, keep] = w, vv.abs().amax(-1)          # a value row's largest is 6 (448) scales: the weight's unit there
        tiles[b] = ((ww * scale).view(H, -1, 128).amax(-1) * 128).sum(-1)
    return out, weight, logit, digits, tiles
