"""The quantised cache without a GPU: the format's definition, sizes, and every refusal (made before anything is enqueued)."""
import ctypes

import pytest
import torch

import kvq_reference as R
from midiemo import _lib, ops
from midiemo.kvcache import QuantKVCache


@pytest.mark.parametrize("bits", [4, 8])
def test_rounding_of_the_definition(bits):
    grid = R.GRID[bits]
    x = torch.cat((grid, -grid, (grid[1:] + grid[:-1]) / 2, torch.tensor([R.TOP[bits]], dtype=torch.float64))).float()
    x = x[None]
    c, s = R.codes_of(x, bits)
    assert float(s) == 1.0
    v = R.values_of(c, s, bits)[0]
    n = len(grid)
    assert torch.equal(v[:n], grid) and torch.equal(v[n:2 * n].abs(), grid)
    assert bool((c[0, 2 * n:-1] % 2 == 0).all())                       # ties to the even code
    if bits == 8:                                                      # the library's own e4m3 rounding says the same
        y = torch.randn(1, 4096) * 40
        y[0, 0] = 448.0
        c, s = R.codes_of(y, 8)
        assert torch.equal(R.values_of(c, s, 8), y.to(torch.float8_e4m3fn).double())


def test_scale_of_the_definition():
    x = torch.zeros(5, 32)
    x[1] = 2.0 ** -97
    x[2, 3] = float("inf")
    x[3, 0] = float("nan")
    x[4, 7] = -5.0
    s = R.scale_of(x, 4)
    assert s[0] == 0 and s[1] == 0 and torch.isnan(s[2]) and torch.isnan(s[3])
    assert s[4] == torch.tensor(5 / 6).bfloat16().float() or s[4] < 5 / 6
    assert 5 / 6 * (1 - 2 ** -7) < float(s[4]) <= 5 / 6


def test_cache_sizes_and_construction():
    c = QuantKVCache(2, 3, 100, 48, 4, device="cpu")
    assert c.max_len == 128 and c.k.shape == (2, 3, 4, 32 * 24) and c.v_scale.shape == (2, 3, 128) and c.nbytes == 2 * 2 * 3 * 128 * (24 + 2)
    w = QuantKVCache.wrap(c.k, c.k_scale, c.v, c.v_scale, 48, 4)
    assert w.k is c.k and w.max_len == 128
    for bad in (dict(head_dim=40), dict(bits=5), dict(batch=0), dict(max_len=0)):
        with pytest.raises(RuntimeError):
            QuantKVCache(**{**dict(batch=1, heads=1, max_len=32, head_dim=32, bits=4, device="cpu"), **bad})
    with pytest.raises(RuntimeError):
        QuantKVCache.wrap(c.k, c.k_scale, c.v, c.v_scale, 64, 4)
    with pytest.raises(RuntimeError):
        QuantKVCache.wrap(c.k, c.k_scale.float(), c.v, c.v_scale, 48, 4)
    with pytest.raises(RuntimeError):
        QuantKVCache.wrap(c.k, c.k_scale[:, :, :64], c.v, c.v_scale, 48, 4)


def test_refusals_of_the_cache():
    c = QuantKVCache(2, 3, 64, 32, 4, device="cpu")
    k = torch.zeros(2, 5, 3, 32)
    q, rel, pad = torch.zeros(2, 3, 32), torch.zeros(64, 32), torch.zeros(2, 64, dtype=torch.bool)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    for call in (lambda: c.write(k, k, 60), lambda: c.write(k, k, -1), lambda: c.write(k[:, :, :2], k, 0), lambda: c.write(k, k.half(), 0),
                 lambda: c.write(k.transpose(2, 3), k.transpose(2, 3), 0), lambda: c.write(torch.zeros(2, 65, 3, 32), torch.zeros(2, 65, 3, 32), i32(0)),
                 lambda: c.write(k, k, i32(0, 1, 2)), lambda: c.write(k, k, torch.zeros(2)), lambda: c.write(k, k, 0, lens=torch.tensor([1, 2])),
                 lambda: c.write(k, k, 0, lens=i32(1)), lambda: c.read(60, 5), lambda: c.read(0, 65), lambda: c.attend(q[:1], 0), lambda: c.attend(q, 64),
                 lambda: c.attend(q, -2), lambda: c.attend(q, 3, rel=rel[:63]), lambda: c.attend(q, 3, rel=rel.half()), lambda: c.attend(q, 3, rel=rel.t()),
                 lambda: c.attend(q, 3, key_pad=pad[:, ::2]), lambda: c.attend(q, 3, key_pad=pad[:1]), lambda: c.attend(q, 3, key_pad=pad[:, :3].contiguous()),
                 lambda: c.attend(q, 3, out=q.half()), lambda: c.attend(q, 3, out=torch.zeros(1, 3, 32).expand(2, 3, 32)), lambda: c.attend(q, 3, nsplit=65),
                 lambda: c.attend(q.transpose(0, 1), 3), lambda: c.append_attend(q, q, q.half(), 3), lambda: c.append_attend(q, q[:1], q[:1], 3),
                 lambda: c.append_attend(q, q, q, -1), lambda: c.append_attend(q, q, q, 64), lambda: c.append_attend(q, q, torch.zeros(3, 2, 32).transpose(0, 1), 3)):
        with pytest.raises(RuntimeError, match="kv cache"):
            call()
    for call in (lambda: c.write(k, k, 0), lambda: c.read(0, 5), lambda: c.append_attend(q, q, q, 3), lambda: c.attend(q, 3, rel=rel, key_pad=pad)):       # right, but no device
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_refusals_of_the_c_abi():
    lib = _lib.load()
    P = 4096                                                           # never touched: the call is refused first
    six = (ctypes.c_int64 * 6)(*[64] * 6)

    def cache(kc=P, B=1, H=1, dh=64, blocks=1, bits=4, vs=P):
        return ctypes.byref(_lib.KVQCache(kc, P, P, vs, B, H, dh, blocks, bits))

    def write(k=P, strides=six, n=1, t=0, t_dev=None, ld_t=0, dtype=_lib.ME_BF16, c=True, **kw):
        return lib.me_kvq_write(cache(**kw) if c else None, k, P, strides, n, t, t_dev, ld_t, None, dtype, None)

    def attn(q=P, E=None, M=0, pad=None, ld_pad=0, out=P, part=None, part_bytes=0, nsplit=1, t=0, ld_t=0, dtype=_lib.ME_BF16, c=True, **kw):
        return lib.me_kvq_attn(cache(**kw) if c else None, q, 64, 64, E, M, pad, ld_pad, out, 64, 64, part, part_bytes, nsplit, t, None, ld_t, dtype, None)

    NULL, SHAPE, TYPE, ALIGN, WS = -5, -2, -1, -3, -6
    assert write(c=False) == NULL and write(vs=None) == NULL and attn(c=False) == NULL
    assert write(k=None) == NULL and write(strides=None) == NULL and write(kc=P + 4) == ALIGN and write(dtype=7) == TYPE
    for bad in (dict(dh=40), dict(bits=2), dict(t=32), dict(t=-1), dict(n=33), dict(n=-1), dict(ld_t=2), dict(H=70000), dict(B=70000), dict(blocks=1 << 26), dict(B=-1)):
        assert write(**bad) == SHAPE, bad
    assert write(B=0) == 0 and write(n=0) == 0                         # nothing to do
    assert attn(q=None) == NULL and attn(out=None) == NULL and attn(dtype=9) == TYPE and attn(kc=P + 8) == ALIGN and attn(E=P + 2, M=64) == ALIGN
    for bad in (dict(dh=128), dict(bits=16), dict(t=32), dict(t=-2), dict(nsplit=0), dict(nsplit=65), dict(E=P, M=31), dict(B=70000), dict(ld_t=3), dict(pad=P, ld_pad=-1)):
        assert attn(**bad) == SHAPE, bad
    need = ops.workspace_bytes(_lib.ME_WS_KVQ_ATTN, 1, 4, 64, torch.bfloat16)
    assert need == 4 * 68 * 4
    assert attn(nsplit=4) == WS and attn(nsplit=4, part=P, part_bytes=need - 1) == WS and attn(out=None, part=P, part_bytes=68 * 4 - 4) == WS
    assert attn(B=0) == 0

    def append(k=P, v=P, ldn=64, t=0, **kw):
        return lib.me_kvq_append_attn(cache(**kw), P, 64, 64, k, v, ldn, 64, None, 0, None, 0, P, 64, 64, None, 0, 1, t, None, 0, _lib.ME_BF16, None)
    assert append(k=None) == NULL and append(v=None) == NULL and append(t=-1) == SHAPE and append(t=32) == SHAPE and append(k=P + 2) == ALIGN and append(v=P + 4) == ALIGN
    assert append(ldn=63) == ALIGN and append(B=0) == 0
    for rel in (0, 1):
        for b, h, n in ((1, 8, 1), (1, 8, 2048), (4, 8, 2048), (64, 16, 1999), (1, 1, 1 << 30), (10 ** 6, 8, 2048), (0, 1, 1)):
            assert 1 <= lib.me_kvq_splits(b, h, n, rel) <= 64
    assert lib.me_kvq_splits(4, 8, 2048, 1) == 16 and lib.me_kvq_splits(4, 8, 2048, 0) == 1 and lib.me_kvq_splits(1, 1, 1 << 30, 0) == 64


def test_layouts_once_checked_survive_a_flush_by_another_thread():
    c = QuantKVCache(1, 1, 32, 64, 4, "cpu")
    flush = lambda *t: c._seen.clear() or 5
    for i in range(300):
        assert c._passed((i, "key"), flush) == 5
    assert len(c._seen) <= 256
