"""The quantised key / value cache on the GPU: codes, scales and read-back bit for bit against the definition in 64 bits, the
attention against it within bounds that follow from the arithmetic, and the calls around them (streams, graphs, ragged batches)."""
import math

import pytest
import torch

import kvq_reference as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def cache(B, H, room, dh, bits):
    from midiemo.kvcache import QuantKVCache
    return QuantKVCache(B, H, room, dh, bits)


def rows(B, n, H, dh, T, seed, kind="plain"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, n, 3, H, dh, generator=g) * torch.exp2(torch.randint(-3, 4, (B, n, 3, H, 1), generator=g).float())
    if kind == "grid":                        # amax and values on few bits: quotients that fall exactly between two codes
        x = torch.randint(-12, 13, x.shape, generator=g).float()
    if kind == "odd":
        r = x.view(-1, dh)
        r[0] = 0.0
        r[1] = 2.0 ** -120 if T != torch.float16 else 0.0
        r[2, 3] = math.inf
        r[3, dh - 1] = math.nan
        r[4, 0] = -math.inf
        r[5] = torch.finfo(T).max
        r[6] = 0.0
        r[6, 1] = -torch.finfo(T).max
        r[7] = torch.finfo(T).tiny * (1 if T != torch.float16 else 4)
        r[8, ::2] = -0.0
    return x.to(T)


def expect_rows(x, bits, T):
    """[B, n, H, dh] -> codes [B, H, n, dh], scales [B, H, n], values of T"""
    c, s = R.codes_of(x.transpose(1, 2), bits)
    return c, s, R.values_of(c, s, bits).to(T).transpose(1, 2)


def same(a, b):
    a, b = a.double(), b.double()
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_scales_next_to_their_borders(bits):
    """f32 rows whose largest value is a scale's exact multiple, or up to three bits off it"""
    scales = torch.arange(0x3f80, 0x4080, dtype=torch.int32) << 16
    amax = (scales.view(torch.float32) * R.TOP[bits]).view(torch.int32)[:, None] + torch.arange(-3, 4, dtype=torch.int32)
    amax = amax.view(torch.float32).reshape(1, -1, 1, 1)                  # 1792 rows
    x = (torch.rand(1, amax.shape[1], 1, 32, generator=torch.Generator().manual_seed(1)) - 0.5) * amax
    x[..., 7] = amax[..., 0]
    c = cache(1, 1, 1792, 32, bits)
    c.write(x.cuda(), x.neg().cuda(), 0)
    codes, scale, value = expect_rows(x, bits, torch.float32)
    assert torch.equal(c.k_scale.cpu().float()[0, 0], scale[0, 0]) and torch.equal(c.v_scale, c.k_scale)
    k, v = c.read(0, 1792)
    assert same(k.cpu(), value) and same(v.cpu(), -value)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dh", [32, 48, 64])
@pytest.mark.parametrize("T", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,pos,kind", [(1, 0, "plain"), (1, 37, "plain"), (1, 63, "grid"), (31, 5, "plain"), (64, 32, "grid"), (77, 45, "odd"), (200, 1, "plain")])
def test_write_and_read_are_the_definition(T, dh, bits, n, pos, kind):
    T, B, H, room = DT[T], 2, 3, 256
    x = rows(B, n, H, dh, T, 100 * n + pos + dh + bits, kind)
    c = cache(B, H, room, dh, bits)
    g = torch.Generator().manual_seed(1)
    held = [torch.randint(0, 100, t.shape, generator=g).to(torch.uint8) for t in (c.k, c.v)]      # what the call may not touch (no NaN among them)
    c.k.copy_(held[0]); c.v.copy_(held[1]); c.k_scale.fill_(3.0); c.v_scale.fill_(5.0)
    d = x.cuda()
    c.write(d[:, :, 1], d[:, :, 2], pos)
    for which, part, scale, code, old, other in (("k", 1, c.k_scale, c.k, held[0], 3.0), ("v", 2, c.v_scale, c.v, held[1], 5.0)):
        ec, es, ev = expect_rows(x[:, :, part], bits, T)
        got = R.unpack(code.cpu(), which, dh, bits)
        before = R.unpack(old, which, dh, bits)
        inside = torch.zeros(room, dtype=torch.bool)
        inside[pos:pos + n] = True
        # a negative value that rounds to zero may have either sign of zero
        top = 1 << (bits - 1)
        fold = lambda t: torch.where((t & (top - 1)) == 0, torch.zeros_like(t), t)
        assert torch.equal(fold(got[:, :, inside]), fold(ec)), which
        assert torch.equal(got[:, :, ~inside], before[:, :, ~inside]), which
        s = scale.cpu().float()
        assert same(s[:, :, inside], es) and bool((s[:, :, ~inside] == other).all())
        back = c.read(pos, n, T)[part - 1].cpu()
        assert same(back, ev), which


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dh", [32, 48, 64])
def test_write_ragged_and_device_positions(dh, bits):
    B, H, n, room = 5, 2, 70, 128
    x = rows(B, n, H, dh, torch.bfloat16, 3)
    pos, lens = [0, 17, 100, 127, 64], [70, 0, 50, 1, 3]          # sequence 2 runs out of the cache
    c = cache(B, H, room, dh, bits)
    p = torch.tensor(pos, dtype=torch.int32, device="cuda")
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    d = x.cuda()
    c.write(d[:, :, 1], d[:, :, 2], p, lens=ln)
    k, v = c.read(p, n, torch.bfloat16, lens=ln)
    for part, back in ((1, k.cpu()), (2, v.cpu())):
        ev = expect_rows(x[:, :, part], bits, torch.bfloat16)[2]
        for b in range(B):
            m = min(lens[b], room - pos[b])
            assert same(back[b, :m], ev[b, :m]) and bool((back[b, m:] == 0).all()), b
    for b in range(B):                                            # nothing outside pos .. pos + lens
        s = c.k_scale[b, 0].cpu()
        used = torch.zeros(room, dtype=torch.bool)
        used[pos[b]:min(room, pos[b] + lens[b])] = True
        assert bool((s[~used] == 0).all()) and bool((s[used] > 0).all())
    one = torch.tensor([3], dtype=torch.int32, device="cuda")      # one position for all
    c.write(d[:, :1, 1], d[:, :1, 2], one)
    assert same(c.read(3, 1, torch.bfloat16)[0].cpu(), expect_rows(x[:, :1, 1], bits, torch.bfloat16)[2])
    out = torch.tensor([-1, 128, 500, -2**31, 127], dtype=torch.int32, device="cuda")   # no place: left out, read as zeros
    before = c.k.clone(), c.v.clone(), c.k_scale.clone()
    c.write(d[:, :1, 1], d[:, :1, 2], out, lens=torch.tensor([1, 1, 1, 1, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(before[0], c.k) and torch.equal(before[1], c.v) and torch.equal(before[2], c.k_scale)
    assert bool((c.read(out, 5, torch.float32)[0][:4] == 0).all())


@pytest.mark.parametrize("T", ["bf16", "f32"])
def test_write_takes_any_strides(T):
    T, B, n, H, dh = DT[T], 2, 40, 3, 48
    x = rows(B, n, H, dh, T, 9)[:, :, 0]
    want = expect_rows(x, 4, T)[2]
    flat = torch.zeros(B * n * H * (dh + 1) + 1, dtype=T, device="cuda")
    odd = flat[1:].view(B, n, H, dh + 1)[..., :dh]                 # neither the base nor the rows are 16-byte aligned
    odd.copy_(x)
    perm = x.permute(2, 0, 1, 3).contiguous().cuda().permute(1, 2, 0, 3)
    for view in (odd, perm):
        c = cache(B, H, 64, dh, 4)
        c.write(view, perm, 7)
        k, v = c.read(7, n, T)
        assert same(k.cpu(), want) and same(v.cpu(), want)
    c.write(x[:1].cuda().expand(B, -1, -1, -1), perm, 0)           # one prompt for all sequences
    assert same(c.read(0, n, T)[0].cpu(), want[:1].expand(B, -1, -1, -1))
    c.write(odd[:, :0], odd[:, :0], 64)                            # no rows
    assert c.read(64, 0)[0].shape == (B, 0, H, dh)


def fill(c, n, T, seed):
    """random rows in the whole cache; float64 values of what it then holds [B, H, n, dh]"""
    x = rows(c.batch, n, c.heads, c.head_dim, T, seed).cuda()
    c.write(x[:, :, 1], x[:, :, 2], 0)
    return [t.cpu().double().transpose(1, 2) for t in c.read(0, n, torch.float32)]


def check(out, q, k, v, pos, rel, pad, T, dh, bits):
    want, weight, logit, digits, tiles = R.attend(q, k, v, pos, rel, pad)
    # logits: products and sums in 32 bits (dh + 16 roundings at most in any chain); weights: exp2 and a few roundings.  An error d of every logit
    # changes the result by at most 2 d of the weighted |v|.
    # 4 bits: four (f32: six) digits in base 32 of a value scaled into [8, 16) leave at most half a unit of the last, 2^-16 / 8 (2^-26 / 8) of the
    # largest: of |q| in the query, of weight times value scale in each tile of 128 keys.
    # 8 bits: the query exact (16-bit types) or, like the weights, in two (f32: three) bfloat16 parts of 8 bits and a sign each, 2^-17 (2^-25) of each value.
    unit = 2.0 ** -24
    d = logit * (dh + 16) * unit
    wide = T == torch.float32
    if bits == 4:
        left = 2.0 ** (-29 if wide else -19)
        d = d + digits * left
        bound = (tiles * left)[..., None]
    else:
        left = 2.0 ** (-25 if wide else -17)
        d = d + logit * left
        bound = weight * left
    bound = bound + want.abs() * torch.finfo(T).eps / 2 + weight * (2 * d + 64 * unit)[..., None]
    if T == torch.float16:
        bound = bound + 2.0 ** -25                                # subnormal results
    err = (out.cpu().double() - want).abs()
    assert bool((err <= bound).all()), (float((err / bound.clamp_min(1e-300)).max()), float(err.max()))
    return want


CASES = [(1, 1, 1), (2, 3, 31), (1, 8, 33), (2, 9, 128), (3, 2, 129), (1, 4, 513), (2, 16, 700), (1, 2, 2048)]


@pytest.mark.parametrize("rel", [True, False])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dh", [32, 48, 64])
@pytest.mark.parametrize("T", ["bf16", "f16", "f32"])
def test_attention_is_the_formula(T, dh, bits, rel):
    T = DT[T]
    for i, (B, H, n) in enumerate(CASES):
        g = torch.Generator().manual_seed(i)
        c = cache(B, H, n, dh, bits)
        k, v = fill(c, n, T, 7 + i)
        q = torch.randn(B, H, dh, generator=g).to(T)
        E = torch.randn(2048, dh, generator=g).to(T) if rel else None
        for ns in (0, 1, 3):
            out = c.attend(q.cuda(), n - 1, rel=E.cuda() if rel else None, nsplit=ns)
            check(out, q, k, v, [n - 1] * B, E, None, T, dh, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dh", [32, 48, 64])
@pytest.mark.parametrize("T", ["bf16", "f16", "f32"])
def test_attention_ragged_padded_and_empty_rows(T, dh, bits):
    T, B, H, n = DT[T], 6, 5, 300
    g = torch.Generator().manual_seed(dh)
    c = cache(B, H, n, dh, bits)
    k, v = fill(c, n, T, 11)
    pos = [299, 0, 130, -1, 255, 40]
    pad = torch.rand(B, n, generator=g) < 0.3
    pad[4] = True                                                 # every key masked
    pad[5, :40] = True                                            # only the newest left
    pad[5, 40] = False
    # a masked key, and what lies behind a sequence's last one, may hold anything: rows of infinities and NaN
    bad = torch.full((B, n, H, dh), math.nan, dtype=T)
    bad[:, ::2] = math.inf
    live = ~pad & (torch.arange(n)[None] <= torch.tensor(pos)[:, None])
    x = torch.where(live.cuda()[:, :, None, None], c.read(0, n, torch.float32)[0], bad.cuda().float())
    y = torch.where(live.cuda()[:, :, None, None], c.read(0, n, torch.float32)[1], bad.cuda().float())
    c.write(x, y, 0)                                              # rows that stand on the code's own values: read back unchanged up to the scale
    k, v = [t.cpu().double().transpose(1, 2) for t in c.read(0, n, torch.float32)]
    q = torch.randn(B, H, dh, generator=g).to(T)
    E = torch.randn(2048, dh, generator=g).to(T)
    p = torch.tensor(pos, dtype=torch.int32, device="cuda")
    for ns in (1, 2, 5):
        for mask in (pad.cuda(), pad.to(torch.uint8).cuda()):
            out = c.attend(q.cuda(), p, rel=E.cuda(), key_pad=mask, nsplit=ns)
            want = check(out, q, k, v, pos, E, pad, T, dh, bits)
            assert bool((out[3] == 0).all()) and bool((out[4] == 0).all()) and bool((want[3:5] == 0).all())
    # a mask narrower than the cache: keys behind it are not masked (sequences 1 and 5 lie inside it)
    out = c.attend(q.cuda(), p, rel=E.cuda(), key_pad=pad[:, :41].contiguous().cuda(), nsplit=2)
    full = c.attend(q.cuda(), p, rel=E.cuda(), key_pad=pad.cuda(), nsplit=2)
    assert torch.equal(out[1], full[1]) and torch.equal(out[5], full[5])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dh", [32, 48, 64])
@pytest.mark.parametrize("T", ["bf16", "f16", "f32"])
def test_append_and_attend_in_one_launch(T, dh, bits):
    """the cache afterwards is the one that write() leaves, bit for bit; the result is the formula over it"""
    T, B, H, n = DT[T], 4, 5, 160
    g = torch.Generator().manual_seed(dh + bits)
    x = rows(B, n, H, dh, T, 17).cuda()
    E = torch.randn(2048, dh, generator=g).to(T)
    for pos in ([0, 1, 2, 31], [32, 63, 64, 127], [128, 129, 159, 100], 0, 133, [-1, 160, 400, 5]):
        a, b = cache(B, H, n, dh, bits), cache(B, H, n, dh, bits)
        for c in (a, b):
            c.write(x[:, :, 1], x[:, :, 2], 0)
        new = rows(B, 1, H, dh, T, 23).cuda()
        kn, vn = new[:, 0, 1].contiguous(), new[:, 0, 2].contiguous()
        p = pos if isinstance(pos, int) else torch.tensor(pos, dtype=torch.int32, device="cuda")
        b.write(kn[:, None], vn[:, None], p)
        q = torch.randn(B, H, dh, generator=g).to(T)
        listed = [pos] * B if isinstance(pos, int) else [min(i, n - 1) for i in pos]
        k, v = [t.cpu().double().transpose(1, 2) for t in b.read(0, n, torch.float32)]
        for rel in (E, None):
            pad = torch.rand(B, n, generator=g) < 0.2
            pad[1, listed[1]] = True                              # the new key itself masked: written, not used
            for ns, mask in ((0, None), (1, pad), (2, None), (7, pad)):
                c = cache(B, H, n, dh, bits)
                for m in ("k", "v", "k_scale", "v_scale"):
                    getattr(c, m).copy_(getattr(a, m))
                out = c.append_attend(q.cuda(), kn, vn, p, rel=None if rel is None else rel.cuda(), key_pad=None if mask is None else mask.cuda(), nsplit=ns)
                for m in ("k", "v"):
                    assert torch.equal(getattr(c, m), getattr(b, m)), (m, pos)
                for m in ("k_scale", "v_scale"):
                    assert torch.equal(getattr(c, m).view(torch.int16), getattr(b, m).view(torch.int16)), (m, pos)
                check(out, q, k, v, listed, rel, mask, T, dh, bits)
    # rows that are not numbers: held as such, and the result says so
    kn[0, 0, 3], vn[1, 1, 0] = math.inf, math.nan
    for ns in (1, 3):
        c = cache(B, H, n, dh, bits)
        c.write(x[:, :, 1], x[:, :, 2], 0)
        out = c.append_attend(q.cuda(), kn, vn, 90, nsplit=ns).cpu()
        assert bool(torch.isnan(out[0, 0]).all()) and bool(torch.isnan(out[1, 1]).all()) and bool(torch.isfinite(out[2:]).all())
        d = cache(B, H, n, dh, bits)
        out = d.append_attend(q.cuda(), kn, vn, 0, nsplit=ns).cpu()      # the only key
        assert bool(torch.isnan(out[0, 0]).all()) and bool(torch.isfinite(out[2:]).all())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T", ["bf16", "f16", "f32"])
def test_a_query_that_is_no_number_gives_none(T, bits):
    c = cache(1, 3, 40, 48, bits)
    fill(c, 40, DT[T], 3)
    E = torch.randn(2048, 48).to(DT[T]).cuda()
    for bad in (math.inf, -math.inf, math.nan):
        q = torch.randn(1, 3, 48).to(DT[T])
        q[0, 1, 47] = bad
        for rel in (None, E):
            for out in (c.attend(q.cuda(), 39, rel=rel), c.append_attend(q.cuda(), q.cuda() * 0 + 1, q.cuda() * 0 + 1, 39, rel=rel)):
                assert bool(torch.isnan(out[0, 1]).all()), bad


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dh", [32, 48, 64])
def test_what_unused_rows_hold_does_not_matter(dh, bits):
    """masked rows and those behind the position: every code and scale there may be anything, numbers or not"""
    B, H, n, pos = 3, 2, 320, 200
    E = torch.randn(n, dh).bfloat16().cuda()
    q = torch.randn(B, H, dh).bfloat16().cuda()
    pad = (torch.rand(B, n) < 0.3).to(torch.uint8)
    pad[2] = 0
    x, y = rows(B, n, H, dh, torch.bfloat16, 5).cuda().unbind(2)[1:]
    got = []
    for junk in (0x00, 0x7f, 0xff, 0x5a):
        c = cache(B, H, n, dh, bits)
        for t in (c.k, c.v):
            t.fill_(junk)
        for t in (c.k_scale, c.v_scale):
            t.view(torch.uint8).fill_(junk)
        for j in range(pos + 1):                                 # only the rows that count are written
            for b in range(B):
                if not pad[b, j]:
                    one = torch.zeros(B, dtype=torch.int32)
                    one[b] = 1
                    c.write(x[:, j : j + 1], y[:, j : j + 1], j, lens=one.cuda())
        p = pad.cuda()
        got.append([c.attend(q, pos, rel=E, key_pad=p), c.attend(q, pos, key_pad=p),
                    c.append_attend(q, x[:, pos + 1].contiguous(), y[:, pos + 1].contiguous(), pos + 1, rel=E, key_pad=p)])
        assert all(bool(torch.isfinite(o).all()) for o in got[-1])
    for g in got[1:]:
        for a, b in zip(got[0], g):
            assert torch.equal(a, b)


def test_attention_values_that_are_not_numbers():
    c = cache(2, 2, 64, 64, 4)
    x = rows(2, 64, 2, 64, torch.bfloat16, 2)
    x[0, 5, 1, 0, 0] = math.inf                                    # a key of sequence 0, head 0
    x[0, 6, 2, 1, 0] = math.nan                                    # a value of sequence 0, head 1
    c.write(x.cuda()[:, :, 1], x.cuda()[:, :, 2], 0)
    q = torch.randn(2, 2, 64).bfloat16()
    q[1, 1, 3] = math.inf
    for ns in (1, 2):
        out = c.attend(q.cuda(), 63, nsplit=ns).cpu()
        assert bool(torch.isnan(out[0]).all()) and bool(torch.isfinite(out[1, 0]).all()) and bool(torch.isnan(out[1, 1]).all())
    # queries at both ends of the type's range: logits stay apart, nothing overflows on the way
    for mag in (2.0 ** -126, 2.0 ** -60, 2.0 ** 30):
        qq = (torch.ones(2, 2, 64) * mag).bfloat16()
        out = c.attend(qq.cuda(), 3).cpu()
        assert bool(torch.isfinite(out).all())


def test_attention_strided_query_and_output():
    B, H, dh = 3, 4, 32
    c = cache(B, H, 96, dh, 4)
    k, v = fill(c, 96, torch.float16, 5)
    big = torch.randn(H, B, dh + 5).half().cuda()
    q = big.permute(1, 0, 2)[..., 2:2 + dh]
    out = torch.full((B, H, 2 * dh), 9.0, dtype=torch.float16, device="cuda")
    r = c.attend(q, 95, out=out[..., dh:])
    assert r.data_ptr() == out[..., dh:].data_ptr() and bool((out[..., :dh] == 9).all())
    check(r, q.cpu(), k, v, [95] * B, None, None, torch.float16, dh, 4)


def test_attention_repeats_bit_for_bit_and_replays():
    """the same call twice; a captured step that moves its own position, replayed with eager work between, on a stream of its own"""
    B, H, dh, n = 4, 8, 64, 512
    c = cache(B, H, n, dh, 4)
    x = rows(B, n, H, dh, torch.bfloat16, 21).cuda()
    q = torch.randn(B, H, dh).bfloat16().cuda()
    E = torch.randn(2048, dh).bfloat16().cuda()
    ref = cache(B, H, n, dh, 4)
    ref.write(x[:, :, 1], x[:, :, 2], 0)
    a, b = ref.attend(q, n - 1, rel=E), ref.attend(q, n - 1, rel=E)
    assert torch.equal(a, b)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    kin, vin = torch.empty(B, 1, H, dh, dtype=torch.bfloat16, device="cuda"), torch.empty(B, 1, H, dh, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    side = torch.cuda.Stream()

    def step():
        c.write(kin, vin, pos)
        c.attend(q, pos, rel=E, out=out)
        pos.add_(1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kin.copy_(x[:, :1, 1]); vin.copy_(x[:, :1, 2])
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for t in range(1, 140):
            kin.copy_(x[:, t:t + 1, 1]); vin.copy_(x[:, t:t + 1, 2])
            graph.replay()
            if t % 23 == 0 or t == 139:
                want = ref.attend(q, torch.tensor([t], dtype=torch.int32, device="cuda"), rel=E)
                side.synchronize()
                assert torch.equal(out, want), t
    torch.cuda.synchronize()
    assert int(pos) == 140
    for m in ("k_scale", "v_scale"):
        assert torch.equal(getattr(c, m)[:, :, :140], getattr(ref, m)[:, :, :140])


def test_two_streams_attend_one_cache():
    c = cache(2, 8, 2048, 64, 4)
    fill(c, 2048, torch.bfloat16, 31)
    qs = [torch.randn(2, 8, 64).bfloat16().cuda() for _ in range(2)]
    want = [c.attend(q, 2047, nsplit=16) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = c.attend(qs[i], 2047, nsplit=16)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_beyond_32_bits():
    """the last sequence of a cache whose codes pass 4 GiB: 68 sequences of 131072 + tokens"""
    B, H, room, dh = 68, 8, 131072, 64
    c = cache(B, H, room, dh, 8)
    assert c.k.numel() > 2 ** 32
    x = rows(1, 200, H, dh, torch.bfloat16, 41).cuda().expand(B, -1, -1, -1, -1)
    p = torch.full((B,), room - 200, dtype=torch.int32, device="cuda")
    c.write(x[:, :, 1], x[:, :, 2], p)
    k, v = c.read(p, 200, torch.float32)
    want = expect_rows(x[:1, :, 1].cpu(), 8, torch.float32)[2]
    assert same(k[-1:].cpu(), want)
    pad = torch.ones(B, room, dtype=torch.uint8, device="cuda")
    pad[:, room - 200:] = 0
    q = torch.randn(B, H, dh).bfloat16()
    out = c.attend(q.cuda(), room - 1, key_pad=pad)
    kk, vv = [t[-1:].cpu().double().transpose(1, 2) for t in (k, v)]
    check(out[-1:], q[-1:], kk, vv, [199], None, None, torch.bfloat16, dh, 8)
