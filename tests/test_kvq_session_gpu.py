"""Quantised caches and min-p sampling in their place: DecodeSession(kv_bits=...) against the model's formulas in 64 bits, the device-resident
loops against single steps, generate() and its command line."""
import math
import os
import subprocess
import sys

import pytest
import torch

import kvq_reference as R
from oracle import ref_model as O

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(cd, mode="continuous_concat", V=1007, d=128, heads=2, layers=2, seed=5):
    from midiemo.models.build_model import build_model
    cfg = O.Cfg(V, layers, heads, d, 2 * d, d_condition=16, conditioning=mode)
    P = O.seeded_params(cfg, seed)
    model, _ = build_model(dict(vocab_size=V, n_layer=layers, n_head=heads, d_model=d, d_inner=2 * d, dropout=0.0,
                                d_condition=16 if mode == "continuous_concat" else -1, conditioning=mode, compute_dtype=cd))
    model.load_state_dict(P)
    return model.to("cuda").eval(), {k: v.double() for k, v in P.items()}, cfg


def ln(x, g, b):
    m = x.mean(-1, keepdim=True)
    return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-6) * g + b


def emulate(P, cfg, sess, tok, cond, t, eps):
    """one position in 64 bits over the session's own cached rows -> logits, and the new rows of every layer before they are quantised"""
    d, dc, H, M = cfg.d_model, cfg.d_condition, cfg.n_head, cfg.max_seq
    pe = torch.as_tensor(sess.m._pe[t].cpu()).double()
    x = torch.cat((P["embedding.weight"][tok] * math.sqrt(d - dc), cond @ P["fc_condition.weight"].t() + P["fc_condition.bias"]), -1) + pe
    B, dh = tok.numel(), d // H
    rows = []
    for i in range(cfg.n_layer):
        p = f"enc_layers.{i}."
        lin = lambda n, y: y @ P[p + n + ".weight"].t() + P[p + n + ".bias"]
        q, k, v = [lin("rga." + n, x).view(B, H, dh) for n in ("Wq", "Wk", "Wv")]
        rows.append((k, v))
        kc, vc = [c.double().cpu().transpose(1, 2) for c in sess.kvq[i].read(0, t + 1, torch.float32)]
        E = P[p + "rga.E"][M - 1 - t:]
        s = ((q[:, :, None] * kc).sum(-1) + q @ E.t()) / math.sqrt(dh)
        a = (torch.softmax(s, -1)[..., None] * vc).sum(2).reshape(B, d)
        o1 = ln(x + lin("rga.fc", a), P[p + "layernorm1.weight"], P[p + "layernorm1.bias"])
        x = ln(o1 + lin("FFN_suf", torch.relu(lin("FFN_pre", o1))), P[p + "layernorm2.weight"], P[p + "layernorm2.bias"])
    return x @ P["fc.weight"].t() + P["fc.bias"], rows


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B,d,heads", [(3, 128, 2), (10, 96, 2), (1, 128, 4)])
def test_session_is_the_model_over_quantised_rows(bits, B, d, heads):
    """exact tier.  The rows the session caches are the quantised projections (a code may differ where 32 and 64 bits fall on two sides of a
    border: by one step, and rarely), and over those rows the step is the formula (f32 arithmetic through two layers: 1e-4 as in the model tests)."""
    from midiemo.decode import DecodeSession
    model, P, cfg = build("fp32", d=d, heads=heads)
    sess = DecodeSession(model, B, kv_bits=bits)
    g = torch.Generator().manual_seed(bits)
    toks = torch.randint(1, cfg.vocab_size, (40, B), generator=g)
    cond = torch.rand(B, 2, generator=g) * 2 - 1
    off = all_ = 0
    for t in range(40):
        got = sess.step(toks[t].cuda(), cond.cuda()).double().cpu()
        want, rows = emulate(P, cfg, sess, toks[t], cond.double(), t, model.LN_EPS)
        assert float((got - want).norm() / want.norm()) < 1e-4, t
        for c, kv in zip(sess.kvq, rows):
            for have, row in zip(c.read(t, 1, torch.float32), kv):
                code, s = R.codes_of(row.float(), bits)
                near = R.values_of(code, s, bits)
                diff = (have.cpu().double()[:, 0] - near).abs()
                step = s.double()[..., None] * (2.0 if bits == 4 else 32.0) * 1.01           # the widest step of the codes
                assert bool((diff <= step).all())
                off += int((diff > s.double()[..., None] * 2.0 ** -6).sum())
                all_ += diff.numel()
    assert off <= 2 + all_ * 2e-3


@pytest.mark.parametrize("cd,bits", [("bf16", 4), ("bf16", 8), ("fp16", 4), ("fp32", 8)])
@pytest.mark.parametrize("B", [2, 9])
def test_device_loops_are_the_single_steps(cd, bits, B):
    """greedy and sampled loops with the position on the device, captured and not, against steps from the host: the same tokens"""
    from midiemo import ops
    from midiemo.decode import DecodeSession
    model, _, cfg = build(cd)
    cond = (torch.rand(B, 2, generator=torch.Generator().manual_seed(1)) * 2 - 1).cuda()
    first = torch.full((B,), 5, dtype=torch.int64, device="cuda")
    special = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    n = 30
    sess = DecodeSession(model, B, kv_bits=bits)
    tok, want = first.clone(), []
    for _ in range(n):
        lg = sess.step(tok, cond)
        nxt = torch.empty(B, dtype=torch.int64, device="cuda")
        ops.greedy_pick(lg, cfg.vocab_size, special, nxt, B)
        want.append(nxt)
        tok = nxt
    want = torch.stack(want, 1)
    for graph in (False, True):
        s2 = DecodeSession(model, B, kv_bits=bits)
        got = torch.cat([s2.greedy_run(first, n // 2, cond, special, use_graph=graph), ], 1)
        got = torch.cat([got, s2.greedy_run(got[:, -1], n - n // 2, cond, special, use_graph=graph)], 1)
        assert torch.equal(got, want), graph
    assert s2.launches_per_token == (1 + 4 * (1 if B <= 8 else 2)) * 2 + 1 + (1 if B <= 8 else 2) + 1
    # sampled, with min-p
    ts = (torch.arange(cfg.vocab_size) % 7 == 0).cuda()
    uni = torch.rand(n, B, generator=torch.Generator().manual_seed(3)).cuda()
    runs = []
    for graph in (False, True):
        s3, rc = DecodeSession(model, B, kv_bits=bits), torch.zeros(B, device="cuda")
        runs.append((s3.sample_run(first, n, cond, special, ts, rc, 1.1, 0.9, 0.5, 0, 0.95, uni, use_graph=graph, min_p=0.02).clone(), rc))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    s4, rc, tok = DecodeSession(model, B, kv_bits=bits), torch.zeros(B, device="cuda"), first.clone()
    import generate as G
    for t in range(n):
        lg = s4.step(tok, cond)
        temp = G.sampling_temperature(tok, rc, ts, 1.1, 0.9, 0.5)
        nxt, nc = torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
        ops.sample_minp(lg, cfg.vocab_size, special, temp, 0, 0.95, 0.02, uni[t], nxt, nc)
        rc = G.update_repeat_counts(rc, nc)
        assert torch.equal(nxt, runs[0][0][:, t]), t
        tok = nxt
    assert torch.equal(rc, runs[0][1])


def test_eight_bits_stay_near_the_unquantised_session():
    """the same tokens through both: a row's 8-bit code is off by at most 2^-4 of each value, so logits move by a small part of their spread"""
    from midiemo.decode import DecodeSession
    model, _, cfg = build("bf16")
    a, b, c = DecodeSession(model, 2), DecodeSession(model, 2, kv_bits=8), DecodeSession(model, 2, kv_bits=4)
    g = torch.Generator().manual_seed(2)
    cond = torch.zeros(2, 2).cuda()
    for t in range(60):
        tok = torch.randint(1, cfg.vocab_size, (2,), generator=g).cuda()
        x, y, z = a.step(tok, cond).clone(), b.step(tok, cond), c.step(tok, cond)
        e8, e4 = float((x - y).norm() / x.norm()), float((x - z).norm() / x.norm())
        assert e8 < 2.0 ** -4 and e4 < 2.0 ** -1, (t, e8, e4)


@pytest.mark.parametrize("mode", ["none", "discrete_token", "continuous_token", "continuous_concat"])
def test_generate_with_a_quantised_cache_and_min_p(mode):
    """both loops of generate() draw the same uniforms: the same songs; condition slots and prefixes go through the quantised cache too"""
    import generate as G
    from midiemo.vocab import get_maps
    V = 1017 if mode == "discrete_token" else 1007
    model, _, cfg = build("bf16", mode=mode, V=V)
    maps = get_maps(n_emotion_bins=5 if mode == "discrete_token" else 0)
    conds = [[0.5, -0.2], [-0.7, 0.9]]
    out = []
    for device_loop in (True, False):
        torch.manual_seed(7)
        out.append(G.generate(model, maps, torch.device("cuda"), "/tmp/none", mode,
                              discrete_conditions=[["<V1>", "<A0>"], ["<V-1>", "<A2>"]] if mode == "discrete_token" else None,
                              continuous_conditions=None if mode == "none" else conds, gen_len=40, max_input_len=64, top_k=50, top_p=0.9, min_p=0.01, kv_bits=4,
                              debug=True, min_n_instruments=0, primers=[["<START>"]] * 2 if mode == "none" else [["<START>"]], return_ids=True,
                              device_loop=device_loop))
    assert out[0].shape == (40, 2) and torch.equal(out[0], out[1])


def test_generate_over_a_wide_vocabulary():
    """more than 4096 symbols: sampled on the device all the same"""
    from midiemo.decode import DecodeSession
    model, _, cfg = build("bf16", V=6000)
    first, rc = torch.full((2,), 5, dtype=torch.int64, device="cuda"), torch.zeros(2, device="cuda")
    uni = torch.rand(12, 2, generator=torch.Generator().manual_seed(3)).cuda()
    cond = torch.zeros(2, 2).cuda()
    runs = [DecodeSession(model, 2).sample_run(first, 12, cond, None, torch.zeros(6000, device="cuda"), rc.clone(), 1.0, 1.0, 0.0, 0, 0.9, uni,
                                               use_graph=g).clone() for g in (True, False)]
    assert torch.equal(runs[0], runs[1]) and int(runs[0].max()) < 6000


def test_refusals_of_the_session():
    import generate as G
    from midiemo.decode import DecodeSession
    from midiemo.vocab import get_maps
    model, _, cfg = build("bf16")
    with pytest.raises(ValueError, match="kv_bits"):
        DecodeSession(model, 1, kv_bits=3)
    s = DecodeSession(model, 1, kv_bits=4)
    with pytest.raises(ValueError, match="min_p"):
        s.sample_run(torch.zeros(1, dtype=torch.int64), 4, torch.zeros(1, 2), None, torch.zeros(1007), torch.zeros(1), 1.0, 1.0, 0.0, 0, 0.9,
                     torch.rand(4, 1), min_p=1.5)
    for bad in (dict(kv_bits=4, use_cache=False), dict(min_p=-1.0)):
        with pytest.raises(ValueError):
            G.generate(model, get_maps(n_emotion_bins=0),
                       torch.device("cuda"), "/tmp/none", "continuous_concat", continuous_conditions=[[0.0, 0.0]], gen_len=4, debug=True, **bad)


def test_command_line(tmp_path):
    model, _, cfg = build("bf16")
    run = tmp_path / "run"
    run.mkdir()
    torch.save({k: v.cpu() for k, v in model.state_dict().items()}, run / "model.pt")
    torch.save(dict(vocab_size=1007, n_layer=2, n_head=2, d_model=128, d_inner=256, dropout=0.0, d_condition=16, conditioning="continuous_concat",
                    compute_dtype="bf16"), run / "model_config.pt")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "generate.py"), "--model_dir", "run", "--output_root", str(tmp_path), "--conditioning", "continuous_concat",
                        "--valence", "0.5", "--arousal", "0.1", "--batch_size", "2", "--gen_len", "40", "--kv_bits", "4", "--minp", "0.05", "--min_n_instruments", "0",
                        "--quiet"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    assert len(list((run / "generations" / "inference").glob("inds_*.pt"))) == 2
