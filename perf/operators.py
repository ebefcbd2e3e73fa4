"""The serving operators of the quantised key / value cache and of min-p sampling: cases, plain forms and exact values.

Three operators, as DecodeSession and generate() use them:

  store   keys and values of new tokens are written to a cache in 4 or 8 bits and read back
  attend  one new query per sequence and head against such a cache, with the learned relative table and a key mask
  sample  one token per row from temperature, top-k, top-p and min-p at a given uniform

The cache.  A row (one token, one head) of dh values is held as dh codes and one scale in bfloat16:
scale = amax / 6 (4 bits) or amax / 448 (8 bits), divided in 32 bits and cut to bfloat16 toward zero; code = x / scale to the
nearest e2m1 (4 bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) or e4m3 (8 bits) value, ties to the even code, larger ones
to the largest; a row with amax below 2^-96 is held as zeros, one with an infinity or a NaN reads back as NaN.  32 tokens form
a block.  Codes of a block lie in the order in which the matrix instructions take them (`k_position`, `v_position`)."""
import math
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TOP = {4: 6.0, 8: 448.0}


def framework():
    """The package, imported where its operators run."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "midi-emotion_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from midiemo import kvcache, ops
    return kvcache, ops


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of 64 songs that are generated side by side: what a layer writes per step
        dict(name="store 64x1 bf16 4bit", op="store", B=64, n=1, pos=1023, H=8, dh=64, dtype="bf16", bits=4, ragged=False),
        # a batch of prompts of different lengths, the odd head dimension of the 768-wide model
        dict(name="store 8x1215 f16 8bit ragged", op="store", B=8, n=1215, pos=0, H=16, dh=48, dtype="f16", bits=8, ragged=True),
        # prompts of the model's full window, a large batch
        dict(name="store 32x2048 bf16 4bit", op="store", B=32, n=2048, pos=0, H=8, dh=64, dtype="bf16", bits=4, ragged=False),
        # the same in the exact tier, behind a first piece that ended inside a block
        dict(name="store 4x777 f32 4bit", op="store", B=4, n=777, pos=45, H=8, dh=32, dtype="f32", bits=4, ragged=True),
        # a single song early in its window: latency alone
        dict(name="attend 1x256 bf16 4bit", op="attend", B=1, L=256, H=8, dh=64, dtype="bf16", bits=4, rel=True, pad=False, ragged=False),
        # the four songs of generate.py's default batch at the end of the window
        dict(name="attend 4x2048 bf16 4bit", op="attend", B=4, L=2048, H=8, dh=64, dtype="bf16", bits=4, rel=True, pad=False, ragged=False),
        # many songs of different lengths, padded keys among them, a song with nothing left after the mask
        dict(name="attend 64x1999 f16 8bit pad", op="attend", B=64, L=1999, H=16, dh=48, dtype="f16", bits=8, rel=True, pad=True, ragged=True),
        # the exact tier
        dict(name="attend 16x1031 f32 4bit", op="attend", B=16, L=1031, H=8, dh=32, dtype="f32", bits=4, rel=True, pad=True, ragged=True),
        # long caches without a relative table: the stream from memory is all
        dict(name="attend 64x16384 bf16 4bit", op="attend", B=64, L=16384, H=8, dh=64, dtype="bf16", bits=4, rel=False, pad=False, ragged=False),
        # the default batch and vocabulary of generate.py
        dict(name="sample 4x1018", op="sample", B=4, V=1018, top_k=0, top_p=0.9, min_p=0.05, steps="bf16"),
        # a batch over a vocabulary of merged events
        dict(name="sample 64x32000", op="sample", B=64, V=32000, top_k=200, top_p=0.95, min_p=0.02, steps="f32"),
        # the widest rows, nothing but min-p and the nucleus
        dict(name="sample 128x131071", op="sample", B=128, V=131071, top_k=0, top_p=0.98, min_p=0.001, steps="bf16"),
    ]


def spread(rng, lo, hi):
    """A whole number from lo to hi, even in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "sample"])
    if op == "sample":
        V = spread(rng, 64, 131072)
        return dict(op=op, B=spread(rng, 1, min(128, 16_000_000 // V)), V=V, top_k=rng.choice([0, 0, spread(rng, 1, V)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]), min_p=rng.choice([0.0, round(10 ** rng.uniform(-3, -0.3), 4)]),
                    steps=rng.choice(["f32", "bf16"]))
    dh, dtype, bits = rng.choice([32, 48, 64]), rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([4, 4, 8])
    H = spread(rng, 1, 16)
    if op == "store":
        n = spread(rng, 1, 2048)
        return dict(op=op, B=spread(rng, 1, max(1, min(64, 30000 // n))), n=n, pos=rng.choice([0, rng.randrange(0, 200)]), H=min(H, 8), dh=dh, dtype=dtype,
                    bits=bits, ragged=rng.random() < 0.5)
    rel = rng.random() < 0.7
    L = spread(rng, 1, 2048 if rel else 16384)
    return dict(op=op, B=spread(rng, 1, max(1, min(64, 4_000_000 // (L * H)))), L=L, H=H, dh=dh, dtype=dtype, bits=bits, rel=rel,
                pad=rng.random() < 0.4, ragged=rng.random() < 0.5)


def lengths(case):
    """Tokens of each sequence: all alike, or up to a quarter fewer."""
    full = case["n"] if case["op"] == "store" else case["L"]
    return [full - (7919 * b) % (full // 4 + 1) if case["ragged"] else full for b in range(case["B"])]


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["B"] * (case["V"] * 4 + 20), "flops": 3.0 * case["B"] * case["V"]}
    size, H, dh = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]], case["H"], case["dh"]
    row = dh * case["bits"] // 8 + 2
    total = sum(lengths(case))
    if case["op"] == "store":       # rows in, cache rows out and in again, the whole read-back out
        return {"bytes": 2 * H * (total * (dh * size + 2 * row) + case["B"] * case["n"] * dh * size), "flops": 8.0 * total * H * dh}
    extra = (case["L"] * dh * size if case["rel"] else 0) + (total if case["pad"] else 0)
    return {"bytes": 2 * H * total * row + 2 * case["B"] * H * dh * size + extra, "flops": total * H * dh * (6.0 if case["rel"] else 4.0)}


# ---------------------------------------------------------------------------------------------------- the cache's format
def k_position(dh, bits):
    """Where in a block's 32 * dh codes the code of (token, dimension) of a key lies: int64 [32, dh] on the CPU."""
    t, d = torch.arange(32)[:, None], torch.arange(dh)[None, :]
    lane, half = t % 16, t // 16
    if dh == 64:
        group, i = 2 * half + d // 32, d % 32 + 0 * t
    elif dh == 32:
        group, i = half + 0 * d, d + 0 * t
    else:
        group = torch.where(d < 32, 2 * half, torch.ones_like(half + d))
        i = torch.where(d < 32, d + 0 * t, 16 * half + d - 32)
    if bits == 4:
        return (group * 16 + lane) * 32 + i
    return (i // 16) * (dh // 16 * 256) + (group * 16 + lane) * 16 + i % 16


def v_position(dh, bits):
    """The same of a value."""
    t, d = torch.arange(32)[:, None], torch.arange(dh)[None, :]
    if bits == 4:
        return d * 32 + t
    return (t // 16) * (dh * 16) + d * 16 + t % 16


def pack(codes, position, bits):
    """Codes uint8 [..., tokens, dh] (tokens a multiple of 32) in the cache's order: uint8 [..., tokens / 32, 32 * dh * bits / 8]."""
    dh = codes.shape[-1]
    blocks = codes.reshape(*codes.shape[:-2], codes.shape[-2] // 32, 32 * dh)
    flat = blocks[..., torch.argsort(position.reshape(-1)).to(codes.device)]
    return flat if bits == 8 else flat[..., 0::2] | (flat[..., 1::2] << 4)


def code_values(packed, position, grid):
    """What the codes stand for, in 32 bits: [..., tokens, dh].  grid: the 16 values of the 4-bit codes, None for 8 bits."""
    if grid is not None:
        values = grid[torch.stack((packed & 15, packed >> 4), -1).flatten(-2).int()]
    else:
        values = packed.view(torch.float8_e4m3fn).float()
    values = values[..., position.reshape(-1)]
    return values.reshape(*packed.shape[:-2], packed.shape[-2] * 32, position.shape[1])


# ---------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEVICE)  # noqa: E731
    uniform = lambda *s: torch.rand(*s, generator=g, device=DEVICE)  # noqa: E731
    state = dict(case)
    if case["op"] == "sample":
        B, V = case["B"], case["V"]
        logits = normal(B, V) * 3
        if case["steps"] == "bf16":                     # a 16-bit head: many equal logits
            logits = logits.bfloat16().float()
        state |= dict(logits=logits, special=torch.arange(3, dtype=torch.int32, device=DEVICE), temp=0.6 + uniform(B), u=uniform(B),
                      ids=torch.empty(B, dtype=torch.int64, device=DEVICE), choices=torch.empty(B, dtype=torch.int32, device=DEVICE))
        return state
    B, H, dh, bits, T = case["B"], case["H"], case["dh"], case["bits"], TYPES[case["dtype"]]
    lens = torch.tensor(lengths(case), dtype=torch.int32, device=DEVICE)
    room = -(-(case["pos"] + case["n"] if case["op"] == "store" else case["L"]) // 32)
    state |= dict(lens=lens, k=torch.zeros(B, H, room, 4 * dh * bits, dtype=torch.uint8, device=DEVICE), k_scale=torch.zeros(B, H, room * 32, dtype=torch.bfloat16, device=DEVICE),
                  v=torch.zeros(B, H, room, 4 * dh * bits, dtype=torch.uint8, device=DEVICE), v_scale=torch.zeros(B, H, room * 32, dtype=torch.bfloat16, device=DEVICE))
    if case["op"] == "store":
        # the key and value parts of a fused projection's output [B, n, 3, H, dh]; every head has a spread of its own
        qkv = (normal(B, case["n"], 3, H, dh) * (0.5 + uniform(1, 1, 3, H, 1)) * (0.5 + uniform(1, 1, 3, 1, dh))).to(T)
        state |= dict(keys=qkv[:, :, 1], values=qkv[:, :, 2])
    else:
        for name, position in (("k", k_position(dh, bits)), ("v", v_position(dh, bits))):
            for b in range(B):                          # one sequence at a time keeps the intermediate arrays small
                y = normal(H, room * 32, dh) * (TOP[bits] / 2.6)
                if bits == 4:
                    codes = torch.bucketize(y.abs(), torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=DEVICE)).to(torch.uint8) | ((y < 0).to(torch.uint8) << 3)
                else:
                    codes = y.clamp(-TOP[8], TOP[8]).to(torch.float8_e4m3fn).view(torch.uint8)
                state[name][b] = pack(codes, position, bits)
            state[name + "_scale"].copy_((0.3 + 0.9 * uniform(B, H, room * 32)) * (2.6 / TOP[bits]))
        pad = uniform(B, case["L"]) < 0.1 if case["pad"] else None
        if case["pad"] and B > 1:
            pad[1] = True
        state |= dict(q=normal(B, H, dh).to(T), pos=lens - 1, table=normal(2048, dh).to(T) if case["rel"] else None,
                      pad=pad.to(torch.uint8) if case["pad"] else None, out=torch.empty(B, H, dh, dtype=T, device=DEVICE),
                      k_at=k_position(dh, bits).to(DEVICE), v_at=v_position(dh, bits).to(DEVICE),
                      grid=torch.tensor(E2M1 + tuple(-x for x in E2M1), device=DEVICE) if bits == 4 else None)
    if own:     # the handle that a session keeps: it holds the same tensors and the workspace of its calls
        state["cache"] = framework()[0].QuantKVCache.wrap(state["k"], state["k_scale"], state["v"], state["v_scale"], dh, bits)
    return state


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return run_own(state)
    return {"store": plain_store, "attend": plain_attend, "sample": plain_sample}[state["op"]](state)


def run_own(s):
    if s["op"] == "store":
        s["cache"].write(s["keys"], s["values"], s["pos"], lens=s["lens"])
        k, v = s["cache"].read(s["pos"], s["n"], s["keys"].dtype, lens=s["lens"])
        return {"keys": k, "values": v}
    if s["op"] == "attend":
        return {"out": s["cache"].attend(s["q"], s["pos"], rel=s["table"], key_pad=s["pad"], out=s["out"])}
    _, ops = framework()
    ops.sample_minp(s["logits"], s["V"], s["special"], s["temp"], s["top_k"], s["top_p"], s["min_p"], s["u"], s["ids"], s["choices"])
    return {"ids": s["ids"], "choices": s["choices"]}


def plain_quantise(x, bits):
    """x [..., dh] -> what the codes stand for (32 bits) and the scale (bfloat16)."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    fine, kept = torch.isfinite(amax), amax >= 2.0 ** -96
    scale = ((amax / TOP[bits]).view(torch.int32) & -65536).view(torch.float32)
    y = torch.where(fine & kept, x.double() / scale.double(), 0.0).clamp(-TOP[bits], TOP[bits])
    if bits == 4:
        # the step at each magnitude is a power of two, so dividing by it is exact and round() settles ties to even
        a = y.abs()
        step = torch.where(a >= 4, 2.0, torch.where(a >= 2, 1.0, 0.5))
    else:
        step = 2.0 ** (torch.log2(y.abs().clamp(min=2.0 ** -6)).floor() - 3)
    value = (torch.round(y / step) * step).float()
    return value, torch.where(fine, torch.where(kept, scale, 0.0), math.nan).bfloat16()


def plain_store(s):
    there = (torch.arange(s["n"], device=DEVICE)[None] < s["lens"][:, None])[:, :, None, None]
    out = {}
    for name in ("keys", "values"):
        value, scale = plain_quantise(s[name], s["bits"])
        out[name] = torch.where(there, value * scale.float(), 0.0).to(s[name].dtype)
    return out


def plain_attend(s):
    L, dh = s["L"], s["dh"]
    k = code_values(s["k"], s["k_at"], s["grid"])[:, :, :L] * s["k_scale"][:, :, :L, None].float()
    q = s["q"].float()
    logits = (k * q[:, :, None]).sum(-1)
    j, pos = torch.arange(L, device=DEVICE), s["pos"].long()
    if s["table"] is not None:
        rows = s["table"].shape[0] - 1 - pos[:, None] + j[None]
        of_row = torch.matmul(q, s["table"].float().t())                            # [B, H, rows of the table]
        logits = logits + torch.gather(of_row, 2, rows.clamp(0, s["table"].shape[0] - 1)[:, None].expand(-1, s["H"], -1))
    logits = logits / math.sqrt(dh)
    open_ = j[None] <= pos[:, None]
    if s["pad"] is not None:
        open_ = open_ & (s["pad"] == 0)
    open_ = open_[:, None]
    top = torch.where(open_, logits, -math.inf).amax(-1, keepdim=True)
    p = torch.where(open_, torch.exp(logits - torch.where(top > -math.inf, top, 0.0)), 0.0)
    v = code_values(s["v"], s["v_at"], s["grid"])[:, :, :L] * s["v_scale"][:, :, :L, None].float()
    total = p.sum(-1)
    out = (p[..., None] * v).sum(2) / torch.where(total > 0, total, 1.0)[..., None]
    return {"out": out.to(s["q"].dtype)}


def plain_sample(s):
    """In 64 bits: the picks lie next to borders."""
    B, V = s["B"], s["V"]
    x = torch.where(torch.isnan(s["logits"]), 0.0, s["logits"])
    x = x.index_fill(1, s["special"].long(), -math.inf).double()
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    e = torch.exp((x - x[:, :1]) / s["temp"].double()[:, None])
    i = torch.arange(V, device=DEVICE)[None]
    if s["top_k"] > 0:
        e = torch.where(i < s["top_k"], e, 0.0)
    if 0 < s["top_p"] < 1:
        e = torch.where((i == 0) | (torch.cumsum(e, 1) <= float(np.float32(s["top_p"])) * e.sum(1, keepdim=True)), e, 0.0)
    e = torch.where(e >= float(np.float32(s["min_p"])), e, 0.0)
    choices = (e > 0).sum(1)
    upto = torch.cumsum(e, 1)
    pick = (upto <= s["u"].double()[:, None] * e.sum(1, keepdim=True)).sum(1)
    pick = torch.minimum(pick, choices - 1)
    return {"ids": torch.gather(order, 1, pick[:, None])[:, 0], "choices": choices.int()}


# ---------------------------------------------------------------------------------------------------- exact values
def nearest(y, bits):
    """y (float64, finite) to the nearest value of the code's type by comparing with all borders between neighbours."""
    if bits == 4:
        grid = torch.tensor(E2M1, dtype=torch.float64, device=y.device)
    else:
        grid = torch.arange(127, dtype=torch.uint8, device=y.device).view(torch.float8_e4m3fn).double()
    border = (grid[1:] + grid[:-1]) / 2
    a = y.abs()
    low, high = torch.bucketize(a, border, right=False), torch.bucketize(a, border, right=True)       # they differ at a tie
    return torch.sign(y) * grid[torch.where(low % 2 == 0, low, high)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        out = {}
        for name in ("keys", "values"):
            x = s[name].double()
            amax = x.abs().amax(-1, keepdim=True).float()
            scale = ((amax / TOP[case["bits"]]).view(torch.int32) & -65536).view(torch.float32).double()
            y = torch.empty_like(x)
            for b in range(case["B"]):
                y[b] = nearest(x[b] / scale[b], case["bits"]) * scale[b] if bool((amax[b] >= 2.0 ** -96).all()) else math.nan
                y[b, int(s["lens"][b]):] = 0
            out[name] = y
        return out
    if case["op"] == "attend":
        out = torch.zeros(case["B"], case["H"], case["dh"], dtype=torch.float64, device=DEVICE)
        for b in range(case["B"]):
            n = int(s["pos"][b]) + 1
            keep = torch.ones(n, dtype=torch.bool, device=DEVICE) if s["pad"] is None else s["pad"][b, :n] == 0
            if not bool(keep.any()):
                continue
            blocks = -(-n // 32)
            part = lambda m: code_values(s[m][b, :, :blocks], s[m + "_at"], s["grid"])[:, :n].double() * s[m + "_scale"][b, :, :n, None].double()  # noqa: E731
            k, q = part("k"), s["q"][b].double()
            if s["table"] is not None:
                k = k + s["table"][2048 - n:].double()[None]
            w = torch.softmax(((k @ q[:, :, None])[:, :, 0] / math.sqrt(case["dh"])).masked_fill(~keep[None], -math.inf), -1)
            out[b] = (w[:, None] @ part("v"))[:, 0]
        return {"out": out}
    ids, choices = np.zeros(case["B"], np.int64), np.zeros(case["B"], np.int32)
    logits, temp, u = (s[m].cpu().numpy().astype(np.float64) for m in ("logits", "temp", "u"))
    for b in range(case["B"]):
        x = np.nan_to_num(logits[b], nan=0.0, posinf=np.inf, neginf=-np.inf)
        x[s["special"].cpu().numpy()] = -np.inf
        order = np.argsort(-x, kind="stable")
        if case["top_k"] > 0:
            order = order[:case["top_k"]]
        w = np.exp((x[order] - x[order[0]]) / temp[b])
        n = len(w)
        if 0 < case["top_p"] < 1:
            n = min(n, max(1, int(np.searchsorted(np.cumsum(w), float(np.float32(case["top_p"])) * w.sum(), side="right"))))
        n = int(np.count_nonzero((w[:n] >= float(np.float32(case["min_p"]))) & (w[:n] > 0)))
        upto = np.cumsum(w[:n])
        choices[b], ids[b] = n, order[min(n - 1, int(np.searchsorted(upto, u[b] * upto[-1], side="right")))]
    return {"ids": ids, "choices": choices}
