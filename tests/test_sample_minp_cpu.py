"""Refusals of me_sample_minp and me_sample_minp_step: made on the host, before anything is enqueued (addresses are never touched)."""
import pytest
import torch

from midiemo import _lib, ops

P = 4096
NULL, SHAPE, WS = -5, -2, -6


def row(logits=P, ld=100, V=100, special=None, n_special=0, temp=P, top_k=0, top_p=0.9, min_p=0.1, u=P, out=P, B=1, ws=None, ws_bytes=0):
    return _lib.load().me_sample_minp(logits, ld, V, special, n_special, temp, top_k, top_p, min_p, u, out, None, B, ws, ws_bytes, None)


def step(prev=P, ts=P, rc=P, pos=P, u_ld=4, V=100, min_p=0.1, B=1):
    return _lib.load().me_sample_minp_step(P, 100, V, None, 0, prev, ts, rc, 1.0, 1.0, 0.5, 0, 0.9, min_p, P, u_ld, pos, 0, P, None, B, None, 0, None)


def test_refusals():
    for bad in (dict(logits=None), dict(temp=None), dict(u=None), dict(out=None), dict(n_special=2)):
        assert row(**bad) == NULL, bad
    for bad in (dict(V=0), dict(ld=99), dict(V=_lib.ME_SAMPLE_MAX_VOCAB + 1, ld=1 << 20), dict(B=-1), dict(min_p=-0.1), dict(min_p=1.5), dict(min_p=float("nan")), dict(n_special=-1)):
        assert row(**bad) == SHAPE, bad
    assert row(B=0) == 0 and row(B=70000) == SHAPE
    need = _lib.load().me_workspace_bytes(_lib.ME_WS_SAMPLE, 3, 50000, 0, 0)
    assert need > 0 and _lib.load().me_workspace_bytes(_lib.ME_WS_SAMPLE, 3, 32512, 0, 0) == 0
    for bad in (dict(), dict(ws=P, ws_bytes=need - 1), dict(ws=P + 8, ws_bytes=need)):
        assert row(B=3, V=50000, ld=50000, **bad) == WS, bad
    for bad in (dict(prev=None), dict(ts=None), dict(rc=None), dict(pos=None)):
        assert step(**bad) == NULL, bad
    for bad in (dict(u_ld=3, B=4), dict(V=0), dict(min_p=2.0)):
        assert step(**bad) == SHAPE, bad
    assert step(B=0) == 0


def test_tensors_that_do_not_fit_are_refused():
    f = lambda *s: torch.zeros(*s)
    ids, special, counts = torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    good = dict(logits=f(3, 9), V=9, special=special, temp=f(3), u=f(3), ids=ids, counts=counts)
    for key, bad in (("logits", f(3, 9).half()), ("logits", f(2, 9)), ("logits", f(3, 8)), ("logits", f(9, 3).t()), ("logits", f(27)), ("temp", f(2)),
                     ("temp", f(3).double()), ("u", f(6)[::2]), ("ids", counts), ("ids", torch.zeros(6, dtype=torch.int64)[::2]), ("special", ids),
                     ("counts", ids), ("counts", special)):
        a = {**good, key: bad}
        with pytest.raises(RuntimeError, match="sampling: "):
            ops.sample_minp(a["logits"], a["V"], a["special"], a["temp"], 0, 0.9, 0.1, a["u"], a["ids"], a["counts"])
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.sample_minp(good["logits"], 9, special, good["temp"], 0, 0.9, 0.1, good["u"], ids, counts)
    marks, prev, table, pos = torch.zeros(9, dtype=torch.uint8), torch.zeros(3, dtype=torch.int64), f(5, 3), torch.zeros(1, dtype=torch.int32)
    for bad in ((prev.int(), marks, table, pos), (prev[:2], marks, table, pos), (prev, marks.bool(), table, pos), (prev, marks[:8], table, pos),
                (prev, marks, f(5, 2), pos), (prev, marks, f(3, 5).t(), pos), (prev, marks, table, pos.long())):
        with pytest.raises(RuntimeError, match="sampling: "):
            ops.sample_minp_step(good["logits"], 9, special, bad[0], bad[1], f(3), 1.0, 1.0, 0.5, 0, 0.9, 0.1, bad[2], bad[3], 0, ids, counts)
