"""Refusals of me_sample_minp and me_sample_minp_step: made on the host, before anything is enqueued (addresses are never touched)."""
from midiemo import _lib

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
