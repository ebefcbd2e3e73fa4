"""Layouts that QuantKVCache takes: dimensions of one entry, whose stride means nothing."""
import pytest
import torch

from midiemo.kvcache import QuantKVCache


def singles(B, H, dh):
    """new rows whose strides differ, or are no multiple of 16 bytes, in dimensions of one entry only"""
    base = torch.randn(B, H, dh)
    other = torch.randn(B * H * dh + 64)
    yield base, other[:B * H * dh].as_strided((B, H, dh), (7 if B == 1 else H * dh, 3 if H == 1 else dh, 1))
    yield other[:B * H * dh].as_strided((B, H, dh), (7 if B == 1 else H * dh, 3 if H == 1 else dh, 1)), base


@pytest.mark.parametrize("B,H", [(1, 3), (2, 1), (1, 1)])
def test_new_rows_of_one_sequence_or_head_pass_the_checks(B, H):
    c = QuantKVCache(B, H, 32, 64, 4, device="cpu")
    q = torch.zeros(B, H, 64)
    for k, v in singles(B, H, 64):
        with pytest.raises(RuntimeError, match="no CPU path"):
            c.append_attend(q, k, v, 3)
    with pytest.raises(RuntimeError, match="kv cache: new rows"):       # real strides have to be equal
        QuantKVCache(2, 3, 32, 64, 4, device="cpu").append_attend(torch.zeros(2, 3, 64), torch.zeros(2, 3, 64), torch.zeros(2, 3, 128)[..., :64], 3)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H", [(1, 3), (2, 1), (1, 1)])
def test_new_rows_of_one_sequence_or_head_are_written(B, H):
    q = torch.randn(B, H, 64, device="cuda")
    for k, v in singles(B, H, 64):
        a, b = QuantKVCache(B, H, 32, 64, 4), QuantKVCache(B, H, 32, 64, 4)
        dk, dv = (torch.zeros(B * H * 64, device="cuda").as_strided(x.shape, x.stride()).copy_(x) for x in (k, v))
        out = a.append_attend(q, dk, dv, 0)
        b.write(dk[:, None], dv[:, None], 0)
        for name in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(a, name), getattr(b, name))
        held = b.read(0, 1)[1][:, 0]
        assert bool(((out - held).abs() <= held.abs() * 2.0 ** -20).all())      # the only key: the value as it is held
