"""What the sampling calls refuse, or take, of layouts and devices beside test_sample_minp_cpu.py."""
import pytest
import torch

from midiemo import ops


def test_rows_too_far_apart_are_refused():
    """a row stride is a C int: 2^32 + 16 would arrive as 16 and read other rows (meta tensors: no memory behind them)"""
    far = torch.empty(2, 2 ** 32 + 16, device="meta")[:, :9]
    one, ids = torch.ones(2), torch.empty(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="2.31 elements apart"):
        ops.sample_minp(far, 9, None, one, 0, 0.9, 0.0, one, ids)
    with pytest.raises(RuntimeError, match="no CPU path"):      # a single row has no next one
        ops.sample_minp(torch.empty(1, 2 ** 32 + 16, device="meta")[:, :9], 9, None, one[:1], 0, 0.9, 0.0, one[:1], ids[:1])


@pytest.mark.gpu
def test_a_single_row_may_have_any_stride():
    x = torch.randn(1, 4, 300, device="cuda")
    one, ids = torch.ones(1, device="cuda"), torch.empty(1, dtype=torch.int64, device="cuda")
    for row in (x[:, 2], x[0, 2].expand(1, 300), x[0, 2].as_strided((1, 300), (7, 1))):
        ops.sample_minp(row, 300, None, one, 1, 1.0, 0.0, one * 0.5, ids)
        assert int(ids) == int(row.argmax())


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["marks", "table", "pos"])
def test_a_step_with_a_tensor_elsewhere_is_refused(which):
    t = dict(marks=torch.zeros(50, dtype=torch.uint8), table=torch.zeros(4, 2), pos=torch.zeros(1, dtype=torch.int32))
    t = {k: v if k == which else v.cuda() for k, v in t.items()}
    prev, rc = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(RuntimeError, match="sampling: "):
        ops.sample_minp_step(torch.zeros(2, 50, device="cuda"), 50, None, prev, t["marks"], rc, 1.0, 1.0, 0.5, 0, 0.9, 0.0, t["table"], t["pos"], 0, prev)
