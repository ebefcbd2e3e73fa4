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


def test_columns_of_one_entry_have_no_stride():
    one, ids = torch.ones(1), torch.empty(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.sample_minp(torch.zeros(1, 4).t(), 1, None, torch.ones(4), 0, 0.9, 0.0, torch.ones(4), torch.empty(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.sample_minp_step(torch.zeros(1, 9), 9, None, ids, torch.zeros(9, dtype=torch.uint8), one, 1.0, 1.0, 0.5, 0, 0.9, 0.0,
                             torch.rand(5).as_strided((5, 1), (1, 5)), torch.zeros(1, dtype=torch.int32), 0, ids)


@pytest.mark.gpu
def test_a_step_of_one_row_reads_its_uniforms_down_the_column():
    x, u = torch.randn(1, 300, device="cuda"), torch.rand(5, device="cuda")
    ts, pos = torch.zeros(300, dtype=torch.uint8, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    got = []
    for table in (u[:, None].contiguous(), u.as_strided((5, 1), (1, 5))):
        prev, out = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.empty(1, dtype=torch.int64, device="cuda")
        ops.sample_minp_step(x, 300, None, prev, ts, torch.zeros(1, device="cuda"), 1.0, 1.0, 0.0, 0, 1.0, 0.0, table, pos, 0, out)
        got.append(int(out))
    want = torch.empty(1, dtype=torch.int64, device="cuda")
    ops.sample_minp(x, 300, None, torch.ones(1, device="cuda"), 0, 1.0, 0.0, u[3:4].contiguous(), want)
    assert got == [int(want)] * 2
