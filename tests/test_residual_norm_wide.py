"""residual_norm on the shapes that few rows of test_residual_norm.py reach: rows
wider than 16384, which stay in memory, with several rows to a block of the
backward pass, and gate rows of rows that several waves share.  Its cases and
bounds; the formulas run in float64 on the device, the tensors being large."""

import pytest
import torch

import test_residual_norm as base

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
WIDE = [16392, 16401]  # whole vectors of every type, and of none


@pytest.fixture(autouse=True)
def formulas_on_the_device(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "cpu", lambda self: self.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("xdt,ydt", base.TYPES)
@pytest.mark.parametrize("C", WIDE)
def test_types(C, xdt, ydt):
    base._run_case((33, C), xdt, ydt, (33, C), "tanh", True)


@pytest.mark.gpu
@pytest.mark.parametrize("C", WIDE)
@pytest.mark.parametrize("kw", [
    dict(post=False), dict(pre=False), dict(post=False, pre=False), dict(y=False),
    dict(use=("new",)), dict(use=("h",)), dict(wdt=F32)])
def test_optional_parts(C, kw):
    branch = kw.get("y") is not False
    base._run_case((33, C), BF16, BF16, (33, 1) if branch else None, "silu" if branch else None,
                   branch, **kw)


@pytest.mark.gpu
def test_number_as_scale_and_type_of_h():
    base._run_case((9, WIDE[0]), F32, BF16, None, None, 0.25)
    base._run_case((9, WIDE[1]), F32, F16, None, None, None, y=False, dtype=F16)


@pytest.mark.gpu
@pytest.mark.parametrize("C", WIDE)
def test_strides_alignment_and_values_that_are_not_finite(C):
    base.test_strides_and_alignment(C)
    base.test_values_that_are_not_finite_stay_in_their_row(C)


@pytest.mark.gpu
@pytest.mark.parametrize("xdt,ydt", [(F32, F32), (F32, BF16)])
@pytest.mark.parametrize("gate", [None, (2, 650, 1), (2, 650, WIDE[1]), (1,), (2, 1, 1),
                                  (2, 1, WIDE[1]), (WIDE[1],)])
def test_several_rows_to_a_block(gate, xdt, ydt):
    """1300 rows on 1024 blocks: a block adds its rows' sums up."""
    base._run_case((2, 650, WIDE[1]), xdt, ydt, gate, gate and "sigmoid", True)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,L", [(650, 2), (433, 3), (2050, 2)])
def test_short_sequences(seqs, L):
    """Gate rows of as many rows as a block has, of more, and of fewer."""
    base._run_case((seqs, L, WIDE[0]), F32, F32, (seqs, 1, WIDE[0]), "tanh", True)
    base._run_case((seqs, L, WIDE[0]), BF16, BF16, (seqs, 1, 1), "silu", True)


@pytest.mark.gpu
@pytest.mark.parametrize("xdt,ydt", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("C,seqs,L", [
    (1032, 2, 1500), (1032, 7, 700), (1032, 600, 2), (1032, 1300, 3), (1035, 9, 111),
    (4096, 2, 1500), (4096, 600, 2), (4096, 700, 3), (4099, 3, 500),
    (9000, 2, 700), (9000, 400, 2), (9001, 5, 111), (16384, 3, 200)])
def test_gate_rows_of_rows_that_waves_share(C, seqs, L, xdt, ydt):
    base._run_case((seqs, L, C), xdt, ydt, (seqs, 1, C), "tanh", True)


@pytest.mark.gpu
@pytest.mark.parametrize("C,cols", [(8, 8), (300, 300), (8, 1)])
def test_more_gate_rows_than_a_grid_is_high(C, cols):
    base._run_case((70000, 2, C), F32, F32, (70000, 1, cols), "sigmoid", True)
