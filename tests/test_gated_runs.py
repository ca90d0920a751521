"""The weight gradient of gated_linear without offsets, a product whose rows are cut into runs
on either tile: what the plan says it runs on, and its values (bounds of test_gated)."""

import ctypes

import pytest

from test_gated import _check, _inputs
from test_grouped import BF16, F16
from torchsplinekan_amd import _lib as lib

WEIGHT = 2
# T, outputs of both weights, K: rows of a tile, of a run (0: all are one), operands that are
# brought onto 16 bytes first
PLANS = [(10001, 3000, 1030, 256, 2560, 2), (8200, 8192, 512, 256, 2752, 0),
         (5000, 2048, 1024, 128, 1728, 0), (4100, 264, 136, 128, 576, 0),
         (2000, 64, 40, 128, 704, 0), (1100, 640, 512, 128, 0, 0)]


def _plan(dtype, T, N, K, dense=True):
    plan = (ctypes.c_int64 * 6)()
    code = lib.OPERATOR_DTYPES[dtype]
    if dense:
        lib.check(lib.LIB.kan_hip_grouped_matmul_dense_plan(code, WEIGHT, 4096, 4096, T, N, K, plan))
    else:
        lib.check(lib.LIB.kan_hip_grouped_matmul_plan(code, WEIGHT, 4096, 4096, 0, T, 1, N, K, plan))
    return list(plan)


@pytest.mark.parametrize("T,N,K,rows,run,align", PLANS)
def test_plans(T, N, K, rows, run, align):
    plan = _plan(BF16, T, N, K)
    assert (plan[0], plan[2], plan[4]) == (rows, run, align)
    assert run == 0 or T % run      # (the last run is a part of one)


def test_offsets_are_planned_otherwise():
    assert _plan(BF16, 8200, 8192, 512) != _plan(BF16, 8200, 8192, 512, dense=False)
    assert lib.LIB.kan_hip_grouped_matmul_dense_plan(1, WEIGHT, None, None, 4, 4, 4, None) \
        == lib.KAN_ERR_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,N,K,rows,run,align", PLANS)
def test_values(T, N, K, rows, run, align, dtype):
    plan = _plan(dtype, T, N, K)
    assert (plan[0], plan[2], plan[4]) == (rows, run, align)
    _check(*_inputs(T, 1, K, N // 2, dtype, seed=T), None, where="cuda")
