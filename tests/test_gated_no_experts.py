"""gated_linear without experts, at widths whose rows would be brought onto 16 bytes."""

import ctypes

import pytest
import torch

from test_grouped import BF16, DTYPES, F16
from torchsplinekan_amd import _lib as lib
from torchsplinekan_amd import gated_linear


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("E,K", [(0, 1023), (1, 0), (0, 0)])
def test_nothing_is_copied(E, K, dtype):
    nbytes = ctypes.c_size_t()
    lib.check(lib.LIB.kan_hip_gated_workspace(lib.OPERATOR_DTYPES[dtype], 4096, 4096, 8192, E, 1024,
                                              K, 0, ctypes.byref(nbytes)))
    assert nbytes.value == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,K", [(8192, 1024, 1023), (8192, 1024, 1024), (20, 3, 5)])
def test_rows_of_no_expert_are_zero(T, N, K, dtype):
    x = torch.randn(T, K, device="cuda").to(dtype).requires_grad_()
    w = torch.zeros(0, 2, N, K, device="cuda", dtype=dtype).requires_grad_()
    for offsets in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
        h = gated_linear(x, w, offsets.cuda())
        assert h.shape == (T, N) and not bool(h.any())
        dx, dw = torch.autograd.grad(h, [x, w], torch.ones_like(h))
        assert not bool(dx.any()) and dw.shape == w.shape
