"""gated_linear's gradients in float16 at upstream gradients far from 1: dg and du
leave the type's range long before dx and dw do.

Bound: dg and du carry one rounding and the results another, each a uniform error of at
most H = 2^-11 relatively, H (2 / 3)^(1/2) normwise; a result below the smallest normal
value is off by up to 2^-25 more.  dg and du themselves, stored so that the largest lies at
2^14 and more, lose what is below 2^-25 / 2^14 of the largest: nothing of this."""

import pytest
import torch

from test_gated import _act, _inputs
from test_grouped import F16, _offsets
from torchsplinekan_amd import _lib as lib
from torchsplinekan_amd import gated_linear

H = 2.0 ** -11


def _gradients(x, w, dh, offsets, act):
    """dx and dw in float64."""
    x, w, dh = x.double(), w.double(), dh.double()
    dx, dw, lo = torch.zeros_like(x), torch.zeros_like(w), 0
    ends = [len(x)] if offsets is None else offsets.tolist()[1:]
    for e, hi in enumerate(ends):
        r = slice(lo, hi)
        g, u = x[r] @ w[e, 0].t(), x[r] @ w[e, 1].t()
        a, slope = _act(g, act)
        d = [dh[r] * u * slope, dh[r] * a]
        dx[r] = d[0] @ w[e, 0] + d[1] @ w[e, 1]
        dw[e, 0], dw[e, 1] = d[0].t() @ x[r], d[1].t() @ x[r]
        lo = hi
    return dx, dw


def _near(got, want):
    error = (got.double() - want).norm()
    return float(error) <= H * (2 / 3) ** 0.5 * float(want.norm()) + 2.0 ** -25 * want.numel() ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -22, 1e-6, 1e-5, 1e-4, 1.0, 30.0, 3e3])
@pytest.mark.parametrize("counts,N,K,act", [
    ([4096], 128, 128, "silu"), ([2000], 129, 77, "gelu"), ([300, 0, 1700], 64, 40, None),
    ([1], 512, 64, "silu"), ([5, 4], 33, 31, "tanh")])
def test_gradients_at_every_size(counts, N, K, act, size):
    """(Weights of 2^-6 of the usual size at the largest gradients, so that dx and dw
    themselves are within the type.)"""
    T, E = sum(counts), len(counts)
    x, w, dh = _inputs(T, E, K, N, F16)
    off = None if E == 1 else _offsets(counts).cuda()
    x, w = x.cuda(), w.cuda()
    dh = (dh.float().cuda() * size).to(F16)
    if size > 1:
        x = (x.float() * 2.0 ** -6).to(F16)
        w[:, 1] = (w[:, 1].float() * 2.0 ** 6).to(F16)   # u as before, h and du small
        w[:, 0] = (w[:, 0].float() * 2.0 ** -2).to(F16)
    want = _gradients(x, w, dh, off, act)
    if not all(float(v.abs().max()) < 6e4 for v in want):
        pytest.skip("results beyond the type")
    x.requires_grad_(), w.requires_grad_()
    h = gated_linear(x, w if off is not None else w[0], off, act=act)
    for got, ref in zip(torch.autograd.grad(h, [x, w], dh), want):
        assert _near(got, ref)


@pytest.mark.gpu
def test_products_beyond_the_type_with_gradients_within():
    """dg and du pass 65504 where dx, over weights that are small, does not."""
    x, w, dh = _inputs(500, 1, 64, 96, F16)
    x, w = x.cuda(), (w.float() * 2.0 ** -8).cuda().to(F16)
    w[:, 1] = (w[:, 1].float() * 2.0 ** 8).to(F16)
    dh = (dh.float() * 3e4).clamp(-6e4, 6e4).cuda().to(F16)
    want = _gradients(x, w, dh, None, None)[0]
    g, u = x.double() @ w[0, 0].double().t(), x.double() @ w[0, 1].double().t()
    assert float((dh.double() * u).abs().max()) > 2 * 65504 and float(want.abs().max()) < 6e4
    x.requires_grad_()
    dx, = torch.autograd.grad(gated_linear(x, w[0], act=None), x, dh)
    assert _near(dx, want)


@pytest.mark.gpu
def test_gradients_that_are_not_finite_leave_the_factor_alone():
    x, w, dh = _inputs(200, 1, 64, 96, F16)
    x, w, dh = x.cuda().requires_grad_(), w[0].cuda(), (dh.float() * 1e-5).cuda().to(F16)
    dh[7, 3], dh[150, 0] = float("inf"), float("nan")
    dx, = torch.autograd.grad(gated_linear(x, w), x, dh)
    keep = [i for i in range(200) if i not in (7, 150)]
    assert _near(dx[keep], _gradients(x.detach(), w[None], dh, None, "silu")[0][keep])
    assert not bool(dx[7].isfinite().all()) and not bool(dx[150].isfinite().all())
    dx, = torch.autograd.grad(gated_linear(x, w), x, torch.zeros_like(dh))
    assert not bool(dx.any())


@pytest.mark.gpu
def test_replays_take_the_factor_of_their_own_gradient():
    x, w, dh = _inputs(300, 1, 64, 96, F16)
    x, w, dh = x.cuda().requires_grad_(), w[0].cuda().requires_grad_(), dh.cuda()
    step = lambda: torch.autograd.grad(gated_linear(x, w), [x, w], dh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for size in (1.0, 2.0 ** -10, 2.0 ** 8):
        dh.mul_(size)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_c_entry_refusals():
    L, p = lib.LIB, 4096
    back, mm = L.kan_hip_gated_backward_scaled, L.kan_hip_grouped_matmul_scaled
    assert back(lib.KAN_DTYPE_BF16, 3, p, p, 4, 16, p, p, None) == lib.KAN_ERR_INVALID
    assert back(lib.KAN_DTYPE_F16, 3, p, p, 4, 16, p, None, None) == lib.KAN_ERR_INVALID
    assert back(lib.KAN_DTYPE_F16, 3, None, p, 4, 16, p, p, None) == lib.KAN_ERR_INVALID
    assert back(lib.KAN_DTYPE_F16, 3, None, None, 0, 16, None, p, None) == lib.KAN_OK

    def call(dtype=lib.KAN_DTYPE_F16, op=1, scale=p, T=0):
        return mm(dtype, op, p, p, p, 0, T, 1, 16, 16, scale, p, None, 0, None)

    assert call() == lib.KAN_OK
    assert call(dtype=lib.KAN_DTYPE_F32) == lib.KAN_ERR_INVALID
    assert call(op=0) == lib.KAN_ERR_INVALID
    assert call(scale=None) == lib.KAN_ERR_INVALID
