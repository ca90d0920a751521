"""layer_norm from float32 to float16, past 2^31 values, and gated_linear past them; the
operators of a training step under the device's autocast.  (Bounds: test_layer_norm,
test_gated.)"""

import pytest
import torch

from test_gated import _expected, _near
from test_layer_norm import BF16, EPS, F16, F32, _check, _inputs
from torchsplinekan_amd import (gated_linear, layer_norm, linear_cross_entropy,
                                linear_distillation)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wdt", [F32, F16])
@pytest.mark.parametrize("C", [7, 64, 136, 256, 301, 1000, 4096, 8192, 9999, 16384, 16385])
def test_layer_norm_of_a_float32_stream_in_float16(C, wdt):
    _check(*_inputs((77, C), F32, F16, wdt, seed=C))


def test_layer_norm_past_2_31_values():
    """Rows as in a call of their own, bit for bit; the weight's and the bias's sums, of
    n / 64 + 64 terms in a chain at most, in float64 a piece at a time."""
    n, C, step = 2200003, 1000, 100000
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(n, C, device="cuda", dtype=BF16).normal_(generator=g).requires_grad_()
    dy = torch.empty(n, C, device="cuda", dtype=BF16).normal_(generator=g)
    w = torch.linspace(0.5, 1.5, C, device="cuda").requires_grad_()
    b = torch.zeros(C, device="cuda").requires_grad_()
    y = layer_norm(x, w, b, eps=EPS)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    for lo in (0, (1 << 31) // C - 500, n - 1000):
        r = slice(lo, lo + 1000)
        xs = x[r].detach().requires_grad_()
        ys = layer_norm(xs, w, b, eps=EPS)
        assert torch.equal(y[r], ys)
        assert torch.equal(dx[r], torch.autograd.grad(ys, xs, dy[r])[0])
    sums = [torch.zeros(C, device="cuda", dtype=torch.float64) for _ in range(4)]
    for lo in range(0, n, step):
        xs, d = x[lo:lo + step].detach().double(), dy[lo:lo + step].double()
        xs = xs - xs.mean(1, keepdim=True)
        xh = xs / (xs.square().mean(1, keepdim=True) + EPS).sqrt()
        for s, v in zip(sums, (d * xh, (d * xh).abs(), d, d.abs())):
            s += v.sum(0)
    # (x hat is off by (C / 64 + 128) 2^-24 H, where H = r X + |x hat| R < 16 here)
    u = 2.0 ** -24
    tol_w = (n / 64 + 64) * u * sums[1] + (C / 64 + 128) * u * 16 * sums[3]
    assert bool(((dw.double() - sums[0]).abs() <= tol_w).all())
    assert bool(((db.double() - sums[2]).abs() <= (n / 64 + 64) * u * sums[3]).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gated_linear_past_2_31_values(dtype):
    T, K, N, step = 600011, 40, 2048, 20000
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(T, K, device="cuda", dtype=dtype).normal_(generator=g)
    w = (torch.empty(2, N, K, device="cuda").normal_(generator=g) / 8).to(dtype)
    dh = torch.empty(T, N, device="cuda", dtype=dtype).normal_(generator=g)
    x.requires_grad_()
    h = gated_linear(x, w)
    dx, = torch.autograd.grad(h, x, dh)
    for lo in (0, (1 << 31) // (2 * N) - step // 2, (1 << 30) // N - step // 2, T - step):
        r = slice(lo, lo + step)
        want = _expected(x[r].detach().double(), w.double(), dh[r].double(), "silu", dtype)
        _near(h[r], want["h"], "h")
        _near(dx[r], want["dx"], "dx")


@pytest.mark.parametrize("cast", [BF16, F16])
def test_autocast_casts_nothing(cast):
    torch.manual_seed(0)
    x = torch.randn(70, 64, device="cuda").requires_grad_()
    w, up = torch.randn(64, device="cuda"), torch.randn(2, 48, 64, device="cuda") / 8
    head, target = torch.randn(100, 64, device="cuda") / 8, torch.randint(100, (70,), device="cuda")
    ids, teacher = torch.randint(100, (70, 3), device="cuda"), torch.randn(70, 3, device="cuda")
    for fn in (lambda: layer_norm(x, w), lambda: gated_linear(x, up),
               lambda: linear_cross_entropy(x, head, target),
               lambda: linear_distillation(x, head, ids, teacher)):
        want = fn()
        grad = torch.autograd.grad(want.sum(), x)[0]
        with torch.autocast("cuda", dtype=cast):
            got = fn()
        assert got.dtype == F32 and torch.equal(got, want)
        assert torch.equal(torch.autograd.grad(got.sum(), x)[0], grad)
