"""layer_norm of rows whose values are all the same, or nearly: the mean of C equal
float32 values rounds, and 1 / sqrt(eps) would show it."""

import pytest
import torch

from torchsplinekan_amd import layer_norm

WIDTHS = [1, 7, 64, 100, 129, 300, 301, 512, 777, 1000, 2048, 4096, 9999, 16384, 16392]
VALUES = [0.1, 1000.1, -3.3e-3, 12345.678, 3.3e7, 1e30, 1e-30]


def _constant(C, where):
    x = torch.tensor(VALUES, device=where).unsqueeze(1).expand(-1, C).contiguous()
    b = torch.linspace(-1, 1, C, device=where)
    y = layer_norm(x, None, b)
    assert torch.equal(y, b.expand(len(VALUES), -1))
    assert not bool(layer_norm(x).any())


def _nearly(C, where):
    """Values of a few units in the last place about a large one: y against float64 within
    the mean's rounding, half a unit there in units of r (as the values themselves lie on
    units), and some 2^-20 of the sums."""
    g = torch.Generator().manual_seed(C)
    for base, unit in ((1000.0, 2.0 ** -14), (1e6, 2.0 ** -4)):
        x = base + unit * torch.randint(-2, 3, (9, C), generator=g)
        v = x.double()
        v = v - v.mean(1, keepdim=True)
        r = 1 / (v.square().mean(1, keepdim=True) + 1e-5).sqrt()
        got = layer_norm(x.to(where)).cpu().double()
        # (a mean that is off by e moves the variance by e^2: r by less than r^3 e^2 / 2)
        e = unit / 2
        tol = r * e + (v * r).abs() * (r * e) ** 2 / 2 + 2.0 ** -20 * (v * r).abs() + 2.0 ** -20
        assert bool(((got - v * r).abs() <= tol).all())


@pytest.mark.parametrize("C", WIDTHS)
def test_cpu(C):
    _constant(C, "cpu")
    _nearly(C, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("C", WIDTHS)
def test_constant_rows(C):
    _constant(C, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("C", WIDTHS)
def test_nearly_constant_rows(C):
    _nearly(C, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("C", [100, 301, 1000, 16392])
def test_gradients_of_constant_rows(C):
    """x hat is zero: dx = (dy - mean dy) / sqrt(eps), dweight zero."""
    x = torch.full((5, C), 1000.1, device="cuda").requires_grad_()
    w = torch.ones(C, device="cuda").requires_grad_()
    dy = torch.randn(5, C, generator=torch.Generator().manual_seed(0)).cuda()
    dx, dw = torch.autograd.grad(layer_norm(x, w, eps=0.25), [x, w], dy)
    want = 2 * (dy.double() - dy.double().mean(1, keepdim=True))
    assert not bool(dw.any())
    tol = 2 * (C / 64 + 32) * 2.0 ** -24 * (dy.abs() + dy.abs().mean(1, keepdim=True)) + 2.0 ** -24 * want.abs()
    assert bool(((dx - want).abs() <= tol).all())
