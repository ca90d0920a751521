"""Calls recorded by torch.jit.trace compute on the inputs they are replayed with, and
make_fx, which cannot record the device kernels, is refused."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from torchsplinekan_amd import (KANExpertStack, KANLinear, _lib, gated_linear, grouped_linear,
                                layer_norm, linear_cross_entropy, linear_distillation,
                                quantize_activation, residual_norm)


class _Twice(torch.autograd.Function):
    """Writes its result past torch's operations, as a launch does."""

    @staticmethod
    def forward(ctx, x):
        y = torch.empty_like(x)
        y.detach().numpy()[:] = 2 * x.detach().numpy()
        return y

    @staticmethod
    def backward(ctx, g):
        return 2 * g


def test_a_traced_call_is_recorded():
    traced = torch.jit.trace(lambda x: _lib.call(_Twice, False, x), (torch.zeros(3),))
    x = torch.arange(1.0, 4.0, requires_grad=True)
    y = traced(x)
    assert torch.equal(y, 2 * x)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.full((3,), 2.0))
    assert not _lib.traced() and _lib.call(_Twice, False, x).grad_fn is None
    assert _lib.call(_Twice, True, x).grad_fn is not None


def test_make_fx_is_refused():
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(lambda x: _lib.call(_Twice, False, x))(torch.zeros(3))
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(lambda x: _lib.call(_Twice, True, x))(torch.zeros(3))


# ---------------------------------------------------------------------------
# device
# ---------------------------------------------------------------------------

def _cases():
    """name: (function of x [T, 64], whose result or results are float tensors)"""
    torch.manual_seed(0)
    w, b = torch.randn(64).cuda(), torch.randn(64).cuda()
    up, head = torch.randn(2, 48, 64).cuda() / 8, torch.randn(100, 64).cuda() / 8
    experts, off = torch.randn(3, 40, 64).cuda() / 8, torch.tensor([0, 9, 9, 20]).cuda()
    target, ids = torch.randint(100, (23,)).cuda(), torch.randint(100, (23, 4)).cuda()
    teacher = torch.randn(23, 4).cuda()
    layer, stack = KANLinear(64, 32).cuda(), KANExpertStack(64, 2, 4, feed_forward=32,
                                                            input_norm=True).cuda()

    def eight(x, format):
        kept = quantize_activation(x, 32, format)
        return kept.dequantize(), kept.scale

    return {
        "layer_norm": lambda x: layer_norm(x, w, b),
        "gated_linear": lambda x: gated_linear(x, up),
        "gated_linear by expert": lambda x: gated_linear(x, experts.reshape(3, 2, 20, 64), off),
        "grouped_linear": lambda x: grouped_linear(x, experts, off),
        "linear_cross_entropy": lambda x: linear_cross_entropy(x, head, target),
        "linear_distillation": lambda x: linear_distillation(x, head, ids, teacher, reduction="none"),
        "residual_norm": lambda x: residual_norm(x, x * 2, pre_weight=w, post_weight=b),
        "quantize_activation int8": lambda x: eight(x, "int8"),
        "quantize_activation e4m3": lambda x: eight(x, "e4m3"),
        "KANLinear": layer,
        "KANExpertStack": stack,
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", [
    "layer_norm", "gated_linear", "gated_linear by expert", "grouped_linear",
    "linear_cross_entropy", "linear_distillation", "residual_norm", "quantize_activation int8",
    "quantize_activation e4m3", "KANLinear", "KANExpertStack"])
@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls_take_new_inputs(name, grad):
    fn = _cases()[name]
    many = lambda r: list(r) if isinstance(r, (tuple, list)) else [r]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(fn, (torch.randn(23, 64, device="cuda"),), check_trace=False)
    for seed in (1, 2):
        x = torch.randn(23, 64, generator=torch.Generator().manual_seed(seed)).cuda()
        # (training's forward of a KAN layer adds in another order than inference's)
        with torch.no_grad():
            for got, want in zip(many(traced(x)), many(fn(x))):
                torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)
        if "quantize" in name:
            continue
        xg = x.requires_grad_()
        got = torch.autograd.grad([r.sum() for r in many(traced(xg))], xg)[0]
        want = torch.autograd.grad([r.sum() for r in many(fn(xg))], xg)[0]
        torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_make_fx_of_device_calls_is_refused():
    x, w = torch.randn(5, 64, device="cuda"), torch.ones(64, device="cuda")
    for fn in (lambda v: layer_norm(v, w), lambda v: quantize_activation(v).dequantize(),
               KANLinear(64, 8).cuda()):
        with pytest.raises(RuntimeError, match="make_fx"), torch.no_grad():
            make_fx(fn)(x)
