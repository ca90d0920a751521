"""Layer norm with its backward pass (no reference counterpart):

    y = weight * (x - mean(x)) / sqrt(mean((x - mean(x))^2) + eps) + bias

Device tensors run on the kernels of csrc/kan_layernorm.hip, forward and
backward; CPU tensors on the same formulas in torch.
"""

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import fused as _fused

_C = _fused._C


def _refuse(*msg) -> None:
    raise RuntimeError("layer_norm: " + "".join(str(m) for m in msg))


def _native():
    if _C is None:
        raise RuntimeError("layer_norm: device tensors need libkan_hip.so; build it with "
                           "`python -m torchsplinekan_amd.build_lib`")
    return _C._lib


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, dtype):
        lib = _native()
        save = ctx is not None and any(ctx.needs_input_grad)
        C = x.shape[-1]
        n = x.numel() // C
        y = torch.empty(x.shape, dtype=dtype, device=x.device)
        stats = torch.empty(2, n, dtype=torch.float32, device=x.device) if save else None
        code = lib.OPERATOR_DTYPES
        wdtype = (weight if weight is not None else bias if bias is not None else y).dtype
        codes = (code[x.dtype], code[dtype], code[wdtype])
        at = [None if t is None else t.data_ptr() for t in (x, weight, bias, y, stats)]
        lib.launch(lib.LIB.kan_hip_layer_norm, x.device, *codes, *at[:3], n, C, eps, *at[3:])
        if save:
            ctx.save_for_backward(x, weight, bias, stats)
            ctx.args = (codes, n, C)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        lib = _native()
        x, weight, bias, stats = ctx.saved_tensors
        codes, n, C = ctx.args
        dy = dy.contiguous()
        grads = [torch.empty_like(t) if t is not None and need else None
                 for t, need in zip((x, weight, bias), ctx.needs_input_grad)]
        nbytes, ws = ctypes.c_size_t(), None
        if grads[1] is not None or grads[2] is not None:
            lib.check(lib.LIB.kan_hip_layer_norm_backward_workspace(n, C, ctypes.byref(nbytes)))
            ws = torch.empty(nbytes.value, dtype=torch.uint8, device=x.device)
        at = [None if t is None else t.data_ptr() for t in (dy, x, weight, stats, *grads, ws)]
        lib.launch(lib.LIB.kan_hip_layer_norm_backward, x.device, *codes, *at[:4], n, C, *at[4:],
                   nbytes.value)
        return (*grads, None, None)


def _composite(x, weight, bias, eps, dtype):
    """The formula in torch (CPU tensors, empty tensors), in float32 or wider."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    v = x.to(wide)
    m = v.mean(-1, keepdim=True)
    v = v - (m + (v - m).mean(-1, keepdim=True))  # (a constant row becomes zero)
    v = v * (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    if weight is not None:
        v = v * weight.to(wide)
    return (v if bias is None else v + bias.to(wide)).to(dtype)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The layer norm of x [..., C] over its last dimension.

    weight, bias [C] (None: 1 and 0) share a type.
    dtype: type of the result (default: x's); x is in that type or in float32.
    Statistics and sums are held in float32.  First-order gradients reach x,
    weight and bias (device tensors refuse forward mode); sums over rows have a
    fixed order."""
    if x.dim() < 1:
        _refuse("x must have at least one dimension")
    C, dtype = x.shape[-1], x.dtype if dtype is None else dtype
    if x.dtype != dtype and x.dtype != torch.float32:
        _refuse("x must be in the result's type or float32, got ", x.dtype, " and ", dtype)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != C:
            _refuse(name, " must have shape [", C, "], got ", list(t.shape))
        if t.device != x.device:
            _refuse("tensors must be on one device")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        _refuse("weight and bias must share a dtype")
    if not x.is_cuda or x.numel() == 0:
        return _composite(x, weight, bias, eps, dtype)
    lib = _native()
    for t in (x, weight, bias):
        if t is not None and t.dtype not in lib.OPERATOR_DTYPES:
            lib.operator_dtype_code(t.dtype, "layer_norm")  # (raises)
    lib.operator_dtype_code(dtype, "layer_norm")
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    save = torch.is_grad_enabled() and (
        x.requires_grad or weight is not None and weight.requires_grad
        or bias is not None and bias.requires_grad)
    return lib.call(_LayerNorm, save, x, weight, bias, float(eps), dtype)
