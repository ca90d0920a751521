"""The norm after a block, its gate and residual scale, and the norm before the
next block, in one pass over a residual stream (no reference counterpart):

    u  = post_weight * y / sqrt(mean(y^2) + eps)      (u = y without post_weight)
    x' = x + scale * gate_act(gate) * u
    h  = pre_weight * x' / sqrt(mean(x'^2) + eps)

Device tensors run on the kernels of csrc/kan_norm.hip, forward and backward;
CPU tensors on the same formulas in torch.
"""

import ctypes
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import fused as _fused

_C = _fused._C
GATE_ACTS = {None: 0, "sigmoid": 1, "tanh": 2, "silu": 3}


def _req(cond: bool, *msg) -> None:
    if not cond:
        raise RuntimeError("residual_norm: " + "".join(str(m) for m in msg))


def _native():
    if _C is None:
        raise RuntimeError("residual_norm: device tensors need libkan_hip.so; build it with "
                           "`python -m torchsplinekan_amd.build_lib`")
    return _C._lib


def _gate_rows(gate: torch.Tensor, x: torch.Tensor) -> int:
    """Rows of a gate (of x's dimensions) whose leading sizes are x's up to one
    point and 1 from there on: each serves a run of consecutive rows of x.  0
    for any other gate."""
    lead, cut, rows = x.shape[:-1], 0, 1
    while cut < len(lead) and gate.shape[cut] == lead[cut]:
        rows *= lead[cut]
        cut += 1
    return rows if all(s == 1 for s in gate.shape[cut:-1]) else 0


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, post, pre, scale, gate_rows, scale_const, act, eps, dtype, wdtype,
                save):
        lib = _native()
        C = x.shape[-1]
        n = x.numel() // C
        new = None if y is None else torch.empty_like(x)
        h = None if pre is None else torch.empty(x.shape, dtype=dtype, device=x.device)
        rstd = torch.empty(2, n, dtype=torch.float32, device=x.device) if save else None
        code = lib.OPERATOR_DTYPES
        codes = (code[x.dtype], code[dtype], code.get(wdtype, lib.KAN_DTYPE_F32))
        gate_cols = 0 if gate is None else gate.shape[-1]
        at = [None if t is None else t.data_ptr()
              for t in (x, y, gate, post, pre, scale, new, h, rstd)]
        lib.launch(lib.LIB.kan_hip_residual_norm, x.device, *codes, *at[:6], scale_const, act,
                   gate_rows, gate_cols, n, C, eps, *at[6:])
        if save:
            ctx.save_for_backward(x, y, gate, post, pre, scale, rstd)
            ctx.args = (codes, gate_rows, gate_cols, scale_const, act, n, C)
            ctx.set_materialize_grads(False)
        return new, h

    @staticmethod
    @once_differentiable
    def backward(ctx, gnew, gh):
        lib = _native()
        x, y, gate, post, pre, scale, rstd = ctx.saved_tensors
        codes, gate_rows, gate_cols, scale_const, act, n, C = ctx.args
        gnew = None if gnew is None else gnew.contiguous()
        gh = None if gh is None else gh.contiguous()
        grads = [torch.empty_like(t) if t is not None and need else None
                 for t, need in zip((x, y, gate, post, pre, scale), ctx.needs_input_grad)]
        if gh is None and grads[4] is not None:
            grads[4].zero_()
        gpre = None if gh is None else grads[4]
        nbytes = ctypes.c_size_t()
        lib.check(lib.LIB.kan_hip_residual_norm_backward_workspace(
            gate_rows, gate_cols, n, C, ctypes.byref(nbytes)))
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=x.device)
        at = [None if t is None else t.data_ptr()
              for t in (gnew, gh, x, y, gate, post, pre, scale, rstd, *grads[:4], gpre, grads[5],
                        ws)]
        lib.launch(lib.LIB.kan_hip_residual_norm_backward, x.device, *codes, *at[:8], scale_const,
                   act, gate_rows, gate_cols, n, C, *at[8:], nbytes.value)
        return (*grads, None, None, None, None, None, None, None)


def _composite(x, y, gate, post, pre, scale, scale_const, act, eps, dtype):
    """The formulas in torch (CPU tensors, empty tensors), in float32 or wider."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32

    def norm(v, w):
        return v * (v.square().mean(-1, keepdim=True) + eps).rsqrt() * w.to(wide)

    new = x.to(wide)
    if y is not None:
        u = y.to(wide) if post is None else norm(y.to(wide), post)
        u = u * (scale_const if scale is None else scale.to(wide))
        if gate is not None:
            g = gate.to(wide)
            u = u * (g if act is None else g.sigmoid() if act == "sigmoid"
                     else g.tanh() if act == "tanh" else g * g.sigmoid())
        new = new + u
    return (x if y is None else new.to(x.dtype),
            None if pre is None else norm(new, pre).to(dtype))


def residual_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None, *,
                  post_weight: Optional[torch.Tensor] = None,
                  pre_weight: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, gate_act: Optional[str] = None,
                  scale: Union[torch.Tensor, float, None] = None, eps: float = 1e-6,
                  dtype: Optional[torch.dtype] = None
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(x', h): the residual stream after a block and the next block's input.

    x [..., C]: the stream before the block, in y's type or float32.
    y [..., C]: the block's output (None: x' is x, only h is taken).
    post_weight [C]: norm of y (None: y is added as it is).
    pre_weight [C]: norm of x' for the next block (None: h is None).
    gate: broadcasts against x, with 1 or C values in its last dimension (one
    for an element, a token, a sequence [B, 1, C], ...), in y's type; gate_act
    None, "sigmoid", "tanh" or "silu" is applied to it.
    scale: residual scale, [C] or a number.
    dtype: type of h without y (default: x's).
    post_weight, pre_weight and a scale tensor share a type.  First-order
    gradients reach every tensor (device tensors refuse forward mode); x' is not kept for them (the backward
    evaluates it again from x and y)."""
    _req(x.dim() >= 1, "x must have at least one dimension")
    shape, C, device = x.shape, x.shape[-1], x.device
    _req(gate_act in GATE_ACTS, "gate_act must be None, 'sigmoid', 'tanh' or 'silu', got ",
         repr(gate_act))
    if y is None:
        _req(post_weight is None and gate is None and scale is None,
             "post_weight, gate and scale need a branch y")
        dtype = x.dtype if dtype is None else dtype
        if pre_weight is None:
            return x, None
    else:
        _req(y.shape == shape, "y must have x's shape ", list(shape), ", got ", list(y.shape))
        _req(dtype is None or dtype == y.dtype, "with y, h is in y's type ", y.dtype)
        dtype = y.dtype
        _req(y.device == device, "tensors must be on one device")
    _req(gate is not None or gate_act is None, "gate_act needs a gate")
    _req(x.dtype == dtype or x.dtype == torch.float32,
         "x must be in the branch's type or float32, got ", x.dtype, " and ", dtype)
    scale_t, scale_const = None, 1.0
    if isinstance(scale, torch.Tensor):
        scale_t = scale
    elif scale is not None:
        scale_const = float(scale)
    wdtype = None
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("scale", scale_t)):
        if t is None:
            continue
        _req(t.dim() == 1 and t.shape[0] == C, name, " must have shape [", C, "], got ",
             list(t.shape))
        _req(wdtype is None or t.dtype == wdtype,
             "post_weight, pre_weight and scale must share a dtype")
        _req(t.device == device, "tensors must be on one device")
        wdtype = t.dtype
    gate_rows = 0
    if gate is not None:
        _req(gate.dtype == dtype, "gate must be in the branch's type ", dtype, ", got ", gate.dtype)
        _req(1 <= gate.dim() <= x.dim() and gate.shape[-1] in (1, C)
             and all(g in (1, s) for g, s in zip(gate.shape[-2::-1], shape[-2::-1])),
             "gate of shape ", list(gate.shape), " does not broadcast against ", list(shape))
        _req(gate.device == device, "tensors must be on one device")
    if not x.is_cuda or x.numel() == 0:
        return _composite(x, y, gate, post_weight, pre_weight, scale_t, scale_const, gate_act, eps,
                          dtype)
    lib = _native()
    for t in (x.dtype, dtype, wdtype):
        if t is not None and t not in lib.OPERATOR_DTYPES:
            lib.operator_dtype_code(t, "residual_norm")  # (raises)
    if gate is not None:
        if gate.dim() < x.dim():
            gate = gate.reshape((1,) * (x.dim() - gate.dim()) + tuple(gate.shape))
        gate_rows = _gate_rows(gate, x)
        if gate_rows == 0:
            # broadcast over leading dimensions: one gate row for every row of
            # x, in float32, so that its gradient is rounded once, after the sum
            new, h = residual_norm(
                x.float(), y.float(), post_weight=post_weight, pre_weight=pre_weight,
                gate=gate.float().expand(*shape[:-1], gate.shape[-1]), gate_act=gate_act,
                scale=scale, eps=eps)
            return new.to(x.dtype), None if h is None else h.to(dtype)
    tensors = [t if t is None or t.is_contiguous() else t.contiguous()
               for t in (x, y, gate, post_weight, pre_weight, scale_t)]
    save = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    args = (gate_rows, scale_const, GATE_ACTS[gate_act], float(eps), dtype, wdtype, save)
    if save or _forward_ad._current_level >= 0:  # (apply refuses forward-mode derivatives)
        new, h = _ResidualNorm.apply(*tensors, *args)
    else:
        new, h = _ResidualNorm.forward(None, *tensors, *args)
    return (x if new is None else new), h
