"""Activations kept in 8 bits between the forward and the backward pass (no
reference counterpart; the reference bounds memory by recomputation only).

``quantize_activation`` keeps a tensor as 8-bit values with one float32 scale
for every group of its last axis; ``checkpoint_8bit`` runs a layer that keeps
nothing but its input, in 8 bits, and runs again in the backward pass: a KAN
layer then holds 1 byte an input instead of the 4 (R + 1) of its basis.
Device tensors run on the kernels of csrc/kan_act8.hip, CPU tensors on the same
formulas in torch.
"""

from contextlib import ExitStack
from dataclasses import dataclass
from typing import Callable, Optional, Sequence

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import fused as _fused

_C = _fused._C
FORMATS = {"int8": (1, 127.0, torch.int8), "e4m3": (2, 448.0, torch.float8_e4m3fn)}
GROUPS = (32, 64, 128, 256)


def _req(cond: bool, *msg) -> None:
    if not cond:
        raise RuntimeError("".join(str(m) for m in msg))


def check_format(who: str, group: int, format: str) -> None:
    _req(format in FORMATS, who, ": format must be 'int8' or 'e4m3', got ", repr(format))
    _req(group in GROUPS, who, ": group must be 32, 64, 128 or 256, got ", group)


def _native(who: str):
    if _C is None:
        raise RuntimeError(f"{who}: device tensors need libkan_hip.so; build it with "
                           "`python -m torchsplinekan_amd.build_lib`")
    return _C._lib


@dataclass(eq=False)
class Activation8:
    """A tensor in 8 bits: q (int8 or float8_e4m3fn, the tensor's shape), scale
    [..., ceil(C / group)] float32, and the type it had.  A group that held an
    infinity or a NaN has scale NaN and comes back as NaN; one whose scale
    would be below the smallest normal float32 comes back as zeros."""

    q: torch.Tensor
    scale: torch.Tensor
    group: int
    format: str
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.q.numel() + 4 * self.scale.numel()

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The tensor, each value q * scale rounded to dtype (default: its own)."""
        dtype = self.dtype if dtype is None else dtype
        if not self.q.is_cuda or self.q.numel() == 0:
            return _dequantize_cpu(self, dtype)
        lib = _native("dequantize_activation")
        out = torch.empty(self.q.shape, dtype=dtype, device=self.q.device)
        C = out.shape[-1]
        lib.launch(lib.LIB.kan_hip_act8_dequantize, out.device,
                   lib.operator_dtype_code(dtype, "dequantize_activation"),
                   FORMATS[self.format][0], self.q.data_ptr(), self.scale.data_ptr(),
                   out.numel() // C, C, self.group, out.data_ptr())
        return out


def _quantize_cpu(x, group, format):
    _, qmax, qdtype = FORMATS[format]
    C = x.shape[-1]
    parts = -(-C // group)
    v = torch.nn.functional.pad(x.float(), (0, parts * group - C)).reshape(*x.shape[:-1], parts,
                                                                           group)
    finite = v.isfinite().all(-1, keepdim=True)
    scale = v.abs().amax(-1, keepdim=True) * (1 / qmax)
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, 0.0, scale)
    u = torch.where((scale > 0) & finite, v * (1 / scale), torch.zeros(()))
    u = u.round() if format == "int8" else u
    q = u.reshape(*x.shape[:-1], parts * group)[..., :C].to(qdtype).contiguous()
    return q, torch.where(finite, scale, torch.nan)[..., 0]


def _dequantize_cpu(a, dtype):
    C = a.q.shape[-1]
    scale = a.scale.repeat_interleave(a.group, -1)[..., :C]
    return (a.q.float() * scale).to(dtype)


def quantize_activation(x: torch.Tensor, group: int = 128, format: str = "int8") -> Activation8:
    """x [..., C] in 8 bits: for every group of `group` (32, 64, 128 or 256)
    consecutive values of the last axis, scale = max|x| * (1 / qmax) (127 for
    "int8", 448 for "e4m3") and q = round(x * (1 / scale)) to nearest, ties to even."""
    who = "quantize_activation"
    check_format(who, group, format)
    _req(x.dim() >= 1, who, ": x must have at least one dimension")
    _req(x.dtype in (torch.float32, torch.bfloat16, torch.float16), who,
         ": only FP32, BF16 and FP16 tensors are supported, got ", x.dtype)
    if not x.is_cuda or x.numel() == 0:
        q, scale = _quantize_cpu(x.detach(), group, format)
        return Activation8(q, scale, group, format, x.dtype)
    lib = _native(who)
    C = x.shape[-1]
    rows, ldx = x.numel() // C, C
    if not x.is_contiguous():
        if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= C:
            ldx = x.stride(0)
        else:
            x = x.contiguous()
    code, _, qdtype = FORMATS[format]
    q = torch.empty(x.shape, dtype=qdtype, device=x.device)
    scale = torch.empty(x.shape[:-1] + (-(-C // group),), dtype=torch.float32, device=x.device)
    lib.launch(lib.LIB.kan_hip_act8_quantize, x.device, lib.OPERATOR_DTYPES[x.dtype], code,
               x.data_ptr(), ldx, rows, C, group, q.data_ptr(), scale.data_ptr())
    return Activation8(q, scale, group, format, x.dtype)


def _autocast_of(device_type: str):
    """(device type, enabled, type) of autocast on device_type and the CPU."""
    return [(t, torch.is_autocast_enabled(t), torch.get_autocast_dtype(t))
            for t in {device_type, "cpu"}]


def _autocast(state) -> ExitStack:
    """Autocast as in `state`.  Casts of weights are not kept where it is on: those of
    a pass without gradients would serve calls beside it, which then lost theirs."""
    stack = ExitStack()
    for device_type, on, dtype in state:
        if on or torch.is_autocast_enabled(device_type):
            stack.enter_context(torch.autocast(device_type, dtype=dtype, enabled=on,
                                               cache_enabled=False))
    return stack


def _fill(rest, tensors):
    """(rest with `tensors` in the places of its Nones, the tensors left over)"""
    left = iter(tensors)
    return [next(left) if r is None else r[0] for r in rest], list(left)


class _Checkpoint8(torch.autograd.Function):
    """Inputs beside x: the tensors among fn's further arguments (rest has None in
    their places, the others as (value,)), then the parameters."""

    @staticmethod
    def forward(ctx, fn, rest, group, format, x, *tensors):
        args, params = _fill(rest, tensors)
        kept = quantize_activation(x, group, format)
        ctx.fn, ctx.rest, ctx.form = fn, rest, (group, format, x.dtype)
        ctx.save_for_backward(kept.q, kept.scale, *tensors[:len(tensors) - len(params)])
        # (fn holds its parameters: references and versions are enough)
        ctx.params, ctx.versions = params, [p._version for p in params]
        ctx.autocast = _autocast_of(x.device.type)
        with torch.no_grad(), _autocast(ctx.autocast):
            return fn(x, *args)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        q, scale, *tensors = ctx.saved_tensors
        _req([p._version for p in ctx.params] == ctx.versions, "checkpoint_8bit: a parameter was "
             "changed in place between the forward and the backward pass")
        needs = ctx.needs_input_grad[4:]
        x = Activation8(q, scale, *ctx.form).dequantize().requires_grad_(needs[0])
        tensors = [t.detach().requires_grad_(need) for t, need in zip(tensors, needs[1:])]
        with torch.enable_grad(), _autocast(ctx.autocast):
            out = ctx.fn(x, *_fill(ctx.rest, tensors)[0])
        outs = [out] if isinstance(out, torch.Tensor) else list(out)
        pairs = [(o, g) for o, g in zip(outs, grads) if g is not None and o.requires_grad]
        wanted = [t for t, need in zip((x, *tensors, *ctx.params), needs) if need]
        got = iter(torch.autograd.grad([o for o, _ in pairs], wanted, [g for _, g in pairs],
                                       allow_unused=True) if pairs and wanted
                   else [None] * len(wanted))
        return (None, None, None, None, *(next(got) if need else None for need in needs))


def checkpoint_8bit(fn: Callable, x: torch.Tensor, *args, group: int = 128, format: str = "int8",
                    params: Optional[Sequence[torch.Tensor]] = None):
    """fn(x, *args), keeping x in 8 bits for the backward pass and nothing that
    fn makes: the backward restores x and runs fn again, under the call's
    autocast, so gradients are those of fn at the restored x (the output is
    exact).  Gradients reach x, tensors in args and `params` (default:
    fn.parameters() of a module), nothing else that fn uses.  fn must give the
    same result each time: no random numbers."""
    check_format("checkpoint_8bit", group, format)
    if params is None:
        params = tuple(fn.parameters()) if isinstance(fn, nn.Module) else ()
    params = tuple({id(p): p for p in params if p.requires_grad}.values())
    tensors = tuple(a for a in args if isinstance(a, torch.Tensor))
    if not (torch.is_grad_enabled()
            and (x.requires_grad or params or any(t.requires_grad for t in tensors))):
        return fn(x, *args)
    rest = [None if isinstance(a, torch.Tensor) else (a,) for a in args]
    return _Checkpoint8.apply(fn, rest, group, format, x, *tensors, *params)
