"""Gated products, h = act(x gate^T) * (x up^T), for all rows alike or by expert
(no reference counterpart).  Device tensors run on the kernels of
csrc/kan_gated.hip and, for the gradients, on the grouped products; CPU tensors
on torch products.
"""

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import fused as _fused
from .grouped import INPUT, WEIGHT, _matmul

_C = _fused._C
ACTS = {None: 0, "sigmoid": 1, "tanh": 2, "silu": 3, "gelu": 4, "relu": 5}


def _refuse(*msg) -> None:
    raise RuntimeError("gated_linear: " + "".join(str(m) for m in msg))


def _native():
    if _C is None:
        raise RuntimeError("gated_linear: device tensors need libkan_hip.so; build it with "
                           "`python -m torchsplinekan_amd.build_lib`")
    return _C._lib


def _bytes(lib, fn, *args) -> int:
    nbytes = ctypes.c_size_t()
    lib.check(fn(*args, ctypes.byref(nbytes)))
    return nbytes.value


class _GatedLinear(torch.autograd.Function):
    """x [T, K], weight [E, 2, N, K], or [2, N, K] without offsets."""

    @staticmethod
    def forward(ctx, x, weight, offsets, act):
        lib = _native()
        save = ctx is not None and any(ctx.needs_input_grad)
        T, K = x.shape
        N, E = weight.shape[-2], 1 if offsets is None else weight.shape[0]
        code = lib.OPERATOR_DTYPES[x.dtype]
        h = x.new_empty(T, N)
        kept = ws = None
        if save:
            kept = torch.empty(_bytes(lib, lib.LIB.kan_hip_gated_kept, code, T, N),
                               dtype=torch.uint8, device=x.device)
        px, pw = lib.ptr(x), lib.ptr(weight)
        nbytes = _bytes(lib, lib.LIB.kan_hip_gated_workspace, code, px, pw, T, E, N, K, int(save))
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        lib.launch(lib.LIB.kan_hip_gated, x.device, code, act, px, pw, lib.ptr(offsets),
                   int(offsets is not None and offsets.dtype == torch.int64), T, E, N, K,
                   lib.ptr(h), lib.ptr(kept), lib.ptr(ws), nbytes)
        if save:
            need_x, need_w = ctx.needs_input_grad[:2]
            ctx.args = (act, T, E, N, K)
            ctx.save_for_backward(x if need_w else None, weight if need_x else None, offsets, kept)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        lib = _native()
        x, weight, offsets, kept = ctx.saved_tensors
        act, T, E, N, K = ctx.args
        need_x, need_w = ctx.needs_input_grad[:2]
        dh = dh.contiguous()
        dpre = dh.new_empty(T, 2 * N)
        code, factor = lib.OPERATOR_DTYPES[dh.dtype], None
        if dh.dtype == torch.float16 and dpre.numel():  # (small or large values would be lost)
            factor = torch.empty(lib.KAN_GATED_SCALE_VALUES, dtype=torch.float32, device=dh.device)
            lib.launch(lib.LIB.kan_hip_gated_backward_scaled, dh.device, code, act, lib.ptr(dh),
                       lib.ptr(kept), T, N, lib.ptr(dpre), factor.data_ptr())
        else:
            lib.launch(lib.LIB.kan_hip_gated_backward, dh.device, code, act, lib.ptr(dh),
                       lib.ptr(kept), T, N, lib.ptr(dpre))
        dx = dw = None
        if need_x:
            dx = _matmul(INPUT, dpre, weight, offsets, dh.new_empty(T, K), T, E, 2 * N, K, factor)
        if need_w:
            shape = (2, N, K) if offsets is None else (E, 2, N, K)
            dw = _matmul(WEIGHT, dpre, x, offsets, dh.new_empty(shape), T, E, 2 * N, K, factor)
        return dx, dw, None, None


def _act(g: torch.Tensor, act: Optional[str]) -> torch.Tensor:
    if act == "gelu":
        return 0.5 * g * torch.erfc(g * -(0.5 ** 0.5))
    return {None: lambda: g, "sigmoid": g.sigmoid, "tanh": g.tanh, "relu": g.relu,
            "silu": lambda: g * g.sigmoid()}[act]()


def _composite(x, weight, offsets, act):
    """Row blocks of each expert with torch products, in float32 or wider."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    T, N = x.shape[0], weight.shape[2]
    bounds = [0, T] if offsets is None else offsets.tolist()
    parts, lo = [], 0
    with torch.autocast(x.device.type, enabled=False):  # (whose products would be narrower)
        for e in range(weight.shape[0]):
            hi = max(lo, min(max(int(bounds[e + 1]), 0), T))
            xe, we = x[lo:hi].to(wide), weight[e].to(wide)
            parts.append(_act(xe @ we[0].t(), act) * (xe @ we[1].t()))
            lo = hi
    parts.append(x.new_zeros(T - lo, N, dtype=wide))
    return torch.cat(parts).to(x.dtype)


def gated_linear(x: torch.Tensor, weight: torch.Tensor, offsets: Optional[torch.Tensor] = None, *,
                 act: Optional[str] = "silu") -> torch.Tensor:
    """act(x gate^T) * (x up^T): both projections, the activation and the product
    of a gated feed-forward block.

    Without offsets: x [..., K] and weight [2, N, K], gate and up: [..., N].
    With offsets: x [T, K], rows sorted by expert, weight [E, 2, N, K] and offsets
    [E + 1] as grouped_linear takes them: [T, N]; rows from offsets[E] on get
    zeros.
    act: None, "sigmoid", "tanh", "silu", "gelu" (of the normal distribution's
    cdf itself) or "relu".
    Sums are held in float32, also under autocast, which casts nothing here.
    Gradients (first order) reach x and weight (device tensors refuse forward
    mode); for them 5 (bfloat16), 6 (float16) or 8 bytes an output are kept.
    Sums over rows have a fixed order."""
    if act not in ACTS:
        _refuse("act must be None, 'sigmoid', 'tanh', 'silu', 'gelu' or 'relu', got ", repr(act))
    shape = weight.shape
    if offsets is None:
        if weight.dim() != 3 or shape[0] != 2:
            _refuse("weight must be [2, N, K], got ", list(shape))
        if x.dim() < 1:
            _refuse("x must have at least one dimension")
    else:
        if x.dim() != 2 or weight.dim() != 4 or shape[1] != 2:
            _refuse("with offsets x must be [T, K] and weight [E, 2, N, K], got ", list(x.shape),
                    " and ", list(shape))
        if offsets.dim() != 1 or offsets.shape[0] != shape[0] + 1:
            _refuse("offsets must be [E + 1] = [", shape[0] + 1, "], got ", list(offsets.shape))
        if offsets.dtype not in (torch.int32, torch.int64):
            _refuse("offsets must be int32 or int64, got ", offsets.dtype)
        if offsets.device != x.device:
            _refuse("x, weight and offsets must be on one device")
    if shape[-1] != x.shape[-1]:
        _refuse("weight.size(-1)=", shape[-1], " must equal K=", x.shape[-1])
    if weight.dtype != x.dtype:
        _refuse("x and weight must share a dtype")
    if weight.device != x.device:
        _refuse("x, weight and offsets must be on one device")
    lead = None
    if x.dim() != 2:
        lead = x.shape[:-1]
        x = x.reshape(lead.numel(), shape[-1])
    if not x.is_cuda:
        h = _composite(x, weight if offsets is not None else weight.unsqueeze(0), offsets, act)
    else:
        lib = _native()
        lib.operator_dtype_code(x.dtype, "gated_linear")
        x, weight = x.contiguous(), weight.contiguous()
        offsets = None if offsets is None else offsets.contiguous()
        save = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
        h = lib.call(_GatedLinear, save, x, weight, offsets, ACTS[act])
    return h if lead is None else h.reshape(lead + (shape[-2],))
