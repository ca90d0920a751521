"""Matrix products grouped by expert with ragged sizes (no reference
counterpart).  Rows are sorted by expert and the group boundaries stay on the
device, so a router's result is used without waiting for it.  Device tensors
run on the kernels of csrc/kan_grouped.hip, CPU tensors on torch products.
"""

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import fused as _fused
from .act8 import FORMATS, Activation8, check_format, quantize_activation

_C = _fused._C
FORWARD, INPUT, WEIGHT = 0, 1, 2


def _req(cond: bool, *msg) -> None:
    if not cond:
        raise RuntimeError("grouped_linear: " + "".join(str(m) for m in msg))


def _native():
    if _C is None:
        raise RuntimeError("grouped_linear: device tensors need libkan_hip.so; build it with "
                           "`python -m torchsplinekan_amd.build_lib`")
    return _C._lib


def _matmul(op: int, a, b, offsets, out, T: int, E: int, N: int, K: int, factor=None):
    """One grouped product into `out`; b may be an Activation8 (WEIGHT), offsets None
    with one group; factor: a float32 tensor whose first value all results are times."""
    lib = _native()
    if out.numel() == 0:
        return out
    code = lib.OPERATOR_DTYPES[out.dtype]
    form, scale, group, ws = 0, None, 0, None
    if isinstance(b, Activation8):
        form, scale, group, b = FORMATS[b.format][0], b.scale.data_ptr(), b.group, b.q
    pa, pb = lib.ptr(a), lib.ptr(b)
    nbytes = ctypes.c_size_t()
    lib.check(lib.LIB.kan_hip_grouped_matmul_workspace(code, op, pa, pb, form, T, E, N, K,
                                                       ctypes.byref(nbytes)))
    if nbytes.value:
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=out.device)
    off64 = int(offsets is not None and offsets.dtype == torch.int64)
    if factor is not None:
        lib.launch(lib.LIB.kan_hip_grouped_matmul_scaled, out.device, code, op, pa, pb,
                   lib.ptr(offsets), off64, T, E, N, K, factor.data_ptr(), out.data_ptr(),
                   lib.ptr(ws), nbytes.value)
        return out
    lib.launch(lib.LIB.kan_hip_grouped_matmul, out.device, code, op, pa, pb, form, scale, group,
               lib.ptr(offsets), off64, T, E, N, K, out.data_ptr(), lib.ptr(ws), nbytes.value)
    return out


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, checkpoint, group):
        T, K = x.shape
        E, N, _ = weight.shape
        y = _matmul(FORWARD, x, weight, offsets, x.new_empty(T, N), T, E, N, K)
        if ctx is None:
            return y
        need_x, need_w = ctx.needs_input_grad[:2]
        keep, scale = x if need_w else None, None
        if need_w and checkpoint is not None:
            kept = quantize_activation(x, group, checkpoint)
            keep, scale = kept.q, kept.scale
        ctx.sizes = (T, E, N, K)
        ctx.form = (group, checkpoint)
        ctx.like = x.new_empty(0)
        ctx.save_for_backward(keep, scale, weight if need_x else None, offsets)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, scale, weight, offsets = ctx.saved_tensors
        T, E, N, K = ctx.sizes
        need_x, need_w = ctx.needs_input_grad[:2]
        dy = dy.contiguous()
        dx = dw = None
        if need_x:
            dx = _matmul(INPUT, dy, weight, offsets, ctx.like.new_empty(T, K), T, E, N, K)
        if need_w:
            if scale is not None:
                x = Activation8(x, scale, *ctx.form, dy.dtype)
            dw = _matmul(WEIGHT, dy, x, offsets, ctx.like.new_empty(E, N, K), T, E, N, K)
        return dx, dw, None, None, None


class _KeptRows(torch.autograd.Function):
    """Values of x in the forward pass; the product's weight gradient sees x as
    it comes back from 8 bits (the CPU form of the checkpoint)."""

    @staticmethod
    def forward(ctx, x, weight, group, format):
        kept = quantize_activation(x, group, format)
        ctx.save_for_backward(weight, kept.q, kept.scale)
        ctx.form = (group, format, x.dtype)
        return x @ weight.t()

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, q, scale = ctx.saved_tensors
        return dy @ weight, dy.t() @ Activation8(q, scale, *ctx.form).dequantize(), None, None


def _composite(x, weight, offsets, checkpoint, group):
    """Row blocks of each expert with torch products, in float32 or wider."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    T, E = x.shape[0], weight.shape[0]
    parts, lo = [], 0
    ends = [min(max(int(v), 0), T) for v in offsets.tolist()[1:]]
    with torch.autocast(x.device.type, enabled=False):  # (whose products would be narrower)
        for e in range(E):
            hi = max(lo, ends[e])
            xe, we = x[lo:hi].to(wide), weight[e].to(wide)
            if checkpoint is None:
                parts.append(xe @ we.t())
            else:
                parts.append(_KeptRows.apply(xe, we, group, checkpoint))
            lo = hi
    parts.append(x.new_zeros(T - lo, weight.shape[1], dtype=wide))
    return torch.cat(parts).to(x.dtype)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *,
                   checkpoint: Optional[str] = None, group: int = 128) -> torch.Tensor:
    """y [T, N] with y[t] = weight[e] x[t], e the expert that row t belongs to.

    x [T, K]: rows sorted by expert.  weight [E, N, K].  offsets [E + 1], int32
    or int64, on x's device: expert e has the rows offsets[e] .. offsets[e + 1]
    - 1; they ascend from 0, and rows from offsets[E] on get zeros.  (Their
    values are not read on the host; the kernels take each within 0 .. T and
    never below the one before.)
    checkpoint "int8" or "e4m3": the weight's gradient reads x from 8 bits
    (groups of `group` values, quantize_activation) and x itself is not kept.
    On the device the restored values take part rounded to x's type, as
    Activation8.dequantize gives them; on the CPU in float32.
    Sums are held in float32, also under autocast, which casts nothing here.
    Gradients (first order) reach x and weight (device tensors refuse forward
    mode); sums over rows have a fixed order."""
    _req(x.dim() == 2 and weight.dim() == 3, "x must be [T, K] and weight [E, N, K], got ",
         list(x.shape), " and ", list(weight.shape))
    _req(weight.shape[2] == x.shape[1], "weight.size(2)=", weight.shape[2], " must equal K=",
         x.shape[1])
    _req(weight.dtype == x.dtype, "x and weight must share a dtype")
    _req(offsets.dim() == 1 and offsets.shape[0] == weight.shape[0] + 1,
         "offsets must be [E + 1] = [", weight.shape[0] + 1, "], got ", list(offsets.shape))
    _req(offsets.dtype in (torch.int32, torch.int64), "offsets must be int32 or int64, got ",
         offsets.dtype)
    _req(weight.device == x.device and offsets.device == x.device,
         "x, weight and offsets must be on one device")
    if checkpoint is not None:
        check_format("grouped_linear", group, checkpoint)
    if not x.is_cuda:
        return _composite(x, weight, offsets, checkpoint, group)
    lib = _native()
    lib.operator_dtype_code(x.dtype, "grouped_linear")
    x, weight, offsets = x.contiguous(), weight.contiguous(), offsets.contiguous()
    save = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
    return lib.call(_GroupedLinear, save, x, weight, offsets, checkpoint, group)
