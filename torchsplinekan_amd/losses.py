"""Losses of the logits x W^T of a last layer, without the logits (no reference
counterpart): the softmax cross entropy over a vocabulary or its classes, and the
distillation from a teacher's top logits.  Device tensors run on the kernels of
csrc/kan_vocab.hip, which keep a maximum and a sum for every row and take the
logits again, a piece of the vocabulary at a time, in the backward pass; CPU
tensors on torch products.
"""

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import fused as _fused

_C = _fused._C
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
MAX_TOP = 1024


def _refuse(*msg) -> None:
    raise RuntimeError("".join(str(m) for m in msg))


def _native(who: str):
    if _C is None:
        raise RuntimeError(f"{who}: device tensors need libkan_hip.so; build it with "
                           "`python -m torchsplinekan_amd.build_lib`")
    return _C._lib


def _workspace(lib, device, fn, *args):
    """(tensor or None, its bytes) of a workspace query"""
    nbytes = ctypes.c_size_t()
    lib.check(fn(*args, ctypes.byref(nbytes)))
    size = nbytes.value
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None, size


class _VocabLoss(torch.autograd.Function):
    """x [T, D], weight [V, D], ids [T, k], teacher [T, k] float32; cross entropy:
    ids [T, 1], teacher None."""

    @staticmethod
    def forward(ctx, x, weight, ids, teacher, ignore, tau, reduction):
        lib = _native("linear_cross_entropy")
        T, D = x.shape
        V, k = weight.shape[0], 0 if teacher is None else ids.shape[1]
        code, L = lib.OPERATOR_DTYPES[x.dtype], lib.LIB
        kept, _ = _workspace(lib, x.device, L.kan_hip_vocab_loss_kept, T, V, k)
        px, pw = x.data_ptr(), weight.data_ptr()
        ws, nbytes = _workspace(lib, x.device, L.kan_hip_vocab_loss_workspace, code, px, pw, T, V,
                                D)
        loss = torch.empty((T,) if reduction == 0 else (), dtype=torch.float32, device=x.device)
        lib.launch(L.kan_hip_vocab_loss, x.device, code, px, pw, ids.data_ptr(),
                   int(ids.dtype == torch.int64), None if teacher is None else teacher.data_ptr(),
                   T, V, D, k, ignore, tau, reduction, loss.data_ptr(), kept.data_ptr(),
                   ws.data_ptr(), nbytes)
        if ctx is not None and any(ctx.needs_input_grad):
            ctx.args = (code, T, V, D, k, ignore, tau, reduction)
            ctx.save_for_backward(x, weight, ids if k == 0 else None, kept)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        lib = _native("linear_cross_entropy")
        x, weight, ids, kept = ctx.saved_tensors
        code, T, V, D, k, ignore, tau, reduction = ctx.args
        dx, dw = [torch.empty_like(t) if need else None
                  for t, need in zip((x, weight), ctx.needs_input_grad)]
        g = g.contiguous()
        px, pw, L = x.data_ptr(), weight.data_ptr(), lib.LIB
        ws, nbytes = _workspace(lib, x.device, L.kan_hip_vocab_loss_backward_workspace, code, px,
                                pw, T, V, D, int(dx is not None), int(dw is not None))
        lib.launch(L.kan_hip_vocab_loss_backward, x.device, code, g.data_ptr(), px, pw,
                   None if ids is None else ids.data_ptr(),
                   int(ids is not None and ids.dtype == torch.int64), kept.data_ptr(), T, V, D, k,
                   ignore, tau, reduction,
                   None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                   ws.data_ptr(), nbytes)
        return dx, dw, None, None, None, None, None


def _composite(x, weight, ids, teacher, ignore, tau, reduction):
    """The definition in torch, logits and all, in float32 or wider."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    V = weight.shape[0]
    there = (ids >= 0) & (ids < V)
    if teacher is None:
        there = there & (ids != ignore)
        bad = ~there & (ids != ignore)
        prob = there.to(wide)
    else:
        bad = ids >= V
        score = torch.where(there, teacher.to(wide) / tau, -torch.inf)
        top = score.amax(1, keepdim=True)
        prob = (score - torch.where(top == -torch.inf, 0.0, top)).exp()
        total = prob.sum(1, keepdim=True)
        prob = prob / torch.where(total == 0, 1.0, total)
    some, bad = ~(prob == 0), bad.any(1)
    counts = some.any(1) | bad
    x = torch.where(counts.unsqueeze(1), x, 0)  # (whatever other rows hold stays out)
    with torch.autocast(x.device.type, enabled=False):  # (whose products would be narrower)
        z = x.to(wide) @ weight.to(wide).t()
    logq = (z / tau).log_softmax(1).gather(1, torch.where(there, ids, 0).long())
    terms = torch.where(some, prob * (torch.where(some, prob, 1.0).log() - logq), 0.0)
    at = bad.nonzero()[:, 0]
    rows = (tau * tau * terms.sum(1)).index_add(0, at, torch.nan * z[at].sum(1))
    if reduction == 0:
        return rows
    loss = rows.sum()
    return loss if reduction == 1 else loss / counts.sum().clamp(min=1)


def _loss(who, x, weight, ids, teacher, ignore, tau, reduction):
    """x [..., D], ids [..., k] as checked by the callers."""
    if reduction not in REDUCTIONS:
        _refuse(who, ": reduction must be 'none', 'sum' or 'mean', got ", repr(reduction))
    if x.dim() < 1 or weight.dim() != 2:
        _refuse(who, ": x must be [..., D] and weight [V, D], got ", list(x.shape), " and ",
                list(weight.shape))
    if weight.shape[1] != x.shape[-1]:
        _refuse(who, ": weight.size(1)=", weight.shape[1], " must equal D=", x.shape[-1])
    if weight.shape[0] < 1:
        _refuse(who, ": weight must have at least one row")
    if weight.dtype != x.dtype:
        _refuse(who, ": x and weight must share a dtype")
    if weight.device != x.device or ids.device != x.device:
        _refuse(who, ": tensors must be on one device")
    lead, code = x.shape[:-1], REDUCTIONS[reduction]
    if x.dim() != 2:
        x = x.reshape(lead.numel(), x.shape[-1])
        ids = ids.reshape(lead.numel(), ids.shape[-1])
    if teacher is not None:
        teacher = teacher.detach().reshape(ids.shape)
    if not x.is_cuda or x.numel() == 0 or ids.numel() == 0:
        loss = _composite(x, weight, ids, teacher, ignore, tau, code)
    else:
        lib = _native(who)
        lib.operator_dtype_code(x.dtype, who)
        x, weight, ids = x.contiguous(), weight.contiguous(), ids.contiguous()
        teacher = None if teacher is None else teacher.float().contiguous()
        save = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
        loss = lib.call(_VocabLoss, save, x, weight, ids, teacher, ignore, tau, code)
    return loss.reshape(lead) if code == 0 and len(lead) != 1 else loss


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """The softmax cross entropy of the logits x weight^T against target, which never
    holds the logits: log sum exp z - z[target], in float32.

    x [..., D]; weight [V, D]; target [...], int32 or int64: 0 .. V - 1, or
    ignore_index for rows that do not count.  Any other value makes its row's loss
    and its gradients NaN (no value of target is read on the host).
    reduction: "none" (the rows' losses [...], 0 for those that do not count),
    "sum", or "mean" over the rows that count (0 without any).  A row that does not
    count may hold anything, NaN too.
    Gradients (first order) reach x and weight (device tensors refuse forward
    mode); their products take the logits' gradient in x's type, and sums are held
    in float32, also under autocast, which casts nothing here."""
    who = "linear_cross_entropy"
    if target.dtype not in (torch.int32, torch.int64):
        _refuse(who, ": target must be int32 or int64, got ", target.dtype)
    if x.dim() < 1 or target.shape != x.shape[:-1]:
        _refuse(who, ": target must have x's leading shape ", list(x.shape[:-1]), ", got ",
                list(target.shape))
    return _loss(who, x, weight, target.unsqueeze(-1), None, int(ignore_index), 1.0, reduction)


def linear_distillation(x: torch.Tensor, weight: torch.Tensor, ids: torch.Tensor,
                        teacher: torch.Tensor, *, temperature: float = 1.0,
                        reduction: str = "mean") -> torch.Tensor:
    """The divergence of a student's softmax from a teacher's top logits,
    temperature^2 sum_j p_j (log p_j - log q[ids_j]), with p the softmax of
    teacher / temperature over a row's ids and q that of x weight^T / temperature
    over all V, in float32 and without the student's logits.

    x [..., D]; weight [V, D]; ids [..., k], int32 or int64, k <= 1024: columns in
    any order (equal ones add); those below 0 are absent, and a row without any, or
    with logits of -inf alone, does not count.  An id from V on makes its row's loss
    and its gradients NaN.
    teacher [..., k]: its logits at ids, float32, bfloat16 or float16; no gradient
    reaches it.  reduction, types and gradients as linear_cross_entropy."""
    who = "linear_distillation"
    if ids.dtype not in (torch.int32, torch.int64):
        _refuse(who, ": ids must be int32 or int64, got ", ids.dtype)
    if x.dim() < 1 or ids.dim() != x.dim() or ids.shape[:-1] != x.shape[:-1]:
        _refuse(who, ": ids must have x's leading shape and k ids each, got ", list(ids.shape),
                " and ", list(x.shape))
    if not 1 <= ids.shape[-1] <= MAX_TOP:
        _refuse(who, ": 1 to ", MAX_TOP, " ids a row, got ", ids.shape[-1])
    if teacher.shape != ids.shape:
        _refuse(who, ": teacher must have ids' shape ", list(ids.shape), ", got ",
                list(teacher.shape))
    if not teacher.is_floating_point():
        _refuse(who, ": teacher must hold floating point logits, got ", teacher.dtype)
    if teacher.device != x.device:
        _refuse(who, ": tensors must be on one device")
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        _refuse(who, ": temperature must be positive and finite, got ", temperature)
    return _loss(who, x, weight, ids, teacher, -1, temperature, reduction)
