"""Mixtures of KAN layers and a residual stack of them (no reference
counterpart; the reference has single layers and plain stacks of them).

``KANExperts`` routes every row to top_k of its experts, each a KAN layer over
knots they share; the routed rows' products run grouped by expert
(``grouped_linear``), and with ``checkpoint`` the rows are kept in 8 bits and
the basis, R + 1 times their size, is evaluated again in the backward pass
(``checkpoint_8bit``).  ``KANExpertStack`` puts such blocks on a residual stream
(``residual_norm``): norm, experts, norm, gate and residual scale; with a gated
feed-forward block (``gated_linear``) beside the experts, a layer norm of what comes
in (``layer_norm``) and a last layer of classes or tokens, whose losses never hold
the logits (``linear_cross_entropy``, ``linear_distillation``).
"""

import math
from typing import Optional, Tuple

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import fused as _fused
from .act8 import check_format, checkpoint_8bit
from .gated import gated_linear
from .grouped import grouped_linear
from .layernorm import layer_norm
from .losses import linear_cross_entropy, linear_distillation
from .reference_backend import compute_basis
from .residual import residual_norm

_C = _fused._C


def route(logits: torch.Tensor, top_k: int):
    """(weights [N, k], order [N k], offsets [E + 1]) of rows that go to the top_k
    experts of logits [N, E] each: weights are the softmax over the chosen
    logits; `order` lists the (row, choice) pairs (as row * k + choice) sorted by
    expert, rows in order, and offsets are the experts' boundaries in it.  Nothing
    is read on the host."""
    N, E = logits.shape
    top, ids = logits.topk(top_k, -1)
    sorted_ids, order = ids.reshape(-1).sort(stable=True)
    bounds = torch.arange(E + 1, device=logits.device, dtype=sorted_ids.dtype)
    offsets = torch.searchsorted(sorted_ids, bounds)
    return top.softmax(-1), order, offsets


class KANExperts(nn.Module):
    """A mixture of num_experts KAN layers [in_features -> out_features] on common
    uniform knots.

    Parameters: router [E, I], base_weight [E, O, I], spline_weight
    [E, O, I, R] (R = grid_size + spline_order); buffer grid [I, G + 2k + 1].
    checkpoint: None, "int8" or "e4m3" (with `group` values a scale): what the
    backward pass keeps of the routed rows (in float32 only).  First-order
    gradients only; device inputs are float32, and autocast changes nothing."""

    def __init__(self, in_features: int, out_features: int, num_experts: int, top_k: int = 2,
                 grid_size: int = 5, spline_order: int = 3, scale_noise: float = 0.1,
                 grid_range: Tuple[float, float] = (-2.0, 2.0),
                 checkpoint: Optional[str] = None, group: int = 128) -> None:
        super().__init__()
        if not 1 <= top_k <= num_experts:
            raise ValueError(f"top_k must be in 1..num_experts={num_experts}, got {top_k}")
        if grid_size < 1 or spline_order not in (1, 2, 3):
            raise ValueError("grid_size must be >= 1 and spline_order 1, 2 or 3, got "
                             f"{grid_size} and {spline_order}")
        if checkpoint is not None:
            check_format("KANExperts", group, checkpoint)
        self.in_features, self.out_features = in_features, out_features
        self.num_experts, self.top_k = num_experts, top_k
        self.grid_size, self.spline_order = grid_size, spline_order
        self.checkpoint, self.group = checkpoint, group
        k, R = spline_order, grid_size + spline_order
        lo, hi = grid_range
        knots = lo + torch.arange(-k, grid_size + k + 1) * ((hi - lo) / grid_size)
        self.register_buffer("grid", knots.expand(in_features, -1).contiguous())
        self.router = nn.Parameter(torch.empty(num_experts, in_features))
        self.base_weight = nn.Parameter(torch.empty(num_experts, out_features, in_features))
        self.spline_weight = nn.Parameter(
            torch.empty(num_experts, out_features, in_features, R))
        bound = 1.0 / math.sqrt(in_features)
        nn.init.normal_(self.router, std=bound)
        nn.init.uniform_(self.base_weight, -bound, bound)
        noise = scale_noise / math.sqrt(R)
        nn.init.uniform_(self.spline_weight, -noise, noise)

    def _expert_rows(self, rows: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        """Every expert's KAN layer on its rows [T, I] -> [T, O]."""
        E, O, I, R = self.spline_weight.shape
        if rows.is_cuda and _C is not None:
            s, H = _fused.native_basis_silu(rows, self.grid, self.spline_order)
        else:
            s, H = F.silu(rows), compute_basis(rows, self.grid, self.spline_order)
        y = grouped_linear(s, self.base_weight, offsets)
        return y + grouped_linear(H.reshape(-1, I * R), self.spline_weight.reshape(E, O, I * R),
                                  offsets)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        with torch.autocast(x.device.type, enabled=False):
            return self._forward(x)

    def _forward(self, x: torch.Tensor) -> torch.Tensor:
        lead, I, k = x.shape[:-1], self.in_features, self.top_k
        xf = x.reshape(-1, I)
        weights, order, offsets = route(F.linear(xf, self.router), k)
        # (each gathered row is its own, so no gradient is added atomically)
        rows = xf.unsqueeze(1).expand(-1, k, -1).reshape(-1, I).index_select(0, order)
        if self.checkpoint is None:
            y = self._expert_rows(rows, offsets)
        else:
            y = checkpoint_8bit(self._expert_rows, rows, offsets, group=self.group,
                                format=self.checkpoint,
                                params=(self.base_weight, self.spline_weight))
        back = torch.empty_like(order)
        back[order] = torch.arange(order.numel(), device=order.device)
        y = y.index_select(0, back).reshape(-1, k, self.out_features)
        return (y * weights.unsqueeze(-1)).sum(1).reshape(lead + (self.out_features,))


class _Block(nn.Module):
    def __init__(self, width: int, residual_scale: float, feed_forward: int, **experts) -> None:
        super().__init__()
        self.pre_weight = nn.Parameter(torch.ones(width))
        self.post_weight = nn.Parameter(torch.ones(width))
        self.scale = nn.Parameter(torch.full((width,), residual_scale))
        self.gate = nn.Linear(width, 1)
        self.experts = KANExperts(width, width, **experts)
        self.gate_up = self.down = None
        if feed_forward > 0:
            self.gate_up = nn.Parameter(torch.empty(2, feed_forward, width))
            self.down = nn.Parameter(torch.empty(width, feed_forward))
            nn.init.normal_(self.gate_up, std=1.0 / math.sqrt(width))
            nn.init.normal_(self.down, std=1.0 / math.sqrt(feed_forward))

    def forward(self, h: torch.Tensor) -> torch.Tensor:
        y = self.experts(h)
        if self.down is not None:
            y = y + F.linear(gated_linear(h, self.gate_up), self.down)
        return y


class KANExpertStack(nn.Module):
    """depth residual blocks x' = x + scale * sigmoid(gate(h)) * norm(block(h)),
    h = norm(x), and a norm of the last x'.  Each block's second norm, gate,
    scale and addition run in one pass with the next block's first norm.
    feed_forward > 0: every block adds a gated feed-forward block of that many
    outputs, which all rows pass, to its experts.  input_norm: x passes a layer
    norm first, with input_eps (eps is the other norms').  num_classes: a last layer
    head [num_classes, width] for logits, loss and distillation_loss.  Further
    arguments go to each KANExperts."""

    def __init__(self, width: int, depth: int, num_experts: int, residual_scale: float = 0.2,
                 eps: float = 1e-6, feed_forward: int = 0, input_norm: bool = False,
                 num_classes: Optional[int] = None, input_eps: float = 1e-5, **experts) -> None:
        super().__init__()
        if depth < 1:
            raise ValueError(f"depth must be >= 1, got {depth}")
        if feed_forward < 0:
            raise ValueError(f"feed_forward must be >= 0, got {feed_forward}")
        if num_classes is not None and num_classes < 1:
            raise ValueError(f"num_classes must be >= 1, got {num_classes}")
        self.blocks = nn.ModuleList([
            _Block(width, residual_scale, feed_forward, num_experts=num_experts, **experts)
            for _ in range(depth)])
        self.norm_weight = nn.Parameter(torch.ones(width))
        self.eps, self.input_eps = eps, input_eps
        self.input_weight = self.input_bias = self.head = None
        if input_norm:
            self.input_weight = nn.Parameter(torch.ones(width))
            self.input_bias = nn.Parameter(torch.zeros(width))
        if num_classes is not None:
            self.head = nn.Parameter(torch.empty(num_classes, width))
            nn.init.normal_(self.head, std=1.0 / math.sqrt(width))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        with torch.autocast(x.device.type, enabled=False):
            return self._forward(x)

    def _forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.input_weight is not None:
            x = layer_norm(x, self.input_weight, self.input_bias, eps=self.input_eps)
        x, h = residual_norm(x, pre_weight=self.blocks[0].pre_weight, eps=self.eps)
        for block, after in zip(self.blocks, [*self.blocks[1:], None]):
            x, h = residual_norm(
                x, block(h), post_weight=block.post_weight, gate=block.gate(h),
                gate_act="sigmoid", scale=block.scale, eps=self.eps,
                pre_weight=self.norm_weight if after is None else after.pre_weight)
        return h

    def _head(self) -> torch.Tensor:
        if self.head is None:
            raise RuntimeError("KANExpertStack: no last layer (num_classes)")
        return self.head

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        """head h of the stack's rows h, [..., num_classes]."""
        head = self._head()
        h = self(x)
        with torch.autocast(x.device.type, enabled=False):
            return F.linear(h, head)

    def loss(self, x: torch.Tensor, target: torch.Tensor, **kw) -> torch.Tensor:
        """linear_cross_entropy of the stack's rows against target [...]; further
        arguments go to it."""
        head = self._head()
        return linear_cross_entropy(self(x), head, target, **kw)

    def distillation_loss(self, x: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor,
                          **kw) -> torch.Tensor:
        """linear_distillation of the stack's rows from a teacher's logits at ids
        [..., k] (`values, ids = teacher.logits(x).topk(k)`); further arguments go to
        it."""
        head = self._head()
        return linear_distillation(self(x), head, ids, teacher, **kw)
