"""The losses at more rows than a launch of a wave each can have (2^26), past 2^31 bytes and
values: every row against the logits written out, piece by piece.

Bound, as of the other sizes: u = 2^-24; a logit of D = 8 products is off by 24 u of
|x| |w|, Z its largest over a row; the loss by twice that, by 16 u of Z (exponentials), and
by 8 u of itself."""

import pytest
import torch

from torchsplinekan_amd import _lib as lib
from torchsplinekan_amd import linear_cross_entropy, linear_distillation

U, STEP = 2.0 ** -24, 1 << 22


def _draw(T, V, D, dtype, high):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, D, generator=g, device="cuda", dtype=dtype)
    w = torch.randn(V, D, generator=g, device="cuda", dtype=dtype)
    return x, w, torch.randint(high, (T,), generator=g, device="cuda", dtype=torch.int32)


def _compare(rows, x, w, ids):
    for lo in range(0, len(x), STEP):
        r = slice(lo, lo + STEP)
        xs, t = x[r].double(), ids[r]
        z = xs @ w.double().t()
        on = t >= 0
        want = z.logsumexp(1) - z.gather(1, t.clamp(min=0).long().unsqueeze(1))[:, 0]
        want = torch.where(on, want, 0.0)
        Z = (xs.abs() @ w.double().abs().t()).amax(1)
        tol = (2 * 24 + 16) * U * Z + 8 * U * want.abs()
        assert bool(((rows[r] - want).abs() <= tol).all()), lo


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,V,D", [
    (torch.bfloat16, (1 << 26) + 37, 40, 8), (torch.float32, (1 << 26) + 37, 33, 8),
    (torch.bfloat16, (1 << 28) + 3, 3, 2)])
def test_cross_entropy(dtype, T, V, D):
    x, w, target = _draw(T, V, D, dtype, V + 1)
    target[target == V] = -100
    with torch.no_grad():
        _compare(linear_cross_entropy(x, w, target, reduction="none"), x, w, target)


@pytest.mark.gpu
def test_distillation_of_one_id_is_its_cross_entropy():
    x, w, ids = _draw((1 << 26) + 37, 40, 8, torch.bfloat16, 41)
    ids -= 1                                    # (-1: absent)
    with torch.no_grad():
        rows = linear_distillation(x, w, ids.unsqueeze(1), torch.randn(len(x), 1, device="cuda"),
                                   reduction="none")
        _compare(rows, x, w, ids)


@pytest.mark.gpu
def test_gradient_of_the_rows():
    """dz W of every row; the rows' own weights."""
    T, V, D = (1 << 26) + 37, 40, 8
    x, w, target = _draw(T, V, D, torch.bfloat16, V)
    x.requires_grad_()
    dx, = torch.autograd.grad(linear_cross_entropy(x, w, target, reduction="sum"), x)
    for lo in range(0, T, STEP):
        r = slice(lo, lo + STEP)
        xs = x[r].detach().double()
        p = (xs @ w.double().t()).softmax(1)
        Z = (xs.abs() @ w.double().abs().t()).amax(1, keepdim=True)
        p.scatter_add_(1, target[r].long().unsqueeze(1), p.new_full((len(p), 1), -1.0))
        want, size = p @ w.double(), p.abs() @ w.double().abs()
        # dz rounded to bfloat16 and off by its logits' errors; then the result's rounding
        tol = (2.0 ** -8 + 2 * (2 * 24 + 16) * U * Z) * size + 2.0 ** -8 * want.abs()
        assert bool(((dx[r].double() - want).abs() <= tol).all()), lo


def test_tiles_beyond_a_grid_are_refused():
    """(2^39 logits: the check of a launch that never takes place; the operands are not read.)"""
    L, p = lib.LIB, 4096
    nbytes = lib.ctypes.c_size_t()
    T, V, D = 1 << 25, 1 << 15, 64
    lib.check(L.kan_hip_vocab_loss_workspace(2, p, p, T, V, D, lib.ctypes.byref(nbytes)))
    rc = L.kan_hip_vocab_loss(2, p, p, p, 0, None, T, V, D, 0, -100, 1.0, 0, p, p, p, nbytes.value,
                              None)
    assert rc == lib.KAN_ERR_LIMIT and "too many tiles" in lib.last_error()
