"""linear_cross_entropy and linear_distillation against their definitions in
float64, losses and gradients.

Bounds, u = 2^-24 and H the half step of the operands' type relative to a value:
  z        a product's sum of D terms in float32: E = (D + 16) u of the sum of
           magnitudes (16: what a matrix instruction truncates inside)
  lse      moved by at most max E / tau by the logits, and relatively to the sum by C u
           (C = V / 64 + 64: a chain of its additions) and by the exponentials'
           arguments, (2 |z - top| / tau + 8) u each
  p        P = (2 |teacher| / tau + C) u relatively
  loss     tau^2 times what these move its terms by, and C u of the terms' magnitudes
  q        relatively by R, the sum of what moves z / tau, lse and its exponential
  dz       q R + p P, then one rounding H of q - p as the operand of the gradients'
           products (float16: of 2^15 (q - p), whose subnormals are 2^-24 apart)
and dx, dw as products over V and over the rows, rounded once.  What is below
float32's smallest normal number, 2^-126, may be lost wherever a value is formed."""

import ctypes

import pytest
import torch
import torch.nn.functional as F

from test_grouped import BF16, DTYPES, F16, F32, HALF_ULP
from torchsplinekan_amd import linear_cross_entropy, linear_distillation

U = 2.0 ** -24


def _inputs(T, V, D, dtype, k=0, seed=0):
    """x, w, target; with k x, w, ids [T, k], teacher [T, k]"""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * 2 * max(D, 1) ** -0.5).to(dtype)
    target = torch.randint(V, (T,), generator=g)
    x = (torch.randn(T, D, generator=g) + 1.5 * w[target].float()).to(dtype)
    if not k:
        return x, w, target
    ids = torch.rand(T, V, generator=g).topk(k, 1).indices
    return x, w, ids, 2 * torch.randn(T, k, generator=g)


def _expected(x, w, ids, teacher, tau, ignore, g, dtype):
    """rows' losses, dx, dw as (value, tolerance) in float64 on x's device; g: the
    gradient of each row's loss; ids [T, k], teacher [T, k] or None."""
    T, D = x.shape
    V = len(w)
    x, w = x.double(), w.double()
    C = V / 64 + 64
    z, E = x @ w.t(), (D + 16) * U * (x.abs() @ w.abs().t())
    there = (ids >= 0) & (ids < V)
    if teacher is None:
        there &= ids != ignore
        p, P = there.double(), torch.zeros_like(ids, dtype=torch.float64)
    else:
        v = torch.where(there, teacher.double() / tau, -torch.inf)
        p = torch.nan_to_num(v.softmax(1))
        P = (2 * torch.where(p > 0, v, 0.0).abs() + C) * U
    counts = (p > 0).any(1)
    zt, Et = z / tau, E / tau
    top, lse = zt.amax(1, keepdim=True), zt.logsumexp(1, keepdim=True)
    q = (zt - lse).exp()
    arg = (2 * (zt - top).abs() + 8) * U
    Elog = Et.amax(1, keepdim=True) + C * U + (q * arg).sum(1, keepdim=True)
    at = torch.where(there, ids, 0)
    logp = torch.where(p > 0, p, 1.0).log()
    zat = zt.gather(1, at)
    terms = torch.where(p > 0, p * (logp - (zat - lse)), 0.0)
    rows = tau ** 2 * terms.sum(1) * counts
    moved = (p * Et.gather(1, at)).sum(1) + Elog[:, 0]
    moved += (p * P * (1 + logp.abs() + (zat - lse).abs())).sum(1)
    moved += C * U * ((p * (logp.abs() + zat.abs())).sum(1) + top[:, 0].abs() + lse[:, 0].abs() + 1)
    Erows = tau ** 2 * moved * counts
    scat = torch.zeros_like(q).scatter_add_(1, at, p)
    spread = torch.zeros_like(q).scatter_add_(1, at, p * P)
    R = torch.expm1(Et + Elog + arg + C * U)
    d = q - scat
    Ed = q * R + spread + 4 * U * (q + scat)
    if dtype != F32:
        Ed = Ed + HALF_ULP[dtype] * (d.abs() + Ed) + (2.0 ** -40 if dtype == F16 else 0.0)
    f = (tau * g * counts)[:, None]
    # (the rows' shares of the largest weight are rounded too)
    Ed = Ed + 2.0 ** -125
    d, Ed = d * f, Ed * f.abs() + 8 * U * (d * f).abs() + 2.0 ** -126
    if dtype == F16:
        Ed = Ed + 2.0 ** -40 * f.abs().max() * (counts[:, None] > 0)
    out = []
    for a, Ea, b, terms in ((d, Ed, w, V), (d.t(), Ed.t(), x, T)):
        value = a @ b
        err = Ea @ b.abs() + (terms + 16) * U * ((a.abs() + Ea) @ b.abs())
        tol = err + HALF_ULP[dtype] * (value.abs() + err) + 2.0 ** -126
        out.append((value, tol + 2.0 ** -25 if dtype == F16 else tol))
    return (rows, Erows + U * rows.abs()), *out


def _near(got, want, what):
    value, tol = want
    bad = ~((got.detach().double().to(value.device) - value).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound"


def _call(x, w, ids, teacher, tau, ignore, reduction):
    if teacher is None:
        return linear_cross_entropy(x, w, ids, ignore_index=ignore, reduction=reduction)
    return linear_distillation(x, w, ids, teacher, temperature=tau, reduction=reduction)


def _check(x, w, ids, teacher=None, tau=1.0, ignore=-100, reductions=("none", "sum", "mean")):
    dtype, T = x.dtype, len(x)
    x, w, ids = x.cuda(), w.cuda(), ids.cuda()
    teacher = None if teacher is None else teacher.cuda()
    ids2 = ids[:, None] if teacher is None else ids
    gen = torch.Generator(device="cuda").manual_seed(1)
    xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
    for reduction in reductions:
        loss = _call(xd, wd, ids, teacher, tau, ignore, reduction)
        assert loss.dtype == F32 and loss.shape == ((T,) if reduction == "none" else ())
        g = torch.randn(loss.shape, generator=gen, device="cuda")
        dx, dw = torch.autograd.grad(loss, [xd, wd], g, retain_graph=True)
        for a, b in zip(torch.autograd.grad(loss, [xd, wd], g), (dx, dw)):
            assert torch.equal(a, b)
        with torch.no_grad():
            assert torch.equal(_call(xd, wd, ids, teacher, tau, ignore, reduction), loss)
        present = (ids2 != ignore if teacher is None
                   else (ids2 >= 0) & (teacher > -torch.inf)).any(1)
        n = present.sum().clamp(min=1)
        rows_g = g.double().expand(T) / (n if reduction == "mean" else 1)
        rows, wx, ww = _expected(x, w, ids2, teacher, tau, ignore, rows_g, dtype)
        if reduction == "none":
            _near(loss, rows, "loss")
        else:
            value, tol = (v.sum() / (n if reduction == "mean" else 1) for v in rows)
            _near(loss, (value, tol + 2 * U * value.abs()), reduction)
        assert dx.dtype == dtype and dw.dtype == dtype
        _near(dx, wx, f"dx of {reduction}")
        _near(dw, ww, f"dw of {reduction}")


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_cpu_cross_entropy_is_torchs(reduction):
    x, w, target = _inputs(12, 9, 5, torch.float64)
    target[[2, 7]] = -100
    x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, target, reduction=reduction)
    want = F.cross_entropy(x @ w.t(), target, reduction=reduction)
    torch.testing.assert_close(loss, want)
    g = torch.randn_like(loss)
    for a, b in zip(torch.autograd.grad(loss, [x, w], g), torch.autograd.grad(want, [x, w], g)):
        torch.testing.assert_close(a, b)


@pytest.mark.parametrize("tau", [1.0, 3.0])
def test_cpu_distillation_is_the_divergence(tau):
    x, w, ids, teacher = _inputs(6, 9, 5, torch.float64, k=4)
    teacher = teacher.double()
    p = (teacher / tau).softmax(1)
    want = tau ** 2 * (p * (p.log() - (x @ w.t() / tau).log_softmax(1).gather(1, ids))).sum(1)
    torch.testing.assert_close(linear_distillation(x, w, ids, teacher, temperature=tau,
                                                   reduction="none"), want)
    x.requires_grad_(), w.requires_grad_()
    ids[1, 2], ids[3] = -1, -1
    ids[4, 1] = ids[4, 0]
    assert torch.autograd.gradcheck(
        lambda a, b: linear_distillation(a, b, ids, teacher, temperature=tau), (x, w))


def test_cpu_rows_that_do_not_count():
    x, w, target = _inputs(4, 7, 3, F32)
    x.requires_grad_(), w.requires_grad_()
    none = linear_cross_entropy(x, w, torch.full((4,), 3), ignore_index=3)
    assert float(none) == 0.0
    for d in torch.autograd.grad(none, [x, w]):
        assert not bool(d.any())
    rows = linear_cross_entropy(x, w, torch.tensor([1, 7, -1, 2]), reduction="none")
    assert rows.isnan().tolist() == [False, True, True, False]
    ids, teacher = torch.tensor([[0, 1], [-1, -1], [2, 7], [3, 3]]), torch.zeros(4, 2)
    rows = linear_distillation(x, w, ids, teacher, reduction="none")
    assert rows.isnan().tolist() == [False, False, True, False] and float(rows[1]) == 0.0
    dead = linear_distillation(x[:1], w, ids[:1], torch.full((1, 2), -torch.inf))
    assert float(dead) == 0.0


def test_cpu_leading_shape_types_and_empty():
    x, w, target = _inputs(6, 7, 3, BF16)
    rows = linear_cross_entropy(x.reshape(2, 3, 3), w, target.reshape(2, 3).int(), reduction="none")
    assert rows.shape == (2, 3) and rows.dtype == F32
    assert float(linear_cross_entropy(x[:0], w, target[:0])) == 0.0
    assert linear_cross_entropy(x[:0], w, target[:0], reduction="none").shape == (0,)
    with torch.autocast("cpu", dtype=BF16):
        assert torch.equal(linear_cross_entropy(x.float(), w.float(), target),
                           linear_cross_entropy(x.float(), w.float(), target))


@pytest.mark.parametrize("make,text", [
    (lambda x, w, t, i, s: linear_cross_entropy(x, w, t.float()), "target must be int32"),
    (lambda x, w, t, i, s: linear_cross_entropy(x, w, t[:2]), "leading shape"),
    (lambda x, w, t, i, s: linear_cross_entropy(x, w[:, :2], t), "must equal D"),
    (lambda x, w, t, i, s: linear_cross_entropy(x, w.to(BF16), t), "share a dtype"),
    (lambda x, w, t, i, s: linear_cross_entropy(x, w[:0], t), "at least one row"),
    (lambda x, w, t, i, s: linear_cross_entropy(x, w[0], t), "weight \\[V, D\\]"),
    (lambda x, w, t, i, s: linear_cross_entropy(x, w, t, reduction="max"), "reduction must"),
    (lambda x, w, t, i, s: linear_distillation(x, w, t, s), "leading shape and k ids"),
    (lambda x, w, t, i, s: linear_distillation(x, w, i.double(), s), "ids must be int32"),
    (lambda x, w, t, i, s: linear_distillation(x, w, i, s[:, :1]), "ids' shape"),
    (lambda x, w, t, i, s: linear_distillation(x, w, i, i), "floating point"),
    (lambda x, w, t, i, s: linear_distillation(x, w, i[:, :0], s[:, :0]), "1 to 1024 ids"),
    (lambda x, w, t, i, s: linear_distillation(x, w, i, s, temperature=0.0), "temperature must"),
    (lambda x, w, t, i, s: linear_distillation(x, w, i, s, temperature=float("nan")),
     "temperature must"),
])
def test_refusals(make, text):
    x, w, ids, teacher = _inputs(4, 7, 3, F32, k=2)
    with pytest.raises(RuntimeError, match=text):
        make(x, w, ids[:, 0], ids, teacher)


def test_c_entry_refusals():
    from torchsplinekan_amd import _lib as lib
    L, n, p = lib.LIB, ctypes.c_size_t(), 4096

    def call(dtype=2, x=p, ids=p, teacher=None, T=4, V=8, D=8, k=0, tau=1.0, red=2, loss=p, kept=p,
             ws=p, size=1 << 40):
        return L.kan_hip_vocab_loss(dtype, x, p, ids, 1, teacher, T, V, D, k, -100, tau, red, loss,
                                    kept, ws, size, None)

    bad = [dict(dtype=1), dict(x=None), dict(ids=None), dict(loss=None), dict(kept=None), dict(T=-1),
           dict(V=0), dict(D=0), dict(k=-1), dict(k=1), dict(teacher=p), dict(tau=0.0), dict(tau=-1.0),
           dict(tau=float("nan")), dict(tau=float("inf")), dict(red=3), dict(kept=p + 4),
           dict(ws=p + 8)]
    for kw in bad:
        assert call(**kw) == lib.KAN_ERR_INVALID, kw
    for kw in (dict(T=1 << 30), dict(V=(1 << 22) + 1), dict(D=(1 << 22) + 1),
               dict(k=1025, teacher=p)):
        assert call(**kw) == lib.KAN_ERR_LIMIT, kw
    assert call(T=0, x=None, ids=None, loss=None, kept=None, ws=None) == lib.KAN_OK
    assert L.kan_hip_vocab_loss_kept(5, 99, 3, ctypes.byref(n)) == lib.KAN_OK
    assert n.value == 4 * (3 * 5 + 4 + 2 * 15)
    assert L.kan_hip_vocab_loss_kept(5, 10, 0, ctypes.byref(n)) == lib.KAN_OK
    assert n.value == 4 * (3 * 5 + 4 + 50)              # (few classes: their logits)
    assert L.kan_hip_vocab_loss_kept(5, 99, 3, None) == lib.KAN_ERR_INVALID
    assert L.kan_hip_vocab_loss_workspace(2, p, p, 4, 8, 8, None) == lib.KAN_ERR_INVALID

    def back(g=p, ids=p, dx=p, dw=p, ws=p, size=1 << 40, T=4):
        return L.kan_hip_vocab_loss_backward(2, g, p, p, ids, 1, p, T, 8, 8, 0, -100, 1.0, 2, dx, dw,
                                             ws, size, None)

    assert back(g=None) == lib.KAN_ERR_INVALID
    assert back(ids=None) == lib.KAN_ERR_INVALID
    assert back(ws=p + 8) == lib.KAN_ERR_INVALID
    assert back(dx=None, dw=None) == lib.KAN_OK
    assert back(T=0) == lib.KAN_OK


# ---------------------------------------------------------------------------
# device
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,D", [(1, 1), (2, 8), (10, 33), (17, 40), (64, 64), (65, 64), (128, 72), (129, 1), (1000, 200),
                                 (1025, 40), (2049, 17)])
@pytest.mark.parametrize("T", [1, 5, 33, 130, 300])
def test_cross_entropy_sizes(T, V, D, dtype):
    x, w, target = _inputs(T, V, D, dtype, seed=V)
    target[1::7] = -100
    _check(x, w, target)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D,k", [(1, 2, 8, 1), (5, 10, 33, 10), (40, 30, 257, 9), (33, 300, 64, 7),
                                     (130, 1000, 72, 64), (70, 2049, 40, 65), (3, 1024, 16, 1024),
                                     (300, 515, 24, 33)])
@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_distillation_sizes(T, V, D, k, tau, dtype):
    x, w, ids, teacher = _inputs(T, V, D, dtype, k=k, seed=V)
    g = torch.Generator().manual_seed(3)
    ids[torch.rand(T, k, generator=g) < 0.2] = -1          # absent, here and there
    ids[T // 2] = -1                                       # a row without any
    teacher[T - 1, : k // 2] = -torch.inf
    _check(x, w, ids.int() if T % 2 else ids, teacher, tau)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_ids_add(dtype):
    x, w, ids, teacher = _inputs(150, 400, 48, dtype, k=12)
    ids[:, 5], ids[:, 9] = ids[:, 2], ids[:, 2]
    _check(x, w, ids, teacher)
    ids[:] = 7
    _check(x, w, ids, teacher, 2.0)


# one size for every kind of tile, rows off 16 bytes among them
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,V,D,rows", [(8000, 4096, 64, 256), (8000, 4095, 61, 256),
                                        (5000, 2048, 72, 192), (5000, 2047, 71, 192),
                                        (8000, 4095, 301, 256), (2000, 1040, 136, 128)])
def test_kinds_of_tiles(T, V, D, rows, dtype):
    from torchsplinekan_amd import _lib as lib
    plan = (ctypes.c_int64 * 6)()
    lib.check(lib.LIB.kan_hip_grouped_matmul_plan(lib.OPERATOR_DTYPES[dtype], 0, 4096, 4096, 0, T, 1,
                                                  V, D, plan))
    assert plan[0] == rows
    x, w, target = _inputs(T, V, D, dtype)
    target[::5] = -100
    _check(x, w, target, reductions=("none", "mean"))
    x, w, ids, teacher = _inputs(T, V, D, dtype, k=20)
    _check(x, w, ids, teacher, 2.0, reductions=("mean",))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,V", [(BF16, 16000, 20000), (F16, 16000, 20003), (F32, 9000, 20000)])
def test_pieces_of_the_vocabulary(dtype, T, V):
    """(Logits of more than a piece's 512 MiB; rows of float64 a part at a time.)"""
    D = 40
    x, w, target = (t.cuda() for t in _inputs(T, V, D, dtype))
    target[::3] = -100
    xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(xd, wd, target, reduction="sum")
    dx, dw = torch.autograd.grad(loss, [xd, wd])
    g = torch.ones(T, dtype=torch.float64, device="cuda")
    total, slack, wv, wt = 0.0, 0.0, 0.0, 0.0
    for lo in range(0, T, 2000):
        r = slice(lo, lo + 2000)
        rows, ex, ew = _expected(x[r], w, target[r, None], None, 1.0, -100, g[r], dtype)
        _near(dx[r], ex, "dx")
        total, slack = total + rows[0].sum(), slack + rows[1].sum()
        wv, wt = wv + ew[0], wt + ew[1]
    _near(loss, (total, slack + 2 * U * total), "loss")
    # (each part's bound holds a rounding and a chain of its own; the chain of all rows
    # is as long as theirs together)
    _near(dw, (wv, wt * 2 + (T + 16) * U * wv.abs()), "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_are_off_by_two_roundings(dtype):
    """(An operand's rounding and the result's, each a uniform error of at most H:
    H (2 / 3)^(1/2) normwise, whatever the rows' common factor.)"""
    x, w, target = (t.cuda() for t in _inputs(3000, 2000, 256, dtype))
    x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, target, reduction="sum")
    got = torch.autograd.grad(loss, [x, w], torch.tensor(1.03, device="cuda"))
    want = _expected(x.detach(), w.detach(), target[:, None], None, 1.0, -100,
                     torch.full((3000,), 1.03, dtype=torch.float64, device="cuda"), dtype)[1:]
    for v, (value, _) in zip(got, want):
        assert float((v.double() - value).norm() / value.norm()) < HALF_ULP[dtype] * (2 / 3) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", [(1, 10), (70, 32), (40, 33), (300, 1500), (3, 5000)])
@pytest.mark.parametrize("ties", [False, True])
def test_rows_that_are_nearly_certain(T, V, ties, dtype):
    """Logits without rounding (sixteenths), targets ahead of the rest by 8 to 25: what
    is left of the loss, 1e-3 and below, is right in its own size, and so are gradients.
    Each exponential's argument is rounded in its product with log2(e) and by log2(e)
    itself, and comes out to 2 ulp: r = (3 |z - top| + 8) u; then a sum of V terms.
    ties: a row's largest logit is there twice (loss log 2 and more)."""
    g = torch.Generator().manual_seed(V + T)
    w = torch.randint(-3, 4, (V, 64), generator=g).float()
    w[:, 0] = 4
    target = torch.randint(1, V, (T,), generator=g)
    x = w[target] / 16
    if ties:
        w[0] = w[int(target[0])]
    z = x.double() @ w.double().t()
    top = z.amax(1, keepdim=True)
    assert bool((z.gather(1, target[:, None]) == top).all()) or ties
    e = (z - top).exp()
    hit = F.one_hot(target, V).double()
    rest = (e * (1 - hit)).sum(1, keepdim=True) if not ties else e.sum(1, keepdim=True) - 1
    rows = (torch.log1p(rest) + top - z.gather(1, target[:, None]))[:, 0]
    r = (3 * (z - top).amin().abs() + 8 + V) * U
    xd, wd = (t.to("cuda", dtype).requires_grad_() for t in (x, w))
    loss = linear_cross_entropy(xd, wd, target.cuda(), reduction="none")
    _near(loss, (rows, 2 * r * rows + 2.0 ** -126), "loss")
    dx, dw = torch.autograd.grad(loss, [xd, wd], torch.ones(T, device="cuda"))
    # q - 1 = ((e - 1) - rest) / (1 + rest), without the difference of nearly equal numbers
    d = ((e - hit) - hit * rest) / (1 + rest)
    H = HALF_ULP[dtype]
    # (float16: dz 2^15 times as large, subnormals 2^-24 apart)
    Ed = d.abs() * (2 * r + (0 if dtype == F32 else H)) + (2.0 ** -39 if dtype == F16 else 0.0)
    for got, a, E, b, terms in ((dx, d, Ed, w, V), (dw, d.t(), Ed.t(), x, T)):
        value = a @ b.double()
        err = (E + (2 * terms + 32) * U * (a.abs() + E)) @ b.double().abs()
        tol = err + H * (value.abs() + err) + (2.0 ** -25 if dtype == F16 else 2.0 ** -126)
        _near(got, (value, tol), "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,V,D", [(1, 2, 115), (3, 120, 128), (64, 9000, 40), (65, 1000, 72),
                                   (2048, 20, 64), (3, 100000, 64)])
@pytest.mark.parametrize("k", [0, 2])
def test_small_problems_round_their_gradients_once(T, V, D, k, dtype):
    """Up to 64 rows, or 4096 and 2^31 products of values, dz goes into its products in two parts:
    what is left of its rounding is H^2 of it, and the gradients' error their own
    rounding.  2^15 dz in float16 has subnormals 2^-24 apart in its second part."""
    x, w, ids, *teacher = _inputs(T, V, D, dtype, k, seed=V)
    x, w, ids = x.cuda(), w.cuda(), ids.cuda()
    teacher = teacher[0].cuda() if teacher else None
    if teacher is None:
        ids = ids[:, None]
    xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = _call(xd, wd, ids if k else ids[:, 0], teacher, 1.0, -100, "sum")
    H = HALF_ULP[dtype]
    got = torch.autograd.grad(loss, [xd, wd], torch.tensor(2.0, device="cuda"))
    g = torch.full((T,), 2.0, dtype=torch.float64, device="cuda")
    # the bound of float32 operands, with the second part's rounding and the last one
    _, *want = _expected(x.float(), w.float(), ids, teacher, 1.0, -100, g, F32)
    z = x.double() @ w.double().t()
    p = torch.zeros_like(z).scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float64)
                                         if teacher is None else teacher.double().softmax(1))
    d = (2 * (z.softmax(1) - p)).abs()
    part = 2 * H * H * d + (2.0 ** -38 if dtype == F16 else 0.0)
    for a, (value, tol), left in zip(got, want, (part @ w.double().abs(),
                                                 part.t() @ x.double().abs())):
        err = tol + 2 * left
        _near(a, (value, err + H * (value.abs() + err) + (2.0 ** -25 if dtype == F16 else 0.0)),
              "gradient")


@pytest.mark.gpu
def test_half_precision_keeps_small_probabilities():
    """A vocabulary whose probabilities are below float16's smallest numbers."""
    T, V, D = 64, 60000, 32
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(T, D, generator=g).to(F16), (torch.randn(V, D, generator=g) * 0.01).to(F16)
    target = torch.randint(100, (T,), generator=g)
    _check(x, w, target, reductions=("sum",))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits(dtype):
    """Far from zero, far apart, and rows that are sure of their answer."""
    x, w, target = _inputs(140, 300, 64, dtype)
    _check(x * 8, w * 8, target)
    far = x.clone()
    far[:, 0], w2 = 100.0, w.clone()
    w2[:, 0] = 50.0 if dtype != F16 else 5.0
    _check(far, w2, target)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_ids_that_are_no_columns_and_values_that_are_not_finite(dtype):
    x, w, target = (t.cuda() for t in _inputs(140, 300, 64, dtype))
    want = linear_cross_entropy(x, w, target, reduction="none")
    bad = target.clone()
    bad[3], bad[50], bad[100] = 300, -7, 1 << 40
    xd = x.clone().requires_grad_()
    rows = linear_cross_entropy(xd, w, bad, reduction="none")
    keep = [i for i in range(140) if i not in (3, 50, 100)]
    assert bool(rows[[3, 50, 100]].isnan().all()) and torch.equal(rows[keep], want[keep])
    dx, = torch.autograd.grad(rows.sum(), xd)
    assert bool(dx[[3, 50, 100]].isnan().all()) and bool(dx[keep].isfinite().all())
    # a row that does not count stays out of everything, whatever it holds
    nan = x.clone()
    nan[9] = float("nan")
    bad = target.clone()
    bad[9] = -100
    nan.requires_grad_()
    wd = w.clone().requires_grad_()
    loss = linear_cross_entropy(nan, wd, bad)
    dx, dw = torch.autograd.grad(loss, [nan, wd])
    assert bool(loss.isfinite()) and not bool(dx[9].any()) and bool(dx.isfinite().all())
    assert bool(dw.isfinite().all())
    # one that counts gives NaN
    assert linear_cross_entropy(nan.detach(), w, target, reduction="none").isnan().nonzero().tolist() \
        == [[9]]
    x2, w2, ids, teacher = (t.cuda() for t in _inputs(140, 300, 64, dtype, k=5))
    want = linear_distillation(x2, w2, ids, teacher, reduction="none")
    ids[3, 2], teacher[7, 1] = 300, float("nan")
    rows = linear_distillation(x2, w2, ids, teacher, reduction="none")
    keep = [i for i in range(140) if i not in (3, 7)]
    assert bool(rows[[3, 7]].isnan().all()) and torch.equal(rows[keep], want[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [20, 700])
def test_a_gradient_that_is_not_finite_stays_in_its_row(V, dtype):
    x, w, target = (t.cuda() for t in _inputs(100, V, 40, dtype))
    x.requires_grad_()
    g = torch.rand(100, device="cuda") + 0.5
    g[50] = 2.0
    loss = linear_cross_entropy(x, w, target, reduction="none")
    want, = torch.autograd.grad(loss, x, g, retain_graph=True)
    others = torch.ones(100, dtype=torch.bool, device="cuda")
    others[[3, 77]] = False
    g[3], g[77] = torch.inf, torch.nan
    got, = torch.autograd.grad(loss, x, g)
    if dtype == F32:
        # (a tile of the product that holds such values is evaluated a second time, without
        # the split of its operands: each result lies within a sum's bound)
        d = (x.double() @ w.double().t()).softmax(1).scatter_add_(
            1, target[:, None], torch.ones(100, 1, dtype=torch.float64, device="cuda"))
        tol = 2 * (V + 16) * U * ((2 * d) @ w.double().abs())
        assert bool(((got.double() - want.double()).abs() <= tol)[others].all())
    else:
        assert torch.equal(got[others], want[others])
    assert not bool(got[~others].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_row_counts(dtype):
    x, w, _ = (t.cuda() for t in _inputs(140, 300, 64, dtype))
    x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(x, w, torch.full((140,), -100, device="cuda"))
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert float(loss) == 0.0 and not bool(dx.any()) and not bool(dw.any())
    rows = linear_distillation(x, w, torch.full((140, 3), -1, device="cuda"),
                               torch.zeros(140, 3, device="cuda"), reduction="none")
    dx, dw = torch.autograd.grad(rows, [x, w], torch.ones_like(rows))
    assert not bool(rows.any()) and not bool(dx.any()) and not bool(dw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_only_one_gradient_shapes_and_strides(dtype):
    x, w, target = (t.cuda() for t in _inputs(60, 200, 48, dtype))
    xd, wd = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(linear_cross_entropy(xd, wd, target), [xd, wd])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xd, w, target), xd)[0], dx)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, wd, target), wd)[0], dw)
    x3 = x.t().contiguous().t().reshape(3, 20, 48).requires_grad_()
    w3 = w.t().contiguous().t().requires_grad_()
    loss = linear_cross_entropy(x3, w3, target.int().reshape(3, 20))
    d3 = torch.autograd.grad(loss, [x3, w3])
    assert torch.equal(d3[0].reshape(60, 48), dx) and torch.equal(d3[1], dw)
    rows = linear_cross_entropy(xd, wd, target, reduction="none")
    spread = torch.autograd.grad(rows.sum(), [xd, wd])         # (a gradient of stride 0)
    whole = torch.autograd.grad(linear_cross_entropy(xd, wd, target, reduction="sum"), [xd, wd])
    for a, b in zip(spread, whole):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_empty_and_refusals():
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    w = torch.zeros(5, 8, device="cuda", requires_grad=True)
    loss = linear_cross_entropy(x, w, torch.zeros(0, dtype=torch.long, device="cuda"))
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert float(loss) == 0.0 and dx.shape == (0, 8) and not bool(dw.any())
    x, t = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    with pytest.raises(RuntimeError, match="FP32, BF16 and FP16"):
        linear_cross_entropy(x.double(), w.double(), t)
    with pytest.raises(RuntimeError, match="one device"):
        linear_cross_entropy(x, w, t.cpu())
    with pytest.raises(RuntimeError, match="one device"):
        linear_distillation(x, w, t[:, None], torch.zeros(4, 1))
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError):
        linear_cross_entropy(fwAD.make_dual(x, torch.ones_like(x)), w, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [0, 6])
def test_other_stream_and_graph(k, dtype):
    inputs = [t.cuda() for t in _inputs(150, 600, 64, dtype, k=k)]
    x, w = inputs[0].requires_grad_(), inputs[1].requires_grad_()

    def step():
        loss = (linear_distillation if k else linear_cross_entropy)(x, w, *inputs[2:])
        return (loss.detach(), *torch.autograd.grad(loss, [x, w]))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        with torch.no_grad():
            x.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
