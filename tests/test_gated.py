"""gated_linear against its formulas in float64, forward and gradients.

Bounds, u = 2^-24 and H the half step of the results' type relative to a value:
  g, u     a sum of K products in float32: E = (K + 16) u of the sum of magnitudes
           (16: what a matrix instruction truncates inside)
  act(g)   F = (g^2 + 16) u relatively (the argument's rounding moves exp(-g) by |g| u
           and exp(-g^2 / 2) by g^2 u), and |act'| <= 1.13 for what g is off
  kept     g and u for the backward pass: 2^-12 of their value in bfloat16, 2^-16
           in float16
  act'(g)  F relatively to its terms' magnitudes (at most 1 + |g|), and |act''| <= 1
           for what g is off (relu: undecided where g is within that of 0)
  dg, du   one more rounding H each, as operands of the gradients' products
and the gradients' products over 2 N (dx) or the rows (dw) as g and u."""

import ctypes

import pytest
import torch

from test_grouped import BF16, DTYPES, F16, F32, HALF_ULP, _counts, _offsets
from torchsplinekan_amd import gated_linear

ACTS = [None, "sigmoid", "tanh", "silu", "gelu", "relu"]
U = 2.0 ** -24


def _act(g, act):
    """(act(g), act'(g))"""
    s, t = torch.sigmoid(g), torch.tanh(g)
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-g * 0.5 ** 0.5)
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * torch.pi) ** -0.5
    return {None: (g, torch.ones_like(g)), "sigmoid": (s, s * (1 - s)), "tanh": (t, 1 - t * t),
            "silu": (g * s, s * (1 + g * (1 - s))),
            "relu": (g.clamp(min=0), (g > 0).to(g.dtype))}[act]


def _inputs(T, E, K, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g).to(dtype)
    w = (torch.randn(E, 2, N, K, generator=g) * 1.5 * max(K, 1) ** -0.5).to(dtype)
    return x, w, torch.randn(T, N, generator=g).to(dtype)


def _rounded(value, err, dtype):
    """What a result in dtype may be off, computed with an error of `err`."""
    tol = err + HALF_ULP[dtype] * (value.abs() + err)
    return tol + 2.0 ** -25 if dtype == F16 else tol


def _expected(X, W, D, act, dtype):
    """{name: (value, tolerance)} of one expert's rows, in float64."""
    N, K = W.shape[1:]
    g, u = X @ W[0].t(), X @ W[1].t()
    Eg, Eu = [(K + 16) * U * (X.abs() @ w.abs().t()) for w in W]
    a, slope = _act(g, act)
    F = (g * g + 16) * U
    Ea = 1.13 * Eg + F * a.abs() + 2.0 ** -120
    r = {"h": (a * u, _rounded(a * u, Ea * (u.abs() + Eu) + a.abs() * Eu + 4 * U * (a * u).abs(),
                               dtype))}
    kept = {F32: 0.0, BF16: 2.0 ** -12, F16: 2.0 ** -16}[dtype]
    Kg, Ku = Eg + kept * (g.abs() + Eg), Eu + kept * (u.abs() + Eu)
    Es = Kg + F * (1 + g.abs())
    if act == "relu":
        Es = torch.where(g.abs() <= Kg, 1.0, Es)
    Ea = 1.13 * Kg + F * a.abs() + 2.0 ** -120
    dg, du = D * u * slope, D * a
    Edg = D.abs() * ((u.abs() + Ku) * (slope.abs() + Es) - (u * slope).abs()) + 4 * U * dg.abs()
    Edu = D.abs() * Ea + 4 * U * du.abs()
    d = torch.cat([dg, du], 1)
    Ed = torch.cat([Edg, Edu], 1)
    if dtype != F32:
        Ed = _rounded(d, Ed, dtype)
    w = W.reshape(2 * N, K)
    dx, dw = d @ w, d.t() @ X
    Ex = Ed @ w.abs() + (2 * N + 16) * U * ((d.abs() + Ed) @ w.abs())
    Ew = Ed.t() @ X.abs() + (len(X) + 16) * U * ((d.abs() + Ed).t() @ X.abs())
    r["dx"] = (dx, _rounded(dx, Ex, dtype))
    r["dw"] = (dw.reshape(W.shape), _rounded(dw, Ew, dtype).reshape(W.shape))
    return r


def _near(got, want, what):
    value, tol = want
    bad = ~((got.detach().double().to(value.device) - value).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound"


def _check(x, w, dh, offsets, act="silu", where="cpu"):
    """offsets None: dense, w [1, 2, N, K]."""
    xd, wd = x.cuda().requires_grad_(), (w if offsets is not None else w[0]).cuda().requires_grad_()
    off = None if offsets is None else offsets.cuda()
    h = gated_linear(xd, wd, off, act=act)
    assert h.dtype == x.dtype and h.shape == dh.shape
    dx, dw = torch.autograd.grad(h, [xd, wd], dh.cuda(), retain_graph=True)
    for a, b in zip(torch.autograd.grad(h, [xd, wd], dh.cuda()), (dx, dw)):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(gated_linear(xd, wd, off, act=act), h)
    dw = dw.reshape(w.shape)
    ends = [len(x)] if offsets is None else offsets.tolist()[1:]
    X, W, D = (t.to(where).double() for t in (x, w, dh))
    lo = 0
    for e, hi in enumerate(ends):
        r = slice(lo, hi)
        want = _expected(X[r], W[e], D[r], act, x.dtype)
        _near(h[r], want["h"], f"h of {e}")
        _near(dx[r], want["dx"], f"dx of {e}")
        _near(dw[e], want["dw"], f"dw of {e}")
        lo = hi
    assert not bool(h[lo:].any()) and not bool(dx[lo:].any())


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("act", ACTS)
def test_cpu_against_formulas_and_differences(act):
    x, w, dh = _inputs(7, 2, 5, 3, torch.float64)
    off = _offsets([4, 2])
    x.requires_grad_(), w.requires_grad_()
    assert torch.autograd.gradcheck(lambda a, b: gated_linear(a, b, off, act=act), (x, w))
    h = gated_linear(x, w, off, act=act)
    g, u = x[:4] @ w[0, 0].t(), x[:4] @ w[0, 1].t()
    torch.testing.assert_close(h[:4], _act(g, act)[0] * u)
    assert not bool(h[6:].any())
    torch.testing.assert_close(gated_linear(x[:4].reshape(2, 2, 5), w[0], act=act).reshape(4, 3),
                               h[:4])


def test_cpu_sums_under_autocast():
    x, w, _ = _inputs(9, 1, 40, 5, F32)
    want = gated_linear(x, w[0])
    with torch.autocast("cpu", dtype=BF16):
        got = gated_linear(x, w[0])
    assert got.dtype == F32 and torch.equal(got, want)


@pytest.mark.parametrize("x,w,off,kw,text", [
    (torch.zeros(4, 5), torch.zeros(3, 6, 5), None, {}, "weight must be"),
    (torch.zeros(4, 5), torch.zeros(6, 5), None, {}, "weight must be"),
    (torch.zeros(4, 5), torch.zeros(2, 6, 4), None, {}, "must equal K"),
    (torch.zeros(4, 5), torch.zeros(2, 6, 5).to(BF16), None, {}, "share a dtype"),
    (torch.zeros(4, 5), torch.zeros(2, 6, 5), None, dict(act="swish"), "act must be"),
    (torch.zeros(4, 5), torch.zeros(2, 6, 5), torch.zeros(2, dtype=torch.int32), {}, "with offsets"),
    (torch.zeros(4, 5), torch.zeros(3, 2, 6, 5), torch.zeros(3, dtype=torch.int32), {},
     "offsets must be"),
    (torch.zeros(4, 5), torch.zeros(3, 2, 6, 5), torch.zeros(4), {}, "int32 or int64"),
])
def test_refusals(x, w, off, kw, text):
    with pytest.raises(RuntimeError, match=text):
        gated_linear(x, w, off, **kw)


def test_c_entry_refusals():
    from torchsplinekan_amd import _lib as lib
    L, n, p = lib.LIB, ctypes.c_size_t(), 4096

    def call(dtype=2, act=3, x=p, off=p, T=64, E=2, N=16, K=16, h=p, kept=None):
        return L.kan_hip_gated(dtype, act, x, p, off, 0, T, E, N, K, h, kept, None, 0, None)

    assert call(dtype=lib.KAN_DTYPE_F64) == lib.KAN_ERR_INVALID
    assert call(act=6) == lib.KAN_ERR_INVALID
    assert call(x=None) == lib.KAN_ERR_INVALID
    assert call(off=None) == lib.KAN_ERR_INVALID
    assert call(h=None) == lib.KAN_ERR_INVALID
    assert call(kept=p + 8) == lib.KAN_ERR_INVALID
    assert call(T=-1) == lib.KAN_ERR_INVALID
    assert call(N=(1 << 21) + 1) == lib.KAN_ERR_LIMIT
    assert call(E=1 << 16) == lib.KAN_ERR_LIMIT
    assert call(x=None, off=None, h=None, T=0) == lib.KAN_OK
    assert call(dtype=0, T=1000) == lib.KAN_ERR_WORKSPACE
    assert L.kan_hip_gated_kept(0, 10, 3, ctypes.byref(n)) == lib.KAN_OK and n.value == 240
    assert L.kan_hip_gated_kept(2, 10, 3, ctypes.byref(n)) == lib.KAN_OK and n.value == 128 + 30
    assert L.kan_hip_gated_kept(3, 10, 3, ctypes.byref(n)) == lib.KAN_OK and n.value == 128 + 60
    assert L.kan_hip_gated_kept(2, 10, 3, None) == lib.KAN_ERR_INVALID
    assert L.kan_hip_gated_workspace(2, p, p, 4, 2, 16, 16, 0, None) == lib.KAN_ERR_INVALID
    back = L.kan_hip_gated_backward
    assert back(1, 3, p, p, 4, 16, p, None) == lib.KAN_ERR_INVALID
    assert back(2, 3, None, p, 4, 16, p, None) == lib.KAN_ERR_INVALID
    assert back(2, 3, p, p + 4, 4, 16, p, None) == lib.KAN_ERR_INVALID
    assert back(2, 3, None, None, 0, 16, None, None) == lib.KAN_OK


# ---------------------------------------------------------------------------
# device
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(1, 1), (1, 70), (33, 1), (8, 8), (16, 48), (64, 32), (100, 60),
                                 (301, 257), (136, 264)])
@pytest.mark.parametrize("T", [1, 5, 16, 17, 70, 300])
def test_dense_sizes(T, K, N, dtype):
    _check(*_inputs(T, 1, K, N, dtype), None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [3, 200])
def test_activations(T, act, dtype):
    x, w, dh = _inputs(T, 1, 96, 40, dtype, seed=1)
    _check(x, w, dh, None, act)
    _check(x * 6, w, dh, None, act)       # g to +-40


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(40, 72), (33, 31)])
@pytest.mark.parametrize("counts", [[1], [5, 0, 1, 40], [0, 0, 70, 0], [64, 128, 130], [300, 3]])
def test_experts(counts, K, N, dtype):
    x, w, dh = _inputs(sum(counts) + 9, len(counts), K, N, dtype)
    _check(x, w, dh, _offsets(counts, torch.int64))     # 9 rows behind the last expert's


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,E,N,K,rows,align", [
    (5000, 1, 1024, 200, 192, 0), (8000, 1, 2048, 64, 256, 0), (1500, 1, 520, 1024, 128, 0),
    (700, 70, 96, 72, 128, 0), (9000, 2, 1001, 531, 192, 3), (8000, 1, 2047, 301, 256, 3),
    (8000, 1, 2047, 61, 256, 0), (16, 2, 200, 513, 16, 0),
    (128, 16, 1024, 256, 16, 0), (700, 3, 130, 77, 128, 0)])
def test_kinds_of_tiles(T, E, N, K, rows, align, dtype):
    from torchsplinekan_amd import _lib as lib
    x, w, dh = _inputs(T, E, K, N, dtype)
    plan = (ctypes.c_int64 * 6)()
    lib.check(lib.LIB.kan_hip_grouped_matmul_plan(lib.OPERATOR_DTYPES[dtype], 0, 4096, 4096, 0, T, E,
                                                  2 * N, K, plan))
    assert (plan[0], plan[4]) == (rows, align)
    _check(x, w, dh, _offsets(_counts(T, E, seed=E)), where="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,N,K,dense", [
    ([17], 256, 4096, True), ([64], 512, 2048, True), ([33], 203, 4100, True),
    ([200], 72, 8192, True), ([40], 8, 2051, True), ([60, 0, 90], 64, 2048, False),
    ([0, 129, 2], 77, 3000, False)])
def test_sums_in_cuts(counts, N, K, dense, dtype):
    """Few tiles and long sums: partial sums that another kernel joins."""
    T, E = sum(counts), len(counts)
    x, w, dh = _inputs(T, E, K, N, dtype)
    from torchsplinekan_amd import _lib as lib
    nbytes = ctypes.c_size_t()
    for keep in (0, 1):
        lib.check(lib.LIB.kan_hip_gated_workspace(
            lib.OPERATOR_DTYPES[dtype], 4096, 4096, T, E, N, K, keep, ctypes.byref(nbytes)))
        assert nbytes.value >= 2 * 4 * T * 2 * N
    _check(x, w, dh, None if dense else _offsets(counts), where="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sums_in_cuts_of_rows_behind_the_last_expert(dtype):
    x, w, _ = _inputs(90, 2, 2048, 40, dtype)
    h = gated_linear(x.cuda(), w.cuda(), torch.tensor([0, 30, 70], device="cuda"), act="sigmoid")
    assert bool(h[:70].any(1).all()) and not bool(h[70:].any())
    for r, e in ((slice(0, 30), 0), (slice(30, 70), 1)):
        want = _expected(x[r].double(), w[e].double(), torch.zeros(1, 40).double(), "sigmoid", dtype)
        _near(h[r], tuple(v.cuda() for v in want["h"]), "h")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_are_off_by_two_roundings(dtype):
    """(An operand's rounding and the result's, each a uniform error of at most H:
    H (2 / 3)^(1/2) normwise; the kept values' bits leave no trace.)"""
    x, w, dh = _inputs(2000, 1, 512, 640, dtype)
    xd, wd = x.cuda().requires_grad_(), w[0].cuda().requires_grad_()
    got = torch.autograd.grad(gated_linear(xd, wd), [xd, wd], dh.cuda())
    want = _expected(x.cuda().double(), w[0].cuda().double(), dh.cuda().double(), "silu", dtype)
    for v, name in zip(got, ("dx", "dw")):
        value = want[name][0]
        assert float((v.double() - value).norm() / value.norm()) < HALF_ULP[dtype] * (2 / 3) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_sizes(dtype):
    for T, K, N in ((0, 8, 8), (5, 0, 8), (5, 8, 0)):
        x = torch.zeros(T, K, dtype=dtype, device="cuda", requires_grad=True)
        w = torch.zeros(2, N, K, dtype=dtype, device="cuda", requires_grad=True)
        h = gated_linear(x, w, act="sigmoid")
        assert h.shape == (T, N) and not bool(h.any())
        dx, dw = torch.autograd.grad(h.sum(), [x, w])
        assert dx.shape == x.shape and dw.shape == w.shape
        assert not bool(dx.any()) and not bool(dw.any())
    x = torch.ones(5, 8, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.zeros(0, 2, 6, 8, dtype=dtype, device="cuda", requires_grad=True)
    h = gated_linear(x, w, torch.zeros(1, dtype=torch.int32, device="cuda"))
    dx, _ = torch.autograd.grad(h.sum(), [x, w])
    assert h.shape == (5, 6) and not bool(h.any()) and not bool(dx.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [4, 150])
def test_offsets_that_say_anything(T, dtype):
    """Taken within 0 .. T and as their running maximum."""
    x, w, _ = _inputs(T, 3, 40, 24, dtype)
    got = gated_linear(x.cuda(), w.cuda(),
                       torch.tensor([-5, 3, 1, 1 << 40], dtype=torch.int64, device="cuda"))
    want = gated_linear(x.cuda(), w.cuda(), torch.tensor([0, 3, 3, T], device="cuda"))
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [4, 150])
def test_strides_and_offsets_of_memory(T, dtype):
    x, w, dh = (t.cuda() for t in _inputs(T, 1, 40, 24, dtype))
    want = gated_linear(x, w[0])
    wide = torch.zeros(T, 50, dtype=dtype, device="cuda")
    wide[:, 3:43] = x
    assert torch.equal(gated_linear(wide[:, 3:43], w[0]), want)
    loose = torch.zeros(w.numel() + 1, dtype=dtype, device="cuda")
    loose[1:] = w.reshape(-1)
    moved = loose[1:].reshape(2, 24, 40)
    torch.testing.assert_close(gated_linear(x, moved), want, rtol=4 * HALF_ULP[dtype],
                               atol=HALF_ULP[dtype])
    xt = x.t().contiguous().t().requires_grad_()
    wt = w[0].transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    h = gated_linear(xt, wt)
    assert torch.equal(h, want)
    g = torch.autograd.grad(h, [xt, wt], dh.t().contiguous().t())
    xc, wc = x.detach().requires_grad_(), w[0].detach().requires_grad_()
    for a, b in zip(g, torch.autograd.grad(gated_linear(xc, wc), [xc, wc], dh)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_that_are_not_finite(dtype):
    """They stay in their rows, and NaN is kept as NaN for the gradients.  (A float32
    tile that meets them evaluates all its rows again, by products that are not
    split: each way is within the bound, not bit for bit the other.)"""
    x, w, dh = (t.cuda() for t in _inputs(150, 1, 64, 40, dtype))
    w = w[0]
    want = gated_linear(x, w)
    bad = x.clone()
    bad[7, 3], bad[90, 0] = float("nan"), float("inf")
    bad.requires_grad_()
    h = gated_linear(bad, w)
    keep = [i for i in range(150) if i not in (7, 90)]
    assert bool(h[7].isnan().all())
    if dtype == F32:
        _near(h[keep], _expected(x[keep].double(), w.double(), dh[keep].double(), "silu", F32)["h"],
              "the other rows")
    else:
        assert torch.equal(h[keep], want[keep])
    dx, = torch.autograd.grad(h, bad, dh)
    assert bool(dx[7].isnan().all()) and bool(dx[keep].isfinite().all())


@pytest.mark.gpu
def test_device_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(2, 6, 8, device="cuda")
    with pytest.raises(RuntimeError, match="FP32, BF16 and FP16"):
        gated_linear(x.double(), w.double())
    with pytest.raises(RuntimeError, match="one device"):
        gated_linear(x, w.cpu())
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError):
        gated_linear(fwAD.make_dual(x, torch.ones_like(x)), w)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 300])
def test_other_stream_and_graph(T):
    x, w, dh = (t.cuda() for t in _inputs(T, 3, 64, 40, BF16))
    off = _offsets([T // 2, 0, T // 3]).cuda()
    x.requires_grad_(), w.requires_grad_()

    def step():
        h = gated_linear(x, w, off)
        return (h.detach(), *torch.autograd.grad(h, [x, w], dh))

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
    for k in range(3):
        with torch.no_grad():
            x.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_sums_in_cuts_in_two_graphs():
    """Two captured calls, replayed in turn with eager ones between them: each has
    partial sums of its own."""
    w = _inputs(1, 1, 4096, 192, BF16)[1][0].cuda()
    xs = [_inputs(T, 1, 4096, 192, BF16, seed=T)[0].cuda() for T in (48, 70)]
    with torch.no_grad():
        want = [gated_linear(x, w) for x in xs]
        torch.cuda.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in xs]
        out = []
        for x, graph in zip(xs, graphs):
            with torch.cuda.graph(graph):
                out.append(gated_linear(x, w))
        for _ in range(3):
            for k in (0, 1):
                graphs[k].replay()
                assert torch.equal(gated_linear(xs[1 - k], w), want[1 - k])
                torch.cuda.synchronize()
                assert torch.equal(out[k], want[k])
                out[k].zero_()
