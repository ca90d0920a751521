"""layer_norm against its formulas in float64, forward and gradients.

Bounds (u = 2^-24, a chain of k float32 operations is off by k u of the sum of
magnitudes).  A sum over a row has at most C / 64 + 32 terms in a chain (a
lane's values, or C / 256 of rows that no registers hold, then a tree), one over
rows at most n / 64 + 64 (a block's rows, then the blocks' partial rows in 16
lanes); L = C / 64 + n / 64 + 128 covers both and the few products between them.
  x - m        off by L u X,             X = |x| + mean|x|
  r            relatively by L u R,      R = mean(|xh| r X)  (of the variance; halved by the root)
  xh           L u H,                    H = r X + |xh| R
and dx, dw and db by the sums of their terms' errors; then one rounding to the
result's type."""

import ctypes

import pytest
import torch

from torchsplinekan_amd import layer_norm

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_ULP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
EPS = 1e-5


def _formulas(x, w, b, dy):
    """{name: (value, magnitude that its error is counted in)} in float64."""
    x, dy = x.double(), dy.double()
    C = x.shape[-1]
    x, dy = x.reshape(-1, C), dy.reshape(-1, C)
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double()
    mean = lambda v: v.mean(-1, keepdim=True)
    xc = x - mean(x)
    r = 1 / (xc.square().mean(-1, keepdim=True) + EPS).sqrt()
    xh, X = xc * r, x.abs() + mean(x.abs())
    R = mean(xh.abs() * r * X)
    H = r * X + xh.abs() * R
    t = dy * w
    ta, xa = t.abs(), xh.abs()
    inner = ta + mean(ta) + xa * mean(ta * xa)
    return {
        "y": (xh * w + b, H * w.abs() + b.abs()),
        "dx": (r * (t - mean(t) - xh * mean(t * xh)),
               r * ((1 + R) * inner + H * mean(ta * xa) + xa * mean(ta * H))),
        "dw": ((dy * xh).sum(0), (dy.abs() * H).sum(0)),
        "db": (dy.sum(0), dy.abs().sum(0)),
    }


def _bound(got, value, mag, n, C, what):
    got = got.detach().cpu()
    value, mag = value.reshape(got.shape), mag.reshape(got.shape)
    chain = (C / 64 + n / 64 + 128) * 2.0 ** -24
    tol = chain * mag + HALF_ULP[got.dtype] * (value.abs() + chain * mag)
    if got.dtype == F16:
        tol = tol + 2.0 ** -25        # (spacing of its subnormals)
    bad = ~((got.double() - value).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound"


def _inputs(shape, xdt, ydt, wdt, weight=True, bias=True, mean=0.3, seed=0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (2 * torch.randn(*shape, generator=g) + mean).to(xdt)
    w = (1 + 0.1 * torch.randn(C, generator=g)).to(wdt) if weight else None
    b = (0.1 * torch.randn(C, generator=g)).to(wdt) if bias else None
    return x, w, b, torch.randn(*shape, generator=g).to(ydt)


def _check(x, w, b, dy):
    n, C = x.numel() // x.shape[-1], x.shape[-1]
    want = _formulas(x, w, b, dy)
    leaves = [None if t is None else t.cuda().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps=EPS, dtype=dy.dtype)
    assert y.dtype == dy.dtype and y.shape == x.shape
    with torch.no_grad():
        assert torch.equal(layer_norm(*leaves, eps=EPS, dtype=dy.dtype), y)
    there = [t for t in leaves if t is not None]
    got = iter(torch.autograd.grad(y, there, dy.cuda(), retain_graph=True))
    again = torch.autograd.grad(y, there, dy.cuda())
    _bound(y, *want["y"], 1, C, "y")
    for name, t, rows in (("dx", leaves[0], 1), ("dw", leaves[1], n), ("db", leaves[2], n)):
        if t is not None:
            v = next(got)
            assert v.dtype == t.dtype and v.shape == t.shape
            _bound(v, *want[name], rows, C, name)
    for t, v in zip(again, torch.autograd.grad(layer_norm(*leaves, eps=EPS, dtype=dy.dtype), there,
                                               dy.cuda())):
        assert torch.equal(t, v)


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------

def test_cpu_against_formulas_and_differences():
    x, w, b, dy = _inputs((3, 5, 7), torch.float64, torch.float64, torch.float64)
    for t in (x, w, b):
        t.requires_grad_()
    y = layer_norm(x, w, b, eps=EPS)
    want = _formulas(x.detach(), w.detach(), b.detach(), dy)
    torch.testing.assert_close(y.reshape(-1, 7), want["y"][0])
    got = torch.autograd.grad(y, [x, w, b], dy)
    for v, name in zip(got, ("dx", "dw", "db")):
        torch.testing.assert_close(v.reshape(want[name][0].shape), want[name][0])
    assert torch.autograd.gradcheck(lambda *t: layer_norm(*t, eps=EPS), (x, w, b))


def test_cpu_result_type_and_empty():
    x, w, b, _ = _inputs((4, 9), F32, BF16, BF16)
    assert layer_norm(x, w, b, dtype=BF16).dtype == BF16
    assert layer_norm(x[:0], w, b).shape == (0, 9)


def test_refusals():
    x = torch.zeros(4, 6)
    with pytest.raises(RuntimeError, match="weight must have shape"):
        layer_norm(x, torch.ones(5))
    with pytest.raises(RuntimeError, match="bias must have shape"):
        layer_norm(x, None, torch.ones(6, 1))
    with pytest.raises(RuntimeError, match="share a dtype"):
        layer_norm(x, torch.ones(6), torch.ones(6, dtype=BF16))
    with pytest.raises(RuntimeError, match="result's type or float32"):
        layer_norm(x.to(BF16), dtype=F32)
    with pytest.raises(RuntimeError, match="at least one dimension"):
        layer_norm(torch.zeros(()))


def test_c_refusals():
    from torchsplinekan_amd import _lib as lib
    L, f32, bf16, n = lib.LIB, lib.KAN_DTYPE_F32, lib.KAN_DTYPE_BF16, ctypes.c_size_t()
    fwd = lambda *c, x=16, y=16, rows=4: L.kan_hip_layer_norm(*c, x, None, None, rows, 8, 1e-5, y,
                                                              None, None)
    assert fwd(lib.KAN_DTYPE_F64, f32, f32) == lib.KAN_ERR_INVALID
    assert fwd(bf16, f32, f32) == lib.KAN_ERR_INVALID
    assert fwd(f32, f32, f32, x=None) == lib.KAN_ERR_INVALID
    assert fwd(f32, f32, f32, y=None) == lib.KAN_ERR_INVALID
    assert fwd(f32, f32, f32, rows=-1) == lib.KAN_ERR_INVALID
    assert fwd(f32, f32, f32, x=None, rows=0) == lib.KAN_OK
    assert L.kan_hip_layer_norm_backward_workspace(4, 8, None) == lib.KAN_ERR_INVALID
    assert L.kan_hip_layer_norm_backward_workspace(-4, 8, ctypes.byref(n)) == lib.KAN_ERR_INVALID
    assert L.kan_hip_layer_norm_backward_workspace(4, 8, ctypes.byref(n)) == lib.KAN_OK
    assert n.value >= 2 * 8 * 4
    bwd = lambda ws, size, dw=16: L.kan_hip_layer_norm_backward(
        f32, f32, f32, 16, 16, None, 16, 4, 8, 16, dw, None, ws, size, None)
    assert bwd(None, 0) == lib.KAN_ERR_WORKSPACE
    assert bwd(16, n.value - 1) == lib.KAN_ERR_WORKSPACE
    assert bwd(8, n.value) == lib.KAN_ERR_INVALID


# ---------------------------------------------------------------------------
# device
# ---------------------------------------------------------------------------

# one width for every shape of a row, whole vectors and odd ends
@pytest.mark.gpu
@pytest.mark.parametrize("C", [1, 7, 64, 100, 128, 136, 201, 256, 257, 512, 1000, 1024, 1025, 2048,
                               4097, 8192, 9999, 16384, 16385])
@pytest.mark.parametrize("xdt,ydt", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16)])
def test_widths(C, xdt, ydt):
    _check(*_inputs((77, C), xdt, ydt, ydt, seed=C))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 9, 1023, 5003])
@pytest.mark.parametrize("C", [64, 301])
def test_rows(n, C):
    _check(*_inputs((n, C), F32, F32, F32, seed=n))
    _check(*_inputs((n, C), BF16, BF16, F32, seed=n))


@pytest.mark.gpu
@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(weight, bias):
    _check(*_inputs((3, 11, 200), F16, F16, F16, weight, bias))


@pytest.mark.gpu
def test_rows_far_from_zero():
    """(The variance is taken of the values less their mean.)"""
    _check(*_inputs((40, 512), F32, F32, F32, mean=1000.0))
    x = torch.full((3, 300), 7.0, device="cuda")
    assert not bool(layer_norm(x).any())


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_rows():
    x, w, b, _ = _inputs((6, 130), F32, F32, F32)
    want = layer_norm(x.cuda(), w.cuda(), b.cuda())
    x[1, 3], x[4, 0] = float("inf"), float("nan")
    got = layer_norm(x.cuda(), w.cuda(), b.cuda())
    assert bool(got[[1, 4]].isnan().all())
    keep = [0, 2, 3, 5]
    assert torch.equal(got[keep], want[keep])


@pytest.mark.gpu
def test_strides_and_offsets():
    x, w, b, dy = _inputs((33, 96), BF16, BF16, BF16)
    wide = torch.zeros(33, 200, dtype=BF16, device="cuda")
    wide[:, 5:101] = x.cuda()
    loose = torch.zeros(33 * 96 + 1, dtype=BF16, device="cuda")
    loose[1:] = x.cuda().reshape(-1)
    w2 = torch.zeros(97, dtype=BF16, device="cuda")
    w2[1:] = w.cuda()
    want = layer_norm(x.cuda(), w.cuda(), b.cuda())
    assert torch.equal(layer_norm(wide[:, 5:101], w.cuda(), b.cuda()), want)
    got = layer_norm(loose[1:].reshape(33, 96), w2[1:], b.cuda())
    torch.testing.assert_close(got, want, rtol=2 ** -7, atol=2 ** -8)
    xt = x.cuda().t().contiguous().t().requires_grad_()
    g = torch.autograd.grad(layer_norm(xt, w.cuda()), xt, dy.cuda().t().contiguous().t())[0]
    xc = x.cuda().requires_grad_()
    assert torch.equal(g, torch.autograd.grad(layer_norm(xc, w.cuda()), xc, dy.cuda())[0])


@pytest.mark.gpu
def test_only_some_gradients():
    x, w, b, dy = _inputs((50, 301), F32, F32, F32)
    all3 = [t.cuda().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*all3), all3, dy.cuda())
    for i in range(3):
        t = [v.cuda().requires_grad_(k == i) for k, v in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(layer_norm(*t), t[i], dy.cuda())[0], want[i])


@pytest.mark.gpu
def test_device_refusals():
    x = torch.zeros(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="FP32, BF16 and FP16"):
        layer_norm(x.double())
    with pytest.raises(RuntimeError, match="one device"):
        layer_norm(x, torch.ones(8))
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError):
        layer_norm(fwAD.make_dual(x, torch.ones_like(x)))


@pytest.mark.gpu
def test_other_stream_and_graph():
    x, w, b, dy = [t.cuda() for t in _inputs((70, 256), BF16, BF16, BF16)]
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        for u, v in zip(out, eager):
            assert torch.equal(u, v)
        del eager
