"""grouped_linear against products in float64, forward and gradients.

Bounds: a sum of L products in float32 is off by at most L + 16 roundings of
2^-24 of the sum of magnitudes (16: what a matrix instruction truncates inside),
plus one rounding to the result's type."""

import ctypes

import pytest
import torch

from _saved import check_kept_is_saved
from torchsplinekan_amd import grouped_linear, quantize_activation

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_ULP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
DTYPES = [F32, BF16, F16]


def _offsets(counts, dtype=torch.int32):
    return torch.tensor([0] + list(counts)).cumsum(0).to(dtype)


def _counts(T, E, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.softmax(torch.randn(E, generator=g) * 1.5, 0)
    return torch.bincount(torch.multinomial(p, T, replacement=True, generator=g),
                          minlength=E).tolist()


def _bound(got, want, mag, terms, what):
    got = got.detach().cpu()
    assert got.shape == want.shape, what
    fp32 = (terms + 16) * 2.0 ** -24 * mag
    tol = fp32 + HALF_ULP[got.dtype] * (want.abs() + fp32)
    if got.dtype == F16:
        tol = tol + 2.0 ** -25
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound"


def _inputs(T, E, K, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g).to(dtype)
    w = (torch.randn(E, N, K, generator=g) * max(K, 1) ** -0.5).to(dtype)
    dy = torch.randn(T, N, generator=g).to(dtype)
    return x, w, dy


def _check(x, w, dy, offsets, ends=None, checkpoint=None, group=128):
    """ends: where the groups end, when the offsets themselves do not say."""
    T, K = x.shape
    E, N, _ = w.shape
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = grouped_linear(xd, wd, offsets.cuda(), checkpoint=checkpoint, group=group)
    assert y.dtype == x.dtype
    dx, dw = torch.autograd.grad(y, [xd, wd], dy.cuda())
    with torch.no_grad():
        assert torch.equal(grouped_linear(xd, wd, offsets.cuda()), y)
    kept = x if checkpoint is None else quantize_activation(x, group, checkpoint).dequantize(F32)
    ends = offsets.tolist()[1:] if ends is None else ends
    X, W, D, Q = x.double(), w.double(), dy.double(), kept.double()
    # (a value q * scale takes part in the 16-bit products rounded to their type)
    extra = 0.0 if checkpoint is None or x.dtype == F32 else HALF_ULP[x.dtype]
    lo = 0
    for e in range(E):
        hi = max(lo, ends[e])
        r = slice(lo, hi)
        _bound(y[r], X[r] @ W[e].t(), X[r].abs() @ W[e].abs().t(), K, f"y of {e}")
        _bound(dx[r], D[r] @ W[e], D[r].abs() @ W[e].abs(), N, f"dx of {e}")
        mag = D[r].abs().t() @ Q[r].abs()
        _bound(dw[e], D[r].t() @ Q[r], mag * (1 + extra * 2.0 ** 24 / (hi - lo + 16)), hi - lo,
               f"dw of {e}")
        lo = hi
    assert not bool(y[lo:].any()) and not bool(dx[lo:].any())


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------

def test_cpu_path_against_differences():
    x, w, dy = _inputs(9, 3, 4, 5, torch.float64)
    off = _offsets([4, 0, 3])
    x.requires_grad_(), w.requires_grad_()
    torch.autograd.gradcheck(lambda a, b: grouped_linear(a, b, off), (x, w))
    y = grouped_linear(x, w, off)
    torch.testing.assert_close(y[:4], x[:4] @ w[0].t())
    assert not bool(y[7:].any())


def test_cpu_checkpoint():
    x, w, dy = _inputs(9, 2, 40, 5, F32)
    off = _offsets([4, 5])
    x.requires_grad_(), w.requires_grad_()
    y = grouped_linear(x, w, off, checkpoint="int8", group=32)
    assert torch.equal(y, grouped_linear(x, w, off))
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    kept = quantize_activation(x[:4], 32).dequantize()
    torch.testing.assert_close(dw[0], dy[:4].t() @ kept)
    torch.testing.assert_close(dx[4:], dy[4:] @ w[1])


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_cpu_sums_under_autocast(checkpoint):
    """Products in float32, as on the device."""
    x, w, _ = _inputs(9, 2, 40, 5, F32)
    off = _offsets([4, 5])
    want = grouped_linear(x, w, off, checkpoint=checkpoint)
    with torch.autocast("cpu", dtype=BF16):
        got = grouped_linear(x, w, off, checkpoint=checkpoint)
    assert got.dtype == F32 and torch.equal(got, want)


def _check_saved(format, dev):
    x, w, dy = (t.to(dev) for t in _inputs(9, 2, 40, 5, F32))
    off = _offsets([4, 5]).to(dev)
    x.requires_grad_(), w.requires_grad_()
    check_kept_is_saved(lambda: grouped_linear(x, w, off, checkpoint=format), [x, w], dy,
                        in_place=[w] if dev == "cpu" else [w, off])


@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_cpu_kept_rows_are_saved_tensors(format):
    _check_saved(format, "cpu")


@pytest.mark.parametrize("x,w,off,kw,text", [
    (torch.zeros(4), torch.zeros(2, 3, 4), torch.zeros(3, dtype=torch.int32), {}, "must be"),
    (torch.zeros(4, 5), torch.zeros(2, 3, 4), torch.zeros(3, dtype=torch.int32), {}, "equal K"),
    (torch.zeros(4, 4), torch.zeros(2, 3, 4).bfloat16(), torch.zeros(3, dtype=torch.int32), {},
     "share a dtype"),
    (torch.zeros(4, 4), torch.zeros(2, 3, 4), torch.zeros(2, dtype=torch.int32), {}, "offsets must"),
    (torch.zeros(4, 4), torch.zeros(2, 3, 4), torch.zeros(3), {}, "int32 or int64"),
    (torch.zeros(4, 4), torch.zeros(2, 3, 4), torch.zeros(3, dtype=torch.int32),
     dict(checkpoint="int4"), "format must"),
    (torch.zeros(4, 4), torch.zeros(2, 3, 4), torch.zeros(3, dtype=torch.int32),
     dict(checkpoint="int8", group=100), "group must"),
])
def test_refusals(x, w, off, kw, text):
    with pytest.raises(RuntimeError, match=text):
        grouped_linear(x, w, off, **kw)


def test_c_entry_refusals():
    lib = pytest.importorskip("torchsplinekan_amd._lib")
    f = lib.LIB.kan_hip_grouped_matmul
    p = 4096
    tail = (8, 2, 16, 16, p, None, 0, None)
    assert f(1, 0, p, p, 0, None, 0, p, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(2, 3, p, p, 0, None, 0, p, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(2, 0, p, p, 1, p, 128, p, 0, *tail) == lib.KAN_ERR_INVALID
    assert "weight product only" in lib.last_error()
    assert f(2, 2, p, p, 5, p, 128, p, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(2, 2, p, p, 1, p, 100, p, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(2, 2, p, p, 1, None, 128, p, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(2, 0, None, p, 0, None, 0, p, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(2, 0, p, p, 0, None, 0, None, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(2, 0, p, p, 0, None, 0, p, 0, -1, 2, 16, 16, p, None, 0, None) == lib.KAN_ERR_INVALID
    assert f(2, 0, p, p, 0, None, 0, p, 0, 8, 1 << 16, 16, 16, p, None, 0,
             None) == lib.KAN_ERR_LIMIT
    assert f(2, 0, None, None, 0, None, 0, None, 0, 0, 2, 16, 16, None, None, 0,
             None) == lib.KAN_OK


def test_workspace_of_sizes_whose_product_passes_64_bits():
    """Restored rows are counted also where T E N K is a multiple of 2^64."""
    lib = pytest.importorskip("torchsplinekan_amd._lib")
    nbytes = ctypes.c_size_t()
    T, E, N, K = 1 << 29, 1 << 13, 1 << 11, 1 << 11
    lib.check(lib.LIB.kan_hip_grouped_matmul_workspace(0, 2, None, None, 1, T, E, N, K,
                                                       ctypes.byref(nbytes)))
    assert nbytes.value >= 4 * T * K


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(1, 1), (1, 70), (33, 1), (8, 8), (16, 48), (64, 64), (100, 60),
                                 (301, 257), (136, 520), (128, 1032)])
@pytest.mark.parametrize("counts", [[1], [5, 0, 1, 40], [0, 0, 70, 0], [64, 128, 130], [300, 3]])
def test_sizes(counts, K, N, dtype):
    x, w, dy = _inputs(sum(counts), len(counts), K, N, dtype)
    _check(x, w, dy, _offsets(counts))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E", [1, 2, 16, 63, 64, 65, 130])
@pytest.mark.parametrize("T", [1, 7, 200, 1500])
def test_experts(T, E, dtype):
    """Numbers of experts on either side of a wave's 64 lanes, most of them
    without rows where T is small."""
    x, w, dy = _inputs(T, E, 40, 72, dtype, seed=E)
    _check(x, w, dy, _offsets(_counts(T, E, seed=T + E), torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,K,N", [(3000, 5, 512, 320), (2500, 3, 257, 1000),
                                     (700, 2, 2048, 96), (5000, 4, 96, 2000)])
def test_larger(T, E, K, N, dtype):
    x, w, dy = _inputs(T, E, K, N, dtype)
    _check(x, w, dy, _offsets(_counts(T, E, seed=1)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,K,N", [(40, 5, 4096, 72), (40, 5, 72, 4096), (300, 2, 2051, 130),
                                     (1, 1, 8000, 8), (130, 3, 9, 3001)])
def test_few_tiles_with_long_sums(T, E, K, N, dtype):
    """Outputs of few tiles: their sums are cut into several."""
    x, w, dy = _inputs(T, E, K, N, dtype)
    _check(x, w, dy, _offsets(_counts(T, E, seed=2)))
    off = [0] + [T // 2] * E                      # rows past the last group
    _check(x, w, dy, torch.tensor(off, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,E,K,N", [(12000, 2, 2047, 1027), (9000, 3, 1536, 2045),
                                     (20001, 2, 1283, 1024)])
def test_large_products_of_rows_off_16_bytes(T, E, K, N, dtype):
    """Products that are long enough to bring their rows onto 16 bytes first."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(E, N, K, generator=g, device="cuda") * K ** -0.5).to(dtype).requires_grad_()
    dy = torch.randn(T, N, generator=g, device="cuda").to(dtype)
    counts = _counts(T, E, seed=3)
    off = _offsets(counts).cuda()
    y = grouped_linear(x, w, off)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    lo = 0
    for e, c in enumerate(counts):
        r = slice(lo, lo + c)
        X, W, D = x[r].detach().double(), w[e].detach().double(), dy[r].double()
        for got, a, b, terms in ((y[r], X, W.t(), K), (dx[r], D, W, N), (dw[e], D.t(), X, c)):
            want, mag = torch.mm(a, b), torch.mm(a.abs(), b.abs())
            tol = (terms + 16) * 2.0 ** -24 * mag * (1 + HALF_ULP[dtype])
            tol = tol + HALF_ULP[dtype] * want.abs() + 2.0 ** -25
            assert bool(((got.double() - want).abs() <= tol).all())
        lo += c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("K,N,group", [(1, 3, 32), (100, 60, 64), (136, 128, 32), (301, 257, 128),
                                       (512, 320, 256), (129, 72, 128)])
def test_kept_rows(K, N, group, format, dtype):
    counts = [37, 0, 200, 1, 64]
    x, w, dy = _inputs(sum(counts), len(counts), K, N, dtype)
    _check(x, w, dy, _offsets(counts), checkpoint=format, group=group)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("T,E,K,N", [(12000, 2, 1032, 4104), (9000, 3, 1024, 5001),
                                     (20001, 2, 1283, 520)])
def test_kept_rows_of_long_products(T, E, K, N, format, dtype):
    """Products that are long enough to restore their 8-bit rows in a pass of
    their own, and ones that bring odd rows onto whole chunks."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    w = torch.zeros(E, N, K, dtype=dtype, device="cuda").requires_grad_()
    dy = torch.randn(T, N, generator=g, device="cuda").to(dtype)
    counts = _counts(T, E, seed=3)
    y = grouped_linear(x, w, _offsets(counts).cuda(), checkpoint=format)
    dw, = torch.autograd.grad(y, w, dy)
    kept = quantize_activation(x, 128, format).dequantize(F32).double()
    lo = 0
    for e, c in enumerate(counts):
        X, D = kept[lo:lo + c], dy[lo:lo + c].double()
        want, mag = torch.mm(D.t(), X), torch.mm(D.abs().t(), X.abs())
        tol = (c + 16) * 2.0 ** -24 * mag + HALF_ULP[dtype] * (want.abs() + mag) + 2.0 ** -25
        assert bool(((dw[e].double() - want).abs() <= tol).all())
        # (a value's rounding to 16 bits is independent of the next one's)
        assert float((dw[e].double() - want).norm() / want.norm()) < 2 * HALF_ULP[dtype]
        lo += c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("K,N", [(96, 72), (77, 65)])
def test_kept_rows_one_to_an_expert(K, N, format, dtype):
    """Nothing is added up: a product of the restored value in x's type (exact in
    float32), rounded once."""
    E = 20
    x, w, dy = _inputs(E, E, K, N, dtype)
    wd = w.cuda().requires_grad_()
    y = grouped_linear(x.cuda(), wd, _offsets([1] * E).cuda(), checkpoint=format, group=32)
    dw, = torch.autograd.grad(y, wd, dy.cuda())
    kept = quantize_activation(x, 32, format).dequantize()
    assert torch.equal(dw.cpu(), (dy.float().unsqueeze(2) * kept.float().unsqueeze(1)).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("T,E,K,N", [(200, 3, 96, 72), (200, 3, 77, 65), (12000, 2, 1032, 4104)])
def test_kept_rows_at_the_end_of_the_range(T, E, K, N, format):
    """Groups that hold bfloat16's largest values, whose scale times 128 is above
    float32's: restored on their way into the tiles, and in a pass of their own.
    (Bounds of test_kept_rows_of_long_products; dy's are 2^-110 of unit size.)"""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, K, generator=g, device="cuda").to(BF16)
    top = torch.finfo(BF16).max
    x[3, 0], x[3, 1], x[T - 2, K - 1] = top, -top, -top
    w = torch.zeros(E, N, K, dtype=BF16, device="cuda").requires_grad_()
    dy = (torch.randn(T, N, generator=g, device="cuda") * 2.0 ** -110).to(BF16)
    counts = _counts(T, E, seed=3)
    y = grouped_linear(x, w, _offsets(counts).cuda(), checkpoint=format, group=32)
    dw, = torch.autograd.grad(y, w, dy)
    kept = quantize_activation(x, 32, format).dequantize(F32).double()
    lo = 0
    for e, c in enumerate(counts):
        X, D = kept[lo:lo + c], dy[lo:lo + c].double()
        want, mag = torch.mm(D.t(), X), torch.mm(D.abs().t(), X.abs())
        tol = (c + 16) * 2.0 ** -24 * mag + HALF_ULP[BF16] * (want.abs() + mag)
        assert bool(((dw[e].double() - want).abs() <= tol).all())
        lo += c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offsets,ends", [
    ([0, 10, 30, 30], [10, 30, 30]),          # rows past the last group
    ([0, 0, 0, 0], [0, 0, 0]),                # no group has any
    ([0, 40, 20, 70], [40, 40, 70]),          # descending: the running maximum
    ([0, -5, 200, 90], [0, 90, 90]),          # outside 0 .. T
])
def test_offsets(offsets, ends, dtype):
    x, w, dy = _inputs(90, 3, 72, 80, dtype)
    for t in (torch.int32, torch.int64):
        _check(x, w, dy, torch.tensor(offsets, dtype=t), ends=ends)


@pytest.mark.gpu
def test_empty():
    off = _offsets([0, 0]).cuda()
    for T, K, N, E in [(0, 8, 8, 2), (5, 0, 8, 2), (5, 8, 0, 2)]:
        x = torch.randn(T, K, device="cuda", requires_grad=True)
        w = torch.randn(E, N, K, device="cuda", requires_grad=True)
        y = grouped_linear(x, w, off)
        assert y.shape == (T, N) and not bool(y.any())
        dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
        assert not bool(dx.any()) and not bool(dw.any())
    y = grouped_linear(torch.randn(5, 8, device="cuda"), torch.randn(0, 3, 8, device="cuda"),
                       _offsets([]).cuda())
    assert y.shape == (5, 3) and not bool(y.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Views: rows that start off 16 bytes, transposed weights, transposed
    gradients, and another stream."""
    x, w, dy = _inputs(150, 3, 64, 72, dtype)
    off = _offsets([50, 20, 80]).cuda()
    want = grouped_linear(x.cuda(), w.cuda(), off)
    big = torch.zeros(150 * 64 + 1, dtype=dtype, device="cuda")
    big[1:] = x.cuda().reshape(-1)
    xv = big[1:].view(150, 64)
    wv = w.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grouped_linear(xv, wv, off)
    torch.cuda.current_stream().wait_stream(side)
    tol = 80 * 2.0 ** -24 + 2 * HALF_ULP[dtype]
    mag = x.double().abs() @ w.double().abs().amax(0).t()
    assert bool(((got.double() - want.double()).abs().cpu() <= tol * mag).all())
    xg, wg = xv.detach().requires_grad_(), w.cuda().requires_grad_()
    dyt = dy.cuda().t().contiguous().t()
    dx, dw = torch.autograd.grad(grouped_linear(xg, wg, off), [xg, wg], dyt)
    lo = 0
    for e, c in enumerate([50, 20, 80]):
        r = slice(lo, lo + c)
        D, X = dy[r].double(), x[r].double()
        _bound(dx[r], D @ w[e].double(), D.abs() @ w[e].double().abs(), 72, "dx")
        _bound(dw[e], D.t() @ X, D.abs().t() @ X.abs(), c, "dw")
        lo += c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(64, 64), (77, 65)])
def test_values_that_are_not_finite(K, N, dtype):
    """A row's infinity or NaN reaches that row's outputs and its expert's
    weight gradient, nothing else."""
    counts = [30, 40, 50]
    x, w, dy = _inputs(120, 3, K, N, dtype)
    x[29, 3] = float("nan")           # the last row of expert 0
    x[30, 5] = float("inf")           # the first of expert 1
    w[1, :, 5] = w[1, :, 5].abs() + 1
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = grouped_linear(xd, wd, _offsets(counts).cuda())
    dx, dw = torch.autograd.grad(y, [xd, wd], dy.cuda())
    bad = ~y.isfinite().all(1).cpu()
    assert bad.nonzero().flatten().tolist() == [29, 30]
    assert bool(y[29].isnan().all()) and bool((y[30] == float("inf")).all())
    assert bool(dx.isfinite().all())
    finite = dw.isfinite().cpu()
    assert bool(finite[2].all())
    assert bool(dw[0, :, 3].isnan().all()) and bool(finite[0, :, 4:].all())
    assert not bool(finite[1, :, 5].any()) and bool(finite[1, :, 6:].all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [40, 4000])
def test_weights_past_32_bit_offsets(dtype, rows):
    """2.3e9 weight values; the last expert has the rows."""
    E, N, K = 70, 4096, 8064
    w = torch.zeros(E, N, K, dtype=dtype, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    w[-1] = (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).to(dtype)
    x = torch.randn(rows, K, generator=g, device="cuda").to(dtype)
    dy = torch.randn(rows, N, generator=g, device="cuda").to(dtype)
    off = _offsets([0] * (E - 1) + [rows]).cuda()
    y = grouped_linear(x, w, off)
    want = torch.mm(x.double(), w[-1].double().t())
    assert float((y.double() - want).norm() / want.norm()) < 2 * HALF_ULP[dtype] + 1e-6
    xg = x.clone().requires_grad_()
    dx, = torch.autograd.grad(grouped_linear(xg, w, off), xg, dy)
    want = torch.mm(dy.double(), w[-1].double())
    assert float((dx.double() - want).norm() / want.norm()) < 2 * HALF_ULP[dtype] + 1e-6
    del w
    wg = torch.empty(E, N, K, dtype=dtype, device="cuda").requires_grad_()
    dw, = torch.autograd.grad(grouped_linear(x, wg, off), wg, dy)
    want = torch.mm(dy.double().t(), x.double())
    assert float((dw[-1].double() - want).norm() / want.norm()) < 2 * HALF_ULP[dtype] + 1e-6
    assert not bool(dw[:-1].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_past_32_bit_offsets(dtype):
    """Outputs and inputs of more than 2^31 values; the last rows are compared."""
    T, E, K, N = 1100000, 2, 2048, 72
    x = torch.zeros(T, K, dtype=dtype, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    x[-500:] = torch.randn(500, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(E, N, K, generator=g, device="cuda") * K ** -0.5).to(dtype)
    off = _offsets([T - 400, 400]).cuda()
    y = grouped_linear(x, w, off)
    want = torch.cat([torch.mm(x[-500:-400].double(), w[0].double().t()),
                      torch.mm(x[-400:].double(), w[1].double().t())])
    assert float((y[-500:].double() - want).norm() / want.norm()) < 2 * HALF_ULP[dtype] + 1e-6
    assert not bool(y[:-500].any())
    wt = w.transpose(1, 2).contiguous().requires_grad_()       # [E, 2048, 72]
    z = torch.zeros(T, N, dtype=dtype, device="cuda")
    z[-500:] = y[-500:]
    out = grouped_linear(z, wt, off)                           # [T, 2048]
    want = torch.mm(z[-400:].double(), wt[1].detach().double().t())
    assert float((out[-400:].detach().double() - want).norm() / want.norm()) \
        < 2 * HALF_ULP[dtype] + 1e-6
    dw, = torch.autograd.grad(out, wt, x)
    want = torch.mm(x[-400:].double().t(), z[-400:].double())
    assert float((dw[1].double() - want).norm() / want.norm()) < 2 * HALF_ULP[dtype] + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_every_time(dtype):
    x, w, dy = _inputs(2000, 9, 200, 264, dtype)
    off = _offsets(_counts(2000, 9, 4)).cuda()
    runs = []
    for _ in range(2):
        xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        y = grouped_linear(xd, wd, off, checkpoint="int8")
        runs.append([y, *torch.autograd.grad(y, [xd, wd], dy.cuda())])
    for u, v in zip(*runs):
        assert torch.equal(u, v)


@pytest.mark.gpu
@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_kept_rows_are_saved_tensors(format):
    _check_saved(format, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("leaf", [0, 1])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_forward_mode_is_refused(leaf, checkpoint):
    from torch.autograd import forward_ad
    x, w, _ = _inputs(9, 2, 32, 5, F32)
    args, off = [x.cuda(), w.cuda()], _offsets([4, 5]).cuda()
    want = grouped_linear(*args, off)
    with forward_ad.dual_level():
        got = grouped_linear(*args, off, checkpoint=checkpoint)
        assert torch.equal(got, want) and not got.requires_grad
        args[leaf] = forward_ad.make_dual(args[leaf], torch.ones_like(args[leaf]))
        with pytest.raises(RuntimeError, match="jvp"):
            grouped_linear(*args, off, checkpoint=checkpoint)


@pytest.mark.gpu
def test_float64_and_other_devices_are_refused():
    x = torch.zeros(2, 4, dtype=torch.float64, device="cuda")
    off = _offsets([2]).cuda()
    with pytest.raises(RuntimeError, match="FP32, BF16 and FP16"):
        grouped_linear(x, torch.zeros(1, 3, 4, dtype=torch.float64, device="cuda"), off)
    with pytest.raises(RuntimeError, match="one device"):
        grouped_linear(x.float(), torch.zeros(1, 3, 4), off)
