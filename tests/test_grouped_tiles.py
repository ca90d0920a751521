"""grouped_linear on every kind of tile: each case pins the plan that it is there
for (rows of a tile, cuts, rows of an item, restored in a pass, operands brought
onto 16 bytes, operands straight into LDS), and its product is held to the bounds
of test_grouped.py element by element, in float64 on the device."""

import ctypes

import pytest
import torch

from test_grouped import BF16, F16, F32, HALF_ULP, _counts, _offsets
from torchsplinekan_amd import quantize_activation
from torchsplinekan_amd.grouped import _matmul

FORWARD, INPUT, WEIGHT = 0, 1, 2
FORMS = {None: 0, "int8": 1, "e4m3": 2}

# (product, 8-bit rows, T, E, N, K, plan)
HALF = [
    (FORWARD, 0, 957, 64, 1680, 34, (192, 1, 0, 0, 0, 0)),
    (FORWARD, 0, 736, 48, 2184, 32, (192, 1, 0, 0, 0, 3)),
    (FORWARD, 0, 5866, 2, 1547, 806, (192, 1, 0, 0, 3, 3)),
    (FORWARD, 0, 386, 48, 2440, 36, (256, 1, 0, 0, 0, 0)),
    (FORWARD, 0, 1755, 70, 1384, 32, (256, 1, 0, 0, 0, 3)),
    (FORWARD, 0, 6603, 2, 1840, 531, (256, 1, 0, 0, 3, 3)),
    (FORWARD, 0, 5321, 2, 1451, 1007, (128, 1, 0, 0, 3, 3)),
    (FORWARD, 0, 82, 2, 32, 1225, (128, 5, 0, 0, 0, 0)),
    (FORWARD, 0, 66, 2, 32, 1304, (128, 5, 0, 0, 0, 3)),
    (INPUT, 0, 848, 2, 1252, 1520, (128, 5, 0, 0, 1, 3)),
    (INPUT, 0, 3963, 2, 1192, 335, (128, 4, 0, 0, 2, 3)),
    (INPUT, 0, 75, 2, 1260, 32, (128, 5, 0, 0, 0, 0)),
    (INPUT, 0, 337, 70, 32, 1694, (192, 1, 0, 0, 0, 0)),
    (INPUT, 0, 381, 100, 32, 1168, (192, 1, 0, 0, 0, 3)),
    (INPUT, 0, 3918, 2, 191, 2080, (192, 1, 0, 0, 1, 3)),
    (INPUT, 0, 8273, 2, 216, 907, (192, 1, 0, 0, 2, 3)),
    (INPUT, 0, 1192, 64, 32, 1703, (256, 1, 0, 0, 0, 0)),
    (INPUT, 0, 13676, 130, 32, 264, (256, 1, 0, 0, 0, 3)),
    (INPUT, 0, 9007, 2, 365, 1321, (256, 1, 0, 0, 3, 3)),
    (WEIGHT, 0, 765, 3, 36, 33, (128, 1, 256, 0, 0, 0)),
    (WEIGHT, 0, 1838, 2, 467, 1264, (128, 1, 512, 0, 1, 3)),
    (WEIGHT, 0, 1341, 2, 1349, 1343, (128, 1, 0, 0, 3, 3)),
    (WEIGHT, 0, 71, 130, 32, 265, (256, 1, 0, 0, 0, 0)),
    (WEIGHT, 0, 159, 130, 264, 32, (256, 1, 0, 0, 0, 3)),
    (WEIGHT, 0, 4026, 32, 279, 976, (256, 1, 0, 0, 1, 3)),
    (WEIGHT, 0, 2624, 24, 1312, 297, (256, 1, 0, 0, 2, 3)),
    (WEIGHT, 0, 18931, 32, 33, 1849, (256, 1, 1024, 0, 0, 0)),
    (WEIGHT, 0, 21317, 32, 40, 2104, (256, 1, 1024, 0, 0, 3)),
    (WEIGHT, 1, 765, 3, 36, 33, (128, 1, 256, 0, 0, 0)),
    (WEIGHT, 1, 875, 2, 32, 40, (128, 1, 256, 0, 0, 1)),
    (WEIGHT, 1, 727, 2, 738, 1840, (128, 1, 0, 0, 1, 1)),
    (WEIGHT, 1, 1908, 2, 808, 674, (128, 1, 512, 0, 2, 1)),
    (WEIGHT, 1, 281, 130, 260, 32, (256, 1, 0, 0, 0, 0)),
    (WEIGHT, 1, 71, 130, 32, 265, (256, 1, 0, 0, 0, 1)),
    (WEIGHT, 1, 4026, 32, 279, 976, (256, 1, 0, 0, 1, 1)),
    (WEIGHT, 1, 2624, 24, 1312, 297, (256, 1, 0, 0, 2, 1)),
    (WEIGHT, 1, 1360, 8, 837, 2070, (256, 1, 0, 0, 3, 1)),
    (WEIGHT, 1, 8192, 16, 1024, 1001, (256, 1, 0, 0, 2, 1)),
    (WEIGHT, 1, 18931, 32, 33, 1849, (256, 1, 1024, 0, 0, 0)),
    (WEIGHT, 1, 21520, 32, 48, 1803, (256, 1, 1024, 0, 0, 1)),
    (WEIGHT, 1, 12907, 5, 2456, 1568, (256, 1, 0, 1, 0, 3)),
    (WEIGHT, 1, 10154, 5, 2503, 2008, (256, 1, 0, 1, 1, 3)),
]
FLOAT = [
    (FORWARD, 0, 66, 2, 40, 459, (128, 2, 0, 0, 0, 0)),
    (INPUT, 0, 69, 2, 464, 37, (128, 2, 0, 0, 0, 0)),
    (WEIGHT, 0, 363, 2, 34, 32, (128, 1, 256, 0, 0, 0)),
    (WEIGHT, 0, 16519, 16, 888, 2152, (256, 1, 0, 0, 0, 0)),
    (WEIGHT, 0, 20000, 16, 1030, 1000, (256, 1, 1024, 0, 0, 0)),
    (WEIGHT, 0, 17420, 16, 561, 1285, (256, 1, 1024, 0, 0, 0)),
    (WEIGHT, 1, 363, 2, 34, 32, (128, 1, 256, 1, 0, 0)),
    (WEIGHT, 1, 17420, 16, 561, 1285, (256, 1, 1024, 1, 0, 0)),
]
CASES = [(code, *c) for code, cases in ((2, HALF), (3, HALF), (0, FLOAT)) for c in cases]


@pytest.mark.parametrize("code,op,kept,T,E,N,K,plan", CASES)
def test_plans(code, op, kept, T, E, N, K, plan):
    lib = pytest.importorskip("torchsplinekan_amd._lib")
    got = (ctypes.c_int64 * 6)()
    lib.check(lib.LIB.kan_hip_grouped_matmul_plan(code, op, None, None, kept, T, E, N, K, got))
    assert tuple(got) == plan
    lib.check(lib.LIB.kan_hip_grouped_matmul_plan(code, op, None, None, 2 * kept, T, E, N, K, got))
    assert tuple(got) == plan


def test_plan_refusals():
    lib = pytest.importorskip("torchsplinekan_amd._lib")
    f, got = lib.LIB.kan_hip_grouped_matmul_plan, (ctypes.c_int64 * 6)()
    assert f(0, 0, None, None, 0, 8, 2, 16, 16, None) == lib.KAN_ERR_INVALID
    assert f(1, 0, None, None, 0, 8, 2, 16, 16, got) == lib.KAN_ERR_INVALID
    assert f(0, 0, None, None, 0, 8, 1 << 16, 16, 16, got) == lib.KAN_ERR_LIMIT


def _uneven(T, E, seed):
    """Counts of a skewed router, with an expert that has none and rows left over."""
    counts = _counts(T - 5, E, seed)
    if E > 2:
        counts[0] += counts[1]
        counts[1] = 0
    return counts


def _run(code, op, form, T, E, N, K):
    dtype = {0: F32, 2: BF16, 3: F16}[code]
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(E, N, K, generator=g, device="cuda") * K ** -0.5).to(dtype)
    dy = torch.randn(T, N, generator=g, device="cuda").to(dtype)
    counts = _uneven(T, E, seed=T)
    off = _offsets(counts).cuda()
    kept = None if form is None else quantize_activation(x, 64, form)
    a, b = {FORWARD: (x, w), INPUT: (dy, w), WEIGHT: (dy, kept or x)}[op]
    shape = {FORWARD: (T, N), INPUT: (T, K), WEIGHT: (E, N, K)}[op]
    out = _matmul(op, a, b, off, torch.full(shape, float("nan"), dtype=dtype, device="cuda"),
                  T, E, N, K)
    # (restored values take part as dequantize gives them, in x's type)
    X = (x if kept is None else kept.dequantize()).double()
    W, D, lo = w.double(), dy.double(), 0
    for e, c in enumerate(counts):
        r = slice(lo, lo + c)
        got, u, v, terms = {FORWARD: (out[r], X[r], W[e].t(), K), INPUT: (out[r], D[r], W[e], N),
                            WEIGHT: (out[e], D[r].t(), X[r], c)}[op]
        want, mag = torch.mm(u, v), torch.mm(u.abs(), v.abs())
        fp32 = (terms + 16) * 2.0 ** -24 * mag
        tol = fp32 + HALF_ULP[dtype] * (want.abs() + fp32) + (2.0 ** -25 if dtype == F16 else 0.0)
        assert bool(((got.double() - want).abs() <= tol).all()), f"expert {e} of {c} rows"
        lo += c
    if op != WEIGHT:
        assert lo == T - 5 and not bool(out[lo:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("code,op,kept,T,E,N,K,plan", CASES)
def test_products(code, op, kept, T, E, N, K, plan):
    for form in ("int8", "e4m3") if kept else (None,):
        _run(code, op, form, T, E, N, K)


@pytest.mark.gpu
@pytest.mark.parametrize("code", [0, 2])
@pytest.mark.parametrize("op", [FORWARD, INPUT, WEIGHT])
def test_as_many_experts_as_there_may_be(op, code):
    """65535 experts, most of them without rows."""
    T, E, N, K = 300, 65535, 8, 12
    dtype = {0: F32, 2: BF16}[code]
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    dy = torch.randn(T, N, generator=g, device="cuda").to(dtype)
    w = torch.randn(E, N, K, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, E, (T,), generator=g, device="cuda").sort().values
    off = torch.searchsorted(ids, torch.arange(E + 1, device="cuda"))
    shape = {FORWARD: (T, N), INPUT: (T, K), WEIGHT: (E, N, K)}[op]
    out = _matmul(op, x if op == FORWARD else dy, x if op == WEIGHT else w, off,
                  torch.empty(shape, dtype=dtype, device="cuda"), T, E, N, K)
    X, D, W = x.double(), dy.double(), w[ids].double()
    if op == WEIGHT:
        want = torch.zeros(E, N, K, dtype=torch.float64, device="cuda")
        want.index_add_(0, ids, D.unsqueeze(2) * X.unsqueeze(1))
    else:
        want = (W * (X.unsqueeze(1) if op == FORWARD else D.unsqueeze(2))).sum(
            2 if op == FORWARD else 1)
    # (12 products at most, of values up to 5 each)
    tol = (12 + 16) * 2.0 ** -24 * 12 * 25 + HALF_ULP[dtype] * want.abs()
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("op,N,K", [(FORWARD, 2, 1 << 22), (INPUT, 1 << 22, 2)])
def test_float32_rows_past_a_buffer_resource(op, N, K):
    """Rows whose tile spans more than 2^31 bytes take 64-bit addresses.  (A sum of
    2^22 terms: chains of 2^13 slabs at most, each rounding 2^-24 of a running sum
    that grows with the root of its length, so 2^-24 2^6.5 of its end; 2^-16 of the
    norm is ten times that.)"""
    T, E = 40, 1
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, K, generator=g, device="cuda")
    w = torch.randn(E, N, K, generator=g, device="cuda")
    dy = torch.randn(T, N, generator=g, device="cuda")
    a = x if op == FORWARD else dy
    out = torch.empty(T, N if op == FORWARD else K, device="cuda")
    _matmul(op, a, w, _offsets([T - 1]).cuda(), out, T, E, N, K)
    b = w[0].double()
    want = torch.mm(a[:-1].double(), b.t() if op == FORWARD else b)
    assert float((out[:-1].double() - want).norm() / want.norm()) < 2.0 ** -16
    assert not bool(out[-1].any())
