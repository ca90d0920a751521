"""residual_norm against its formulas in float64, forward and gradients.

Bounds: every result is a chain of float32 operations on its terms' magnitudes,
so its error stays within (chain length) 2^-24 of the same formula evaluated on
magnitudes (`_formulas(..., magnitude=True)`), plus one rounding to the result's
type.  A chain is at most C / 64 terms in a lane, n / 64 rows in a block's
partial sum, and 64 for the trees, the elementary functions (expf, tanhf: a few
roundings) and the remaining products."""

import pytest
import torch

from torchsplinekan_amd import residual_norm

EPS = 1e-6
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAMES = ("x", "y", "gate", "post", "pre", "scale")


def _act(g, act):
    s = torch.sigmoid(g)
    t = torch.tanh(g)
    return {None: (g, torch.ones_like(g)), "sigmoid": (s, s * (1 - s)), "tanh": (t, 1 - t * t),
            "silu": (g * s, s * (1 + g * (1 - s)))}[act]


def _sum_to(v, shape):
    lead = v.dim() - len(shape)
    v = v.sum(tuple(range(lead))) if lead else v
    dims = tuple(i for i, s in enumerate(shape) if s == 1 and v.shape[i] != 1)
    return v.sum(dims, keepdim=True) if dims else v


def _formulas(t, act, scale, dnew, dh, magnitude=False):
    """Results in float64 from the closed formulas; magnitude: the same with
    every term's magnitude."""
    f = (lambda v: v.abs()) if magnitude else (lambda v: v)
    sub = (lambda a, b: a + b) if magnitude else (lambda a, b: a - b)
    d = {k: None if v is None else v.detach().cpu().double() for k, v in t.items()}
    x, y, post, pre = d["x"], d["y"], d["post"], d["pre"]
    sc = d["scale"] if d["scale"] is not None else torch.tensor(
        1.0 if scale is None else float(scale), dtype=torch.float64)
    r = {}
    true_new = new = f(x)
    if y is not None:
        r1 = (y.square().mean(-1, keepdim=True) + EPS).rsqrt() if post is not None else 1.0
        yh = y * r1
        u = yh * post if post is not None else y
        a, slope = (_act(d["gate"], act) if d["gate"] is not None
                    else (torch.ones((), dtype=torch.float64), None))
        true_new = x + sc * a * u
        new = f(x) + f(sc * a * u)
    r["new"] = new
    r2 = (true_new.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = new * r2
    if pre is not None:
        r["h"] = xh * f(pre)
    if dnew is None and dh is None:
        return r
    total = torch.zeros_like(x) if dnew is None else f(dnew.cpu().double())
    if dh is not None:
        g = f(dh.cpu().double())
        tt = g * f(pre)
        total = total + r2 * sub(tt, xh * (tt * xh).mean(-1, keepdim=True))
        r["dpre"] = _sum_to(g * xh, pre.shape)
    r["dx"] = total
    if y is None:
        return r
    v = total * f(sc * a)
    if post is not None:
        w = v * f(post)
        r["dy"] = r1 * sub(w, f(yh) * (w * f(yh)).mean(-1, keepdim=True))
        r["dpost"] = _sum_to(v * f(yh), post.shape)
    else:
        r["dy"] = v
    if d["scale"] is not None:
        r["dscale"] = _sum_to(total * f(a * u), d["scale"].shape)
    if slope is not None:
        # (a slope such as 1 - t^2 is a difference of values up to 1)
        slope = slope.abs().clamp(min=1.0) if magnitude else slope
        r["dgate"] = _sum_to(total * f(sc * u) * slope, d["gate"].shape)
    return r


def _make(shape, xdt, ydt, gate, with_scale, post=True, pre=True, y=True, wdt=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    wdt = wdt or ydt
    rnd = lambda *s: torch.randn(*s, generator=g)
    t = dict.fromkeys(NAMES)
    t["x"] = (2 * rnd(*shape)).to(xdt)
    if y:
        t["y"] = rnd(*shape).to(ydt)
        t["post"] = (1 + 0.1 * rnd(C)).to(wdt) if post else None
        t["scale"] = (0.2 + 0.05 * rnd(C)).to(wdt) if with_scale is True else None
        t["gate"] = rnd(*gate).to(ydt) if gate is not None else None
    t["pre"] = (1 + 0.1 * rnd(C)).to(wdt) if pre else None
    return t, rnd(*shape).to(xdt), rnd(*shape).to(ydt)


def _call(t, act, scale, dtype=None):
    return residual_norm(t["x"], t["y"], post_weight=t["post"], pre_weight=t["pre"],
                         gate=t["gate"], gate_act=act,
                         scale=t["scale"] if t["scale"] is not None else scale, eps=EPS,
                         dtype=dtype)


def _check(got, want, mag, rows, C, what):
    got = got.detach().cpu()
    assert got.shape == want.shape, what
    chain = (C / 64 + rows / 64 + 64) * 2.0 ** -24
    tol = chain * mag + HALF_ULP[got.dtype] * (want.abs() + chain * mag)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25        # (spacing of its subnormals)
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound"


def _run_case(shape, xdt, ydt, gate, act, with_scale, use=("new", "h"), dtype=None, **kw):
    t, dnew, dh = _make(shape, xdt, ydt, gate, with_scale, **kw)
    scale = with_scale if isinstance(with_scale, float) else None
    dev = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    new, h = _call(dev, act, scale, dtype)
    outs, gs = [], []
    if t["y"] is not None and "new" in use:
        outs, gs = outs + [new], gs + [dnew.cuda()]
    if h is not None and "h" in use:
        outs, gs = outs + [h], gs + [dh.cuda()]
    names = [k for k in NAMES if dev[k] is not None]
    grads = torch.autograd.grad(outs, [dev[k] for k in names], gs, allow_unused=True)
    args = (t, act, scale, dnew if len(outs) and outs[0] is new else None,
            dh if h is not None and "h" in use else None)
    want, mag = _formulas(*args), _formulas(*args, magnitude=True)
    rows, C = t["x"].numel() // shape[-1], shape[-1]
    assert new.dtype == xdt
    _check(new, want["new"], mag["new"], 0, C, "new")
    if h is not None:
        assert h.dtype == (dtype or ydt)
        _check(h, want["h"], mag["h"], 0, C, "h")
    for k, g in zip(names, grads):
        if "d" + k not in want:
            assert g is None or not bool(g.any()), k
            continue
        assert g.dtype == t[k].dtype
        _check(g, want["d" + k], mag["d" + k], rows, C, "d" + k)
    # without gradients: the same values
    with torch.no_grad():
        n2, h2 = _call(dev, act, scale, dtype)
    assert torch.equal(n2, new) and (h is None or torch.equal(h2, h))


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("act", [None, "sigmoid", "tanh", "silu"])
@pytest.mark.parametrize("gate", [None, (2, 5, 7), (2, 5, 1), (2, 1, 7), (7,), (2, 1, 1)])
def test_formulas_against_differences(gate, act):
    """The closed formulas' gradients against central differences of their
    values (float64), and autograd of the CPU path against both."""
    if gate is None and act is not None:
        pytest.skip("an activation needs a gate")
    t, dnew, dh = _make((2, 5, 7), torch.float64, torch.float64, gate, True)
    want = _formulas(t, act, None, dnew, dh)

    def loss(u):
        r = _formulas(u, act, None, None, None)
        return float((r["new"] * dnew).sum() + (r["h"] * dh).sum())

    g = torch.Generator().manual_seed(5)
    step = 1e-5
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in t.items()}
    new, h = _call(leaf, act, None)
    names = [k for k in NAMES if t[k] is not None]
    auto = dict(zip(names, torch.autograd.grad([new, h], [leaf[k] for k in names], [dnew, dh])))
    for k in names:
        v = torch.randn(t[k].shape, generator=g, dtype=torch.float64)
        up, down = dict(t), dict(t)
        up[k], down[k] = t[k] + step * v, t[k] - step * v
        slope = (loss(up) - loss(down)) / (2 * step)
        # truncation step^2 of third derivatives (up to 1e3 here), rounding 1e-14 / step
        assert abs(float((want["d" + k] * v).sum()) - slope) < 1e-6 * max(1.0, abs(slope)), k
        torch.testing.assert_close(auto[k], want["d" + k], rtol=1e-10, atol=1e-10)


def test_optional_parts_on_the_cpu():
    t, _, _ = _make((3, 4), F32, F32, None, True)
    x, y = t["x"], t["y"]
    new, h = residual_norm(x, y)
    assert h is None
    torch.testing.assert_close(new, x + y)
    same, h = residual_norm(x, pre_weight=t["pre"])
    assert same is x
    torch.testing.assert_close(h, x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * t["pre"])
    assert residual_norm(x) == (x, None)
    new, h = residual_norm(x, pre_weight=t["pre"], dtype=BF16)
    assert new is x and h.dtype == BF16
    new, h = residual_norm(x[:0], y[:0], pre_weight=t["pre"])
    assert new.shape == h.shape == (0, 4)


@pytest.mark.parametrize("kw,text", [
    (dict(y=torch.zeros(3, 5)), "x's shape"),
    (dict(post_weight=torch.ones(4)), "need a branch"),
    (dict(y=torch.zeros(3, 4), gate=torch.zeros(3, 3)), "does not broadcast"),
    (dict(y=torch.zeros(3, 4), gate=torch.zeros(2, 4)), "does not broadcast"),
    (dict(y=torch.zeros(3, 4), gate=torch.zeros(1, 3, 4)), "does not broadcast"),
    (dict(y=torch.zeros(3, 4), gate=torch.zeros(3, 4), gate_act="relu"), "gate_act must be"),
    (dict(y=torch.zeros(3, 4), gate_act="silu"), "needs a gate"),
    (dict(y=torch.zeros(3, 4), gate=torch.zeros(3, 4, dtype=BF16)), "branch's type"),
    (dict(y=torch.zeros(3, 4), pre_weight=torch.ones(5)), "must have shape"),
    (dict(y=torch.zeros(3, 4), pre_weight=torch.ones(4), scale=torch.ones(4, dtype=BF16)),
     "share a dtype"),
    (dict(y=torch.zeros(3, 4), dtype=BF16), "in y's type"),
])
def test_refusals(kw, text):
    kw = dict(kw)
    with pytest.raises(RuntimeError, match=text):
        residual_norm(torch.zeros(3, 4), kw.pop("y", None), **kw)
    with pytest.raises(RuntimeError, match="branch's type or float32"):
        residual_norm(torch.zeros(3, 4, dtype=BF16), torch.zeros(3, 4))


def test_c_entry_refusals():
    """Refused before any launch: no device is needed, no pointer is read."""
    lib = pytest.importorskip("torchsplinekan_amd._lib")
    f = lib.LIB.kan_hip_residual_norm
    b = lib.LIB.kan_hip_residual_norm_backward
    p = 4096
    tail = (8, 16, 1e-6, p, p, None, None)
    assert f(1, 1, 1, p, p, None, p, p, p, 1.0, 0, 0, 0, *tail) == lib.KAN_ERR_INVALID
    assert "FP32, BF16 or FP16" in lib.last_error()
    assert f(2, 3, 0, p, p, None, p, p, p, 1.0, 0, 0, 0, *tail) == lib.KAN_ERR_INVALID
    assert "branch's type" in lib.last_error()
    assert f(0, 0, 0, p, p, p, p, p, p, 1.0, 0, 3, 16, *tail) == lib.KAN_ERR_INVALID
    assert "divide n" in lib.last_error()
    assert f(0, 0, 0, p, p, p, p, p, p, 1.0, 4, 8, 16, *tail) == lib.KAN_ERR_INVALID
    assert f(0, 0, 0, p, None, None, p, p, None, 1.0, 0, 0, 0, *tail) == lib.KAN_ERR_INVALID
    assert f(0, 0, 0, p, p, None, p, None, p, 1.0, 0, 0, 0, *tail) == lib.KAN_ERR_INVALID
    assert "go together" in lib.last_error()
    assert f(0, 0, 0, None, p, None, p, p, p, 1.0, 0, 0, 0, *tail) == lib.KAN_ERR_INVALID
    # no rows, no columns: nothing to do
    assert f(0, 0, 0, None, None, None, None, p, None, 1.0, 0, 0, 0, 0, 16, 1e-6, None, None,
             None, None) == lib.KAN_OK
    # gradients of operands that are not there, and no workspace
    args = (0, 0, 0, p, p, p, p, None, p, p, p, 1.0, 0, 0, 0, 8, 16, p)
    assert b(*args, p, p, p, p, p, p, None, 0, None) == lib.KAN_ERR_INVALID
    assert "absent operand" in lib.last_error()
    assert b(*args, p, p, None, p, p, p, None, 0, None) == lib.KAN_ERR_WORKSPACE


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]


@pytest.mark.gpu
@pytest.mark.parametrize("xdt,ydt", TYPES)
@pytest.mark.parametrize("C", [1, 2, 7, 64, 65, 120, 128, 301, 512, 1000, 1024, 1025, 2048, 4096, 4104, 8192,
                               8200, 16385])
def test_widths(C, xdt, ydt):
    _run_case((5, C), xdt, ydt, (5, C), "sigmoid", True)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 513, 1500, 5003])
@pytest.mark.parametrize("C", [40, 264, 1304])
def test_rows(n, C):
    _run_case((n, C), BF16, BF16, None, None, True)
    _run_case((n, C + 1), F32, F32, (n, 1), "tanh", True)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "sigmoid", "tanh", "silu"])
@pytest.mark.parametrize("gate", [(3, 40, 96), (3, 40, 1), (3, 1, 96), (96,), (1,), (3, 1, 1),
                                  (40, 96), (1, 40, 1)])
@pytest.mark.parametrize("xdt,ydt", TYPES[:1] + TYPES[3:4])
def test_gates(gate, act, xdt, ydt):
    _run_case((3, 40, 96), xdt, ydt, gate, act, True)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,L", [(1, 3000), (2, 1500), (7, 700), (600, 2), (1300, 3), (9, 111)])
@pytest.mark.parametrize("cols", [1, 136, 131])
def test_gate_rows_against_blocks(seqs, L, cols):
    """Gate rows longer and shorter than the rows a block has."""
    C = cols if cols > 1 else 72
    _run_case((seqs, L, C), F32, F32, (seqs, 1, cols), "tanh", True)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [72, 73, 9000])
@pytest.mark.parametrize("kw", [
    dict(post=False), dict(pre=False), dict(post=False, pre=False), dict(y=False),
    dict(use=("new",)), dict(use=("h",)), dict(wdt=F32)])
def test_optional_parts(C, kw):
    _run_case((33, C), BF16, BF16, None if kw.get("y") is False else (33, 1),
              None if kw.get("y") is False else "silu", kw.get("y") is not False, **kw)


@pytest.mark.gpu
def test_number_as_scale_and_type_of_h():
    _run_case((9, 48), F32, BF16, None, None, 0.25)
    _run_case((9, 48), F32, F16, None, None, None, y=False, dtype=F16)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [64, 65, 9000])
def test_strides_and_alignment(C):
    """Views that are neither contiguous nor aligned, and their gradients."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(20, C + 3, generator=g).cuda()
    x = base[:, 1:C + 1].requires_grad_()
    yt = torch.randn(C, 20, generator=g).cuda()
    y = yt.t().requires_grad_()
    w = torch.randn(C + 1, generator=g).cuda()[1:].requires_grad_()
    new, h = residual_norm(x, y, post_weight=w, pre_weight=w)
    ref = [v.detach().clone().contiguous().requires_grad_() for v in (x, y, w)]
    new2, h2 = residual_norm(ref[0], ref[1], post_weight=ref[2], pre_weight=ref[2])
    torch.testing.assert_close(new, new2, rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(h, h2, rtol=1e-6, atol=1e-6)
    dn = torch.randn(C, 20, generator=g).cuda().t()      # a transposed gradient
    ga = torch.autograd.grad([new, h], [x, y, w], [dn, dn])
    gb = torch.autograd.grad([new2, h2], ref, [dn.contiguous(), dn.contiguous()])
    for u, v in zip(ga, gb):
        torch.testing.assert_close(u, v, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [64, 2048, 9000])
def test_values_that_are_not_finite_stay_in_their_row(C):
    t, dnew, dh = _make((6, C), F32, F32, (6, C), True)
    for row, bad in ((1, float("nan")), (3, float("inf"))):
        t["y"][row, C // 2] = bad
    t["x"][4] = 0.0
    t["y"][4] = 0.0                      # a row of zeros: h = 0, no NaN
    dev = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    new, h = _call(dev, "tanh", None)
    gx, gy = torch.autograd.grad([new, h], [dev["x"], dev["y"]], [dnew.cuda(), dh.cuda()])
    for v in (new, h, gx, gy):
        ok = v.isfinite().all(-1).cpu()
        assert ok.tolist() == [True, False, True, False, True, True]
    assert not bool(h[4].any())


@pytest.mark.gpu
@pytest.mark.parametrize("C", [2048, 2047])
def test_rows_past_32_bit_offsets(C):
    """More than 2^31 values; the last rows against the same rows alone."""
    n, last = 1100000, 300
    g = torch.Generator(device="cuda").manual_seed(0)
    parts = [torch.randn(last, C, generator=g, device="cuda").to(BF16) for _ in range(4)]
    x, y, dn, dh = (torch.zeros(n, C, dtype=BF16, device="cuda") for _ in range(4))
    for whole, part in zip((x, y, dn, dh), parts):
        whole[-last:] = part
    w = torch.ones(C, device="cuda", dtype=BF16)

    def once(x, y, dn, dh):
        x, y = x.requires_grad_(), y.requires_grad_()
        new, h = residual_norm(x, y, post_weight=w, pre_weight=w)
        return [new, h, *torch.autograd.grad([new, h], [x, y], [dn, dh])]

    for u, v in zip(once(x, y, dn, dh), once(*parts)):
        assert torch.equal(u[-last:], v)
        assert not bool(u[:-last].any())


@pytest.mark.gpu
def test_same_bits_every_time_and_on_another_stream():
    t, dnew, dh = _make((4, 600, 520), BF16, BF16, (4, 1, 520), True)
    dev = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    names = [k for k in NAMES if dev[k] is not None]

    def once():
        new, h = _call(dev, "tanh", None)
        return [new, h, *torch.autograd.grad([new, h], [dev[k] for k in names],
                                             [dnew.cuda(), dh.cuda()])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(first, second):
        assert torch.equal(u, v)


@pytest.mark.gpu
def test_float64_is_refused_on_the_device():
    x = torch.zeros(2, 4, dtype=torch.float64, device="cuda")
    with pytest.raises(RuntimeError, match="FP32, BF16 and FP16"):
        residual_norm(x, x)


@pytest.mark.gpu
@pytest.mark.parametrize("leaf", NAMES)
def test_forward_mode_is_refused(leaf):
    """A dual tensor raises, with and without gradients; other tensors inside a
    level give what they give outside."""
    from torch.autograd import forward_ad
    t, _, _ = _make((6, 40), F32, F32, (6, 1), True)
    dev = {k: v.cuda() for k, v in t.items()}
    new, h = _call(dev, "silu", None)
    with forward_ad.dual_level():
        for u, v in zip(_call(dev, "silu", None), (new, h)):
            assert torch.equal(u, v) and not u.requires_grad
        dev[leaf] = forward_ad.make_dual(dev[leaf], torch.ones_like(dev[leaf]))
        with pytest.raises(RuntimeError, match="jvp"):
            _call(dev, "silu", None)
        with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
            _call(dev, "silu", None)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x = torch.randn(2, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    _, h = residual_norm(x, x * 1, pre_weight=w)
    g, = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
