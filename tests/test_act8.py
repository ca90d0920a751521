"""Activations in 8 bits: the device kernels give the same 8-bit values, scales
and restored values as the formulas evaluated on the CPU (every operation is a
correctly rounded one, so they agree bit for bit), and the formulas keep their
error bounds."""

import pytest
import torch
import torch.nn as nn

from _saved import check_kept_is_saved
from torchsplinekan_amd import KANLinear, checkpoint_8bit, quantize_activation
from torchsplinekan_amd.act8 import FORMATS, GROUPS

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _values(rows, C, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=g) * 10 ** (torch.rand(rows, 1, generator=g) * 4 - 2)
    return x.to(dtype)


@pytest.mark.parametrize("format", ["int8", "e4m3"])
@pytest.mark.parametrize("C,group", [(1, 32), (31, 32), (128, 128), (130, 64), (300, 256)])
def test_error_bounds(C, group, format):
    """int8: half a step of scale; e4m3: a 16th of the value (half of its last
    of 3 bits), or half the smallest step 2^-9 of scale; and the roundings of
    the scale, its reciprocal and the products (4 in float32)."""
    x = _values(7, C, F32)
    a = quantize_activation(x, group, format)
    assert a.q.shape == x.shape and a.scale.shape == (7, -(-C // group))
    step = a.scale.repeat_interleave(group, 1)[:, :C]
    err = (a.dequantize() - x).abs()
    if format == "int8":
        bound = 0.5 * step
    else:
        bound = torch.maximum(x.abs() / 16, step * 2.0 ** -10)
    assert bool((err <= bound * (1 + 1e-6) + x.abs() * 4 * 2.0 ** -24).all())
    assert a.nbytes == x.numel() + 4 * a.scale.numel()


@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_special_groups(format):
    x = torch.zeros(6, 64)
    x[1, :32] = 1e-39                  # below the smallest scale: zeros
    above = 1.5 * FORMATS[format][1] * torch.finfo(F32).tiny
    x[1, 32:] = above
    x[2, 3] = float("nan")
    x[3, 40] = float("-inf")
    x[4, 5] = -3.0e38
    x[5, 6] = 5.0
    for dev in ["cpu"] + (["cuda"] if torch.cuda.is_available() else []):
        a = quantize_activation(x.to(dev), 32, format)
        back = a.dequantize().cpu()
        assert not bool(back[0].any()) and not bool(a.scale[0].any())
        assert not bool(back[1, :32].any())
        assert bool(((back[1, 32:] - above).abs() < 1e-6 * above).all())
        assert bool(back[2, :32].isnan().all()) and not bool(back[2, 32:].any())
        assert bool(back[3, 32:].isnan().all()) and not bool(back[3, :32].any())
        assert float(back[4, 5]) == pytest.approx(-3.0e38, rel=1e-6)
        assert float(back[5, 6]) == 5.0


@pytest.mark.parametrize("kw,text", [
    (dict(group=48), "group must be"), (dict(format="int4"), "format must be")])
def test_refusals(kw, text):
    with pytest.raises(RuntimeError, match=text):
        quantize_activation(torch.zeros(2, 4), **kw)
    with pytest.raises(RuntimeError, match=text):
        checkpoint_8bit(nn.Linear(4, 4), torch.zeros(2, 4), **kw)
    with pytest.raises(RuntimeError, match="FP32, BF16 and FP16"):
        quantize_activation(torch.zeros(2, 4, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="at least one dimension"):
        quantize_activation(torch.zeros(()))


def test_c_entry_refusals():
    lib = pytest.importorskip("torchsplinekan_amd._lib")
    q, d = lib.LIB.kan_hip_act8_quantize, lib.LIB.kan_hip_act8_dequantize
    p = 4096
    assert q(1, 1, p, 8, 4, 8, 32, p, p, None) == lib.KAN_ERR_INVALID
    assert q(0, 3, p, 8, 4, 8, 32, p, p, None) == lib.KAN_ERR_INVALID
    assert q(0, 1, p, 8, 4, 8, 48, p, p, None) == lib.KAN_ERR_INVALID
    assert "group must be" in lib.last_error()
    assert q(0, 1, p, 7, 4, 8, 32, p, p, None) == lib.KAN_ERR_INVALID
    assert q(0, 1, None, 8, 4, 8, 32, p, p, None) == lib.KAN_ERR_INVALID
    assert q(0, 1, p, 8, -1, 8, 32, p, p, None) == lib.KAN_ERR_INVALID
    assert d(0, 1, p, p, 4, 8, 32, None, None) == lib.KAN_ERR_INVALID
    assert d(0, 1, None, None, 0, 8, 32, None, None) == lib.KAN_OK


def _net(dev="cpu"):
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(24, 40), nn.SiLU(), nn.Linear(40, 8)).to(dev)


@pytest.mark.parametrize("need_x", [True, False])
@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_checkpoint_is_the_layer_at_the_restored_input(need_x, format):
    """Output as without it; gradients those of the layer at the restored x."""
    net, x = _net(), _values(9, 24, F32).requires_grad_(need_x)
    y = checkpoint_8bit(net, x, group=32, format=format)
    assert torch.equal(y, net(x))
    g = torch.randn_like(y)
    inputs = ([x] if need_x else []) + list(net.parameters())
    got = torch.autograd.grad(y, inputs, g)
    xr = quantize_activation(x, 32, format).dequantize().requires_grad_(need_x)
    want = torch.autograd.grad(net(xr), ([xr] if need_x else []) + list(net.parameters()), g)
    for u, v in zip(got, want):
        assert torch.equal(u, v)


def test_checkpoint_other_calls():
    net = _net()
    x = _values(3, 24, F32)
    with torch.no_grad():
        assert not checkpoint_8bit(net, x).requires_grad
    # a function with further arguments, several outputs, one of them unused
    w = torch.randn(24, requires_grad=True)
    f = lambda v, s: (v * w * s, v.sum())
    xr = x.clone().requires_grad_()
    a, b = checkpoint_8bit(f, xr, 2.0, params=[w])
    gw, gx = torch.autograd.grad(a.sum(), [w, xr])
    back = quantize_activation(x).dequantize()
    torch.testing.assert_close(gw, 2 * back.sum(0))
    torch.testing.assert_close(gx, (2 * w).expand(3, 24).detach())


@pytest.mark.parametrize("around", ["both", "forward", "backward"])
def test_checkpoint_keeps_the_forward_pass_autocast(around):
    """Gradients are those of the layer at the restored input under the forward
    pass's autocast, whatever surrounds the backward pass."""
    net, x = _net(), _values(9, 24, F32).requires_grad_()
    inputs = [x, *net.parameters()]
    g = torch.randn(9, 8)

    def cast(on):
        return torch.autocast("cpu", dtype=BF16, enabled=on)

    xr = quantize_activation(x, 32).dequantize().requires_grad_()
    with cast(around != "backward"):
        plain, want = net(x), net(xr)
    with cast(around != "backward"):
        y = checkpoint_8bit(net, x, group=32)
    assert y.dtype == (F32 if around == "backward" else BF16) and torch.equal(y, plain)
    with cast(around != "forward"):  # (which the products of both backward passes see)
        want = torch.autograd.grad(want, [xr, *net.parameters()], g.to(y.dtype))
        got = torch.autograd.grad(y, inputs, g.to(y.dtype))
    for u, v in zip(got, want):
        assert u.dtype == v.dtype and torch.equal(u, v)


def test_checkpoint_counts_a_parameter_once():
    """A tied weight that stands in params twice has one gradient."""
    x, w = _values(6, 24, F32), torch.randn(24, requires_grad=True)
    y = checkpoint_8bit(lambda v: v * w, x, group=32, params=[w, w])
    got, = torch.autograd.grad(y.sum(), [w])
    torch.testing.assert_close(got, quantize_activation(x, 32).dequantize().sum(0))


def test_checkpoint_passes_tensor_arguments():
    """Gradients reach tensor arguments, alone or beside x's, and one that fn gives
    back stays the caller's own."""
    x, s = _values(6, 24, F32), torch.randn(24, requires_grad=True)
    back = quantize_activation(x, 32).dequantize()
    for need_x in (False, True):
        xr = x.clone().requires_grad_(need_x)
        y = checkpoint_8bit(lambda v, t, n: (v * t * n).sin(), xr, s, 2.0, group=32)
        assert torch.equal(y, (x * s * 2).sin())
        got, = torch.autograd.grad(y.sum(), [s], retain_graph=need_x)
        torch.testing.assert_close(got, (2 * back * (2 * back * s).cos()).sum(0))
        if need_x:
            torch.testing.assert_close(torch.autograd.grad(y.sum(), [xr])[0],
                                       2 * s.detach() * (2 * back * s.detach()).cos())
    xr, t = x.clone().requires_grad_(), torch.ones(3)
    y, out = checkpoint_8bit(lambda v, t: (v * 2, t), xr, t, group=32)
    assert t.is_leaf and not t.requires_grad and torch.equal(out, t)
    z = s * 3                                   # (not a leaf)
    y = checkpoint_8bit(lambda v, t: v * t, xr, z, group=32)
    torch.testing.assert_close(torch.autograd.grad(y.sum(), [s])[0], 3 * back.sum(0))


def test_checkpoint_leaves_autocast_of_other_calls():
    """The layer used beside its checkpoint, in one autocast region, keeps its
    gradients (casts of weights made without gradients are not kept for it)."""
    net, x = _net(), _values(9, 24, F32)
    with torch.autocast("cpu", dtype=BF16):
        first = checkpoint_8bit(net, x, group=32)
        beside = net(x)
        got = torch.autograd.grad(beside.float().sum() + first.float().sum(),
                                  list(net.parameters()))
    for v in got:
        assert bool(v.any())
    with torch.autocast("cpu", dtype=BF16):
        a = torch.autograd.grad(net(x).float().sum(), list(net.parameters()))
        xr = quantize_activation(x, 32).dequantize()
        b = torch.autograd.grad(net(xr).float().sum(), list(net.parameters()))
    for v, u, w in zip(got, a, b):
        assert torch.equal(v, u + w)


@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_checkpoint_saves_what_it_keeps(format):
    net, x, shift = _net(), _values(9, 24, F32).requires_grad_(), torch.zeros(8)
    params = list(net.parameters())
    check_kept_is_saved(
        lambda: checkpoint_8bit(lambda v, s: net(v) + s, x, shift, format=format, params=params),
        [x, *params], torch.randn(9, 8), in_place=[params[0], params[3], shift])
    with pytest.raises(RuntimeError, match="second time"):
        y = checkpoint_8bit(net, x)
        for _ in range(2):
            y.sum().backward()


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

def _same(x, group, format):
    dev, cpu = quantize_activation(x.cuda(), group, format), quantize_activation(x, group, format)
    assert torch.equal(dev.scale.cpu(), cpu.scale)
    assert torch.equal(dev.q.cpu().view(torch.uint8), cpu.q.view(torch.uint8))
    for dtype in (x.dtype, F32, BF16, F16):
        u, v = dev.dequantize(dtype).cpu(), cpu.dequantize(dtype)
        assert u.dtype == dtype and torch.equal(u, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 7), (2, 8), (1, 256), (5, 301), (64, 512),
                                    (1000, 40), (33, 1032), (7, 4099)])
@pytest.mark.parametrize("format", list(FORMATS))
def test_same_bits_as_the_formulas(rows, C, group, dtype, format):
    _same(_values(rows, C, dtype), group, format)


@pytest.mark.gpu
@pytest.mark.parametrize("format", list(FORMATS))
def test_ties_and_every_half_precision_value(format):
    """All finite float16 values, group by group, and multiples of half a step."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(F16)
    _same(torch.where(bits.isfinite(), bits, torch.zeros((), dtype=F16)).reshape(512, 128), 128,
          format)
    x = (torch.arange(-254, 255, dtype=F32) / 2).repeat(3, 1)
    _same(torch.cat([x, torch.full((3, 3), 127.0)], 1), 256, format)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [64, 61])
def test_views(C):
    x = _values(40, 2 * C + 1, F32).cuda()
    for v in (x[:, 1:C + 1], x[::2, :C], x.t()[:C], x[:, :C].reshape(4, 10, C), x[0, :C],
              x[:1, 3:C + 3]):
        a, b = quantize_activation(v, 32), quantize_activation(v.contiguous().clone(), 32)
        assert a.q.shape == v.shape
        assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale)
        assert torch.equal(a.dequantize(), b.dequantize())


@pytest.mark.gpu
@pytest.mark.parametrize("C", [2048, 2047])
def test_values_past_32_bit_offsets(C):
    x = torch.zeros(1100000, C, dtype=BF16, device="cuda")
    x[-300:] = _values(300, C, BF16).cuda()
    a, b = quantize_activation(x), quantize_activation(x[-300:].clone())
    assert torch.equal(a.q[-300:], b.q) and torch.equal(a.scale[-300:], b.scale)
    back = a.dequantize()
    assert torch.equal(back[-300:], b.dequantize()) and not bool(back[:-300].any())


@pytest.mark.gpu
def test_special_groups_on_the_device():
    test_special_groups("int8")
    test_special_groups("e4m3")
    empty = quantize_activation(torch.empty(0, 5, device="cuda"))
    assert empty.dequantize().shape == (0, 5)


@pytest.mark.gpu
def test_checkpointed_kan_layer():
    """A KAN layer keeps 8 bits of its input: gradients are those of the layer
    at the restored input, bit for bit, and the memory held between the passes
    is the 8-bit input's and the output's."""
    torch.manual_seed(0)
    layer = KANLinear(256, 64, grid_size=10, backend="cuda").cuda()
    x = (torch.rand(4096, 256) * 2 - 1).cuda().requires_grad_()
    g = torch.randn(4096, 64).cuda()
    torch.autograd.grad(layer(x), x, g)      # (first-use allocations)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = checkpoint_8bit(layer, x)
    held = torch.cuda.memory_allocated() - before
    assert held <= 4096 * 256 + 4096 * 2 * 4 + 4096 * 64 * 4 + 4096
    got = torch.autograd.grad(y, [x, *layer.parameters()], g)
    xr = quantize_activation(x).dequantize().requires_grad_()
    want = torch.autograd.grad(layer(xr), [xr, *layer.parameters()], g)
    for u, v in zip(got, want):
        assert torch.equal(u, v)


@pytest.mark.gpu
@pytest.mark.parametrize("inside", [True, False])
def test_checkpoint_under_autocast_on_the_device(inside):
    """As on the CPU, the backward pass running on a thread of its own: gradients of
    the layer at the restored input under the call's autocast, and a layer used
    beside its checkpoint keeps its own."""
    net, x = _net("cuda"), _values(64, 24, F32).cuda().requires_grad_()
    params, g = list(net.parameters()), torch.randn(64, 8, device="cuda").to(BF16)
    xr = quantize_activation(x, 32).dequantize().requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        want = net(xr)
        y = checkpoint_8bit(net, x, group=32)
        assert y.dtype == BF16 and torch.equal(y, net(x))
        if inside:
            got = torch.autograd.grad(y, [x, *params], g)
            want = torch.autograd.grad(want, [xr, *params], g)
    if not inside:
        got = torch.autograd.grad(y, [x, *params], g)
        want = torch.autograd.grad(want, [xr, *params], g)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    with torch.autocast("cuda", dtype=BF16):
        checkpoint_8bit(net, x, group=32)
        beside = net(x)
    for v in torch.autograd.grad(beside, params, g):
        assert bool(v.any())
