"""KANExperts and KANExpertStack, where residual_norm, grouped_linear and
checkpoint_8bit run together: against KAN layers applied expert by expert,
against the same model in float64, and captured in a HIP graph."""

import copy

import pytest
import torch
import torch.nn.functional as F

from torchsplinekan_amd import KANExperts, KANExpertStack, grouped_linear, residual_norm
from torchsplinekan_amd.experts import route
from torchsplinekan_amd.reference_backend import compute_basis


def _plain(m, x):
    """Every expert on every row, weighted by the routed probabilities."""
    logits = x @ m.router.t()
    top, ids = logits.topk(m.top_k, -1)
    p = torch.zeros_like(logits).scatter(-1, ids, top.softmax(-1))
    H = compute_basis(x, m.grid, m.spline_order)
    y = torch.einsum("ni,eoi->neo", F.silu(x), m.base_weight)
    y = y + torch.einsum("nir,eoir->neo", H, m.spline_weight)
    return (y * p.unsqueeze(-1)).sum(1)


def _model(seed=0, **kw):
    torch.manual_seed(seed)
    return KANExperts(12, 7, 5, **kw)


@pytest.mark.parametrize("top_k", [1, 2, 5])
def test_mixture_is_the_sum_of_its_experts(top_k):
    m = _model(top_k=top_k).double()
    x = torch.randn(33, 12, dtype=torch.float64).requires_grad_()
    y, want = m(x), _plain(m, x)
    torch.testing.assert_close(y, want)
    g = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, *m.parameters()], g)
    ref = torch.autograd.grad(want, [x, *m.parameters()], g)
    for u, v in zip(got, ref):
        torch.testing.assert_close(u, v)
    assert m(x.reshape(3, 11, 12)).shape == (3, 11, 7)


def test_route():
    logits = torch.tensor([[0.0, 3.0, 1.0], [2.0, 0.0, 1.0], [0.0, 5.0, 4.0]])
    w, order, offsets = route(logits, 2)
    assert offsets.tolist() == [0, 1, 3, 6]
    assert order.tolist() == [2, 0, 4, 1, 3, 5]
    torch.testing.assert_close(w, torch.stack([t.topk(2).values.softmax(-1) for t in logits]))


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_checkpoint_keeps_the_output(form):
    a, b = _model(), _model(checkpoint=form, group=32)
    b.load_state_dict(a.state_dict())
    x = torch.randn(40, 12)
    assert torch.equal(a(x), b(x))
    g = torch.randn(40, 7)
    ga = torch.autograd.grad(a(x), list(a.parameters()), g)
    gb = torch.autograd.grad(b(x), list(b.parameters()), g)
    assert torch.equal(ga[0], gb[0])       # the router sees the exact rows
    for u, v in zip(ga[1:], gb[1:]):       # the layers the restored ones
        assert not torch.equal(u, v)
        assert float((u - v).norm() / u.norm()) < 0.1


def test_stack_trains_on_the_cpu():
    torch.manual_seed(1)
    net = KANExpertStack(12, 2, 4, top_k=2, checkpoint="int8", group=32)
    x, t = torch.randn(64, 12), torch.randn(64, 12)
    opt = torch.optim.Adam(net.parameters(), lr=1e-2)
    losses = []
    for _ in range(30):
        opt.zero_grad()
        loss = F.mse_loss(net(x), t)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.7 * losses[0]
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in net.parameters())


def _same_under_autocast(net, x):
    """Output and gradients bit for bit those outside autocast."""
    g = torch.randn(x.shape[:-1] + (x.shape[-1],), device=x.device)
    want, wgrads = _grads(net, x, g)
    with torch.autocast(x.device.type, dtype=torch.bfloat16):
        got = net(x)
    assert got.dtype == torch.float32 and torch.equal(got, want)
    for u, v in zip(torch.autograd.grad(got, [x, *net.parameters()], g), wgrads):
        assert torch.equal(u, v)


@pytest.mark.parametrize("form", [None, "int8"])
def test_autocast_changes_nothing(form):
    torch.manual_seed(2)
    net = KANExpertStack(12, 2, 4, top_k=2, checkpoint=form, group=32)
    _same_under_autocast(net, torch.randn(40, 12).requires_grad_())
    _same_under_autocast(KANExperts(12, 12, 3, checkpoint=form),
                         torch.randn(40, 12).requires_grad_())


def test_refusals():
    with pytest.raises(ValueError, match="top_k"):
        KANExperts(4, 4, 2, top_k=3)
    with pytest.raises(ValueError, match="spline_order"):
        KANExperts(4, 4, 2, spline_order=4)
    with pytest.raises(RuntimeError, match="format must"):
        KANExperts(4, 4, 2, checkpoint="int4")
    with pytest.raises(ValueError, match="depth"):
        KANExpertStack(4, 0, 2)


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

def _grads(net, x, g):
    y = net(x)
    return y, torch.autograd.grad(y, [x, *net.parameters()], g)


@pytest.mark.gpu
@pytest.mark.parametrize("width,depth,experts,top_k,rows", [(64, 2, 8, 2, 700), (33, 1, 3, 1, 65),
                                                            (48, 3, 4, 4, 128), (16, 2, 70, 2, 9)])
def test_stack_on_the_device_against_float64(width, depth, experts, top_k, rows):
    """The device model in float32 against the CPU one in float64.  Float32's
    2^-24 through a block's chain of some 1000 operations, normwise: 1e-4 holds
    a wide margin for the routing's softmax, and a wrong formula misses it by
    orders of magnitude."""
    torch.manual_seed(width)
    net = KANExpertStack(width, depth, experts, top_k=top_k, scale_noise=0.5)
    x = torch.randn(rows, width)
    g = torch.randn(rows, width)
    ref = copy.deepcopy(net).double()
    xr = x.double().requires_grad_()
    want, wgrads = _grads(ref, xr, g.double())
    dev = net.cuda()
    xd = x.cuda().requires_grad_()
    got, grads = _grads(dev, xd, g.cuda())
    for u, v in zip([got, *grads], [want, *wgrads]):
        assert float((u.detach().cpu().double() - v.detach()).norm()) < 1e-4 * max(
            1e-12, float(v.detach().norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("form", [None, "int8"])
def test_autocast_changes_nothing_on_the_device(form):
    torch.manual_seed(2)
    net = KANExpertStack(48, 2, 4, top_k=2, checkpoint=form).cuda()
    _same_under_autocast(net, torch.randn(200, 48, device="cuda").requires_grad_())


@pytest.mark.gpu
def test_checkpointed_stack_on_the_device():
    """The same output bit for bit, little memory held between the passes, and
    the same bits in every run."""
    torch.manual_seed(0)
    kw = dict(top_k=2, grid_size=10)
    net = KANExpertStack(256, 2, 8, **kw).cuda()
    kept = KANExpertStack(256, 2, 8, checkpoint="int8", **kw).cuda()
    kept.load_state_dict(net.state_dict())
    x = torch.randn(4096, 256, device="cuda")
    g = torch.randn(4096, 256, device="cuda")

    def held(m):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = m(x.requires_grad_())
        return y, torch.cuda.memory_allocated() - before

    y0, full = held(net)
    y1, little = held(kept)
    assert torch.equal(y0, y1)
    # of each block's 2 x 4096 routed rows the plain stack keeps the basis
    # (13 + 1) x 256 floats, the other 256 bytes and two scales
    assert full - little > 2 * 8192 * 256 * 13 * 4
    first = torch.autograd.grad(y1, list(kept.parameters()), g)
    again = torch.autograd.grad(kept(x), list(kept.parameters()), g)
    for u, v in zip(first, again):
        assert torch.equal(u, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_operators_replay(dtype):
    """residual_norm and grouped_linear with their gradients in a HIP graph:
    every replay on new inputs and new group sizes gives the eager bits."""
    torch.manual_seed(0)
    T, E, C = 700, 6, 136
    x = torch.randn(T, C, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn(E, C, C, device="cuda") * C ** -0.5).to(dtype).requires_grad_()
    gate = torch.randn(T, 1, device="cuda").to(dtype).requires_grad_()
    weight = torch.ones(C, device="cuda", dtype=dtype).requires_grad_()
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    dy = torch.randn(T, C, device="cuda").to(dtype)
    leaves = [x, w, gate, weight]

    def step():
        _, h = residual_norm(x, pre_weight=weight)
        y = grouped_linear(h, w, off, checkpoint="int8")
        new, h = residual_norm(x, y, post_weight=weight, pre_weight=weight, gate=gate,
                               gate_act="silu", scale=0.5)
        return [new, h, *torch.autograd.grad([new, h], leaves, [dy, dy])]

    def draw(seed):
        g = torch.Generator().manual_seed(seed)
        ids = torch.randint(0, E - seed % 2, (T,), generator=g)
        off[1:].copy_(torch.bincount(ids, minlength=E).cumsum(0))
        with torch.no_grad():
            x.copy_(torch.randn(T, C, generator=g))

    draw(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 5):
        draw(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        for u, v in zip(got, step()):
            assert torch.equal(u, v)
