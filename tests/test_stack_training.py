"""A stack of routed KAN layers with its layer norm, gated feed-forward blocks and
last layer, where layer_norm, gated_linear, linear_cross_entropy and
linear_distillation run together: against the same model written out in torch, in
float64 on the CPU, and captured in a HIP graph."""

import copy

import pytest
import torch
import torch.nn.functional as F

from torchsplinekan_amd import (KANExpertStack, gated_linear, layer_norm, linear_cross_entropy,
                                linear_distillation)


def _net(width=24, classes=17, seed=0, **kw):
    torch.manual_seed(seed)
    net = KANExpertStack(width, 2, 4, feed_forward=40, input_norm=True, num_classes=classes,
                         top_k=2, scale_noise=0.5, **kw)
    with torch.no_grad():
        net.input_bias.normal_(std=0.1)
    return net


def _plain(net, x):
    """The stack written out."""
    def rms(v, w):
        return v / (v.square().mean(-1, keepdim=True) + net.eps).sqrt() * w

    x = F.layer_norm(x, x.shape[-1:], net.input_weight, net.input_bias)
    for b in net.blocks:
        h = rms(x, b.pre_weight)
        y = b.experts(h) + F.linear(F.silu(h @ b.gate_up[0].t()) * (h @ b.gate_up[1].t()), b.down)
        x = x + b.scale * torch.sigmoid(b.gate(h)) * rms(y, b.post_weight)
    return rms(x, net.norm_weight)


def _targets(net, x, k=5):
    g = torch.Generator().manual_seed(3)
    rows = x.shape[:-1]
    target = torch.randint(net.head.shape[0], rows, generator=g)
    target.view(-1)[::6] = -100
    ids = torch.rand(*rows, net.head.shape[0], generator=g).topk(k, -1).indices
    ids[..., 0, :2] = -1
    return target, ids, 2 * torch.randn(ids.shape, generator=g)


def _losses(net, x, target, ids, teacher):
    return [net.loss(x, target), net.distillation_loss(x, ids, teacher, temperature=2.0)]


def test_losses_are_those_of_the_model_written_out():
    net = _net().double()
    x = torch.randn(3, 20, 24, dtype=torch.float64).requires_grad_()
    target, ids, teacher = _targets(net, x)
    z = _plain(net, x) @ net.head.t()
    torch.testing.assert_close(net.logits(x), z)
    p = torch.where(ids < 0, -torch.inf, teacher.double() / 2).softmax(-1)
    logq = (z / 2).log_softmax(-1).gather(-1, ids.clamp(min=0))
    want = [F.cross_entropy(z.reshape(60, 17), target.reshape(60)),
            4 * (p * (p.clamp(min=1e-300).log() - logq)).sum(-1).mean()]
    leaves = [x, *net.parameters()]
    for got, ref in zip(_losses(net, x, target, ids, teacher), want):
        torch.testing.assert_close(got, ref)
        for a, b in zip(torch.autograd.grad(got, leaves), torch.autograd.grad(ref, leaves,
                                                                              retain_graph=True)):
            torch.testing.assert_close(a, b)


def test_gradients_against_differences():
    net = _net(width=6, classes=5).double()
    x = torch.randn(4, 6, dtype=torch.float64)
    target, ids, teacher = _targets(net, x, k=3)
    g = torch.Generator().manual_seed(5)
    for loss in (lambda: net.loss(x, target), lambda: net.distillation_loss(x, ids, teacher)):
        params = [net.head, net.blocks[0].gate_up, net.blocks[1].down, net.input_weight]
        grads = torch.autograd.grad(loss(), params)
        for p, d in zip(params, grads):
            v = torch.randn(p.shape, generator=g, dtype=torch.float64)
            with torch.no_grad():
                p += 1e-6 * v
                up = loss()
                p -= 2e-6 * v
                down = loss()
                p += 1e-6 * v
            torch.testing.assert_close((d * v).sum(), (up - down) / 2e-6, rtol=1e-5, atol=1e-7)


def test_defaults_are_the_stack_as_it_was():
    torch.manual_seed(1)
    net = KANExpertStack(12, 2, 4)
    assert not any(n.split(".")[-1] in ("gate_up", "down", "head", "input_weight")
                   for n, _ in net.named_parameters())
    x = torch.randn(5, 12)
    with pytest.raises(RuntimeError, match="num_classes"):
        net.loss(x, torch.zeros(5, dtype=torch.long))
    with pytest.raises(RuntimeError, match="num_classes"):
        net.logits(x)
    with pytest.raises(ValueError, match="feed_forward"):
        KANExpertStack(12, 2, 4, feed_forward=-1)
    with pytest.raises(ValueError, match="num_classes"):
        KANExpertStack(12, 2, 4, num_classes=0)


def test_teacher_trains_a_student_on_the_cpu():
    teacher, student = _net(seed=1), _net(seed=2, checkpoint="int8", group=32)
    x = torch.randn(64, 24)
    with torch.no_grad():
        values, ids = teacher.logits(x).topk(4)
    opt = torch.optim.Adam(student.parameters(), lr=1e-3)
    for _ in range(3):
        opt.zero_grad()
        student.distillation_loss(x, ids, values, temperature=2.0).backward()
        opt.step()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in student.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("width,classes,rows", [(64, 10, 700), (33, 1000, 65), (16, 3, 9)])
def test_on_the_device_against_float64(width, classes, rows):
    """The device model in float32 against the CPU one in float64, normwise: 2^-24
    through a chain of some 1000 operations, as of the stack without these parts."""
    net = _net(width, classes)
    x = torch.randn(rows, width)
    target, ids, teacher = _targets(net, x, k=min(5, classes))
    ref = copy.deepcopy(net).double()
    xr = x.double().requires_grad_()
    dev, xd = net.cuda(), x.cuda().requires_grad_()
    for want, got in zip(_losses(ref, xr, target, ids, teacher),
                         _losses(dev, xd, target.cuda(), ids.cuda(), teacher.cuda())):
        wgrads = torch.autograd.grad(want, [xr, *ref.parameters()])
        grads = torch.autograd.grad(got, [xd, *dev.parameters()])
        for u, v in zip([got, *grads], [want, *wgrads]):
            assert float((u.detach().cpu().double() - v.detach()).norm()) < 1e-4 * max(
                1e-12, float(v.detach().norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_training_step_replays(dtype):
    """The operators one after the other with their gradients in a HIP graph: every
    replay on new rows, targets and group sizes gives the eager bits."""
    torch.manual_seed(0)
    T, E, C, V = 700, 3, 136, 1030
    dev = dict(device="cuda", dtype=dtype)
    x = torch.randn(T, C, **dev).requires_grad_()
    w, b = torch.ones(C, **dev).requires_grad_(), torch.zeros(C, **dev).requires_grad_()
    up = (torch.randn(E, 2, 264, C, **dev) * C ** -0.5).requires_grad_()
    down = (torch.randn(C, 264, **dev) * 264 ** -0.5).requires_grad_()
    head = (torch.randn(V, C, **dev) * C ** -0.5).requires_grad_()
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    target = torch.zeros(T, dtype=torch.long, device="cuda")
    ids = torch.zeros(T, 6, dtype=torch.int32, device="cuda")
    teacher = torch.randn(T, 6, device="cuda")
    leaves = [x, w, b, up, down, head]

    def step():
        h = layer_norm(x, w, b)
        h = h + gated_linear(h, up, off) @ down.t()
        losses = [linear_cross_entropy(h, head, target), linear_distillation(h, head, ids, teacher)]
        return [t.detach() for t in losses] + list(torch.autograd.grad(losses, leaves))

    def draw(seed):
        g = torch.Generator().manual_seed(seed)
        count = torch.bincount(torch.randint(0, E - seed % 2, (T,), generator=g), minlength=E)
        off[1:].copy_(count.cumsum(0))
        target.copy_(torch.randint(-1, V, (T,), generator=g))
        target[target < 0] = -100
        ids.copy_(torch.randint(-1, V, (T, 6), generator=g))
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


@pytest.mark.gpu
def test_two_calls_at_once_and_graphs_keep_workspaces_of_their_own():
    """Two streams with the same operators on other data, and two captured steps
    replayed in turn: each as alone."""
    torch.manual_seed(0)
    jobs = []
    for seed in range(2):
        x = torch.randn(900, 256, device="cuda", dtype=torch.bfloat16).requires_grad_()
        w = (torch.randn(5000, 256, device="cuda") / 16).bfloat16().requires_grad_()
        up = (torch.randn(2, 512, 256, device="cuda") / 16).bfloat16().requires_grad_()
        target = torch.randint(5000, (900,), device="cuda")
        dh = torch.randn(900, 512, device="cuda", dtype=torch.bfloat16)
        one = torch.ones((), device="cuda")

        def step(x=x, w=w, up=up, target=target, dh=dh, one=one):
            loss = linear_cross_entropy(layer_norm(x), w, target)
            h = gated_linear(x, up)
            return [loss.detach(), h.detach(),
                    *torch.autograd.grad([loss, h], [x, w, up], [one, dh])]

        jobs.append(step)
    want = [[t.clone() for t in step()] for step in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        got = []
        for step, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                got.append(step())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for u, v in zip(a, b):
                assert torch.equal(u, v)
    del got
    graphs, outs = [], []
    for step in jobs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            for u, v in zip(a, b):
                assert torch.equal(u, v)
