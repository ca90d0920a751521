"""KANExpertStack's logits and losses go through the module's call, with its hooks, and its
norms each have their eps."""

import torch
import torch.nn.functional as F

from torchsplinekan_amd import KANExpertStack


def test_hooks_run_for_logits_and_losses():
    torch.manual_seed(0)
    net, seen = KANExpertStack(8, 1, 2, num_classes=5), []
    net.register_forward_pre_hook(lambda m, args: seen.append("before"))
    net.register_forward_hook(lambda m, args, out: 2 * out)
    x = torch.randn(4, 8)
    h = net(x)
    torch.testing.assert_close(net.logits(x), h @ net.head.t())
    values, ids = net.logits(x).topk(2)
    net.loss(x, torch.tensor([0, 1, 2, 3]))
    net.distillation_loss(x, ids, values.detach())
    assert seen == ["before"] * 5


def test_logits_under_autocast_are_those_without():
    torch.manual_seed(0)
    net, x = KANExpertStack(8, 1, 2, num_classes=5), torch.randn(4, 8)
    want = net.logits(x)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = net.logits(x)
    assert got.dtype == torch.float32 and torch.equal(got, want)


def test_the_input_norm_has_an_eps_of_its_own():
    torch.manual_seed(0)
    kw = dict(num_experts=2, eps=0.5, input_norm=True, input_eps=0.25)
    net, x = KANExpertStack(8, 1, **kw).double(), torch.randn(4, 8, dtype=torch.float64)
    plain = KANExpertStack(8, 1, num_experts=2, eps=0.5).double()
    plain.load_state_dict(net.state_dict(), strict=False)
    for eps in (0.25, 2.0):
        net.input_eps = eps
        torch.testing.assert_close(net(x), plain(F.layer_norm(x, (8,), eps=eps)))
    assert KANExpertStack(8, 1, 2, input_norm=True).input_eps == 1e-5
