"""Check of what an operator keeps in 8 bits between its passes."""

import weakref

import pytest
import torch


class _Held:
    def __init__(self, t):
        self.t = t


def check_kept_is_saved(run, inputs, g, in_place=()):
    """run's 8-bit rows and scales pass through saved-tensor hooks and are gone
    after the backward pass; its gradients are what they are without hooks.  A
    tensor of in_place that is changed between the passes raises."""
    want = torch.autograd.grad(run(), inputs, g)
    held = []

    def pack(t):
        h = _Held(t.detach().clone())
        held.append((t.dtype, tuple(t.shape), weakref.ref(h)))
        return h

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda h: h.t):
        y = run()
    kept = [h for h in held if h[0] in (torch.int8, torch.float8_e4m3fn)]
    assert kept and all(r() is not None for _, _, r in kept)
    got = torch.autograd.grad(y, inputs, g)
    assert all(r() is None for _, _, r in held)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, inputs, g)
    for t in in_place:
        y = run()
        with torch.no_grad():
            t.add_(1)
        with pytest.raises(RuntimeError, match="in place|inplace"):
            torch.autograd.grad(y, inputs, g)
        with torch.no_grad():
            t.sub_(1)
