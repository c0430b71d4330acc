"""A captured backward pass of the block norms whose leaves are held by something else than an earlier call of theirs."""
import gc

import pytest
import torch

from fluidnet_amd.models.block_norm import gated_residual

pytestmark = pytest.mark.gpu


def _setup():
    g = torch.Generator().manual_seed(1)
    w, b = (torch.rand(264, generator=g).cuda().requires_grad_() for _ in range(2))
    return w, b, torch.randn(40, 264, generator=g).cuda(), torch.ones(40, 264, device="cuda")


def _held(how, w, b):
    if how == "another operation's graph":
        return (w * 2).sum() + b.exp().sum()
    if how == "one leaf only":
        return b.exp()
    if how == "the node itself":
        return torch.autograd.graph.get_gradient_edge(w).node, torch.autograd.graph.get_gradient_edge(b).node
    return gated_residual(torch.zeros(2, 264, device="cuda"), torch.ones(2, 264, device="cuda"), post_weight=w[:], pre_weight=b)


@pytest.mark.parametrize("how", ["another operation's graph", "one leaf only", "the node itself", "a view's graph"])
def test_a_leaf_that_is_held_on_the_default_stream(how):
    """Refused before torch orders a gradient after the default stream; without what held it, captured and replayed."""
    w, b, x, up = _setup()
    once = lambda: gated_residual(x, x, post_weight=w, pre_weight=b)[1]  # noqa: E731
    want = torch.autograd.grad(once(), [w, b], up)
    held = _held(how, w, b)
    torch.cuda.synchronize()
    for backward in (lambda h: h.backward(up), lambda h: torch.autograd.grad(h, [w, b], up)):
        with pytest.raises(RuntimeError, match="are alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                backward(once())
        torch.cuda.synchronize()
    assert w.grad is None and b.grad is None
    del held
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(once(), [w, b], up)
    for k in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), k


def test_leaves_that_are_not_asked_for_may_be_held():
    """Only b's gradient is handed out: whoever holds w is not in the way."""
    w, b, x, up = _setup()
    once = lambda: gated_residual(x, x, post_weight=w, pre_weight=b)[1]  # noqa: E731
    want, = torch.autograd.grad(once(), [b], up)
    held = (w * 2).sum()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(once(), [b], up)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert held.requires_grad
