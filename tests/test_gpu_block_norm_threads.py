"""One graph of the block norms, several threads."""
import threading

import pytest
import torch

from fluidnet_amd.models.block_norm import gated_residual

pytestmark = pytest.mark.gpu


def _graph():
    g = torch.Generator().manual_seed(2)
    leaves = [torch.randn(s, generator=g).cuda().requires_grad_() for s in ((40, 96), (40, 96), (40, 1), (96,), (96,))]
    x, branch, gate, w1, w2 = leaves
    return leaves, gated_residual(x, branch, gate, post_weight=w1, pre_weight=w2, kind="layer", gate_act="sigmoid"), torch.randn(40, 96, generator=g).cuda()


def _threads(n, work):
    """What work(k) returned or raised on each of n threads that start together."""
    got, start = [None] * n, threading.Barrier(n)

    def run(k):
        start.wait()
        try:
            got[k] = work(k)
        except RuntimeError as e:
            got[k] = e
    ts = [threading.Thread(target=run, args=(k,)) for k in range(n)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
    assert not any(t.is_alive() for t in ts)
    return got


def test_backward_passes_at_once():
    leaves, (y, h), up = _graph()
    want = torch.autograd.grad([y, h], leaves, [up, up], retain_graph=True)
    torch.cuda.synchronize()
    for got in _threads(4, lambda k: [torch.autograd.grad([y, h], leaves, [up, up], retain_graph=True) for _ in range(25)]):
        assert not isinstance(got, Exception), got
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for grads in got for a, b in zip(grads, want))


def test_a_pass_that_releases_next_to_others():
    """Each pass gives the gradients or says that they are used up; the hooks of saved tensors run inside as well."""
    for hooks in (False, True):
        for _ in range(10):
            if hooks:
                with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):
                    leaves, (y, h), up = _graph()
            else:
                leaves, (y, h), up = _graph()
            want = torch.autograd.grad([y, h], leaves, [up, up], retain_graph=True)
            torch.cuda.synchronize()
            got = _threads(3, lambda k: torch.autograd.grad([y, h], leaves, [up, up]))
            torch.cuda.synchronize()
            assert sum(not isinstance(r, Exception) for r in got) >= 1
            for r in got:
                if isinstance(r, Exception):
                    assert "second time" in str(r)
                else:
                    assert all(torch.equal(a, b) for a, b in zip(r, want))
