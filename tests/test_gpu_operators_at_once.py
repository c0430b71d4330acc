"""The block norms and the list operators at once on several streams, eagerly and as replayed graphs, and at the largest counts of rows and samples."""
import pytest
import torch

from fluidnet_amd.models.block_norm import gated_residual, pre_norm
from fluidnet_amd.training.grad_clip import clip_grad_norm_
from fluidnet_amd.training.optim import ClipAdam

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _network(seed, dtype):
    """Parameters and one training step: a residual block with its norms, clipping apart and inside of Adam."""
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).cuda().to(dtype)) for s in ((160, 160), (160,), (160,), (3, 0))]
    x = torch.randn(30, 7, 160, generator=g).cuda().to(dtype)
    gate = torch.randn(30, 1, 160, generator=g).cuda().to(dtype)
    up = [torch.randn(30, 7, 160, generator=g).cuda().to(dtype) for _ in range(2)]
    opt = ClipAdam(ps, 1e-2, max_norm=0.5)

    def step():
        y, h = gated_residual(x, x @ ps[0], gate, post_weight=ps[1], pre_weight=ps[2], kind="layer", gate_act="sigmoid")
        grads = torch.autograd.grad([y, h], ps[:3], up)
        for p, v in zip(ps, grads):
            p.grad = v
        ps[3].grad = torch.zeros_like(ps[3])
        clip_grad_norm_(ps, 1.0)
        opt.step()
        return [p.detach().clone() for p in ps]
    return ps, opt, step


def test_training_steps_on_two_streams():
    want = []
    for seed, dtype in ((1, torch.float32), (2, BF16)):
        step = _network(seed, dtype)[2]
        want.append([step() for _ in range(6)])
    torch.cuda.synchronize()
    steps = [_network(1, torch.float32)[2], _network(2, BF16)[2]]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(steps[k]())
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for s, t in zip(a, b) for p, q in zip(s, t))


def test_graphs_replayed_on_two_streams():
    """Two captured steps (forward, backward, clipping, Adam), each with workspaces of its own, replayed at once next to eager work."""
    runs = []
    for seed, dtype in ((1, torch.float32), (2, BF16)):
        ps, opt, step = _network(seed, dtype)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        runs.append((ps, opt, graph, step))             # step holds the inputs that the graph reads
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    eager = _network(3, BF16)[2]
    for _ in range(5):
        for s, (_, _, graph, _) in zip(streams, runs):
            with torch.cuda.stream(s):
                graph.replay()
        eager()
    torch.cuda.synchronize()
    for (ps, opt, _, _), (seed, dtype) in zip(runs, ((1, torch.float32), (2, BF16))):
        step = _network(seed, dtype)[2]
        for _ in range(6):
            want = step()
        assert all(torch.equal(p, q) for p, q in zip(ps, want)) and opt.step_count == 6


def _tail(t, n):
    return t.reshape(-1, *t.shape[1:])[-n:].clone()


def test_the_most_rows():
    """2^31 - 1 rows of one element: the last ones as if they were alone."""
    rows, last = (1 << 31) - 1, 64
    tail = torch.randn(last, 1, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    x = torch.full((rows, 1), 0.5, dtype=BF16, device="cuda")
    x[-last:] = tail
    w, up = torch.full((1,), 0.75, device="cuda"), torch.full((1, 1), 0.25, dtype=BF16, device="cuda")

    def run(x):
        x = x.detach().requires_grad_()
        h = pre_norm(x, w, eps=0.1)
        return _tail(h.detach(), last), _tail(torch.autograd.grad(h, x, up.expand(x.shape))[0], last)
    for a, b in zip(run(x), run(tail)):
        assert torch.equal(a, b)
    del x
    torch.cuda.empty_cache()


def test_the_most_samples():
    """2^30 - 1 samples of two rows of one element, each with its gate: the last ones as if they were alone, and the weights' sums (of 1/2
    and 1 times powers of two: the last samples' gates are 2, the others 1) as exact as partial sums of 2^20 are."""
    n, last = (1 << 30) - 1, 64
    x = torch.ones(n, 2, 1, dtype=BF16, device="cuda")
    gate = torch.ones(n, 1, 1, dtype=BF16, device="cuda")
    gate[-last:] = 2.0
    x[-last:, 1] = -0.5
    up = torch.ones((1, 1, 1), dtype=BF16, device="cuda")

    def run(x, gate):
        branch, gate, scale = x.detach().requires_grad_(), gate.detach().requires_grad_(), torch.ones(1, device="cuda", requires_grad=True)
        y, _ = gated_residual(x, branch, gate, scale, post=False, pre=False)
        d_branch, d_gate, d_scale = torch.autograd.grad(y, [branch, gate, scale], up.expand(x.shape))
        return _tail(y.detach(), last), _tail(d_branch, last), _tail(d_gate, last), d_scale
    (*got, scale), (*want, _) = run(x, gate), run(_tail(x, last), _tail(gate, last))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    total = 2.0 * (n - last) + last * 2 * (1 - 0.5)
    assert abs(float(scale) - total) <= 1e-4 * total
    del x, gate
    torch.cuda.empty_cache()
