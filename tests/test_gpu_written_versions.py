"""Autograd is told of everything that the list operators write in place: a value that a graph has kept and that was written since raises."""
import pytest
import torch

from fluidnet_amd.training.grad_clip import clip_grad_norm_, clip_grads_with_norm_
from fluidnet_amd.training.optim import ClipAdam, clip_adam_

pytestmark = pytest.mark.gpu


def _lists(dtype):
    p, g, m, v = ([torch.full((n,), x, device="cuda", dtype=t) for n in (3, 5, 0)] for x, t in ((1.0, dtype), (0.5, dtype), (0.1, torch.float32), (0.2, torch.float32)))
    return p, g, m, v, None if dtype is torch.float32 else [t.float() for t in p]


@pytest.mark.parametrize("max_norm", [None, 0.1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_versions_after_a_step(dtype, max_norm):
    p, g, m, v, w = _lists(dtype)
    clock = torch.tensor([0.0, 1.0, 1.0], dtype=torch.float64, device="cuda")
    written = [*p, *m, *v, *(w or []), clock]
    before, grads = [t._version for t in written], [t._version for t in g]
    clip_adam_(p, g, m, v, clock, masters=w, lr=1e-3, max_norm=max_norm)
    assert all(t._version > k for t, k in zip(written, before))
    assert [t._version for t in g] == grads                          # only read


def test_masters_of_fp32_parameters_are_not_written():
    p, g, m, v, _ = _lists(torch.float32)
    w = [t.clone() for t in p]
    clip_adam_(p, g, m, v, torch.tensor([0.0, 1.0, 1.0], dtype=torch.float64, device="cuda"), masters=w, lr=1e-3)
    assert all(t._version == 0 and (t == 1).all() for t in w)


@pytest.mark.parametrize("which", ["params", "exp_avg", "exp_avg_sq", "master", "clock"])
def test_a_graph_that_kept_the_old_value_raises(which):
    p, g, m, v, w = _lists(torch.bfloat16)
    clock = torch.tensor([0.0, 1.0, 1.0], dtype=torch.float64, device="cuda")
    kept = {"params": p[0], "exp_avg": m[0], "exp_avg_sq": v[0], "master": w[0], "clock": clock}[which]
    x = torch.ones(3, device="cuda", requires_grad=True)
    loss = (x * kept).sum()
    clip_adam_(p, g, m, v, clock, masters=w, lr=1e-3)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_clipped_gradients():
    for clip in (lambda ps: clip_grad_norm_(ps, 0.1), lambda ps: clip_grad_norm_(ps, 0.1, error_if_nonfinite=True),
                 lambda ps: clip_grads_with_norm_(ps, 0.1, torch.ones((), device="cuda"))):
        ps = [torch.nn.Parameter(torch.zeros(4, 3, device="cuda", dtype=t)) for t in (torch.float32, torch.float16)]
        wide = torch.ones(4, 9, device="cuda")
        ps[0].grad, ps[1].grad = wide[:, 2:5], torch.ones(4, 3, device="cuda", dtype=torch.float16)
        before = [q.grad._version for q in ps]
        clip(ps)
        assert all(q.grad._version > k for q, k in zip(ps, before)) and wide._version > 0


def test_a_parameter_that_only_the_step_wrote_keeps_its_master():
    p = torch.nn.Parameter(torch.full((16,), 3.0, device="cuda", dtype=torch.bfloat16))
    opt = ClipAdam([p], 1e-4, max_norm=None)
    for _ in range(3):
        p.grad = torch.ones_like(p)
        opt.step()
    assert (opt._w[0] < 3.0 - 2e-4).all() and (p == 3.0).all()        # three steps of 1e-4, below half a step of bf16 at 3
