"""ClipAdam's state: parameters without elements, a module that was moved to another device, states of other parameters.  On the CPU, where the
parameters only say that they lie on a GPU."""
import pytest
import torch

from fluidnet_amd.engine import runtime as rt
from fluidnet_amd.training.optim import ClipAdam


class _Says(torch.nn.Parameter):
    """A parameter in host memory that calls itself a GPU's."""
    is_cuda = True


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def _params(*shapes, dtype=torch.float32):
    return [_Says(torch.arange(float(torch.Size(s).numel())).reshape(s).to(dtype)) for s in shapes]


@pytest.mark.parametrize("shape", [(5, 0), (0, 5), (0,), (0, 0), (3, 0, 2), (2, 3, 0), (1, 0)], ids=str)
def test_parameters_of_no_elements(host, shape):
    opt = ClipAdam(_params((4,), shape), 1e-3)
    opt._init_state()
    assert opt._m[1].shape == shape and opt.step_count == 0


def test_parameters_that_are_not_dense_are_refused(host):
    for view in (torch.zeros(4, 6)[:, ::2], torch.zeros(1, 4).expand(3, 4)):
        p = _Says(view)
        assert p.stride() == view.stride()
        with pytest.raises(ValueError, match="must be dense"):
            ClipAdam([p], 1e-3)._init_state()


def test_state_follows_a_module_to_another_device(host, monkeypatch):
    params = _params((3, 2), (4,), dtype=torch.bfloat16)
    opt = ClipAdam(params, 1e-3, betas=(0.8, 0.9))
    opt._init_state()
    for k in range(2):
        opt._m[k].fill_(0.25 + k)
        opt._v[k].fill_(0.5 + k)
        opt._w[k].mul_(1 + 1e-4)           # still rounds to its parameter
    opt._clock.copy_(torch.tensor([3.0, 0.8 ** 3, 0.9 ** 3], dtype=torch.float64))
    opt.param_groups[0]["lr"] = 7e-4
    opt.push_lr()
    kept = {n: [t.clone() for t in getattr(opt, n)] for n in ("_m", "_v", "_w")}
    # the clock claims to lie on another device than the parameters, as it does after a move; the move itself would need two GPUs
    class Elsewhere(torch.Tensor):
        device = torch.device("meta")
    opt._clock = opt._clock.as_subclass(Elsewhere)
    opt._init_state()
    assert type(opt._clock) is torch.Tensor and opt._clock.device == params[0].device
    for n, ts in kept.items():
        assert all(torch.equal(a, b) for a, b in zip(getattr(opt, n), ts)), n
    assert opt.step_count == 3 and opt._clock.tolist() == [3.0, 0.8 ** 3, 0.9 ** 3] and float(opt._lr) == 7e-4


def _state(opt):
    return [t.clone() for ts in (opt._m, opt._v, opt._w) for t in ts if t is not None] + [opt._clock.clone(), opt._lr.clone()]


@pytest.mark.parametrize("wrong", [
    lambda sd: sd["exp_avg"].__setitem__(0, torch.ones(1, 2)),                    # would be broadcast over the rows
    lambda sd: sd["exp_avg_sq"].__setitem__(1, torch.ones(())),                   # would be broadcast over everything
    lambda sd: sd["exp_avg"].__setitem__(1, torch.ones(5)),
    lambda sd: sd["master"].__setitem__(0, torch.ones(2)),
    lambda sd: sd["exp_avg_sq"].pop(),
    lambda sd: sd["master"].pop(),
    lambda sd: sd["exp_avg"].append(torch.ones(4)),
])
def test_states_of_other_parameters_are_refused(host, wrong):
    """Before anything of the optimizer's own is written."""
    opt = ClipAdam(_params((3, 2), (4,), dtype=torch.bfloat16), 1e-3)
    opt._init_state()
    before, sd = _state(opt), opt.state_dict()
    sd["step"], sd["lr"] = 9, 5e-2
    wrong(sd)
    with pytest.raises(ValueError, match="parameter"):
        opt.load_state_dict(sd)
    assert opt.step_count == 0 and opt.param_groups[0]["lr"] == 1e-3
    assert all(torch.equal(a, b) for a, b in zip(before, _state(opt)))


def test_a_state_loads_into_other_types_and_layouts(host):
    """fp32 parameters take the moments of bf16 ones and ignore their masters; the other way round the master is the parameter."""
    a, b = ClipAdam(_params((3, 2), dtype=torch.bfloat16), 1e-3), ClipAdam(_params((3, 2)), 1e-3)
    for opt in (a, b):
        opt._init_state()
    a._m[0].fill_(0.5)
    b.load_state_dict(a.state_dict())
    assert torch.equal(b._m[0], a._m[0]) and b._w == [None]
    b._m[0].fill_(0.25)
    a.load_state_dict(b.state_dict())
    assert torch.equal(a._m[0], b._m[0]) and torch.equal(a._w[0], a.params[0].detach().float())
