"""ClipAdam.step on what ClipAdam's state has to carry over: parameters without elements, states saved and loaded."""
import pytest
import torch

from fluidnet_amd.training.optim import ClipAdam

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_parameters_of_no_elements(dtype):
    """A layer of no inputs next to others: its bias is stepped, its weight has nothing to step; the others step as without it."""
    make = lambda: [torch.nn.Parameter(torch.ones(s, device="cuda", dtype=dtype)) for s in ((7,), (3, 0), (0, 3), (0, 0))]  # noqa: E731
    with_empty, alone = make(), make()[:1]
    for ps in (with_empty, alone):
        for p in ps:
            p.grad = torch.full_like(p, 0.5)
        opt = ClipAdam(ps, 1e-2, max_norm=0.3)
        opt.step()
        assert abs(float(opt.grad_norm) - 0.5 * 7 ** 0.5) < 1e-6
    assert torch.equal(with_empty[0], alone[0]) and not torch.equal(alone[0], torch.ones_like(alone[0]))
    only = make()[1:]
    for p in only:
        p.grad = torch.zeros_like(p)
    opt = ClipAdam(only, 1e-2, max_norm=0.3)
    opt.step()
    assert float(opt.grad_norm) == 0.0 and opt.step_count == 1


def test_a_loaded_state_goes_on():
    """Saved after three steps and loaded into a new optimizer of the same parameters, the next step is the same, bit for bit."""
    g = torch.Generator().manual_seed(3)
    start = [torch.randn(s, generator=g) for s in ((9, 4), (130,), (2, 0))]
    grads = [[torch.randn(p.shape, generator=g) for p in start] for _ in range(4)]
    ends = []
    for again in (False, True):
        ps = [torch.nn.Parameter(p.cuda().bfloat16()) for p in start]
        opt = ClipAdam(ps, 1e-2, max_norm=1.0)
        for k, gs in enumerate(grads):
            for p, v in zip(ps, gs):
                p.grad = v.cuda().bfloat16()
            if again and k == 3:
                sd, opt = opt.state_dict(), ClipAdam(ps, 1e-2, max_norm=1.0)
                opt.load_state_dict(sd)
            opt.step()
        ends.append([*(p.detach() for p in ps), *opt._m, *opt._v, *opt._w])
    assert all(torch.equal(a, b) for a, b in zip(*ends))
    with pytest.raises(ValueError, match="shape"):
        ClipAdam([torch.nn.Parameter(torch.zeros(9, 1, device="cuda")), *ps[1:]], 1e-2).load_state_dict(sd)
