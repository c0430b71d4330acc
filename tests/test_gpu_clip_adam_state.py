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
