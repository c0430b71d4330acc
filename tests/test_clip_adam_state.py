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
