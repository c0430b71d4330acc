"""Calls of the list operators' C entries that Python never makes."""
import ctypes
import math

import numpy as np
import pytest
import torch

from fluidnet_amd.engine import runtime as rt
from fluidnet_amd.training.grad_clip import _STRIDED

pytestmark = pytest.mark.gpu
NORM_2, NORM_1, NORM_INF = 0, 1, 2


def _scale(tensors, out, *, partials=None, kind=NORM_2, norm=None, max_norm=1.0, strided=b""):
    a = np.array([t.data_ptr() for t in tensors], "u8"), np.array([t.numel() for t in tensors], "i8"), np.zeros(len(tensors), "i4")
    buf = ctypes.cast(ctypes.c_char_p(strided), ctypes.c_void_p) if strided else None
    rc = rt.lib().fnet_list_scale(len(tensors), *(x.ctypes.data for x in a), len(strided) // 112, buf, partials.data_ptr() if partials is not None else None,
                                  0 if partials is None else partials.numel(), kind, norm.data_ptr() if norm is not None else None, max_norm,
                                  out.data_ptr() if out is not None else None, rt.raw_stream(0))
    torch.cuda.synchronize()
    return rc


@pytest.mark.parametrize("tensors", [0, 1, 3])
def test_the_norm_of_a_list_of_nothing_is_stored(tensors):
    """Partial sums of other tensors (of other ranks, say), and nothing to scale here: the norm is stored all the same."""
    empty = [torch.zeros(0, device="cuda") for _ in range(tensors)]
    sums = torch.tensor([4.0, 5.0, 7.0], dtype=torch.float64, device="cuda")
    for kind, want in ((NORM_2, 4.0), (NORM_1, 16.0), (NORM_INF, 7.0)):
        out = torch.full((2,), -3.0, device="cuda")
        assert _scale(empty, out, partials=sums, kind=kind) == 0
        assert out.tolist() == [want, -3.0]
    out = torch.full((2,), -3.0, device="cuda")
    assert _scale(empty, out, norm=torch.tensor(2.5, device="cuda")) == 0
    assert out.tolist() == [2.5, -3.0]
    assert _scale(empty, None, norm=torch.tensor(2.5, device="cuda")) == 0


def test_the_norm_is_stored_once_with_something_to_scale():
    for dense, strided in ((True, False), (False, True), (True, True)):
        t, wide, out = torch.full((6,), 3.0, device="cuda"), torch.full((4, 5), 3.0, device="cuda"), torch.full((2,), -3.0, device="cuda")
        rec = _STRIDED.pack(wide.data_ptr(), 0, 2, 4, 2, 0, 0, 0, 0, 5, 1, 0, 0, 0, 0) if strided else b""
        assert _scale([t] if dense else [], out, norm=torch.tensor(2.0, device="cuda"), strided=rec) == 0
        assert out.tolist() == [2.0, -3.0]
        coef = 1 / (2.0 + 1e-6)
        assert math.isclose(t[0].item(), 3 * coef if dense else 3.0, rel_tol=2.0 ** -22)
        assert math.isclose(wide[3, 1].item(), 3 * coef if strided else 3.0, rel_tol=2.0 ** -22) and (wide[:, 2:] == 3.0).all()
