"""Refusals of gradient clipping and of the Adam step over a list of parameters, in Python and at the C entry points; none reaches the GPU."""
import ctypes
import math
import struct

import numpy as np
import pytest
import torch

from fluidnet_amd.engine import runtime as rt
from fluidnet_amd.training.grad_clip import _STRIDED, _collapsed, clip_grad_norm_, clip_grads_with_norm_, total_grad_norm
from fluidnet_amd.training.optim import _ADAM, ClipAdam, clip_adam_


def _param(grad=True):
    p = torch.nn.Parameter(torch.ones(4))
    if grad:
        p.grad = torch.ones(4)
    return p


def test_nothing_to_clip():
    for got in (clip_grad_norm_([], 1.0), clip_grad_norm_([_param(False)], 1.0), total_grad_norm([])):
        assert float(got) == 0.0 and got.shape == ()
    clip_grads_with_norm_([], 1.0, torch.ones(()))


@pytest.mark.parametrize("error,match,call", [
    (RuntimeError, "no CPU fallback", lambda: clip_grad_norm_([_param()], 1.0)),
    (RuntimeError, "no CPU fallback", lambda: total_grad_norm(torch.ones(3))),
    (RuntimeError, "no CPU fallback", lambda: clip_grads_with_norm_(_param(), 1.0, torch.ones(()))),
    (RuntimeError, "no CPU fallback", lambda: ClipAdam([_param()], 1e-3).step()),
    (NotImplementedError, "norm_type", lambda: clip_grad_norm_([_param()], 1.0, norm_type=3)),
    (ValueError, "max_norm", lambda: clip_grad_norm_([_param()], -1.0)),
    (ValueError, "max_norm", lambda: clip_grad_norm_([_param()], float("nan"))),
    (ValueError, "no parameters", lambda: ClipAdam([], 1e-3)),
    (ValueError, "twice", lambda: ClipAdam([_param()] * 2, 1e-3)),
    (TypeError, "groups", lambda: ClipAdam([{"params": [_param()]}], 1e-3)),
    (ValueError, "equally long", lambda: clip_adam_([], [], [], [], torch.zeros(3), lr=1.0)),
    (ValueError, "equally long", lambda: clip_adam_([_param()], [], [], [], torch.zeros(3), lr=1.0)),
    (ValueError, "betas", lambda: clip_adam_(*[[_param()]] * 4, torch.zeros(3), lr=1.0, betas=(1.0, 0.9))),
    (ValueError, "betas", lambda: clip_adam_(*[[_param()]] * 4, torch.zeros(3), lr=1.0, weight_decay=-1)),
])
def test_python_refuses(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_collapsed_layouts():
    t = torch.zeros(4, 6, 5)
    assert _collapsed(t) == [[1, 120]]
    assert _collapsed(t.permute(2, 0, 1)) == [[1, 120]]
    assert _collapsed(t[:, 1:4]) == [[30, 4], [1, 15]]
    assert _collapsed(t[..., ::2]) == [[5, 24], [2, 3]]
    assert _collapsed(t[:1].expand(3, 6, 5)) is None
    assert _collapsed(torch.zeros(10).as_strided((4, 4), (2, 1))) is None          # rows that overlap
    assert _collapsed(torch.zeros(())) == [] and _collapsed(torch.zeros(1, 1)) == []


class _Host:
    def __init__(self, ptrs=(256, 4096), numels=(8, 8), dtypes=(0, 0)):
        self.a = (np.array(ptrs, "u8"), np.array(numels, "i8"), np.array(dtypes, "i4"))

    def args(self):
        return (len(self.a[0]), *(x.ctypes.data for x in self.a))


def _norm(h, *, strided=b"", kind=0, ws=64, cap=4096, out=True):
    n = ctypes.c_int32()
    buf = ctypes.cast(ctypes.c_char_p(strided), ctypes.c_void_p) if strided else None
    return rt.lib().fnet_list_norm_partials(*h.args(), len(strided) // 112, buf, kind, ws, cap, ctypes.byref(n) if out else None, None, 0.9, 0.9, None)


def test_c_norm_refuses():
    for h in (_Host(dtypes=(0, 3)), _Host(dtypes=(-1, 0)), _Host(numels=(8, -1)), _Host(ptrs=(0, 4096)), _Host(ptrs=(257, 4096), dtypes=(1, 0)),
              _Host(ptrs=(258, 4096))):
        assert _norm(h) == -1
    h = _Host()
    assert _norm(h, kind=3) == -1 and _norm(h, kind=-1) == -1 and _norm(h, ws=None) == -1 and _norm(h, out=False) == -1
    assert _norm(h, cap=1) == -1                                 # two launches' worth of blocks do not fit
    for bad in ((0, 0, 1), (64, 5, 1), (64, 0, 0), (64, 0, 7), (66, 0, 1)):
        assert _norm(h, strided=_STRIDED.pack(*bad, 4, 0, 0, 0, 0, 0, 2, 0, 0, 0, 0, 0)) == -1
    assert _norm(h, strided=_STRIDED.pack(64, 0, 1, 0, 0, 0, 0, 0, 0, 2, 0, 0, 0, 0, 0)) == -1      # no elements
    assert _norm(h, strided=_STRIDED.pack(64, 0, 1, 4, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)) == -1      # stride 0
    L = rt.lib()
    assert L.fnet_list_norm_finish(None, 1, 0, 64, None) == -1 and L.fnet_list_norm_finish(64, 1, 3, 64, None) == -1 and L.fnet_list_norm_finish(64, -1, 0, 64, None) == -1
    assert L.fnet_list_clock(None, 0.9, 0.9, None) == -1


def test_c_scale_refuses():
    scale = lambda h, part=64, n=1, kind=0, norm=None, most=1.0: rt.lib().fnet_list_scale(*h.args(), 0, None, part, n, kind, norm, most, None, None)  # noqa: E731
    assert scale(_Host(), part=None) == -1 and scale(_Host(), norm=64) == -1 and scale(_Host(), most=-1.0) == -1
    assert scale(_Host(), most=math.nan) == -1 and scale(_Host(), n=-1) == -1 and scale(_Host(), kind=3) == -1
    for ptrs, numels in (((256, 256), (8, 8)), ((256, 284), (8, 8)), ((4096, 4080), (8, 8)), ((512, 4096, 540), (8, 8, 8))):
        h = _Host(ptrs=ptrs, numels=numels, dtypes=[0] * len(ptrs))
        assert scale(h) == -5, ptrs
        assert "share memory" in rt.lib().fnet_strerror(-5).decode()


def test_c_adam_refuses():
    def adam(p=(0x1000, 0x2000), g=(0x3000, 0x4000), m=(0x5000, 0x6000), v=(0x7000, 0x8000), w=(0, 0), numel=(8, 8), dtype=(0, 0), lr=1.0, b1=0.9,
             b2=0.9, eps=1e-8, wd=0.0, most=1.0, part=64, clock=64, n=1):
        a = [np.array(x, "u8") for x in (p, g, m, v, w)]
        d = np.array(numel, "i8"), np.array(dtype, "i4")
        h = _ADAM.pack(lr, b1, b2, eps, wd, most, part, clock, 0, 0, n)
        return rt.lib().fnet_list_adam(len(p), *(x.ctypes.data for x in a), *(x.ctypes.data for x in d), h, None)
    assert struct.calcsize("=6d4Qi4x") == _ADAM.size == 88
    for over in (dict(p=(0, 0x2000)), dict(g=(0, 0x4000)), dict(m=(0, 0x6000)), dict(v=(0x7002, 0x8000)), dict(dtype=(1, 0)), dict(dtype=(4, 0)),
                 dict(numel=(-1, 8)), dict(lr=math.inf), dict(lr=math.nan), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(wd=math.inf),
                 dict(most=math.nan), dict(part=0), dict(clock=0), dict(n=-1), dict(p=(0x1002, 0x2000))):
        assert adam(**over) == -1, over
    for over in (dict(p=(0x1000, 0x1010)), dict(m=(0x5000, 0x5000)), dict(v=(0x5004, 0x8000)), dict(dtype=(1, 1), w=(0x1000, 0x9000))):
        assert adam(**over) == -5, over
    # a gradient is read while other blocks write, so it may lie in nothing that is written
    for over in (dict(g=(0x5000, 0x4000)), dict(g=(0x3000, 0x1ffc)), dict(g=(0x101c, 0x4000), most=-1.0), dict(g=(0x701c, 0x4000)),
                 dict(dtype=(1, 1), w=(0xa000, 0x9000), g=(0x901e, 0x4000))):
        assert adam(**over) == -5, over
