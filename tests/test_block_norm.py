"""Refusals of the norms around a residual block, in Python and at the C entry points; none of them reaches the GPU."""
import ctypes
import struct

import pytest
import torch

from fluidnet_amd.engine import runtime as rt
from fluidnet_amd.models.block_norm import gated_residual, pre_norm

X = torch.zeros(2, 3, 8)
_ARGS = struct.Struct("=7q8i2f22Qq")             # struct FnetBlockNorm (include/fluidnet_hip.h)


@pytest.mark.parametrize("match,call", [
    ("no CPU fallback", lambda: pre_norm(X)),
    ("no CPU fallback", lambda: gated_residual(X, X, torch.zeros(2, 1, 8))),
    ("float32, bfloat16 or float16", lambda: pre_norm(X.double())),
    ("last axis", lambda: pre_norm(torch.zeros(3, 0))),
    ("last axis", lambda: pre_norm(torch.zeros(()))),
    ("last axis", lambda: pre_norm(torch.zeros(1, 16385))),
    ("kind", lambda: pre_norm(X, kind="batch")),
    ("gate_act", lambda: gated_residual(X, X, gate_act="relu")),
    ("eps", lambda: pre_norm(X, eps=-1.0)),
    ("eps", lambda: pre_norm(X, eps=float("nan"))),
    ("branch must be like x", lambda: gated_residual(X, X[:1])),
    ("branch must be like x", lambda: gated_residual(X, X.half())),
    ("needs a branch", lambda: gated_residual(X, None)),
    ("post=True", lambda: gated_residual(X, X, post=False, post_weight=torch.ones(8))),
    ("pre=True", lambda: gated_residual(X, X, pre=False, pre_bias=torch.ones(8))),
    ("shape", lambda: pre_norm(X, torch.ones(7))),
    ("must be float32 or", lambda: pre_norm(X, torch.ones(8).half())),
    ("one type", lambda: gated_residual(X.half(), X.half(), post_weight=torch.ones(8), pre_weight=torch.ones(8).half())),
    ("gate of shape", lambda: gated_residual(X, X, torch.ones(3, 8))),
    ("gate of shape", lambda: gated_residual(X, X, torch.ones(1))),
    ("gate of shape", lambda: gated_residual(X, X, torch.ones(1, 3, 8))),
    ("gate must be", lambda: gated_residual(X, X, torch.ones(8).double())),
])
def test_python_refuses(match, call):
    with pytest.raises((ValueError, RuntimeError), match=match):
        call()


BASE = dict(rows=4, tokens=2, xs=8, bs=8, gs=8, dys=8, dhs=8, width=8, dtype=1, pdt=0, gdt=1, kind=0, post=1, gk=0, ga=0, a=1.0, eps=1e-6, x=64,
            branch=64, gate=0, scale=0, pw=64, pb=0, nw=64, nb=0, y=64, h=64, stats=64, dy=64, dh=64, dx=64, db=64, dg=0, ds=0, dpw=64, dpb=0,
            dnw=64, dnb=0, ws=0, wsn=0)


def _pack(**over):
    return _ARGS.pack(*{**BASE, **over}.values())


@pytest.mark.parametrize("over", [
    dict(dtype=3), dict(dtype=-1), dict(pdt=2), dict(gdt=2), dict(width=0), dict(width=16385), dict(rows=-1), dict(rows=1 << 31), dict(kind=2),
    dict(eps=-1.0), dict(eps=float("nan")), dict(gk=5, gate=64), dict(gk=1), dict(gate=64), dict(gk=3, gate=64, tokens=3), dict(gk=3, gate=64, tokens=0),
    dict(ga=3), dict(branch=0), dict(post=0), dict(x=0), dict(x=63), dict(xs=-1), dict(pw=62), dict(stats=2), dict(a=float("nan")),
])
def test_c_entry_refuses(over):
    L = rt.lib()
    assert L.fnet_block_norm_fwd(_pack(**over), None) == -1
    assert L.fnet_block_norm_bwd(_pack(**over), None) == -1
    n = ctypes.c_int64(7)
    assert L.fnet_block_norm_workspace(_pack(**over), ctypes.byref(n)) == -1


def test_c_entry_refuses_by_direction():
    L = rt.lib()
    for over in (dict(y=0), dict(h=0), dict(branch=0, pw=0, post=0, y=64), dict(y=63)):
        assert L.fnet_block_norm_fwd(_pack(**over), None) == -1, over
    for over in (dict(stats=0), dict(dh=0), dict(dg=64), dict(dx=63), dict(dpw=62), dict(post=0, pw=0), dict(ws=0)):
        assert L.fnet_block_norm_bwd(_pack(**{"rows": 4096, "tokens": 2, **over}), None) == -1, over
    n = ctypes.c_int64()
    assert L.fnet_block_norm_workspace(_pack(rows=4096), ctypes.byref(n)) == 0 and n.value > 0
    assert L.fnet_block_norm_bwd(_pack(rows=4096, ws=64, wsn=n.value - 1), None) == -1
    assert L.fnet_block_norm_bwd(_pack(rows=4096, ws=72, wsn=n.value), None) == -1
    assert L.fnet_block_norm_workspace(_pack(rows=0), ctypes.byref(n)) == 0 and n.value == 0
    assert L.fnet_block_norm_workspace(_pack(), None) == -1 and L.fnet_block_norm_fwd(None, None) == -1
