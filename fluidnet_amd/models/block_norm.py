"""Norms around a residual block, with its gate and residual scale, on the HIP kernels of libfluidnet_hip (fnet_block_norm_*).

The reference's blocks normalise each channel over the pixels (ml/models/unet.py:17-28, 42-80) and add the residual as it is.  Here the
norm runs over the LAST axis (the channels of a token, or of a pixel of a channels-last image), and what surrounds a block

    h = pre_norm(x)                                   before the first block
    x, h = gated_residual(x, block(h), gate, scale)   after every block: the residual sum and the norm before the next block

is one kernel forward and one (plus a small sum over rows) backward:

    u = N(branch) * post_weight + post_bias           (post=False: u = branch)
    y = x + residual_scale * scale * act(gate) * u
    h = N(y) * pre_weight + pre_bias                  (pre=False: not computed)

with N(v) = v / sqrt(mean v^2 + eps) (kind="rms") or (v - mean) / sqrt(var + eps) (kind="layer").  h is the norm of y before y is rounded to
its type, statistics and sums are 32-bit, and every sum over rows has a fixed order: the same call gives the same bits.

x and branch: [..., C], fp32, bf16 or fp16, 1 <= C <= 16384, any number of rows (none included).  The last axis is dense and the rows evenly
spaced, or the operand is copied first; slices of the last axis are taken as they are.  Weights, biases and scale: [C], all of them in fp32 or
all in x's type.  gate, in fp32 or x's type: like x (a value per element), [..., 1] (per token), [B, 1, .., 1, C] for x [B, .., C] (per sample)
or [C] (per channel); gate_act "identity", "sigmoid" or "tanh".  A NaN or infinity stays in its row (and in the sums over rows).
There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Literal, Optional, Tuple

import torch
import torch.nn as nn

from ..engine import runtime as rt
from ..engine.elements import ELEM

NormKind = Literal["rms", "layer"]
GateAct = Literal["identity", "sigmoid", "tanh"]

MAX_WIDTH = 16384
_KIND = {"rms": 0, "layer": 1}
_ACT = {"identity": 0, "sigmoid": 1, "tanh": 2}
_NONE, _ELEMENT, _TOKEN, _SAMPLE, _CHANNEL = range(5)
# struct FnetBlockNorm (include/fluidnet_hip.h)
_ARGS = struct.Struct("=7q8i2f22Qq")


class _Spec:
    """What a call is, apart from its tensors."""
    __slots__ = ("rows", "tokens", "width", "dtype", "param_dtype", "gate_dtype", "kind", "post", "pre", "gate_kind", "gate_act",
                 "residual_scale", "eps")


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The tensor (copied if its last axis is not dense or its rows are not evenly spaced) and its row stride."""
    if t.is_contiguous():
        return t, t.shape[-1]
    size, stride = t.shape, t.stride()
    if stride[-1] == 1 or size[-1] == 1:
        step, n = None, 1                     # distance of neighbouring rows, rows in the axes looked at so far
        for d in range(t.ndim - 2, -1, -1):
            if size[d] == 1:
                continue
            if step is None:
                step = stride[d]
            elif stride[d] != step * n:
                break
            n *= size[d]
        else:
            return t, (size[-1] if step is None else step)
    return t.contiguous(), size[-1]


def _param_type(name: str, t: Optional[torch.Tensor], C: int, x: torch.Tensor, seen):
    if t is None:
        return seen
    if t.shape != (C,) or t.device != x.device:
        raise ValueError(f"{name} must have shape ({C},) on {x.device} (got {tuple(t.shape)} on {t.device})")
    if t.dtype is not torch.float32 and t.dtype is not x.dtype:
        raise ValueError(f"{name} must be float32 or {x.dtype} (got {t.dtype})")
    if seen is not None and t.dtype is not seen:
        raise ValueError("weights, biases and scale must all have one type")
    return t.dtype


def _gate_kind(gate: torch.Tensor, x: torch.Tensor) -> int:
    g, s = gate.shape, x.shape
    if len(g) == 1 and g[0] == s[-1] and len(s) > 1:
        return _CHANNEL
    if g == s:
        return _ELEMENT
    if len(g) == len(s):
        if g[:-1] == s[:-1] and g[-1] == 1:
            return _TOKEN
        if g[-1] == s[-1]:
            if len(s) > 2 and g[0] == s[0] and all(n == 1 for n in g[1:-1]):
                return _SAMPLE
            if all(n == 1 for n in g[:-1]):
                return _CHANNEL
    raise ValueError(f"gate of shape {tuple(g)} for x of shape {tuple(s)}: expected x's shape, [..., 1], [B, 1, .., C] or [C]")


def _spec(x, branch, gate, scale, pw, pb, nw, nb, kind, post, pre, gate_act, residual_scale, eps) -> _Spec:
    code = ELEM.get(x.dtype)
    if code is None:
        raise ValueError(f"x must be float32, bfloat16 or float16 (got {x.dtype})")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"the last axis must have 1 to {MAX_WIDTH} elements (got shape {tuple(x.shape)})")
    if kind not in _KIND or gate_act not in _ACT:
        raise ValueError(f"kind must be one of {tuple(_KIND)} and gate_act one of {tuple(_ACT)} (got {kind!r}, {gate_act!r})")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    C = x.shape[-1]
    s = _Spec()
    s.width, s.dtype = C, code
    s.rows = x.numel() // C
    if s.rows >= 1 << 31:
        raise ValueError("at most 2^31 - 1 rows")
    s.tokens = s.rows // x.shape[0] if x.ndim > 1 and x.shape[0] else s.rows
    if branch is None:
        if gate is not None or scale is not None:
            raise ValueError("a gate or scale needs a branch")
        post = False
    else:
        if branch.shape != x.shape or branch.dtype is not x.dtype or branch.device != x.device:
            raise ValueError(f"branch must be like x: {tuple(x.shape)} {x.dtype} on {x.device} (got {tuple(branch.shape)} {branch.dtype} on {branch.device})")
    if not post and (pw is not None or pb is not None):
        raise ValueError("post_weight / post_bias need post=True")
    if not pre and (nw is not None or nb is not None):
        raise ValueError("pre_weight / pre_bias need pre=True")
    seen = None
    for name, t in (("scale", scale), ("post_weight", pw), ("post_bias", pb), ("pre_weight", nw), ("pre_bias", nb)):
        seen = _param_type(name, t, C, x, seen)
    s.param_dtype = 0 if seen is None else ELEM[seen]
    s.gate_kind, s.gate_dtype = _NONE, 0
    if gate is not None:
        if gate.device != x.device or (gate.dtype is not torch.float32 and gate.dtype is not x.dtype):
            raise ValueError(f"gate must be float32 or {x.dtype} on {x.device} (got {gate.dtype} on {gate.device})")
        s.gate_kind, s.gate_dtype = _gate_kind(gate, x), ELEM[gate.dtype]
    s.kind, s.post, s.pre, s.gate_act = _KIND[kind], bool(post), bool(pre), _ACT[gate_act]
    s.residual_scale, s.eps = float(residual_scale), float(eps)
    if not x.is_cuda:
        raise RuntimeError("fluidnet_amd block norms run on MI355X only (got a CPU tensor); there is no CPU fallback")
    return s


def _gate_rows(s: _Spec, gate: Optional[torch.Tensor]) -> Tuple[Optional[torch.Tensor], int]:
    """The gate and the distance of its rows (of its values, for one per token)."""
    if gate is None:
        return None, 0
    if s.gate_kind in (_ELEMENT, _TOKEN):
        return _rows(gate)
    if s.gate_kind == _SAMPLE and gate.stride(-1) == 1:
        return gate, gate.stride(0)
    return gate.contiguous(), s.width


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _forward(s: _Spec, x, branch, gate, scale, pw, pb, nw, nb, keep: bool):
    """(y, h, stats) of prepared operands."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if branch is not None else None
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if s.pre else None
    stats = torch.empty((4, s.rows), dtype=torch.float32, device=x.device) if keep and (s.post or s.pre) else None
    if s.rows and (y is not None or h is not None):
        (xt, xs), (bt, bs), (gt, gs) = _rows(x), (_rows(branch) if branch is not None else (None, 0)), _gate_rows(s, gate)
        params = [_dense(t) for t in (scale, pw, pb, nw, nb)]
        a = _ARGS.pack(s.rows, s.tokens, xs, bs, gs, 0, 0, s.width, s.dtype, s.param_dtype, s.gate_dtype, s.kind, s.post, s.gate_kind, s.gate_act,
                       s.residual_scale, s.eps, xt.data_ptr(), _ptr(bt), _ptr(gt), *map(_ptr, params), _ptr(y), _ptr(h), _ptr(stats),
                       0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        rt.call_on(x, "fnet_block_norm_fwd", a)
    return y, h, stats


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, x, branch, gate, scale, pw, pb, nw, nb):
        ctx.set_materialize_grads(False)
        y, h, stats = _forward(s, x, branch, gate, scale, pw, pb, nw, nb, True)
        ctx.s = s
        ctx.save_for_backward(x, branch, gate, scale, pw, pb, nw, nb, stats)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        s = ctx.s
        x, branch, gate, scale, pw, pb, nw, nb, stats = ctx.saved_tensors
        none = (None,) * 9
        if dy is None and dh is None:
            return none
        _, nx, nbr, ng, nsc, npw, npb, nnw, nnb = ctx.needs_input_grad
        new = lambda t, need: torch.empty(t.shape, dtype=t.dtype, device=t.device) if need and t is not None else None  # noqa: E731
        if s.rows == 0:
            return (None, *(None if not n or t is None else torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t, n in
                            zip((x, branch, gate, scale, pw, pb, nw, nb), ctx.needs_input_grad[1:])))
        # without a gradient of h, the gradient of x is that of y
        dx = (dy if dh is None else new(x, True)) if nx else None
        db, dg, dsc, dpw, dpb = new(branch, nbr), new(gate, ng), new(scale, nsc), new(pw, npw), new(pb, npb)
        zero = lambda t, need: torch.zeros(t.shape, dtype=t.dtype, device=t.device) if need and t is not None else None  # noqa: E731
        dnw, dnb = (new(nw, nnw), new(nb, nnb)) if dh is not None else (zero(nw, nnw), zero(nb, nnb))
        if (dh is not None and (nx or nnw or nnb)) or any(t is not None for t in (db, dg, dsc, dpw, dpb)):
            (xt, xs), (bt, bs), (gt, gs) = _rows(x), (_rows(branch) if branch is not None else (None, 0)), _gate_rows(s, gate)
            (dyt, dys), (dht, dhs) = (_rows(t) if t is not None else (None, 0) for t in (dy, dh))
            params = [_dense(t) for t in (scale, pw, pb, nw, nb)]
            with_dh = dh is not None

            def pack(ws, n):
                return _ARGS.pack(s.rows, s.tokens, xs, bs, gs, dys, dhs, s.width, s.dtype, s.param_dtype, s.gate_dtype, s.kind, s.post,
                                  s.gate_kind, s.gate_act, s.residual_scale, s.eps, xt.data_ptr(), _ptr(bt), _ptr(gt), *map(_ptr, params), 0, 0,
                                  _ptr(stats), _ptr(dyt), _ptr(dht), _ptr(dx) if with_dh else 0, _ptr(db), _ptr(dg), _ptr(dsc), _ptr(dpw),
                                  _ptr(dpb), _ptr(dnw) if with_dh else 0, _ptr(dnb) if with_dh else 0, ws, n)
            need = ctypes.c_int64()
            rt.check(rt.lib().fnet_block_norm_workspace(pack(0, 0), ctypes.byref(need)), "fnet_block_norm_workspace")
            ws = torch.empty(need.value, dtype=torch.uint8, device=x.device) if need.value else None
            rt.call_on(x, "fnet_block_norm_bwd", pack(_ptr(ws), need.value))
        return None, dx, db, dg, dsc, dpw, dpb, dnw, dnb


def _run(s: _Spec, x, branch, gate, scale, pw, pb, nw, nb):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, branch, gate, scale, pw, pb, nw, nb)):
        return _BlockNormFn.apply(s, x, branch, gate, scale, pw, pb, nw, nb)
    y, h, _ = _forward(s, x, branch, gate, scale, pw, pb, nw, nb, False)
    return y, h


def pre_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, kind: NormKind = "rms",
             eps: float = 1e-6) -> torch.Tensor:
    """N(x) * weight + bias: the norm before the first block."""
    s = _spec(x, None, None, None, None, None, weight, bias, kind, False, True, "identity", 1.0, eps)
    return _run(s, x, None, None, None, None, None, weight, bias)[1]


def gated_residual(x: torch.Tensor, branch: torch.Tensor, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, *,
                   post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                   pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None, kind: NormKind = "rms",
                   post: bool = True, pre: bool = True, gate_act: GateAct = "identity", residual_scale: float = 1.0,
                   eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, h): the residual sum with the branch normalised, gated and scaled, and the norm of it that the next block takes (None with
    pre=False).  Differentiable with respect to every tensor."""
    if branch is None:
        raise ValueError("gated_residual needs a branch (pre_norm is the form without one)")
    s = _spec(x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, kind, post, pre, gate_act, residual_scale, eps)
    return _run(s, x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias)


class PreNorm(nn.Module):
    """pre_norm with its parameters."""

    def __init__(self, width: int, *, kind: NormKind = "rms", bias: bool = False, eps: float = 1e-6) -> None:
        super().__init__()
        self.kind, self.eps = kind, eps
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return pre_norm(x, self.weight, self.bias, kind=self.kind, eps=self.eps)


class GatedResidual(nn.Module):
    """gated_residual with its parameters.  scale_init: start value of a learned scale per channel (None: none); channel_gate: start value of
    a learned gate per channel, instead of a gate given to forward."""

    def __init__(self, width: int, *, kind: NormKind = "rms", bias: bool = False, post: bool = True, pre: bool = True,
                 scale_init: Optional[float] = None, channel_gate: Optional[float] = None, gate_act: GateAct = "identity",
                 residual_scale: float = 1.0, eps: float = 1e-6) -> None:
        super().__init__()
        self.kind, self.post, self.pre, self.gate_act, self.residual_scale, self.eps = kind, post, pre, gate_act, residual_scale, eps

        def param(value, wanted=True):
            return nn.Parameter(torch.full((width,), float(value))) if wanted else None
        self.post_weight, self.post_bias = param(1, post), param(0, post and bias)
        self.pre_weight, self.pre_bias = param(1, pre), param(0, pre and bias)
        self.scale = None if scale_init is None else param(scale_init)
        self.gate = None if channel_gate is None else param(channel_gate)

    def forward(self, x: torch.Tensor, branch: torch.Tensor, gate: Optional[torch.Tensor] = None):
        if gate is not None and self.gate is not None:
            raise ValueError("this module has a gate of its own")
        return gated_residual(x, branch, self.gate if gate is None else gate, self.scale, post_weight=self.post_weight, post_bias=self.post_bias,
                              pre_weight=self.pre_weight, pre_bias=self.pre_bias, kind=self.kind, post=self.post, pre=self.pre,
                              gate_act=self.gate_act, residual_scale=self.residual_scale, eps=self.eps)


__all__ = ["pre_norm", "gated_residual", "PreNorm", "GatedResidual", "MAX_WIDTH"]
