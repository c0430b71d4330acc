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
There is no CPU fallback, and no second derivative (asking for one raises).

Both directions can be captured into a graph.  A captured backward pass that hands gradients to leaves (into .grad or out of
torch.autograd.grad) raises while outputs of an eager call from the same leaves on the default stream are alive: torch orders a leaf's gradient
after the stream on which the leaf was first used, the default stream cannot take part in a capture, and the process would end.  Drop those
outputs first, or make the eager calls on a side stream.  (Outputs of other operations on the same leaves are the caller's to drop.)
"""
from __future__ import annotations

import ctypes
import struct
import weakref
from typing import Literal, Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

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
    __slots__ = ("rows", "tokens", "width", "param_dtype", "gate_dtype", "pre", "post", "gate_kind", "fixed")


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The tensor (copied if its last axis is not dense or its rows are not evenly spaced) and its row stride."""
    size = t.shape
    if t.is_contiguous():
        return t, size[-1]
    stride = t.stride()
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


def _param_type(name: str, t: torch.Tensor, C: int, x: torch.Tensor, seen):
    if t.shape != (C,) or t.get_device() != x.get_device():
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
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= MAX_WIDTH:
        raise ValueError(f"the last axis must have 1 to {MAX_WIDTH} elements (got shape {tuple(shape)})")
    if kind not in _KIND or gate_act not in _ACT:
        raise ValueError(f"kind must be one of {tuple(_KIND)} and gate_act one of {tuple(_ACT)} (got {kind!r}, {gate_act!r})")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    s = _Spec()
    s.width = C = shape[-1]
    s.rows = rows = x.numel() // C
    if rows >= 1 << 31:
        raise ValueError("at most 2^31 - 1 rows")
    if branch is None:
        if gate is not None or scale is not None:
            raise ValueError("a gate or scale needs a branch")
        post = False
    elif branch.shape != shape or branch.dtype is not x.dtype or branch.get_device() != x.get_device():
        raise ValueError(f"branch must be like x: {tuple(shape)} {x.dtype} on {x.device} (got {tuple(branch.shape)} {branch.dtype} on {branch.device})")
    if not post and (pw is not None or pb is not None):
        raise ValueError("post_weight / post_bias need post=True")
    if not pre and (nw is not None or nb is not None):
        raise ValueError("pre_weight / pre_bias need pre=True")
    seen = None
    if scale is not None:
        seen = _param_type("scale", scale, C, x, seen)
    if pw is not None:
        seen = _param_type("post_weight", pw, C, x, seen)
    if pb is not None:
        seen = _param_type("post_bias", pb, C, x, seen)
    if nw is not None:
        seen = _param_type("pre_weight", nw, C, x, seen)
    if nb is not None:
        seen = _param_type("pre_bias", nb, C, x, seen)
    gate_kind, gate_dtype, s.tokens = _NONE, 0, rows
    if gate is not None:
        if gate.get_device() != x.get_device() or (gate.dtype is not torch.float32 and gate.dtype is not x.dtype):
            raise ValueError(f"gate must be float32 or {x.dtype} on {x.device} (got {gate.dtype} on {gate.device})")
        gate_kind, gate_dtype = _gate_kind(gate, x), ELEM[gate.dtype]
        if gate_kind == _SAMPLE and rows:
            s.tokens = rows // shape[0]
            if s.tokens == 1:                 # a row of values per row
                gate_kind = _ELEMENT
    s.gate_kind, s.pre, s.post = gate_kind, bool(pre), bool(post)
    s.fixed = (C, code, 0 if seen is None else ELEM[seen], gate_dtype, _KIND[kind], s.post, gate_kind, _ACT[gate_act], float(residual_scale), float(eps))
    if not x.is_cuda:
        raise RuntimeError("fluidnet_amd block norms run on MI355X only (got a CPU tensor); there is no CPU fallback")
    return s


def _gate_rows(s: _Spec, gate: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The gate and the distance of its rows (of its values, for one per token)."""
    if s.gate_kind == _ELEMENT or s.gate_kind == _TOKEN:
        return _rows(gate)
    if s.gate_kind == _SAMPLE and gate.stride(-1) == 1:
        return gate, gate.stride(0)
    return gate.contiguous(), s.width


def _operands(s: _Spec, x, branch, gate, scale, pw, pb, nw, nb):
    """What the kernels read besides gradients, as they take it: strides, addresses and the tensors these belong to."""
    x, xs = _rows(x)
    b = g = c = d = e = f = h = bs = gs = 0
    if branch is not None:
        branch, bs = _rows(branch)
        b = branch.data_ptr()
        if gate is not None:
            gate, gs = _gate_rows(s, gate)
            g = gate.data_ptr()
        if scale is not None:
            scale = scale.contiguous()
            c = scale.data_ptr()
        if pw is not None:
            pw = pw.contiguous()
            d = pw.data_ptr()
        if pb is not None:
            pb = pb.contiguous()
            e = pb.data_ptr()
    if nw is not None:
        nw = nw.contiguous()
        f = nw.data_ptr()
    if nb is not None:
        nb = nb.contiguous()
        h = nb.data_ptr()
    return (xs, bs, gs), (x.data_ptr(), b, g, c, d, e, f, h), (x, branch, gate, scale, pw, pb, nw, nb)


_NO_GRADS = (0,) * 12
_DENSE = torch.contiguous_format


def _forward(s: _Spec, x, branch, gate, scale, pw, pb, nw, nb, keep: bool):
    """(y, h, stats): stats (means and deviations, for the backward) if they are kept."""
    y = torch.empty_like(x, memory_format=_DENSE) if branch is not None else None
    h = torch.empty_like(x, memory_format=_DENSE) if s.pre else None
    stats = x.new_empty((4, s.rows), dtype=torch.float32) if keep and (s.post or s.pre) else None
    if s.rows and (y is not None or h is not None):
        strides, ptrs, _keep = _operands(s, x, branch, gate, scale, pw, pb, nw, nb)
        a = _ARGS.pack(s.rows, s.tokens, *strides, 0, 0, *s.fixed, *ptrs, 0 if y is None else y.data_ptr(), 0 if h is None else h.data_ptr(),
                       0 if stats is None else stats.data_ptr(), *_NO_GRADS)
        rt.call_on(x, "fnet_block_norm_fwd", a)
    return y, h, stats


def _backward(ctx, dy, dh):
    s = ctx.s
    x, branch, gate, scale, pw, pb, nw, nb, stats = ctx.saved_tensors
    _, nx, nbr, ng, nsc, npw, npb, nnw, nnb = ctx.needs_input_grad
    if dy is None and dh is None:
        return (None,) * 9
    make = torch.empty_like if s.rows else torch.zeros_like
    with_h = dh is not None
    # without a gradient of h, the gradient of x is that of y
    dx = None if not nx else make(x, memory_format=_DENSE) if with_h else dy
    db = make(branch, memory_format=_DENSE) if nbr and branch is not None else None
    dg = make(gate, memory_format=_DENSE) if ng and gate is not None else None
    sums = dg is not None
    dsc = dpw = dpb = dnw = dnb = None
    if nsc and scale is not None:
        dsc, sums = make(scale, memory_format=_DENSE), True
    if npw and pw is not None:
        dpw, sums = make(pw, memory_format=_DENSE), True
    if npb and pb is not None:
        dpb, sums = make(pb, memory_format=_DENSE), True
    norm = make if with_h else torch.zeros_like
    if nnw and nw is not None:
        dnw, sums = norm(nw, memory_format=_DENSE), True
    if nnb and nb is not None:
        dnb, sums = norm(nb, memory_format=_DENSE), True
    if s.rows and (with_h or db is not None or dg is not None or sums):
        strides, ptrs, _keep = _operands(s, x, branch, gate, scale, pw, pb, nw, nb)
        py = ys = ph = hs = px = p0 = p1 = 0
        if dy is not None:
            dy, ys = _rows(dy)
            py = dy.data_ptr()
        if with_h:
            dh, hs = _rows(dh)
            ph = dh.data_ptr()
            px = 0 if dx is None else dx.data_ptr()
            p0 = 0 if dnw is None else dnw.data_ptr()
            p1 = 0 if dnb is None else dnb.data_ptr()
        a = (s.rows, s.tokens, *strides, ys, hs, *s.fixed, *ptrs, 0, 0, 0 if stats is None else stats.data_ptr(), py, ph, px,
             0 if db is None else db.data_ptr(), 0 if dg is None else dg.data_ptr(), 0 if dsc is None else dsc.data_ptr(),
             0 if dpw is None else dpw.data_ptr(), 0 if dpb is None else dpb.data_ptr(), p0, p1)
        n = 0
        if sums:                              # partial sums of what is summed over rows
            need = ctypes.c_int64()
            rt.check(rt.lib().fnet_block_norm_workspace(_ARGS.pack(*a, 0, 0), ctypes.byref(need)), "fnet_block_norm_workspace")
            n = need.value
        ws = x.new_empty(n, dtype=torch.uint8) if n else None
        a = _ARGS.pack(*a, 0 if ws is None else ws.data_ptr(), n)
        rt.call_on(x, "fnet_block_norm_bwd", a)
    return None, dx, db, dg, dsc, dpw, dpb, dnw, dnb


_backward_once = once_differentiable(_backward)


_on_default = weakref.WeakSet()              # nodes of the graphs that are alive and were made on the default stream


def _leaf_nodes(node) -> dict:
    """The nodes of leaves in the graph below `node`, by the leaf's identity."""
    seen, todo, leaves = {node}, [node], {}
    while todo:
        for below, _ in todo.pop().next_functions:
            if below is not None and below not in seen:
                seen.add(below)
                todo.append(below)
                if hasattr(below, "variable"):
                    leaves[id(below.variable)] = below
    return leaves


def _wanted(node) -> bool:
    try:
        return torch._C._will_engine_execute_node(node)
    except RuntimeError:                      # torch.autograd.grad is asked for this leaf's
        return True


def _check_capture(ctx) -> None:
    """While a graph is captured: raises if a leaf's gradient would be ordered after the default stream (see above)."""
    eager = [node for node in (ref() for ref in list(_on_default.data)) if node is not None]
    if not eager:
        return
    mine = {leaf for leaf, node in _leaf_nodes(ctx).items() if _wanted(node)}
    if mine and any(mine & _leaf_nodes(node).keys() for node in eager):
        raise RuntimeError("outputs of an earlier call from the same leaves, made on the default stream, are alive: drop them before capturing "
                           "a backward pass")


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, x, branch, gate, scale, pw, pb, nw, nb):
        ctx.set_materialize_grads(False)
        y, h, stats = _forward(s, x, branch, gate, scale, pw, pb, nw, nb, True)
        ctx.s = s
        if rt.raw_stream(x.get_device()) == 0:
            _on_default.add(ctx)
        ctx.save_for_backward(x, branch, gate, scale, pw, pb, nw, nb, stats)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        if torch.cuda.is_current_stream_capturing():
            _check_capture(ctx)
        # with create_graph the gradients are marked as having no derivative of their own; without it nobody can ask for one
        return _backward_once(ctx, dy, dh) if torch.is_grad_enabled() else _backward(ctx, dy, dh)


def _run(s: _Spec, *operands):
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                return _BlockNormFn.apply(s, *operands)
    y, h, _ = _forward(s, *operands, False)
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
