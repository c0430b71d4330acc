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

Both directions can be captured into a graph, the backward pass together with its forward pass.  A captured backward pass that hands gradients
to leaves (into .grad or out of torch.autograd.grad) raises while anything holds a leaf's node that was made on the default stream: outputs of
an eager call on the same leaves, of these operators or of any other, or a gradient edge.  torch orders a leaf's gradient after the stream on
which its node was made, the default stream cannot take part in a capture, and the process would end.  Drop those outputs first, or make the
eager calls on a side stream.
"""
from __future__ import annotations

from typing import Literal, Optional, Tuple

import torch
import torch.nn as nn

from ..engine import runtime as rt

NormKind = Literal["rms", "layer"]
GateAct = Literal["identity", "sigmoid", "tanh"]

MAX_WIDTH = 16384
_KIND = {"rms": 0, "layer": 1}
_ACT = {"identity": 0, "sigmoid": 1, "tanh": 2}


def _code(codes: dict, name: str, value: str) -> int:
    code = codes.get(value)
    if code is None:
        raise ValueError(f"{name} must be one of {tuple(codes)} (got {value!r})")
    return code


def _run(*args):
    """Checks, launch and autograd node, in native code (csrc/torch_ops.cpp)."""
    global _run
    _run = rt.torch_ops().block_norm
    return _run(*args)


def pre_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, kind: NormKind = "rms",
             eps: float = 1e-6) -> torch.Tensor:
    """N(x) * weight + bias: the norm before the first block."""
    return _run(x, None, None, None, None, None, weight, bias, _code(_KIND, "kind", kind), False, True, 0, 1.0, eps)[1]


def gated_residual(x: torch.Tensor, branch: torch.Tensor, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, *,
                   post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                   pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None, kind: NormKind = "rms",
                   post: bool = True, pre: bool = True, gate_act: GateAct = "identity", residual_scale: float = 1.0,
                   eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(y, h): the residual sum with the branch normalised, gated and scaled, and the norm of it that the next block takes (None with
    pre=False).  Differentiable with respect to every tensor."""
    if branch is None:
        raise ValueError("gated_residual needs a branch (pre_norm is the form without one)")
    return _run(x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, _code(_KIND, "kind", kind), post, pre,
                _code(_ACT, "gate_act", gate_act), residual_scale, eps)


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
