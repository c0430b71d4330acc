"""clip_grad_norm_ + Adam on the flat parameter / gradient buffers of fluidnet_amd.UNet, as two HIP launches
(GRAD_NORM, ADAM in csrc/fnet_optim.hip) with the clip coefficient computed on the device -- replaces
torch.nn.utils.clip_grad_norm_ + torch.optim.Adam.step of ml/training/trainer.py:190-195 (88 norms + ~10 foreach kernels and
one host sync in the reference).  Same arithmetic: betas (0.9, 0.999), eps 1e-8, no weight decay, no amsgrad.

clip_adam_ / ClipAdam are the same step for the separate parameters of any module (csrc/fnet_tensor_list.hip), with decoupled weight decay
and 32-bit masters of 16-bit parameters."""
from __future__ import annotations

import math
import struct
from typing import Dict, Iterable, List, Optional, Sequence, Union

import numpy as np
import torch

from ..engine import runtime as rt
from ..engine.runtime import OPC
from .grad_clip import TensorList, _collapsed, _max_norm


class FusedClipAdam:
    def __init__(self, model, lr: float, max_norm: Optional[float] = 1.0, betas=(0.9, 0.999), eps: float = 1e-8) -> None:
        self.model = model
        self.max_norm = max_norm
        self.betas, self.eps = betas, eps
        self.param_groups = [{"lr": float(lr)}]        # torch-optimizer-shaped, for schedulers / logging
        self.step_count = 0
        self._m: Optional[torch.Tensor] = None
        self._v: Optional[torch.Tensor] = None
        self._normsq: Optional[torch.Tensor] = None

    def _state(self):
        p = self.model.flat_params
        if self._m is None or self._m.device != p.device or self._m.numel() != p.numel():
            self._m = torch.zeros_like(p)
            self._v = torch.zeros_like(p)
            self._normsq = torch.zeros(2, dtype=torch.float64, device=p.device)
        return p, self.model.flat_grads, self._m, self._v, self._normsq

    def zero_grad(self, set_to_none: bool = True) -> None:
        self.model.flat_grads.zero_()
        for q in self.model.parameters():
            q.grad = None

    @torch.no_grad()
    def step(self) -> None:
        p, g, m, v, nsq = self._state()
        if not p.is_cuda:
            raise RuntimeError("FusedClipAdam runs on MI355X only; there is no CPU fallback")
        self.model._attach_grads()
        self.step_count += 1
        b1, b2 = self.betas
        n = p.numel()
        ops = np.zeros(2, dtype=rt.OP_DTYPE)
        nsq.zero_()
        ops[0]["op"] = OPC["GRAD_NORM"]
        ops[0]["i"][:2] = [n & 0x7FFFFFFF, n >> 31]
        ops[0]["p"][:2] = [g.data_ptr(), nsq.data_ptr()]
        ops[1]["op"] = OPC["ADAM"]
        ops[1]["i"][:2] = [n & 0x7FFFFFFF, n >> 31]
        ops[1]["f"][:8] = [self.param_groups[0]["lr"], b1, b2, self.eps, 1.0 - b1 ** self.step_count,
                           math.sqrt(1.0 - b2 ** self.step_count), self.max_norm or 0.0, 1.0]
        ops[1]["p"][:5] = [p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), nsq.data_ptr() if self.max_norm else 0]
        rt.run_ops(ops if self.max_norm else ops[1:])
        p.add_(0)          # bump flat_params' autograd version so that engines refresh their bf16 weight copies

    def state_dict(self) -> Dict:
        p, g, m, v, _ = self._state()
        return {"step": self.step_count, "lr": self.param_groups[0]["lr"], "exp_avg": m.detach().cpu(), "exp_avg_sq": v.detach().cpu(),
                "betas": self.betas, "eps": self.eps, "max_norm": self.max_norm}

    def load_state_dict(self, sd: Dict) -> None:
        p, g, m, v, _ = self._state()
        self.step_count = int(sd["step"])
        self.param_groups[0]["lr"] = float(sd["lr"])
        m.copy_(sd["exp_avg"])
        v.copy_(sd["exp_avg_sq"])


# ---------------------------------------------------------------------------------------------------------------- lists of parameters
def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors are dense and element k of one lies where element k of the other does."""
    if a.shape != b.shape or a.is_neg() or b.is_neg():
        return False
    if a.is_contiguous() and b.is_contiguous():
        return True
    return _collapsed(a) in ([], [[1, a.numel()]]) and all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


# struct FnetAdamList (include/fluidnet_hip.h)
_ADAM = struct.Struct("=6d4Qi4x")


def _check_layouts(params, grads, exp_avgs, exp_avg_sqs, masters) -> None:
    """Tensor by tensor what clip_adam_ asks of a whole list: raises for the first one that does not fit; dense tensors in another order pass."""
    for k, (p, g, m, v, w) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, masters)):
        if w is None and p.dtype is not torch.float32:
            raise ValueError(f"parameter {k} is not float32 and needs an fp32 master")
        if p.dtype is not g.dtype or p.get_device() != g.get_device() or not _same_layout(p, g):
            raise ValueError(f"parameter {k} and its gradient must be dense tensors of one type, layout and device (got "
                             f"{tuple(p.shape)} {p.stride()} {p.dtype} {p.device}, {tuple(g.shape)} {g.stride()} {g.dtype} {g.device})")
        for name, t in (("exp_avg", m), ("exp_avg_sq", v)) + ((("master", w),) if p.dtype is not torch.float32 else ()):
            if t.dtype is not torch.float32 or t.get_device() != p.get_device() or not _same_layout(p, t):
                raise ValueError(f"{name} {k} must be a float32 tensor laid out like its parameter: {tuple(p.shape)} {p.stride()} on {p.device}")


def clip_adam_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], clock: torch.Tensor, *, masters: Optional[Sequence[torch.Tensor]] = None,
               lr: Union[float, torch.Tensor], betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
               max_norm: Optional[float] = None) -> Optional[torch.Tensor]:
    """One Adam step of a list of parameters on gradients clipped to the global 2-norm max_norm (None: not clipped), in place.

        c = min(1, max_norm / (norm + 1e-6));  m = b1 m + (1 - b1) c g;  v = b2 v + (1 - b2) (c g)^2
        w = w (1 - lr weight_decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    The gradients are not changed: the clipped ones are never written.  Returns the norm before clipping (0-dim, fp32, on the device; None
    without clipping).  params[k] and grads[k] are of one type (fp32, bf16 or fp16); exp_avgs and exp_avg_sqs are fp32; all of them are dense and
    laid out alike.  Parameters that are not fp32 need an fp32 master each: the master is updated and the parameter is its rounding (masters
    of fp32 parameters are not looked at).  Parameters, moments and masters that share memory, with each other or with a gradient, are
    refused.  clock: three fp64 values on the device, t, beta1^t and beta2^t of the steps done so far; the call advances it.  lr: a number,
    or one fp64 value on the device, which a captured step reads anew at every replay.  Two launches for up to 80 parameters."""
    params, grads, exp_avgs, exp_avg_sqs = list(params), list(grads), list(exp_avgs), list(exp_avg_sqs)
    n = len(params)
    masters = [None] * n if masters is None else list(masters)
    if not n or any(len(x) != n for x in (grads, exp_avgs, exp_avg_sqs, masters)):
        raise ValueError("params, grads, exp_avgs, exp_avg_sqs (and masters) must be equally long and not empty")
    b1, b2 = (float(b) for b in betas)
    if not (0 <= b1 < 1 and 0 <= b2 < 1 and eps >= 0 and weight_decay >= 0):
        raise ValueError(f"betas must lie in [0, 1), eps and weight_decay must not be negative (got {betas}, {eps}, {weight_decay})")
    if max_norm is not None:
        max_norm = _max_norm(max_norm)
    lst, ops = TensorList(grads), rt.torch_ops()
    if not ops.adam_fits(params, grads, exp_avgs, exp_avg_sqs, masters):
        _check_layouts(params, grads, exp_avgs, exp_avg_sqs, masters)
    dev = lst.first.get_device()
    for name, t, count in (("clock", clock, 3),) + ((("lr", lr, 1),) if isinstance(lr, torch.Tensor) else ()):
        if t.dtype is not torch.float64 or t.numel() != count or t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be {count} float64 value(s) on {lst.first.device}")
    address = [ops.addresses(ts) for ts in (params, exp_avgs, exp_avg_sqs, masters)]
    total, ws = None, None
    if max_norm is not None:
        total = torch.empty((), dtype=torch.float32, device=lst.first.device)
        ws = lst.workspace()
    a = _ADAM.pack(0.0 if isinstance(lr, torch.Tensor) else float(lr), b1, b2, eps, weight_decay, -1.0 if max_norm is None else max_norm,
                   0 if ws is None else ws.data_ptr(), clock.data_ptr(), lr.data_ptr() if isinstance(lr, torch.Tensor) else 0,
                   0 if total is None else total.data_ptr(), 0 if ws is None else lst.capacity)
    rt.call_on(lst.first, "fnet_list_adam", n, address[0], lst.ptrs, address[1], address[2], address[3], lst.numels, lst.codes, a)
    ops.written(params, exp_avgs, exp_avg_sqs, masters, clock)
    return total


class ClipAdam:
    """clip_adam_ with its state, for the parameters of any module: the counterpart of FusedClipAdam (same attributes and schedule hooks).

    Parameters without a gradient are left as they are in a step, moments too; t counts the optimizer's steps.  16-bit parameters have fp32
    masters, made from them at the first step and again when a parameter has been written by something else since the last one (which its
    version counter tells: load_state_dict, in-place operations; after writing through .data call refresh()).  step() can be captured into
    a graph after one eager step: step count and learning rate are on the device, set param_groups[0]["lr"] and call push_lr() between replays.  A
    replay does not look for parameters written by something else: call refresh() after such a write.  One clipping norm, learning rate and
    weight decay for all parameters: parameter groups are refused."""

    def __init__(self, params: Iterable[torch.nn.Parameter], lr: float, max_norm: Optional[float] = 1.0, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0) -> None:
        self.params: List[torch.Tensor] = list(params)
        if not self.params:
            raise ValueError("ClipAdam got no parameters")
        if not all(isinstance(p, torch.Tensor) for p in self.params):
            raise TypeError("ClipAdam takes parameters, not groups of them")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("a parameter appears twice")
        self.max_norm = None if max_norm is None else _max_norm(max_norm)
        self.betas, self.eps, self.weight_decay = betas, eps, weight_decay
        self.param_groups = [{"lr": float(lr)}]
        self.grad_norm: Optional[torch.Tensor] = None       # of the last step, before clipping
        self._m: Optional[List[torch.Tensor]] = None

    def _init_state(self) -> None:
        dev = self.params[0].device
        if self._m is not None and self._clock.device == dev:
            return
        for k, p in enumerate(self.params):
            if not p.is_cuda:
                raise RuntimeError("ClipAdam runs on MI355X only; there is no CPU fallback")
            if _collapsed(p) not in ([], [[1, p.numel()]]):
                raise ValueError(f"parameter {k} must be dense (shape {tuple(p.shape)}, strides {p.stride()})")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("ClipAdam: make one eager step before capturing one")
        old = self._packed() if self._m is not None else None          # the module was moved to another device
        self._m = [torch.zeros_like(p, dtype=torch.float32) for p in self.params]
        self._v = [torch.zeros_like(p, dtype=torch.float32) for p in self.params]
        self._w = [None if p.dtype is torch.float32 else p.detach().float() for p in self.params]
        self._clock = torch.tensor([0.0, 1.0, 1.0], dtype=torch.float64, device=dev)
        self._lr = torch.tensor(self.param_groups[0]["lr"], dtype=torch.float64, device=dev)
        self._lr_pushed = self.param_groups[0]["lr"]
        self._seen = rt.torch_ops().marks(self.params)
        if old is not None:
            self.load_state_dict(old)

    @torch.no_grad()
    def refresh(self) -> None:
        """Makes the masters anew from the parameters."""
        self._init_state()
        for w, p in zip(self._w, self.params):
            if w is not None:
                w.copy_(p)
        self._seen = rt.torch_ops().marks(self.params)

    def push_lr(self) -> None:
        """Copies param_groups[0]["lr"] to the device, where a captured step reads it."""
        self._init_state()
        if self.param_groups[0]["lr"] != self._lr_pushed:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("ClipAdam: the learning rate changed; call push_lr() before capturing the step")
            self._lr_pushed = self.param_groups[0]["lr"]
            self._lr.fill_(self._lr_pushed)

    def zero_grad(self, set_to_none: bool = True) -> None:
        for p in self.params:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()

    @torch.no_grad()
    def step(self) -> None:
        self._init_state()
        self.push_lr()
        marks = rt.torch_ops().marks(self.params)
        if marks != self._seen:
            for k, (p, w) in enumerate(zip(self.params, self._w)):
                if w is not None and marks[16 * k:16 * k + 16] != self._seen[16 * k:16 * k + 16]:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("ClipAdam: a parameter was written since the last step; call refresh() before capturing the step")
                    w.copy_(p)
        lists = (self.params, [p.grad for p in self.params], self._m, self._v, self._w)
        have = [k for k, g in enumerate(lists[1]) if g is not None]
        if not have:
            return
        if len(have) < len(self.params):
            lists = [[ts[k] for k in have] for ts in lists]
        params, grads, m, v, w = lists
        if not rt.torch_ops().adam_fits(params, grads, m, v, w):
            grads = [g if _same_layout(p, g) else torch.empty_like(p).copy_(g) for p, g in zip(params, grads)]
        self.grad_norm = clip_adam_(params, grads, m, v, self._clock, masters=w, lr=self._lr, betas=self.betas, eps=self.eps,
                                    weight_decay=self.weight_decay, max_norm=self.max_norm)
        self._seen = rt.torch_ops().marks(self.params)

    @property
    def step_count(self) -> int:
        return 0 if self._m is None else int(self._clock[0].item())

    def state_dict(self) -> Dict:
        self._init_state()
        return self._packed()

    def _packed(self) -> Dict:
        cpu = lambda ts: [None if t is None else t.detach().cpu() for t in ts]  # noqa: E731
        return {"step": self.step_count, "lr": self.param_groups[0]["lr"], "exp_avg": cpu(self._m), "exp_avg_sq": cpu(self._v),
                "master": cpu(self._w), "betas": self.betas, "eps": self.eps, "max_norm": self.max_norm, "weight_decay": self.weight_decay}

    @torch.no_grad()
    def load_state_dict(self, sd: Dict) -> None:
        self._init_state()
        for name in ("exp_avg", "exp_avg_sq", "master"):
            if len(sd[name]) != len(self.params):
                raise ValueError(f"the state's {name} is of {len(sd[name])} parameters, this optimizer has {len(self.params)}")
            for k, (t, p) in enumerate(zip(sd[name], self.params)):
                if (t is not None or name != "master") and t.shape != p.shape:
                    raise ValueError(f"the state's {name} {k} has shape {tuple(t.shape)}, the parameter {tuple(p.shape)}")
        t = int(sd["step"])
        self._clock.copy_(torch.tensor([t, self.betas[0] ** t, self.betas[1] ** t], dtype=torch.float64))
        self.param_groups[0]["lr"] = float(sd["lr"])
        self.push_lr()
        for mine, theirs in ((self._m, sd["exp_avg"]), (self._v, sd["exp_avg_sq"])):
            for a, b in zip(mine, theirs):
                a.copy_(b)
        for w, b, p in zip(self._w, sd["master"], self.params):
            if w is not None:
                # a master that does not round to its parameter is not this parameter's (the model was loaded from elsewhere)
                w.copy_(p if b is None else torch.where(b.to(w.device).to(p.dtype) == p, b.to(w.device), p.float()))
        self._seen = rt.torch_ops().marks(self.params)
