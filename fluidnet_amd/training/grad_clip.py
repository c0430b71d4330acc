"""The global norm of many gradients and their clipping, on the HIP kernels of libfluidnet_hip (fnet_list_*).

torch.nn.utils.clip_grad_norm_ as ml/training/trainer.py:192-195 calls it, for the parameters of any module: fp32, bf16 and fp16 gradients
in one list, dense in any layout or strided views of larger buffers (up to six axes), no elements, odd sizes, any alignment.  (The UNet's own
parameters lie in one flat buffer; FusedClipAdam clips that inside its step.)  One launch per 240 dense gradients, of all types, sums the norm,
one scales, and each strided gradient has two of its own (many of them are better packed); nothing is copied to the host, so all can be
captured into a graph.

Norms are summed in 64 bits in a fixed order: the same gradients give the same bits, and neither a large gradient's square nor the tail of a
long list is lost.  Clipping multiplies in 32 bits and rounds once.  All gradients must lie on one device (one process per GPU).
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Iterable, List, Union

import torch

from ..engine import runtime as rt
from ..engine.elements import ELEM

_KIND = {2.0: 0, 1.0: 1, math.inf: 2}
_MAXDIM = 6
# struct FnetStridedTensor (include/fluidnet_hip.h)
_STRIDED = struct.Struct("=Q2i12q")


def _collapsed(t: torch.Tensor):
    """Sizes and strides of a tensor's memory, largest stride first, neighbouring axes merged; None if elements share memory."""
    if t.numel() == 0:
        return [[1, 0]]
    axes = sorted(((st, n) for n, st in zip(t.shape, t.stride()) if n != 1), reverse=True)
    out: List[List[int]] = []
    for st, n in axes:
        if out and out[-1][0] == st * n:
            out[-1] = [st, out[-1][1] * n]
        else:
            out.append([st, n])
    reach = 1                                   # what lies below an axis must fit between two of its steps
    for st, n in reversed(out):
        if st < reach:
            return None
        reach += (n - 1) * st
    return out


class TensorList:
    """Addresses, element counts and types of the tensors of a call, as the C ABI takes them.  Lives for the call only."""

    def __init__(self, tensors: List[torch.Tensor], what: str = "gradient") -> None:
        self.first = tensors[0]
        table = rt.torch_ops().tensor_table(tensors)
        if table is None:
            self._refuse(tensors, what)
        strided = []
        if not table[0]:
            tensors, strided = self._split(tensors, what)
            table = rt.torch_ops().tensor_table(tensors)
        self.n, self.n_strided = len(tensors), len(strided)
        _, self.ptrs, self.numels, self.codes = table           # as bytes
        self.strided = b"".join(strided) if strided else None
        self.capacity = 2048 + self.n // 64 + 256 * self.n_strided + 8

    @staticmethod
    def _refuse(tensors, what):
        first = tensors[0]
        if not first.is_cuda:
            raise RuntimeError(f"fluidnet_amd runs on MI355X only (got a CPU {what}); there is no CPU fallback")
        k, t = next((k, t) for k, t in enumerate(tensors) if t.dtype not in ELEM or t.device != first.device or t.is_neg())
        raise ValueError(f"{what} {k} must be a float32, bfloat16 or float16 tensor on {first.device} and no negated view (got {t.dtype} on {t.device})")

    @staticmethod
    def _split(tensors, what):
        """The dense tensors, and the records of those that are no dense block of memory."""
        dense, strided = [], []
        for k, t in enumerate(tensors):
            axes = [[1, t.numel()]] if t.is_contiguous() else _collapsed(t)
            if axes is None or len(axes) > _MAXDIM:
                raise ValueError(f"{what} {k}: elements that share memory, or more than {_MAXDIM} separate axes (shape {tuple(t.shape)}, "
                                 f"strides {t.stride()})")
            if len(axes) > 1 or (axes and axes[0][0] != 1):
                pad = [0] * (_MAXDIM - len(axes))
                strided.append(_STRIDED.pack(t.data_ptr(), ELEM[t.dtype], len(axes), *(n for _, n in axes), *pad, *(st for st, _ in axes), *pad))
            else:
                dense.append(t)
        if len(set(strided)) != len(strided):
            raise ValueError(f"a {what} appears twice")
        return dense, strided

    def args(self):
        return self.n, self.ptrs, self.numels, self.codes, self.n_strided, self.strided

    def workspace(self) -> torch.Tensor:
        """Room for the partial sums of the norm."""
        return torch.empty(self.capacity, dtype=torch.float64, device=self.first.device)

    def partials(self, kind: int):
        """(workspace, how many partial sums are in it)."""
        ws = self.workspace()
        used = ctypes.c_int32()
        rt.call_on(self.first, "fnet_list_norm_partials", *self.args(), kind, ws.data_ptr(), self.capacity, ctypes.byref(used), 0, 0.0, 0.0)
        return ws, used.value

    def norm(self, kind: int) -> torch.Tensor:
        ws, used = self.partials(kind)
        out = torch.empty((), dtype=torch.float32, device=self.first.device)
        rt.call_on(self.first, "fnet_list_norm_finish", ws.data_ptr(), used, kind, out.data_ptr())
        return out


def _norm_kind(norm_type) -> int:
    kind = _KIND.get(float(norm_type))
    if kind is None:
        raise NotImplementedError(f"fluidnet_amd: norm_type must be 1, 2 or inf (got {norm_type})")
    return kind


def _max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative (got {max_norm})")
    return max_norm


def _grads(parameters) -> List[torch.Tensor]:
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return [g for g in [p.grad for p in parameters] if g is not None]


def total_grad_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of `tensors` (gradients, or anything else), a 0-dim fp32 tensor on their device.  0 for an empty list, on
    the CPU (as torch.nn.utils.get_total_norm)."""
    kind = _norm_kind(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    return TensorList(tensors, "tensor").norm(kind) if tensors else torch.tensor(0.0)


def _scale(lst: TensorList, max_norm: float, kind: int, partials: int, used: int, norm: int, out: int) -> None:
    rt.call_on(lst.first, "fnet_list_scale", *lst.args(), partials, used, kind, norm, max_norm, out)


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the gradients of `parameters` in place by min(1, max_norm / (norm + 1e-6)) and returns the norm that they had (0-dim, fp32, on
    their device).  Parameters without a gradient are passed over.  A norm that is not finite scales as torch does (gradients become 0 or NaN),
    or raises with error_if_nonfinite=True, which waits for the GPU.  (Finite gradients whose norm is beyond 32 bits are scaled by the norm as it is,
    though the value returned is infinite.)  Dense gradients that share memory are refused, and a strided one that appears twice; of strided
    gradients that overlap otherwise, with each other or with a dense one, the common elements are scaled once for each, as torch does."""
    kind, max_norm = _norm_kind(norm_type), _max_norm(max_norm)
    grads = _grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    lst = TensorList(grads)
    if error_if_nonfinite:
        total = lst.norm(kind)
        if not bool(torch.isfinite(total)):
            raise RuntimeError(f"the total norm of order {norm_type} of the gradients is not finite, so they cannot be clipped")
        _scale(lst, max_norm, kind, 0, 0, total.data_ptr(), 0)
    else:
        ws, used = lst.partials(kind)
        total = torch.empty((), dtype=torch.float32, device=lst.first.device)
        _scale(lst, max_norm, kind, ws.data_ptr(), used, 0, total.data_ptr())
    torch.autograd.graph.increment_version(grads)
    return total


def clip_grads_with_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, total_norm: torch.Tensor) -> None:
    """The scaling alone, by a norm that is known: one element, on the gradients' device (for instance a norm reduced over ranks)."""
    max_norm = _max_norm(max_norm)
    grads = _grads(parameters)
    if not grads:
        return
    lst = TensorList(grads)
    if total_norm.numel() != 1 or total_norm.device != lst.first.device:
        raise ValueError(f"total_norm must be one value on {lst.first.device} (got shape {tuple(total_norm.shape)} on {total_norm.device})")
    norm = total_norm.detach().reshape(()).to(torch.float32)
    _scale(lst, max_norm, 0, 0, 0, norm.data_ptr(), 0)
    torch.autograd.graph.increment_version(grads)


__all__ = ["total_grad_norm", "clip_grad_norm_", "clip_grads_with_norm_"]
