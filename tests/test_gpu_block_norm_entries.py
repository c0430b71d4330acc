"""Calls of the block norms' C entries that Python never makes."""
import ctypes

import pytest
import torch

from fluidnet_amd.engine import runtime as rt
from test_block_norm import _pack

pytestmark = pytest.mark.gpu
ELEMENT, SAMPLE = 1, 3


def _args(rows, width, x, branch, gate, out, **over):
    """A call on dense fp32 operands with a gate and the outputs of a dict; everything else is absent."""
    none = dict.fromkeys(("gate", "scale", "pw", "pb", "nw", "nb", "y", "h", "stats", "dy", "dh", "dx", "db", "dg", "ds", "dpw", "dpb", "dnw", "dnb", "ws"), 0)
    strides = dict.fromkeys(("xs", "bs", "gs", "dys", "dhs"), width)
    at = {k: v.data_ptr() for k, v in out.items()}
    return {**none, **strides, **dict(rows=rows, width=width, dtype=0, pdt=0, gdt=0, kind=1, post=1, a=0.7, eps=1e-6, x=x.data_ptr(), branch=branch.data_ptr(),
                                      gate=gate.data_ptr(), ga=1), **at, **over}


@pytest.mark.parametrize("rows,width", [(1, 5), (3000, 8), (1500, 300), (700, 1100), (600, 2300)])
def test_one_token_a_sample_is_a_gate_per_element(rows, width):
    """Both directions give the bits of the same call with a gate per element; one row behind each output stays as it was."""
    g = torch.Generator().manual_seed(rows)
    x, branch, gate, dy, dh = (torch.randn(rows, width, generator=g).cuda() for _ in range(5))
    L, st = rt.lib(), rt.raw_stream(0)

    def run(kind, tokens):
        make = lambda *s: torch.full(s, 7.5, device="cuda")  # noqa: E731
        fwd = {"y": make(rows + 1, width), "h": make(rows + 1, width), "stats": make(4 * rows + 1)}
        assert L.fnet_block_norm_fwd(_pack(**_args(rows, width, x, branch, gate, fwd, gk=kind, tokens=tokens)), st) == 0
        bwd = {"dx": make(rows + 1, width), "db": make(rows + 1, width), "dg": make(rows + 1, width), "ds": make(width + 1), "dpw": make(width + 1), "dnw": make(width + 1)}
        a = _args(rows, width, x, branch, gate, bwd, gk=kind, tokens=tokens, stats=fwd["stats"].data_ptr(), dy=dy.data_ptr(), dh=dh.data_ptr())
        n = ctypes.c_int64()
        assert L.fnet_block_norm_workspace(_pack(**a), ctypes.byref(n)) == 0
        ws = torch.empty(n.value + 16, dtype=torch.uint8, device="cuda")
        assert L.fnet_block_norm_bwd(_pack(**{**a, "ws": ws.data_ptr(), "wsn": n.value}), st) == 0
        torch.cuda.synchronize()
        for k, v in {**fwd, **bwd}.items():
            assert (v[rows:] == 7.5).all() if v.ndim == 2 else v[-1] == 7.5, k
        return {**fwd, **bwd}
    want, got = run(ELEMENT, rows), run(SAMPLE, 1)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_groups_behind_the_last_of_nearly_2_31_rows():
    """The last step of the last sample begins at row 2^31 - 3, so its fourth group would have row 2^31, which must be no row at all.  Operands
    of stride 0 make room for so many rows; only the statistics (34 GB) have a place per row.  Sums of ones: up to 2^24 per lane they are exact,
    the 4096 partial sums of 2^19 add up with at most 4096 roundings of 2^-24 in order, less than 1e-3 of the sum."""
    rows, tokens, width = (1 << 31) - 2, 357_913_941, 257          # six samples; tokens % 4 == 1
    assert rows % tokens == 0 and (rows - tokens) % 4 == 1
    one = torch.ones(width, device="cuda")
    stats = torch.ones(4 * rows, device="cuda")
    out = {"ds": torch.zeros(width, device="cuda"), "dg": torch.zeros(rows // tokens, width, device="cuda")}
    a = _args(rows, width, one, one, one, out, gk=SAMPLE, tokens=tokens, ga=0, kind=0, a=1.0, dy=one.data_ptr(), stats=stats.data_ptr(), xs=0, bs=0, gs=0, dys=0)
    n = ctypes.c_int64()
    L = rt.lib()
    assert L.fnet_block_norm_workspace(_pack(**a), ctypes.byref(n)) == 0
    ws = torch.empty(n.value + 16, dtype=torch.uint8, device="cuda")
    assert L.fnet_block_norm_bwd(_pack(**{**a, "ws": ws.data_ptr(), "wsn": n.value}), rt.raw_stream(0)) == 0
    torch.cuda.synchronize()
    assert ((out["ds"].double() - rows).abs() <= 1e-3 * rows).all() and ((out["dg"].double() - tokens).abs() <= 1e-3 * tokens).all()
    del stats
    torch.cuda.empty_cache()
