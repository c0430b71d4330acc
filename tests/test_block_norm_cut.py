"""How the C entries of the block norms cut the rows of calls that Python never makes; host only."""
import ctypes

import pytest

from fluidnet_amd.engine import runtime as rt
from test_block_norm import _pack

ELEMENT, SAMPLE = 1, 3


def _workspace(**over):
    n = ctypes.c_int64(-1)
    assert rt.lib().fnet_block_norm_workspace(_pack(dg=64, **over), ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("rows", [1, 63, 4096, 100_003, (1 << 31) - 1500, (1 << 31) - 1])
@pytest.mark.parametrize("width", [1, 8, 300, 2100, 16384])
def test_one_token_a_sample_is_a_gate_per_element(rows, width):
    """A gate per sample counts its samples in 32 bits and adds the grid to the count, which passes 2^31 where a sample is one row and there are
    nearly 2^31 of them.  Such a gate has a row of values per row: it is cut like one, by rows."""
    size = dict(rows=rows, width=width, gate=64, gdt=0)
    assert _workspace(gk=SAMPLE, tokens=1, **size) == _workspace(gk=ELEMENT, tokens=rows, **size)


def test_more_tokens_keep_their_samples():
    """Two tokens a sample: at most 2^30 samples, so a grid more stays below 2^31.  The cut is by samples, one segment each."""
    by_sample, by_row = (_workspace(gk=k, tokens=2, rows=4096, width=8, gate=64) for k in (SAMPLE, ELEMENT))
    assert by_sample > by_row
    assert _workspace(gk=SAMPLE, tokens=2, rows=(1 << 31) - 2, width=1, gate=64) > 0
