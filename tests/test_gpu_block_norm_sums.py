"""The gradients of the block norms that are sums over rows, at row counts where many blocks add them up, bit for bit.

Every operand is chosen so that no operation rounds: rows of +1 and -1 (in neighbouring pairs of both signs, so that every mean is 0 and every
deviation 1 with eps = 0), weights, gates and scales that are powers of two, upstream gradients of small whole numbers.  A sum is then a whole
number (times a power of two) below 2^24, whatever the order, and every row adds at least 1/8 to each of them, so a row that is lost or
added twice shows.  Widths that are no power of two have means that round; there the sums without a norm are exact and the others
are held to the roundings on their path."""
import pytest
import torch

import block_norm_ref as ref
from fluidnet_amd.models.block_norm import gated_residual, pre_norm

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
BRANCH_SUMS, PRE_SUMS = ("gate", "scale", "post_weight", "post_bias"), ("pre_weight", "pre_bias")
A = 0.5


def _signs(g, *shape):
    """+1 and -1; neighbours 2k and 2k + 1 of a row differ (a single element at an odd row's end is +1)."""
    s = torch.randint(0, 2, (*shape[:-1], (shape[-1] + 1) // 2, 1), generator=g) * 2.0 - 1
    return torch.cat([s, -s], -1).reshape(*shape[:-1], -1)[..., :shape[-1]].contiguous()


def _power(g, *shape):
    return 2.0 ** torch.randint(-1, 2, shape, generator=g)


def case(shape, dtype, gate, *, post, bias, param_dtype=F32, seed=0):
    """(operands, dy): the gradient of y alone, on the branch's side.  dy has the sign of the branch, so that nothing cancels in d z."""
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    s = _signs(g, *shape)
    up = torch.randint(1, 4, shape, generator=g).float()
    t = {"x": torch.zeros(shape), "branch": s if post else s * torch.randint(1, 3, shape, generator=g), "scale": _power(g, C), "post": post, "pre": False}
    gs = {"none": None, "element": shape, "token": (*shape[:-1], 1), "sample": (shape[0], *[1] * (len(shape) - 2), C), "channel": (C,)}[gate]
    if gs:
        t["gate"] = _power(g, *gs)
    if post:
        t["post_weight"] = _power(g, C)
        if bias:
            t["post_bias"] = 0.25 * torch.randint(0, 2, (C,), generator=g) + 0.125      # below every weight: the two never cancel
    params = ("scale", "post_weight", "post_bias")
    return {k: v.to(param_dtype if k in params else dtype) if isinstance(v, torch.Tensor) else v for k, v in t.items()}, (up * s).to(dtype)


def pre_case(shape, dtype, *, branch, param_dtype=F32, seed=0):
    """(operands, dh): the second norm's weights; with a branch of zeros, or without one."""
    g = torch.Generator().manual_seed(seed)
    s = _signs(g, *shape)
    t = {"x": s.to(dtype), "pre_weight": _power(g, shape[-1]).to(param_dtype), "pre_bias": _power(g, shape[-1]).to(param_dtype), "post": False, "pre": True}
    if branch:
        t["branch"] = torch.zeros(shape, dtype=dtype)
    return t, (torch.randint(1, 4, shape, generator=g) * s).to(dtype)


def sums(t, kind, dy, dh):
    """The gradients in 64 bits, in the types that the operator gives them."""
    want = ref.reference(t, kind, "identity", A, 0.0, dy, dh)
    return {n: want["d_" + n].to(t[n].dtype) for n in BRANCH_SUMS + PRE_SUMS if t.get(n) is not None}


def run(t, kind, dy, dh):
    d = {k: v.cuda().requires_grad_(k in BRANCH_SUMS + PRE_SUMS) if isinstance(v, torch.Tensor) else v for k, v in t.items()}
    if d.get("branch") is None:
        y, h = None, pre_norm(d["x"], d["pre_weight"], d["pre_bias"], kind=kind, eps=0.0)
    else:
        y, h = gated_residual(d["x"], d["branch"], d.get("gate"), d.get("scale"), post_weight=d.get("post_weight"), post_bias=d.get("post_bias"),
                              pre_weight=d.get("pre_weight"), pre_bias=d.get("pre_bias"), kind=kind, post=d["post"], pre=d["pre"], residual_scale=A, eps=0.0)
    names = [n for n in BRANCH_SUMS + PRE_SUMS if d.get(n) is not None]
    got = torch.autograd.grad(y if dh is None else h, [d[n] for n in names], (dy if dh is None else dh).cuda())
    return {n: v.cpu() for n, v in zip(names, got)}


def compare(t, kind, dy, dh):
    want, got = sums(t, kind, dy, dh), run(t, kind, dy, dh)
    for n in want:
        assert got[n].dtype == want[n].dtype and got[n].shape == want[n].shape, n
        bad = got[n] != want[n]
        assert not bad.any(), f"{n}: {int(bad.sum())} of {bad.numel()} differ, first {got[n][bad][0].item()} for {want[n][bad][0].item()}"


# every layout of rows: 8 to 64 lanes, 2 and 4 waves, 8 and 16 waves, 16 elements a lane
ROWS = [(40_000, 8), (40_000, 64), (20_000, 128), (12_000, 256), (9000, 512), (6000, 1024), (4000, 2048), (2500, 4096), (1500, 8192), (700, 16384)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", ROWS)
@pytest.mark.parametrize("kind,dtype,bias", [("layer", BF16, True), ("rms", F32, False), ("rms", F16, True), ("layer", F32, False)], ids=str)
def test_sums_over_all_rows(rows, width, kind, dtype, bias):
    """Without a gate, with one per channel, per token and per element: what a block adds up and what the blocks' sums add up to."""
    for k, gate in enumerate(("none", "channel", "token", "element")):
        t, dy = case((rows, width), dtype, gate, post=True, bias=bias, param_dtype=dtype if k % 2 else F32, seed=width + k)
        compare(t, kind, dy, None)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", ROWS)
@pytest.mark.parametrize("kind,dtype", [("layer", BF16), ("rms", F32), ("rms", F16)], ids=str)
def test_sums_of_the_second_norm(rows, width, kind, dtype):
    for branch in (False, True):
        t, dh = pre_case((rows, width), dtype, branch=branch, param_dtype=(F32, dtype)[branch], seed=width)
        compare(t, kind, None, dh)


# more samples than blocks (a block goes through several), and fewer (a sample is cut into several parts)
SAMPLES = [(20_000, 2, 8), (5000, 2, 64), (4000, 3, 128), (3000, 5, 256), (3000, 2, 512), (1700, 3, 1024), (1700, 3, 2048), (900, 2, 4096), (600, 2, 8192),
           (600, 2, 16384), (3, 9000, 64), (10, 600, 1024), (7, 300, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SAMPLES, ids=str)
@pytest.mark.parametrize("kind,dtype,bias", [("layer", BF16, True), ("rms", F32, False)], ids=str)
def test_sums_of_samples(shape, kind, dtype, bias):
    """A gate per sample is part of what its rows add, so that each sample's share of the weights' sums has a factor of its own."""
    for post in (True, False):
        t, dy = case(shape, dtype, "sample", post=post, bias=bias, param_dtype=(dtype, F32)[post], seed=shape[2])
        compare(t, kind, dy, None)


ODD = [(9000, 7), (9000, 40), (9000, 101), (9000, 200), (6000, 333), (6000, 640), (6000, 1300), (3000, 2049), (3000, 2309), (1500, 4507), (1200, 6000), (600, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", ODD)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_sums_of_odd_widths(rows, width, dtype):
    """Without a norm the sums are exact at any width.  With the second norm (rms: deviation 1) its factor is off by a few steps of 2^-24,
    and a sum of positive terms by one a step on its path: rows of a lane (rows / 256 at most), groups of a block, partial sums of a lane."""
    for gate in ("channel", "token", "element"):
        t, dy = case((rows, width), dtype, gate, post=False, bias=False, seed=width)
        compare(t, "rms", dy, None)
    t, dy = case((rows // 5, 5, width), dtype, "sample", post=False, bias=False, seed=width)
    compare(t, "rms", dy, None)
    t, dh = pre_case((rows, width), dtype, branch=False, seed=width)
    want, got = sums(t, "rms", None, dh), run(t, "rms", None, dh)
    assert torch.equal(got["pre_bias"], want["pre_bias"])
    path = 8 + -(-rows // 256) + 32 + 64
    assert ((got["pre_weight"].double() - want["pre_weight"].double()).abs() <= path * 2.0 ** -24 * want["pre_weight"].abs()).all()


def _changed(a, b):
    return ((a.double() - b.double()).abs() >= 1 / 32).all()


def test_a_lost_row_shows():
    """Of the operands above, by the definition alone: without any one row every sum over rows is another one."""
    for gate in ("none", "channel", "token", "element"):
        for bias in (True, False):
            t, dy = case((64, 16), F32, gate, post=True, bias=bias, seed=3)
            want = sums(t, "layer", dy, None)
            for row in (0, 17, 63):
                less = dy.clone()
                less[row] = 0
                for n, v in sums(t, "layer", less, None).items():
                    by_row = n == "gate" and gate in ("token", "element")
                    assert _changed(v[row], want[n][row]) if by_row else _changed(v, want[n]), (gate, n)
    t, dy = case((30, 2, 16), F32, "sample", post=True, bias=True, seed=4)
    want = sums(t, "rms", dy, None)
    for sample in (0, 29):
        less = dy.clone()
        less[sample, 1] = 0
        got = sums(t, "rms", less, None)
        assert all(_changed(got[n][sample] if n == "gate" else got[n], want[n][sample] if n == "gate" else want[n]) for n in got)
    t, dh = pre_case((64, 16), F32, branch=False, seed=5)
    less = dh.clone()
    less[40] = 0
    a, b = sums(t, "layer", None, dh), sums(t, "layer", None, less)
    assert _changed(a["pre_weight"], b["pre_weight"]) and _changed(a["pre_bias"], b["pre_bias"])


def test_nothing_rounds():
    """The largest sum in its smallest unit: |d z| 3 (6 without a norm), weight, gate and scale 2, bias 1/4, residual scale 1/2; unit 1/32."""
    for rows in [r for r, _ in ROWS + ODD] + [s[0] * s[1] for s in SAMPLES] + [w for _, w in ROWS + ODD]:
        assert rows * 0.5 * 2 * max(3 * 2 + 3 / 4, 6) * 32 <= 2 ** 24
