"""The norms around a residual block (fluidnet_amd/models/block_norm.py) against their definition in 64 bits: types, widths from 1 to the
largest of every row layout, gates of every shape, strides, no rows, values that are not finite, other streams, graphs."""
import gc
import itertools

import pytest
import torch
import torch.utils.checkpoint

import block_norm_ref as ref
from fluidnet_amd.models.block_norm import MAX_WIDTH, GatedResidual, PreNorm, gated_residual, pre_norm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def operands(shape, dtype=F32, *, gate="none", scale=False, bias=False, post=True, pre=True, branch=True, weights=True, param_dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": (rnd(*shape) * 2 + 0.5).to(dtype), "post": post and branch, "pre": pre}
    if branch:
        t["branch"] = (rnd(*shape) - 0.3).to(dtype)
        gs = {"none": None, "element": shape, "token": (*shape[:-1], 1), "sample": (shape[0], *[1] * (len(shape) - 2), C), "channel": (C,),
              "channel-wide": (*[1] * (len(shape) - 1), C)}[gate]
        if gs:
            t["gate"] = rnd(*gs).to(dtype if gate in ("element", "token", "sample") else param_dtype)
        if scale:
            t["scale"] = (0.5 + 0.2 * rnd(C)).to(param_dtype)
        if post and weights:
            t["post_weight"] = (1 + 0.2 * rnd(C)).to(param_dtype)
            if bias:
                t["post_bias"] = (0.2 * rnd(C)).to(param_dtype)
    if pre and weights:
        t["pre_weight"] = (1 + 0.2 * rnd(C)).to(param_dtype)
        if bias:
            t["pre_bias"] = (0.2 * rnd(C)).to(param_dtype)
    dy = (0.3 * rnd(*shape)).to(dtype) if branch else None
    dh = (0.3 * rnd(*shape)).to(dtype) if pre else None
    return t, dy, dh


def call(t, kind, act, a, eps):
    if t.get("branch") is None:
        return None, pre_norm(t["x"], t.get("pre_weight"), t.get("pre_bias"), kind=kind, eps=eps)
    return gated_residual(t["x"], t["branch"], t.get("gate"), t.get("scale"), post_weight=t.get("post_weight"), post_bias=t.get("post_bias"),
                          pre_weight=t.get("pre_weight"), pre_bias=t.get("pre_bias"), kind=kind, post=t["post"], pre=t["pre"], gate_act=act,
                          residual_scale=a, eps=eps)


def gpu(t, grad=False):
    return {k: v.cuda().requires_grad_(grad) if isinstance(v, torch.Tensor) else v for k, v in t.items()}


def both(t, dy, dh, kind="rms", act="identity", a=0.7, eps=1e-6, on=None):
    """Forward and backward against the definition; `on` lays the operands out on the GPU in a way of its own."""
    want, tol = ref.reference(t, kind, act, a, eps, dy, dh), ref.tolerance(t, kind, act, a, eps, dy, dh)
    d = gpu(t, True) if on is None else on(t)
    y, h = call(d, kind, act, a, eps)
    names = [n for n in ref.NAMES if d.get(n) is not None]
    outs = [(o, g.cuda()) for o, g in ((y, dy), (h, dh)) if o is not None and g is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [d[n] for n in names], [g for _, g in outs], allow_unused=True)
    got = {"y": y, "h": h, **{"d_" + n: v for n, v in zip(names, grads)}}
    for k, v in got.items():
        if want.get(k) is None:
            assert v is None or not v.any(), k
            continue
        assert v.dtype == (d[k[2:]] if k.startswith("d_") else d["x"]).dtype and v.shape == want[k].shape, k
        ref.check(v, want[k], tol[k], k)
    with torch.no_grad():                      # the serving form gives the same bits
        y2, h2 = call(d, kind, act, a, eps)
    assert (y is None or torch.equal(y, y2)) and (h is None or torch.equal(h, h2))


WIDTHS = [1, 2, 7, 8, 9, 63, 64, 65, 128, 129, 200, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096, 4099, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_widths(width, dtype):
    k = WIDTHS.index(width)
    rows = 37 if width <= 512 else 5
    t, dy, dh = operands((rows, width), dtype, gate=("none", "element", "token")[k % 3], bias=k % 2 == 0, seed=width)
    both(t, dy, dh, kind=("rms", "layer")[(k // 2) % 2], act=("identity", "sigmoid", "tanh")[k % 3])


@pytest.mark.parametrize("gate", ["none", "element", "token", "sample", "channel", "channel-wide"])
@pytest.mark.parametrize("act", ["identity", "sigmoid", "tanh"])
@pytest.mark.parametrize("shape", [(3, 50, 40), (5, 2, 7, 72), (2, 300, 520), (1, 4, 1100)], ids=str)
def test_gates(gate, act, shape):
    if gate == "none" and act != "identity":
        pytest.skip("nothing to activate")
    i = ("none", "element", "token", "sample", "channel", "channel-wide").index(gate)
    t, dy, dh = operands(shape, (BF16, F32)[i % 2], gate=gate, scale=i % 2 == 1, bias=True, param_dtype=(F32, F32, BF16)[i % 3] if i % 2 == 0 else F32, seed=i)
    both(t, dy, dh, kind=("layer", "rms")[shape[0] % 2], act=act)


@pytest.mark.parametrize("post,pre,branch", [(True, False, True), (False, True, True), (False, False, True), (False, True, False), (True, True, True)])
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_parts(post, pre, branch, weights, kind):
    for shape, dtype in (((6, 33, 96), BF16), ((70, 640), F32)):
        t, dy, dh = operands(shape, dtype, gate="token" if branch else "none", scale=branch and weights, bias=weights, post=post, pre=pre,
                             branch=branch, weights=weights)
        both(t, dy, dh, kind=kind, act="sigmoid")


def test_a_single_vector():
    """x of one axis: one row, with a gate per element or one value."""
    for gate, width in (("element", 70), ("token", 300)):
        t, dy, dh = operands((width,), BF16, gate="element", bias=True)
        if gate == "token":
            t["gate"] = t["gate"][:1]
        both(t, dy, dh, kind="layer", act="tanh")
        both(t, dy, dh, on=lambda t: {k: v.cuda().repeat_interleave(2)[::2].detach().requires_grad_(True) if isinstance(v, torch.Tensor) else v
                                      for k, v in t.items()})


@pytest.mark.parametrize("shape", [(0, 64), (4, 0, 1024), (0, 3, 8), (1, 1), (1, 4096), (8192, 8), (3, 1, 16), (17, 1, 33), (1100, 2, 40), (2100, 3, 24)],
                         ids=str)
def test_rows(shape):
    """No rows, one row, many; per-sample gates with one, two and three tokens per sample, and more samples than blocks."""
    gate = "sample" if len(shape) == 3 else "channel"
    t, dy, dh = operands(shape, BF16, gate=gate, scale=True, bias=True)
    if 0 not in shape:
        return both(t, dy, dh, kind="layer", act="tanh")
    d = gpu(t, True)
    y, h = call(d, "layer", "tanh", 1.0, 1e-6)
    assert y.shape == h.shape == torch.Size(shape)
    names = [n for n in ref.NAMES if n in d]
    for n, g in zip(names, torch.autograd.grad([y, h], [d[n] for n in names], [dy.cuda(), dh.cuda()])):
        assert g.shape == d[n].shape and g.dtype == d[n].dtype and not g.any(), n


@pytest.mark.parametrize("width,rows", [(1300, 6000), (1100, 9000), (640, 6000), (2049, 3000), (4507, 1500), (6000, 1200), (9000, 600), (500, 9000), (40, 40_000)])
def test_many_rows(width, rows):
    """More rows than the GPU holds blocks of, for rows of 2, 3, 5, 9, 12 and 16 waves: the partial sums of every block."""
    t, dy, dh = operands((rows, width), BF16, gate="channel", bias=True, seed=width)
    both(t, dy, dh, kind="layer", act="sigmoid")
    t, dy, dh = operands((10, rows // 10, width), F32 if width < 2000 else F16, gate="sample", scale=True, seed=width)
    both(t, dy, dh, act="tanh")


@pytest.mark.parametrize("shape", [(2500, 2, 40), (3000, 2, 520), (1700, 3, 1300), (900, 2, 2309), (600, 2, 8200)], ids=str)
def test_many_samples(shape):
    """Several samples to a block, each with its gate: the sums over all of them, in every layout of rows."""
    for kind, act, dtype, bias in (("layer", "sigmoid", BF16, True), ("rms", "tanh", F32, False)):
        t, dy, dh = operands(shape, dtype, gate="sample", scale=True, bias=bias, seed=shape[2])
        both(t, dy, dh, kind=kind, act=act)


def test_no_second_derivative():
    t, dy, dh = operands((3, 16), F32)
    d = gpu(t, True)
    y, h = call(d, "rms", "identity", 1.0, 1e-6)
    g, = torch.autograd.grad([y, h], [d["x"]], [dy.cuda().requires_grad_(True), dh.cuda()], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_node_is_an_ordinary_one():
    """What autograd promises of any operation: operands changed in place are noticed, a graph is used up by a backward pass, saved tensors go
    through hooks (checkpointing among them), subsets of gradients, leaves that appear twice."""
    t, dy, dh = operands((6, 48), F32, gate="element", scale=True, bias=True)
    dyg, dhg = dy.cuda(), dh.cuda()
    names = [n for n in ref.NAMES if n in t]

    def once(d):
        return call(d, "layer", "tanh", 1.0, 1e-6)

    def grads(d, out, which=names, **kw):
        return torch.autograd.grad(out, [d[n] for n in which], [dyg, dhg], **kw)
    d = gpu(t, True)
    out = once(d)
    want = grads(d, out, retain_graph=True)
    for n, g in zip(names, want):
        assert torch.equal(grads(d, out, [n], retain_graph=True)[0], g), n
    grads(d, out)
    with pytest.raises(RuntimeError, match="second time"):
        grads(d, out)
    out = once(d)
    with torch.no_grad():
        d["branch"].add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        grads(d, out)
    d = gpu(t, True)
    with torch.autograd.graph.save_on_cpu():
        out = once(d)
    assert all(torch.equal(a, b) for a, b in zip(grads(d, out), want))
    out = torch.utils.checkpoint.checkpoint(lambda *v: once({**d, **dict(zip(names, v))}), *(d[n] for n in names), use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(grads(d, out), want))
    # x as its own branch: its gradient is the sum of both
    x, b = d["x"].detach().requires_grad_(), d["x"].detach().clone().requires_grad_()
    one = torch.autograd.grad(gated_residual(x, x), x, [dyg, dhg])[0]
    two = torch.autograd.grad(gated_residual(d["x"], b), [d["x"], b], [dyg, dhg])
    assert torch.equal(one, two[0] + two[1])
    with torch.inference_mode():
        y, h = once(gpu(t))
    assert y.is_inference() and torch.equal(h, out[1].detach())


def test_other_transforms_are_refused():
    x, w = torch.randn(4, 32, device="cuda"), torch.ones(32, device="cuda")
    with pytest.raises(NotImplementedError, match="forward-mode"), torch.autograd.forward_ad.dual_level():
        pre_norm(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), w)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: pre_norm(v, w))(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: pre_norm(v, w).sum())(x)
    with pytest.raises(TypeError, match="must be a tensor"):
        pre_norm(x, 1.0)


def test_capture_of_a_shape_that_never_ran():
    """The first call of a shape asks the runtime how many blocks fit, also while a graph is captured."""
    t, dy, dh = operands((700, 3333), BF16, gate="channel", bias=True)
    d = gpu(t, True)
    dyg, dhg = dy.cuda(), dh.cuda()
    names = [n for n in ref.NAMES if n in d]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = call(d, "layer", "tanh", 1.0, 1e-6)
        out = [y, h, *torch.autograd.grad([y, h], [d[n] for n in names], [dyg, dhg])]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        y, h = call(gpu(t, True), "layer", "tanh", 1.0, 1e-6)
        assert torch.equal(out[0], y) and torch.equal(out[1], h)
        want, tol = ref.reference(t, "layer", "tanh", 1.0, 1e-6, dy, dh), ref.tolerance(t, "layer", "tanh", 1.0, 1e-6, dy, dh)
        for n, v in zip(names, out[2:]):
            ref.check(v, want["d_" + n], tol["d_" + n], n)


def test_one_gradient_at_a_time():
    """Only dy, only dh, and one operand that needs a gradient: every other one is not computed, the one is as always."""
    t, dy, dh = operands((9, 70), F32, gate="element", scale=True, bias=True)
    for use_dy, use_dh in ((True, False), (False, True)):
        both(t, dy if use_dy else None, dh if use_dh else None, kind="layer", act="sigmoid")
    full = ref.reference(t, "layer", "tanh", 0.7, 1e-6, dy, dh)
    tol = ref.tolerance(t, "layer", "tanh", 0.7, 1e-6, dy, dh)
    for n in ref.NAMES:
        d = gpu(t)
        d[n].requires_grad_(True)
        y, h = call(d, "layer", "tanh", 0.7, 1e-6)
        g, = torch.autograd.grad([y, h], [d[n]], [dy.cuda(), dh.cuda()])
        ref.check(g, full["d_" + n], tol["d_" + n], n)


def _sliced(t, names, pad=3):
    """Operands as slices of the last axis of wider buffers, at an odd offset."""
    d = gpu(t)
    for n in names:
        v = d[n]
        wide = torch.full((*v.shape[:-1], v.shape[-1] + 2 * pad), float("nan"), dtype=v.dtype, device="cuda")
        wide[..., pad:-pad] = v
        d[n] = wide[..., pad:-pad]
    return {k: v.detach().requires_grad_(True) if isinstance(v, torch.Tensor) else v for k, v in d.items()}


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("width", [24, 101, 2000])
def test_strides(dtype, width):
    t, dy, dh = operands((4, 11, width), dtype, gate="element", bias=True)
    both(t, dy, dh, on=lambda t: _sliced(t, ("x", "branch", "gate")))
    t, dy, dh = operands((4, 11, width), dtype, gate="sample", bias=True)
    both(t, dy, dh, on=lambda t: _sliced(t, ("x", "gate", "post_weight", "pre_bias")))
    # a channels-first image seen channels last, rows of a larger batch, a transposed batch: copied, not misread
    def swapped(t):
        d = gpu(t)
        d["x"] = d["x"].transpose(0, 1).contiguous().transpose(0, 1)
        d["branch"] = d["branch"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
        return {k: v.detach().requires_grad_(True) if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    both(t, dy, dh, on=swapped)


def test_broadcast_operands_and_gradients():
    """Stride 0: an expanded x and the gradients that a sum sends back."""
    t, _, _ = operands((6, 5, 48), F32, gate="token")
    t["x"] = t["x"][:1, :1].clone()
    d = gpu(t, True)
    x = d["x"].expand(6, 5, 48)
    y, h = gated_residual(x, d["branch"], d["gate"], post_weight=d["post_weight"], pre_weight=d["pre_weight"])
    (y.sum() + h.sum()).backward()
    w = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in t.items()}
    w["x"] = t["x"].expand(6, 5, 48).clone()
    one = torch.ones(6, 5, 48)
    want, tol = ref.reference(w, "rms", "identity", 1.0, 1e-6, one, one), ref.tolerance(w, "rms", "identity", 1.0, 1e-6, one, one)
    # the 30 copies' gradients are added by torch: 30 more operations on the sum of their magnitudes
    ref.check(d["x"].grad, want["d_x"].sum((0, 1), keepdim=True), tol["d_x"].sum((0, 1), keepdim=True) + 30 * 2.0 ** -24 * want["d_x"].abs().sum((0, 1), keepdim=True), "x")
    for n in ("branch", "gate", "post_weight", "pre_weight"):
        ref.check(d[n].grad, want["d_" + n], tol["d_" + n], n)


def test_same_tensor_twice():
    """x is its own branch: both gradients arrive."""
    t, dy, dh = operands((7, 90), F32)
    t["branch"] = t["x"]
    want, tol = ref.reference(dict(t, branch=t["x"].clone()), "rms", "identity", 1.0, 1e-6, dy, dh), ref.tolerance(t, "rms", "identity", 1.0, 1e-6, dy, dh)
    d = gpu({k: v for k, v in t.items() if k != "branch"}, True)
    d["branch"] = d["x"]
    y, h = call(d, "rms", "identity", 1.0, 1e-6)
    g, = torch.autograd.grad([y, h], [d["x"]], [dy.cuda(), dh.cuda()])
    ref.check(g, want["d_x"] + want["d_branch"], tol["d_x"] + tol["d_branch"] + 2.0 ** -23 * (want["d_x"].abs() + want["d_branch"].abs()), "x")


def test_rows_far_from_zero_and_zero_rows():
    """A mean 1e4 deviations away (the variance is taken about it), a row of zeros, a constant row."""
    t, dy, dh = operands((8, 640), F32, bias=True)
    t["x"] += 1e4
    t["branch"] -= 1e4
    t["x"][1], t["branch"][1] = 0, 0
    t["x"][2], t["branch"][2] = 0, 3.0
    both(t, dy, dh, kind="layer")
    both(t, dy, dh, kind="rms")


@pytest.mark.parametrize("width", [40, 1500])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_values_that_are_not_finite_stay_in_their_row(width, kind):
    t, dy, dh = operands((12, width), BF16, gate="element")
    clean = gpu(t, True)
    y0, h0 = call(clean, kind, "sigmoid", 1.0, 1e-6)
    names = ("x", "branch", "gate")
    g0 = torch.autograd.grad([y0, h0], [clean[n] for n in names], [dy.cuda(), dh.cuda()])
    for row, (name, value) in enumerate([("x", float("nan")), ("branch", float("nan")), ("x", float("inf")), ("branch", -float("inf")), ("gate", float("nan"))]):
        t[name][2 * row + 1, width // 2] = value
    d = gpu(t, True)
    y, h = call(d, kind, "sigmoid", 1.0, 1e-6)
    g = torch.autograd.grad([y, h], [d[n] for n in names], [dy.cuda(), dh.cuda()])
    fine = torch.tensor([0, 2, 4, 6, 8, 10, 11], device="cuda")
    for a, b in zip((y, h, *g), (y0, h0, *g0)):
        assert torch.equal(a[fine], b[fine])
    want = ref.reference(t, kind, "sigmoid", 1.0, 1e-6)
    for got, k in ((y, "y"), (h, "h")):
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want[k])), k


def test_against_differences():
    """Central differences of the 64-bit definition along random directions.  A step of s = 1e-5 leaves s^2 f''' / 6 of the cut series and
    2^-53 |f| / s of the rounding, both below 1e-8 of the magnitudes here; the kernel's own error is that of its type, summed."""
    for kind, gate, act in itertools.product(("rms", "layer"), ("element", "sample", "channel"), ("sigmoid", "tanh")):
        t, dy, dh = operands((3, 6, 40), F32, gate=gate, scale=True, bias=True, seed=len(gate))
        d = gpu(t, True)
        y, h = call(d, kind, act, 0.6, 1e-5)
        names = [n for n in ref.NAMES if n in d]
        grads = torch.autograd.grad([y, h], [d[n] for n in names], [dy.cuda(), dh.cuda()])
        tol = ref.tolerance(t, kind, act, 0.6, 1e-5, dy, dh)
        f64 = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in t.items()}

        def loss(**moved):
            y, h = ref.forward({**f64, **moved}, kind, act, 0.6, 1e-5)
            return float((y * dy.double()).sum() + (h * dh.double()).sum())
        for n, g in zip(names, grads):
            v = torch.randn(f64[n].shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
            diff = (loss(**{n: f64[n] + 1e-5 * v}) - loss(**{n: f64[n] - 1e-5 * v})) / 2e-5
            got = float((g.cpu().double() * v).sum())
            bound = float(((tol["d_" + n] + 2.0 ** -24 * g.cpu().double().abs()) * v.abs()).sum()) + 1e-6 * float((g.cpu().double() * v).abs().sum() + 1)
            assert abs(got - diff) <= bound, (kind, gate, act, n, got, diff)


def test_same_bits_every_time():
    t, dy, dh = operands((40, 60, 264), BF16, gate="sample", scale=True, bias=True)
    def once():
        d = gpu(t, True)
        y, h = call(d, "layer", "sigmoid", 1.0, 1e-6)
        return [y, h, *torch.autograd.grad([y, h], [d[n] for n in ref.NAMES if n in d], [dy.cuda(), dh.cuda()])]
    a, b = once(), once()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_streams():
    """Two calls at once on two streams, each with its own workspace."""
    t, dy, dh = operands((64, 40, 200), F32, gate="channel", bias=True)
    t2, _, _ = operands((64, 40, 200), F32, gate="channel", bias=True, seed=5)

    def once(t):
        d = gpu(t, True)
        y, h = call(d, "layer", "tanh", 1.0, 1e-6)
        return [y, h, *torch.autograd.grad([y, h], [d[n] for n in ref.NAMES if n in d], [dy.cuda(), dh.cuda()])]
    want = [once(t), once(t2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for k, (s, v) in enumerate(zip(streams, (t, t2))):
            with torch.cuda.stream(s):
                got[k] = once(v)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_graph_forward_and_backward():
    """Captured once, replayed on new values with eager work between; every replay is compared."""
    t, dy, dh = operands((5, 30, 520), BF16, gate="sample", scale=True, bias=True)
    d = gpu(t, True)
    dyg, dhg = dy.cuda(), dh.cuda()
    names = [n for n in ref.NAMES if n in d]

    def once(d):
        y, h = call(d, "layer", "sigmoid", 1.0, 1e-6)
        return [y, h, *torch.autograd.grad([y, h], [d[n] for n in names], [dyg, dhg])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(d)
    for seed in range(4):
        new, _, _ = operands((5, 30, 520), BF16, gate="sample", scale=True, bias=True, seed=seed + 10)
        with torch.no_grad():
            for n in names:
                d[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        want = once(gpu(new, True))
        assert all(torch.equal(p, q) for p, q in zip(out, want)), seed


@pytest.mark.parametrize("through", [False, True], ids=["leaf", "view"])
def test_captured_backward_next_to_an_eager_graph(through):
    """A captured backward pass of leaves whose eager graph on the default stream is alive is refused before torch hands anything to a leaf; with
    that graph dropped, or made on a side stream, it is captured and accumulates at every replay."""
    w = torch.rand(264, device="cuda").requires_grad_()
    b = torch.rand(264, device="cuda").requires_grad_()
    x = torch.randn(40, 264, device="cuda")
    up = torch.ones(40, 264, device="cuda")
    param = (lambda: (w[:], b[:])) if through else (lambda: (w, b))

    def once():
        pw, pb = param()
        return gated_residual(x, x, post_weight=pw, pre_weight=pb)[1]
    eager = once()
    eager.backward(up)
    want, w.grad, b.grad = (w.grad, b.grad), torch.zeros_like(w), torch.zeros_like(b)
    for t in (w, b):
        torch.autograd.graph.get_gradient_edge(t).node.metadata["eager"] = True
    torch.cuda.synchronize()
    for backward in (lambda h: h.backward(up), lambda h: torch.autograd.grad(h, [w, b], up), lambda h: torch.autograd.grad(h, [b], up)):
        with pytest.raises(RuntimeError, match="are alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                backward(once())
        torch.cuda.synchronize()
    assert not w.grad.any() and not b.grad.any()
    del eager
    gc.collect()
    # the leaves' nodes are new ones: nothing of the eager graph is left that the capture below could meet
    assert not any(torch.autograd.graph.get_gradient_edge(t).node.metadata for t in (w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once().backward(up)
    torch.cuda.current_stream().wait_stream(side)
    w.grad.zero_()
    b.grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once().backward(up)
    for k in (1, 2, 3):
        graph.replay()
        torch.cuda.synchronize()
        for a, g in zip((w, b), want):
            # k equal terms added up in fp32: each addition is off by half a step at most
            assert ((a.grad.double() - k * g.double()).abs() <= k * 2.0 ** -23 * k * g.double().abs()).all(), k


def test_large_offsets():
    """Rows that begin behind 2^31 elements of their buffer."""
    wide = 1 << 21
    n = 1100                                          # 1100 * 2^21 = 2.3e9 elements of 2 bytes
    buf = torch.empty(n * wide, dtype=BF16, device="cuda").view(n, wide)
    x = buf[:, 5:5 + 96]
    g = torch.Generator(device="cuda").manual_seed(1)
    x.copy_(torch.randn(n, 96, generator=g, device="cuda"))
    w = torch.rand(96, device="cuda")
    assert torch.equal(pre_norm(x, w), pre_norm(x.clone(memory_format=torch.contiguous_format), w))


def test_more_than_2_31_elements():
    """Rows behind 2^31 elements, forward and backward, operands of a stride of their own among them: the last rows as if they were alone."""
    rows, width, last = 265_000, 8192, 3                  # 2.17e9 elements, 4.3 GB each
    x = torch.empty(rows, width, dtype=BF16, device="cuda").fill_(0.5)
    tail = torch.randn(last, width, generator=torch.Generator().manual_seed(7)).to(BF16).cuda()
    x[-last:] = tail
    w = torch.rand(width, device="cuda")
    up = torch.full((1, width), 0.25, dtype=BF16, device="cuda").expand(rows, width)

    def run(x, up):
        x = x.detach().requires_grad_()
        y, h = gated_residual(x, x.detach(), post_weight=w, pre_weight=w, residual_scale=0.5)
        return y.detach()[-last:], h.detach()[-last:], torch.autograd.grad([y, h], x, [up, up])[0][-last:]
    for a, b in zip(run(x, up), run(tail, up[-last:])):
        assert torch.equal(a, b)
    del x
    torch.cuda.empty_cache()


def test_modules():
    m = GatedResidual(96, kind="layer", bias=True, scale_init=0.1, channel_gate=0.0, gate_act="tanh").cuda()
    first = PreNorm(96, kind="layer", bias=True).cuda()
    x = torch.randn(4, 10, 96, device="cuda")
    y, h = m(x, first(x))
    assert torch.equal(y, x)                          # a tanh gate of zero lets nothing through
    (h.square().mean()).backward()
    assert m.gate.grad.abs().sum() > 0 and m.pre_weight.grad is not None
    with pytest.raises(ValueError, match="gate of its own"):
        m(x, x, x)


def test_width_limit():
    with pytest.raises(ValueError, match=str(MAX_WIDTH)):
        pre_norm(torch.zeros(2, MAX_WIDTH + 1, device="cuda"))
