"""The global gradient norm, clipping and the clipped Adam step over lists of tensors against their definitions in 64 bits."""
import math

import pytest
import torch

from fluidnet_amd.engine.runtime import FluidNetHipError
from fluidnet_amd.training.grad_clip import clip_grad_norm_, clip_grads_with_norm_, total_grad_norm
from fluidnet_amd.training.optim import ClipAdam, clip_adam_

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _list(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=g)).to(dtypes[k % len(dtypes)]).cuda() for k, n in enumerate(sizes)]


def _params(grads):
    ps = []
    for v in grads:
        p = torch.nn.Parameter(torch.zeros(v.shape, dtype=v.dtype, device="cuda"))
        p.grad = v
        ps.append(p)
    return ps


def _norm64(tensors, p):
    flat = torch.cat([t.double().reshape(-1).cpu() for t in tensors]).abs()
    return float(flat.max()) if p == math.inf else float((flat ** p).sum() ** (1 / p))


def _check_norm(got, tensors, p):
    """64-bit sums of at most 2^27 terms: 2^-26 of the norm at worst; then one rounding to 32 bits."""
    want = _norm64(tensors, p)
    if want >= 2.0 ** 128 - 2.0 ** 103:        # beyond half a step above the largest 32-bit value: it rounds to infinity
        assert math.isinf(float(got))
        return
    assert got.dtype == F32 and got.shape == () and abs(float(got) - want) <= (2.0 ** -24 + 2.0 ** -26) * want + 2.0 ** -149, (float(got), want)


def _check_scaled(after, before, coef):
    """The coefficient is rounded to 32 bits, the product to 32 bits and to its type."""
    for k, (a, b) in enumerate(zip(after, before)):
        want, f = b.double() * coef, torch.finfo(a.dtype)
        err = (a.double() - want).abs()
        assert bool((err <= (f.eps / 2 + 2 ** -23) * want.abs() + f.tiny).all()), (k, float(err.max()))


SIZES = {
    "one": [1], "tiny": [1, 2, 3, 5, 7], "vector edges": [7, 8, 9, 15, 16, 17, 2047, 2048, 2049], "chunk edges": [8191, 8192, 8193, 16383, 16384, 16385],
    "many": [k % 13 + 1 for k in range(1000)], "table edge 240": [3] * 240, "table edge 241": [3] * 241, "large": [3_000_001, 1, 700_000, 0, 12],
}


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=str)
@pytest.mark.parametrize("name", list(SIZES))
def test_norm_and_clip(name, dtypes, p):
    grads = _list(SIZES[name], dtypes, seed=len(name))
    before = [g.clone() for g in grads]
    _check_norm(total_grad_norm(grads, p), grads, p)
    want = _norm64(grads, p)
    total = clip_grad_norm_(_params(grads), 0.25 * want, norm_type=p)
    _check_norm(total, before, p)
    _check_scaled(grads, before, 0.25 * want / (want + 1e-6))
    kept = [g.clone() for g in grads]
    clip_grad_norm_(_params(grads), 2 * want, norm_type=p)            # below the limit nothing changes, not by a bit
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))


def test_packed_views_at_every_offset():
    """Gradients packed into one bucket: any start, and nothing between or behind them is touched."""
    for dtype in (F32, BF16, F16):
        buf = torch.randn(40_000, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
        before = buf.clone()
        views, at, inside = [], 1, torch.zeros(40_000, dtype=torch.bool)
        for k in range(60):
            n = (37 * k * k) % 1201 + 1
            views.append(buf[at:at + n])
            inside[at:at + n] = True
            at += n + k % 3
        want = _norm64(views, 2.0)
        total = clip_grad_norm_(_params(views), 0.5)
        _check_norm(total, [before[inside.cuda()]], 2.0)
        assert torch.equal(buf[~inside.cuda()], before[~inside.cuda()])
        _check_scaled([buf[inside.cuda()]], [before[inside.cuda()]], 0.5 / (want + 1e-6))


def test_strided_gradients():
    """Dense in another order, slices of larger buffers (one launch each), and what lies between the slices."""
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(30, 50, 8, generator=g).cuda()
    before = wide.clone()
    grads = [wide[:, :20, 1:6], wide[:, 25:, ::2], torch.randn(16, 9, 3, 3, generator=g).cuda().to(memory_format=torch.channels_last),
             torch.randn(12, 7, generator=g).cuda().t(), torch.randn(5, generator=g).half().cuda(), torch.randn(6, 4, generator=g).bfloat16().cuda()[:, 1]]
    copies = [v.clone() for v in grads]
    for p in (2.0, 1.0, math.inf):
        _check_norm(total_grad_norm(grads, p), grads, p)
    ps = []
    for v in grads:                            # .grad of another layout than the parameter's is taken as it is
        q = torch.nn.Parameter(torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device="cuda"))
        q.grad = v
        ps.append(q)
    want = _norm64(copies, 2.0)
    _check_norm(clip_grad_norm_(ps, 1.0), copies, 2.0)
    _check_scaled([v.contiguous() for v in grads], [v.contiguous() for v in copies], 1 / (want + 1e-6))
    mask = torch.ones_like(wide, dtype=torch.bool)
    mask[:, :20, 1:6] = False
    mask[:, 25:, ::2] = False
    assert torch.equal(wide[mask], before[mask])
    only = [torch.nn.Parameter(torch.zeros(20, 5, device="cuda"))]
    only[0].grad = torch.randn(20, 9, generator=g).cuda()[:, 2:7]
    kept = only[0].grad.clone()
    _check_norm(clip_grad_norm_(only, 0.1), [kept], 2.0)


def test_refusals():
    t = torch.zeros(10, device="cuda")
    with pytest.raises(FluidNetHipError, match="share memory"):
        clip_grad_norm_(_params([t, t]), 1.0)
    with pytest.raises(FluidNetHipError, match="share memory"):
        clip_grad_norm_(_params([t[:6], t[5:]]), 1.0)
    _check_norm(total_grad_norm([t + 1, t + 1]), [t + 1, t + 1], 2.0)
    wide = torch.ones(6, 4, device="cuda")
    with pytest.raises(ValueError, match="twice"):
        clip_grad_norm_(_params([wide[:, 1], wide[:, 1]]), 1.0)
    for bad in (torch.zeros(3, device="cuda", dtype=torch.float64), torch.zeros(3, device="cuda", dtype=torch.int32), torch.zeros(3),
                torch.zeros(1, 4, device="cuda").expand(3, 4), torch.zeros([3] * 7, device="cuda").permute(6, 5, 4, 3, 2, 1, 0)[::2, ::2, ::2, ::2, ::2, ::2, ::2]):
        with pytest.raises((ValueError, RuntimeError)):
            total_grad_norm([t, bad])
    with pytest.raises(ValueError, match="total_norm"):
        clip_grads_with_norm_(_params([t]), 1.0, torch.ones(()))
    with pytest.raises(ValueError, match="total_norm"):
        clip_grads_with_norm_(_params([t]), 1.0, torch.ones(2, device="cuda"))


def test_values_that_are_not_finite():
    """As torch scales by such a norm; with error_if_nonfinite the gradients stay as they were."""
    for value in (math.nan, math.inf, -math.inf):
        for p in (2.0, 1.0, math.inf):
            grads = _list([500, 9], (F32, BF16))
            grads[0][77] = value
            theirs = [g.clone() for g in grads]
            kept = [g.clone() for g in grads]
            with pytest.raises(RuntimeError, match="not finite"):
                clip_grad_norm_(_params(grads), 1.0, norm_type=p, error_if_nonfinite=True)
            assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(grads, kept))
            want = torch.nn.utils.clip_grad_norm_(_params(theirs), 1.0, norm_type=p)
            got = clip_grad_norm_(_params(grads), 1.0, norm_type=p)
            assert torch.equal(got.nan_to_num(7), want.float().nan_to_num(7)), (value, p)
            assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(grads, theirs)), (value, p)


def test_large_and_small_gradients():
    """Squares beyond 32 bits, and a long list of small gradients behind a large one."""
    big = [torch.full((1000,), 1e30, device="cuda"), torch.full((8,), -3e38, device="cuda")]
    _check_norm(total_grad_norm(big), big, 2.0)
    small = [torch.full((1 << 20,), 1e-3, device="cuda"), torch.tensor([4096.0], device="cuda")]
    _check_norm(total_grad_norm(small), small, 2.0)
    none = [torch.zeros(5, device="cuda"), torch.zeros(0, device="cuda")]
    assert float(clip_grad_norm_(_params(none), 1.0)) == 0.0 and not none[0].any()
    empty = [torch.zeros(0, device="cuda")]
    assert float(clip_grad_norm_(_params(empty), 1.0)) == 0.0 and float(total_grad_norm(empty)) == 0.0
    ones = [torch.ones(4, device="cuda")]
    clip_grad_norm_(_params(ones), 0.0)
    assert not ones[0].any()


def test_a_tensor_of_several_table_entries():
    """More than 2^30 elements: the part behind the border is summed and scaled like the rest."""
    n = (1 << 30) + 12345
    g = torch.zeros(n, dtype=BF16, device="cuda")
    g[5], g[(1 << 30) - 1], g[1 << 30], g[-1] = 1.0, 2.0, 4.0, 8.0
    total = clip_grad_norm_(_params([g]), 1.0)
    assert abs(float(total) - math.sqrt(85)) < 1e-6 * 10
    at = torch.tensor([5, (1 << 30) - 1, 1 << 30, n - 1], device="cuda")
    _check_scaled([g[at]], [torch.tensor([1.0, 2.0, 4.0, 8.0], device="cuda").to(BF16)], 1 / (math.sqrt(85) + 1e-6))
    assert int((g != 0).sum()) == 4


def test_error_if_nonfinite_and_given_norm():
    grads = _list([300, 40], (F32, F16))
    before = [g.clone() for g in grads]
    want = _norm64(before, 2.0)
    clip_grad_norm_(_params(grads), 0.5, error_if_nonfinite=True)
    _check_scaled(grads, before, 0.5 / (want + 1e-6))
    again = [g.clone() for g in before]
    clip_grads_with_norm_(_params(again), 0.5, torch.tensor([4.0], dtype=torch.float64, device="cuda"))
    _check_scaled(again, before, 0.5 / (4.0 + 1e-6))
    v = before[0]._version
    clip_grad_norm_(_params([before[0]]), 1e-3)
    assert before[0]._version > v                      # autograd sees that the gradient was written


# ---------------------------------------------------------------------------------------------------------------- Adam
def _state(sizes, dtype, seed=0, shapes=None):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n, s: (s * torch.randn(n, generator=g)).cuda()  # noqa: E731
    p, gr = [rnd(n, 1.0).to(dtype) for n in sizes], [rnd(n, 0.1).to(dtype) for n in sizes]
    m, v = [rnd(n, 0.01) for n in sizes], [rnd(n, 0.01).square() for n in sizes]
    w = None if dtype is F32 else [q.float() + 1e-4 * q.float() for q in p]
    return p, gr, m, v, w


def _adam64(p, g, m, v, w, t, lr, b1, b2, eps, wd, max_norm):
    """The step in 64 bits on the CPU: new (weight, m, v), the update's size without cancellation in m, and the norm."""
    d = lambda ts: [x.detach().cpu().double() for x in ts]  # noqa: E731
    g, m, v, w = d(g), d(m), d(v), d(p if w is None else w)
    norm = math.sqrt(sum(float((x * x).sum()) for x in g))
    c = 1.0 if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
    m0, m = m, [b1 * a + (1 - b1) * c * x for a, x in zip(m, g)]
    v = [b2 * a + (1 - b2) * (c * x) ** 2 for a, x in zip(v, g)]
    rate = [lr / (1 - b1 ** t) / (torch.sqrt(y / (1 - b2 ** t)) + eps) for y in v]
    w = [a * (1 - lr * wd) - r * x for a, x, r in zip(w, m, rate)]
    return w, m, v, [r * (b1 * x.abs() + (1 - b1) * c * y.abs()) for r, x, y in zip(rate, m0, g)], norm


def _check_adam(got, want, g, lr, b1=0.9, wd=0.0):
    """Every 32-bit operation rounds by 2^-24: some eight on the way to m and v (of the sum of their two terms), sixteen more to the
    update, whose magnitude before m's two terms cancel is `size`; two on the weight."""
    (p, m, v, w), (w64, m64, v64, size) = got, want
    for k in range(len(p)):
        mm, vv = m[k].cpu().double(), v[k].cpu().double()
        tm = 8 * 2.0 ** -24 * (m64[k].abs() + 2 * (1 - b1) * g[k].cpu().double().abs()) + 1e-45
        assert bool(((mm - m64[k]).abs() <= tm).all()), ("m", k)
        assert bool(((vv - v64[k]).abs() <= 8 * 2.0 ** -24 * v64[k] + 1e-45).all()), ("v", k)
        master = (p[k] if w is None else w[k]).cpu().double()
        step = (w64[k] - master).abs()
        up = 24 * 2.0 ** -24 * size[k] + 2.0 ** -23 * w64[k].abs()
        assert bool((step <= up).all()), ("w", k, float((step - up).max()))
        if w is not None:
            assert torch.equal(p[k], w[k].to(p[k].dtype))             # the parameter is the master's rounding


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e9])
@pytest.mark.parametrize("name", ["one", "tiny", "vector edges", "chunk edges", "many", "large", "table edge"])
def test_adam_step(name, dtype, max_norm):
    sizes = {"table edge": [5] * 80 + [4096] * 2, **SIZES}[name]
    p, g, m, v, w = _state(sizes, dtype, seed=3)
    kept = [x.clone() for x in g]
    lr, wd = 1e-3, 0.1 if max_norm else 0.0
    clock = torch.tensor([6.0, 0.9 ** 6, 0.999 ** 6], dtype=torch.float64, device="cuda")
    *want, norm = _adam64(p, g, m, v, w, 7, lr, 0.9, 0.999, 1e-8, wd, max_norm)
    total = clip_adam_(p, g, m, v, clock, masters=w, lr=lr, weight_decay=wd, max_norm=max_norm)
    assert (total is None) if max_norm is None else abs(float(total) - norm) <= 2.0 ** -23 * norm
    _check_adam((p, m, v, w), want, g, lr, wd=wd)
    assert all(torch.equal(a, b) for a, b in zip(g, kept))            # the gradients stay
    assert torch.allclose(clock.cpu(), torch.tensor([7.0, 0.9 ** 7, 0.999 ** 7], dtype=torch.float64), rtol=1e-14, atol=0)


def test_adam_refusals():
    p, g, m, v, w = _state([8, 8], BF16)
    clock = torch.tensor([0.0, 1.0, 1.0], dtype=torch.float64, device="cuda")
    kw = dict(lr=1e-3, max_norm=1.0)
    for args, extra, match in (
            ((p, g, m, v, clock), {}, "needs an fp32 master"), ((p, [x.float() for x in g], m, v, clock), dict(masters=w), "one type"),
            ((p, g, [x.half() for x in m], v, clock), dict(masters=w), "float32"), ((p, g, m, v, clock.float()), dict(masters=w), "clock"),
            ((p, g, m, v, clock[:2]), dict(masters=w), "clock"), ((p, g, m, [x[:4] for x in v], clock), dict(masters=w), "laid out"),
            ((p, g, m, v, clock), dict(masters=w, lr=torch.ones((), device="cuda")), "lr"),
            (([x[::2] for x in p], [x[::2] for x in g], m, v, clock), dict(masters=w), "dense")):
        with pytest.raises(ValueError, match=match):
            clip_adam_(*args, **{**kw, **extra})
    with pytest.raises(FluidNetHipError, match="share memory"):
        clip_adam_(p, g, m, m, clock, masters=w, **kw)
    with pytest.raises(FluidNetHipError, match="share memory"):
        clip_adam_([p[0], p[0]], g, m, v, clock, masters=w, **kw)


def test_refused_step_changes_nothing():
    """A step that is refused for what it would write leaves the clock as it was, too; gradients may share memory among themselves only."""
    p, g, m, v, w = _state([8, 8, 0], F32)
    clock = torch.tensor([3.0, 0.9 ** 3, 0.999 ** 3], dtype=torch.float64, device="cuda")
    before = [t.clone() for t in (*p, *g, *m, *v, clock)]
    for args in (([p[0], p[0], p[2]], g, m, v), (p, [m[1], g[1], g[2]], m, v), (p, [g[0], p[0], g[2]], m, v), (p, g, m, m)):
        for max_norm in (1.0, None):
            with pytest.raises(FluidNetHipError, match="share memory"):
                clip_adam_(*args, clock, lr=1e-3, max_norm=max_norm)
    assert all(torch.equal(a, b) for a, b in zip(before, (*p, *g, *m, *v, clock)))
    clip_adam_(p, [g[0], g[0], g[2]], m, v, clock, lr=1e-3, max_norm=1.0)
    assert clock[0].item() == 4.0 and not torch.equal(m[0], before[6])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_optimizer_against_torch(dtype):
    """Ten steps of ClipAdam and of torch's clip_grad_norm_ + AdamW in 64 bits on the same gradients.  Each step adds at most the bound of one
    step (see _check_adam); a parameter in another memory layout, one without a gradient, learning rate changes, state saved and loaded."""
    g = torch.Generator().manual_seed(0)
    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(5)).cuda().to(dtype)) for s in ((40, 30), (7,), (6, 5, 3, 3), (2,))]  # noqa: E731
    ps = make()
    ps[2] = torch.nn.Parameter(ps[2].detach().to(memory_format=torch.channels_last))
    ref = [torch.nn.Parameter(p.detach().cpu().double()) for p in ps]
    opt, theirs = ClipAdam(ps, 1e-2, max_norm=1.0, weight_decay=0.05), torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.05)
    for step in range(10):
        if step == 4:
            for o in (opt, theirs):
                o.param_groups[0]["lr"] = 3e-3
        if step == 6:                          # into a new optimizer
            sd = opt.state_dict()
            opt = ClipAdam(ps, 1e-2, max_norm=1.0, weight_decay=0.05)
            opt.load_state_dict(sd)
            assert opt.step_count == 6 and opt.param_groups[0]["lr"] == 3e-3
        opt.zero_grad()
        for p, r in zip(ps[:3], ref[:3]):
            grad = torch.randn(p.shape, generator=g)
            p.grad = grad.cuda().to(dtype)
            r.grad = p.grad.cpu().double()
        opt.step()
        torch.nn.utils.clip_grad_norm_(ref, 1.0)
        theirs.step()
    assert abs(float(opt.grad_norm) - math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps[:3]))) < 1e-4
    for k, (p, r, w) in enumerate(zip(ps[:3], ref, opt._w)):
        have = (p if w is None else w).detach().cpu().double()
        assert bool(((have - r.detach()).abs() <= 10 * (160 * 2.0 ** -24 * 1e-2 / 0.1 + 2.0 ** -23 * r.detach().abs())).all()), k
    assert torch.equal(ps[3].cpu(), make()[3].cpu()) and opt.step_count == 10


def test_master_follows_a_parameter_written_from_outside():
    p = torch.nn.Parameter(torch.ones(16, device="cuda", dtype=BF16))
    opt = ClipAdam([p], 1e-3, max_norm=None)
    p.grad = torch.ones_like(p)
    opt.step()
    with torch.no_grad():
        p.fill_(5.0)
    p.grad = torch.ones_like(p)
    opt.step()
    assert float((opt._w[0] - 5.0).abs().max()) < 2e-3 and float((p.detach() - 5.0).abs().max()) < 0.02
    p.data.fill_(-2.0)
    opt.refresh()
    p.grad = torch.ones_like(p)
    opt.step()
    assert float((opt._w[0] + 2.0).abs().max()) < 4e-3


def test_optimizer_takes_gradients_of_any_layout():
    """A gradient that is a slice of a wider buffer, or transposed, gives the step of its contiguous copy."""
    g = torch.Generator().manual_seed(8)
    a, b = ([torch.nn.Parameter(torch.randn(6, 5, generator=torch.Generator().manual_seed(1)).cuda()) for _ in range(2)] for _ in range(2))
    wide = torch.randn(6, 12, generator=g).cuda()
    a[0].grad, a[1].grad = wide[:, 2:7], torch.randn(5, 6, generator=g).cuda().t()
    for p, q in zip(a, b):
        q.grad = p.grad.contiguous()
    for ps in (a, b):
        ClipAdam(ps, 1e-2, max_norm=0.1).step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_graphs_of_clip_and_step():
    """A captured clip and a captured optimizer step, replayed on new gradients with eager work between; the step count goes on, the learning
    rate is read anew.  Compared with the eager calls, bit for bit; two graphs that were captured one after the other do not share anything."""
    sizes = [5, 1000, 70_000]
    grads = _list(sizes, (F32, BF16, F16))
    ps = _params(grads)
    mine = [torch.nn.Parameter(torch.ones(n, device="cuda", dtype=BF16)) for n in sizes]
    other = [torch.nn.Parameter(torch.ones(n, device="cuda", dtype=BF16)) for n in sizes]
    for a in (mine, other):
        for p in a:
            p.grad = torch.zeros_like(p)
    opt, eager = ClipAdam(mine, 1e-2, max_norm=0.7), ClipAdam(other, 1e-2, max_norm=0.7)
    opt.step()
    eager.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grad_norm_(ps, 1e9)
    torch.cuda.current_stream().wait_stream(side)
    clip_graph, step_graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(clip_graph):
        total = clip_grad_norm_(ps, 0.5)
    with torch.cuda.graph(step_graph):
        opt.step()
    for seed in range(4):
        new = _list(sizes, (F32, BF16, F16), seed=20 + seed, scale=0.1 + seed)
        with torch.no_grad():
            for a, b in zip(grads, new):
                a.copy_(b)
            for a, b, c in zip(mine, other, new):
                a.grad.copy_(c)
                b.grad.copy_(c)
        for o in (opt, eager):
            o.param_groups[0]["lr"] = 1e-2 / (seed + 1)
        opt.push_lr()
        step_graph.replay()
        clip_graph.replay()
        torch.cuda.synchronize()
        want = clip_grad_norm_(_params(new), 0.5)
        assert torch.equal(total, want) and all(torch.equal(a, b) for a, b in zip(grads, new))
        eager.step()
        assert all(torch.equal(a, b) for a, b in zip(mine, other)) and all(torch.equal(a, b) for a, b in zip(opt._v, eager._v))
        assert torch.equal(opt.grad_norm, eager.grad_norm)
    assert opt.step_count == eager.step_count == 5
    fresh = ClipAdam([torch.nn.Parameter(torch.ones(3, device="cuda"))], 1e-2)
    fresh.params[0].grad = torch.ones(3, device="cuda")
    with pytest.raises(RuntimeError, match="eager step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.zeros(1, device="cuda").add_(1)
            fresh.step()
