"""What is measured of the block norms, of gradient clipping over many tensors and of the clipped Adam step over a list of parameters.

Three operators:
  block  the norms around a residual block: u = N(branch) * w_post + b_post;  y = x + a * scale * act(gate) * u;
         h = N(y) * w_pre + b_pre  (N: RMS or layer norm over the last axis), forward alone (serving) or with every gradient (training)
  clip   the global norm of the gradients of a list of parameters, and their clipping in place
  adam   one Adam step of a list of parameters on the clipped gradients

`own = False` computes them with elementary torch operations in 32 bits; `own = True` makes the calls of fluidnet_amd.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new token of one sequence: serving, where the launch is all there is
        dict(name="block-one-token", op="block", batch=1, tokens=1, width=4096, dtype="bf16", kind="rms", gate="none", act="identity",
             scale=False, bias=False, post=True, pre=True, branch=True, train=False),
        # a serving batch, one token each, gated per token
        dict(name="block-token-batch", op="block", batch=96, tokens=1, width=8192, dtype="bf16", kind="rms", gate="token", act="sigmoid",
             scale=False, bias=False, post=True, pre=True, branch=True, train=False),
        # a whole prompt before its first answer
        dict(name="block-prompt", op="block", batch=1, tokens=8191, width=4096, dtype="bf16", kind="rms", gate="none", act="identity",
             scale=True, bias=False, post=True, pre=True, branch=True, train=False),
        # a training batch whose blocks are gated per sample
        dict(name="block-train-sample-gate", op="block", batch=16, tokens=1024, width=2048, dtype="bf16", kind="rms", gate="sample",
             act="identity", scale=False, bias=False, post=True, pre=True, branch=True, train=True),
        # the bottleneck of the medium UNet at 128 x 128 and batch 64, channels last: 16 x 16 pixels of 256 channels, learned layer scale
        dict(name="block-train-pixels", op="block", batch=64, tokens=256, width=256, dtype="bf16", kind="layer", gate="channel", act="tanh",
             scale=False, bias=True, post=False, pre=True, branch=True, train=True),
        # odd sizes in 32 bits, every operand present
        dict(name="block-train-odd", op="block", batch=3, tokens=677, width=1001, dtype="f32", kind="layer", gate="element", act="sigmoid",
             scale=True, bias=True, post=True, pre=True, branch=True, train=True),
        # the first norm of a network: nothing to add yet
        dict(name="norm-train", op="block", batch=4, tokens=2048, width=1024, dtype="f16", kind="layer", gate="none", act="identity",
             scale=False, bias=True, post=False, pre=True, branch=False, train=True),
        # the gradients of the medium UNet: 88 tensors, views of one buffer
        dict(name="clip-unet", op="clip", spec="unet", width=32, depth=3, dtype="f32", layout="aligned", p=2.0),
        # a transformer's gradients, packed into one bucket without padding
        dict(name="clip-layers", op="clip", spec="layers", width=2048, depth=8, dtype="bf16", layout="packed", p=2.0),
        # some separate gradients of odd sizes and both types
        dict(name="clip-odd", op="clip", spec="odd", count=41, largest=300_000, spread=5, dtype="mixed", layout="separate", p=2.0),
        # the training step of the medium UNet with separate parameters
        dict(name="adam-unet", op="adam", spec="unet", width=32, depth=3, dtype="f32", layout="aligned", clip=True, decay=0.0),
        # a transformer in 16 bits with 32-bit masters
        dict(name="adam-layers", op="adam", spec="layers", width=1024, depth=8, dtype="bf16", layout="packed", clip=True, decay=0.1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["block", "block", "clip", "adam"])
    if op == "block":
        width = _log(rng, 16, 8192)
        if rng.random() < 0.5:
            width = max(16, width // 64 * 64)
        rows = _log(rng, 1, max(1, min(65536, 33_000_000 // width)))
        batch = min(rows, _log(rng, 1, 64))
        branch = rng.random() < 0.85
        post = branch and rng.random() < 0.7
        gate = rng.choice(["none", "element", "token", "sample", "channel"]) if branch else "none"
        return dict(op=op, batch=batch, tokens=max(1, rows // batch), width=width, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    kind=rng.choice(["rms", "layer"]), gate=gate, act=rng.choice(["identity", "sigmoid", "tanh"]) if gate != "none" else "identity",
                    scale=branch and rng.random() < 0.3, bias=rng.random() < 0.4, post=post, pre=not branch or rng.random() < 0.85 or not post,
                    branch=branch, train=rng.random() < 0.6)
    if op == "clip":
        spec = rng.choice(["unet", "layers", "odd"])
        c = dict(op=op, spec=spec, dtype=rng.choice(["f32", "bf16", "f16", "mixed"]), layout=rng.choice(["aligned", "packed"]),
                 p=rng.choice([2.0, 2.0, 2.0, 1.0, math.inf]))
    else:
        spec = rng.choice(["unet", "layers", "odd"])
        c = dict(op=op, spec=spec, dtype=rng.choice(["f32", "bf16", "f16"]), layout=rng.choice(["aligned", "packed"]), clip=rng.random() < 0.75,
                 decay=rng.choice([0.0, 0.01, 0.1]))
    if spec == "unet":
        c.update(width=4 * rng.randint(2, 16), depth=rng.randint(1, 3))
    elif spec == "layers":
        c.update(width=_log(rng, 64, 1400 if op == "clip" else 700), depth=rng.randint(1, 12))
    else:
        c.update(count=_log(rng, 1, 400), largest=_log(rng, 100, 1_000_000), spread=rng.randint(0, 10**6))
    return c


def _shapes(c):
    """The shapes of a parameter list, in order."""
    if c["spec"] == "unet":                 # the UNet's own list: 3 x 3 convolutions without bias, affine norms, residual blocks
        def block(i, o):
            return [(o, i, 3, 3), (o,), (o,), (o, o, 3, 3), (o,), (o,)]
        w, got, skips = c["width"], [(c["width"], 6, 3, 3), (c["width"],)], []
        for _ in range(c["depth"]):
            got += block(w, 2 * w) + block(2 * w, 2 * w) + [(2 * w, 2 * w, 3, 3), (2 * w,)]
            w *= 2
            skips.append(w)
        got += block(w, w)
        for s in reversed(skips):
            got += block(w + s, s // 2) + block(s // 2, s // 2)
            w = s // 2
        return got + [(3, w, 1, 1), (3,)]
    if c["spec"] == "layers":               # two norms, four square projections, two wide ones per layer
        w = c["width"]
        return [s for _ in range(c["depth"]) for s in [(w,), (w, w), (w, w), (w, w), (w, w), (w,), (4 * w, w), (w, 4 * w)]]
    r = random.Random(c["spread"])
    return [(_log(r, 1, c["largest"]),) for _ in range(c["count"])]


def _types(c, n):
    return [(torch.bfloat16, torch.float32)[k % 2] if c["dtype"] == "mixed" else DTYPES[c["dtype"]] for k in range(n)]


# ---------------------------------------------------------------------------------------------------------------- the inputs
def _views(shapes, types, layout, fill):
    """Tensors of these shapes and types whose values `fill(n)` gives (32 bits): views of one buffer per type, each at a multiple of eight
    elements ("aligned") or wherever the one before ends ("packed"), or separate tensors.  Returns the tensors and what holds them."""
    numels = [math.prod(s) for s in shapes]
    if layout == "separate":
        got = [fill(n).to(t).view(s) for s, n, t in zip(shapes, numels, types)]
        return got, got
    got, held = [None] * len(shapes), []
    for t in sorted(set(types), key=str):
        at, where = 0, []
        for k in range(len(shapes)):
            if types[k] is t:
                where.append((k, at))
                at += -(-numels[k] // 8) * 8 if layout == "aligned" else numels[k]
        flat = fill(at).to(t)
        held.append(flat)
        for k, o in where:
            got[k] = flat[o:o + numels[k]].view(shapes[k])
    return got, held


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "block":
        B, N, C, T = case["batch"], case["tokens"], case["width"], DTYPES[case["dtype"]]
        s = {"case": case}
        # a residual stream has a few channels far larger than the others and grows with depth; a branch is of order one
        s["x"] = (normal(B, N, C) * (1 + 2 * normal(C).abs()) + 0.1 * normal(C)).to(T)
        if case["branch"]:
            s["branch"] = (normal(B, N, C) * (0.2 + normal(B, N, 1).abs()) + 0.05).to(T)
            shape = {"none": None, "element": (B, N, C), "token": (B, N, 1), "sample": (B, 1, C), "channel": (C,)}[case["gate"]]
            if shape:
                s["gate"] = normal(*shape) if case["gate"] == "channel" else normal(*shape).to(T)   # a channel's gate is a parameter
            if case["scale"]:
                s["scale"] = 0.1 + 0.05 * normal(C)
            if case["post"]:
                s["post_weight"] = 1 + 0.1 * normal(C)
                if case["bias"]:
                    s["post_bias"] = 0.1 * normal(C)
        if case["pre"]:
            s["pre_weight"] = 1 + 0.1 * normal(C)
            if case["bias"]:
                s["pre_bias"] = 0.1 * normal(C)
        if case["train"]:
            for k in _INPUTS:
                if k in s:
                    s[k].requires_grad_(True)
            if case["branch"]:
                s["dy"] = (1e-2 * normal(B, N, C)).to(T)
            if case["pre"]:
                s["dh"] = (1e-2 * normal(B, N, C)).to(T)
        return s

    shapes = _shapes(case)
    types = _types(case, len(shapes))
    grads, held = _views(shapes, types, case["layout"], lambda n: 1e-3 * normal(n))
    if case["op"] == "clip":
        params = [torch.nn.Parameter(torch.empty(s, dtype=t, device="cuda")) for s, t in zip(shapes, types)]
        for p, v in zip(params, grads):
            p.grad = v
        total = sum(math.prod(s) for s in shapes)
        size = {2.0: 1e-3 * math.sqrt(total), 1.0: 8e-4 * total, math.inf: 1e-3}[case["p"]]
        return {"case": case, "params": params, "held": held, "max_norm": 0.5 * size}
    s = {"case": case, "grads": grads}
    s["params"], s["held"] = _views(shapes, types, case["layout"], lambda n: 0.05 * normal(n))
    f32 = [torch.float32] * len(shapes)
    s["exp_avgs"], s["held_m"] = _views(shapes, f32, case["layout"], lambda n: 1e-4 * normal(n))
    s["exp_avg_sqs"], s["held_v"] = _views(shapes, f32, case["layout"], lambda n: 1e-7 * normal(n).square())
    if case["dtype"] != "f32":
        s["masters"], s["held_w"] = _views(shapes, f32, case["layout"], lambda n: 0 * normal(n))
        for w, p in zip(s["masters"], s["params"]):
            w.copy_(p)
    steps = 100                              # a run some way on: the step count and the powers of both betas
    s["clock"] = torch.tensor([steps, 0.9**steps, 0.999**steps], dtype=torch.float64, device="cuda")
    s["max_norm"] = 0.5e-3 * math.sqrt(sum(math.prod(x) for x in shapes)) if case["clip"] else None
    return s


_INPUTS = ("x", "branch", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")
_LR, _EPS_ADAM, _EPS, _A = 1e-3, 1e-8, 1e-6, 0.5


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"block": _run_block, "clip": _run_clip, "adam": _run_adam}[state["case"]["op"]](state)


def _block_plain(s):
    c = s["case"]

    def norm(v, weight, bias):
        if c["kind"] == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS) * weight
        return v if bias is None else v + bias

    y = x = s["x"].float()
    if c["branch"]:
        u = s["branch"].float()
        if c["post"]:
            u = norm(u, s["post_weight"], s.get("post_bias"))
        if "gate" in s:
            gate = s["gate"].float()
            u = u * {"identity": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[c["act"]](gate)
        if "scale" in s:
            u = u * s["scale"]
        y = x + _A * u
    T = s["x"].dtype
    return (y.to(T) if c["branch"] else None), (norm(y, s["pre_weight"], s.get("pre_bias")).to(T) if c["pre"] else None)


def _block_own(s):
    from fluidnet_amd.models.block_norm import gated_residual, pre_norm
    c = s["case"]
    if not c["branch"]:
        return None, pre_norm(s["x"], s["pre_weight"], s.get("pre_bias"), kind=c["kind"], eps=_EPS)
    return gated_residual(s["x"], s["branch"], s.get("gate"), s.get("scale"), post_weight=s.get("post_weight"), post_bias=s.get("post_bias"),
                          pre_weight=s.get("pre_weight"), pre_bias=s.get("pre_bias"), kind=c["kind"], post=c["post"], pre=c["pre"],
                          gate_act=c["act"], residual_scale=_A, eps=_EPS)


def _run_block(s):
    if not s["case"]["train"]:
        with torch.no_grad():
            y, h = _block_own(s) if own else _block_plain(s)
        return {"y": y, "h": h}
    y, h = _block_own(s) if own else _block_plain(s)
    outs = [(o, s[d]) for o, d in ((y, "dy"), (h, "dh")) if o is not None]
    names = [k for k in _INPUTS if k in s]
    grads = torch.autograd.grad([o for o, _ in outs], [s[k] for k in names], [d for _, d in outs])
    return {"y": y, "h": h, **{"d_" + k: v for k, v in zip(names, grads)}}


def _norm_plain(grads, p):
    flat = torch.cat([v.reshape(-1).float() for v in grads]).abs()
    if p == math.inf:
        return flat.max()
    return flat.sum(dtype=torch.float64).float() if p == 1 else flat.square().sum(dtype=torch.float64).sqrt().float()


def _run_clip(s):
    p = s["case"]["p"]
    s["max_norm"] *= 0.9995                  # so that every pass over the same buffers has something to clip
    if own:
        from fluidnet_amd.training.grad_clip import clip_grad_norm_
        total = clip_grad_norm_(s["params"], s["max_norm"], norm_type=p)
    else:
        grads = [q.grad for q in s["params"]]
        total = _norm_plain(grads, p)
        coef = torch.clamp(s["max_norm"] / (total + 1e-6), max=1.0)
        [v.copy_(v.float() * coef) for v in grads]
    return {"norm": total, "grads": s["held"]}


def _run_adam(s):
    c = s["case"]
    if own:
        from fluidnet_amd.training.optim import clip_adam_
        total = clip_adam_(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["clock"], masters=s.get("masters"), lr=_LR,
                           betas=(0.9, 0.999), eps=_EPS_ADAM, weight_decay=c["decay"], max_norm=s["max_norm"])
    else:
        total = _adam_plain(s, c["decay"])
    return {"norm": total, "params": s["held"], "masters": s.get("held_w"), "exp_avg": s["held_m"], "exp_avg_sq": s["held_v"], "clock": s["clock"]}


def _adam_plain(s, decay):
    def one(tensors):
        return torch.cat([v.reshape(-1).float() for v in tensors])

    def back(tensors, flat):
        [t.copy_(v.view(t.shape)) for t, v in zip(tensors, flat.split([t.numel() for t in tensors]))]

    clock = s["clock"]
    clock.copy_(torch.stack([clock[0] + 1, clock[1] * 0.9, clock[2] * 0.999]))
    grad, total = one(s["grads"]), None
    if s["max_norm"] is not None:
        total = _norm_plain(s["grads"], 2.0)
        grad = grad * torch.clamp(s["max_norm"] / (total + 1e-6), max=1.0)
    m, v, w = one(s["exp_avgs"]), one(s["exp_avg_sqs"]), one(s.get("masters") or s["params"])
    m = 0.9 * m + 0.1 * grad
    v = 0.999 * v + 0.001 * grad * grad
    step, root = (_LR / (1 - clock[1])).float(), torch.sqrt(1 - clock[2]).float()
    w = w * (1 - _LR * decay) - step * m / (torch.sqrt(v) / root + _EPS_ADAM)
    back(s["exp_avgs"], m)
    back(s["exp_avg_sqs"], v)
    back(s["params"], w)
    if "masters" in s:
        back(s["masters"], w)
    return total


# ---------------------------------------------------------------------------------------------------------------- work and definition
def work(case):
    if case["op"] == "block":
        rows, C, b = case["batch"] * case["tokens"], case["width"], torch.finfo(DTYPES[case["dtype"]]).bits // 8
        gate = {"none": 0, "element": rows * C * b, "token": rows * b, "sample": case["batch"] * C * b, "channel": 4 * C}[case["gate"]]
        tensors = (1 + case["branch"]) + (case["branch"] + case["pre"])                      # x, branch; y, h
        vectors = 4 * C * ((case["post"] + case["pre"]) * (1 + case["bias"]) + case["scale"])
        flops = rows * C * 16
        if case["train"]:                                                                     # dy, dh; d_x, d_branch
            tensors += (case["branch"] + case["pre"]) + (1 + case["branch"])
            gate, vectors, flops = 2 * gate, 2 * vectors, 3 * flops
        return {"bytes": tensors * rows * C * b + gate + vectors, "flops": flops}
    shapes = _shapes(case)
    types = _types(case, len(shapes))
    numels = [math.prod(s) for s in shapes]
    held = sum(n * torch.finfo(t).bits // 8 for n, t in zip(numels, types))
    if case["op"] == "clip":
        return {"bytes": 2 * held, "flops": 3 * sum(numels)}
    master = 0 if case["dtype"] == "f32" else 8 * sum(numels)
    reads_p = held if case["dtype"] == "f32" else 0                                           # with a master the 16-bit copy is only written
    return {"bytes": held + reads_p + held + 16 * sum(numels) + master, "flops": 15 * sum(numels)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"block": _exact_block, "clip": _exact_clip, "adam": _exact_adam}[case["op"]](case, s)


def _exact_block(c, s):
    """From the formulas and their derivatives, in 64 bits."""
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    C = c["width"]
    x = d["x"].reshape(-1, C)

    def statistics(v):
        mu = v.sum(1, keepdim=True) / C if c["kind"] == "layer" else torch.zeros_like(v[:, :1])
        r = 1 / torch.sqrt(((v - mu) ** 2).sum(1, keepdim=True) / C + _EPS)
        return r, (v - mu) * r

    def through(r, hat, q):                  # the derivative of a norm, applied to q
        q2 = q - hat * (q * hat).sum(1, keepdim=True) / C
        return r * (q2 - q.sum(1, keepdim=True) / C if c["kind"] == "layer" else q2)

    rows, y, out = x.shape[0], x, {"y": None, "h": None}
    one = torch.ones(1, 1, dtype=torch.float64, device=x.device)
    if c["branch"]:
        o = d["branch"].reshape(-1, C)
        u = o
        if c["post"]:
            r_o, o_hat = statistics(o)
            u = o_hat * d["post_weight"] + d.get("post_bias", 0.0)
        g = one
        if "gate" in d:
            g = d["gate"].expand(s["x"].shape).reshape(-1, C)
        act = {"identity": g, "sigmoid": 1 / (1 + torch.exp(-g)), "tanh": torch.tanh(g)}[c["act"]] if "gate" in d else one
        slope = {"identity": torch.ones_like(g), "sigmoid": act * (1 - act), "tanh": 1 - act**2}[c["act"]] if "gate" in d else one
        scale = d.get("scale", one)
        y = x + _A * scale * act * u
        out["y"] = y.view(s["x"].shape)
    if c["pre"]:
        r_y, y_hat = statistics(y)
        out["h"] = (y_hat * d["pre_weight"] + d.get("pre_bias", 0.0)).view(s["x"].shape)
    if not c["train"]:
        return out
    dy = d["dy"].reshape(-1, C) if c["branch"] else torch.zeros_like(x)
    if c["pre"]:
        dh = d["dh"].reshape(-1, C)
        dy = dy + through(r_y, y_hat, dh * d["pre_weight"])
        out["d_pre_weight"] = (dh * y_hat).sum(0)
        if "pre_bias" in d:
            out["d_pre_bias"] = dh.sum(0)
    out["d_x"] = dy.view(s["x"].shape)
    if c["branch"]:
        e = _A * dy
        if "scale" in d:
            out["d_scale"] = (e * act * u).sum(0)
        if "gate" in d:
            dg = e * scale * u * slope
            out["d_gate"] = {"element": lambda: dg, "token": lambda: dg.sum(1), "channel": lambda: dg.sum(0),
                             "sample": lambda: dg.view(c["batch"], -1, C).sum(1)}[c["gate"]]().reshape(d["gate"].shape)
        du = e * scale * act
        if c["post"]:
            out["d_post_weight"] = (du * o_hat).sum(0)
            if "post_bias" in d:
                out["d_post_bias"] = du.sum(0)
            du = through(r_o, o_hat, du * d["post_weight"])
        out["d_branch"] = (du + torch.zeros_like(x)).view(s["x"].shape)
    assert rows == c["batch"] * c["tokens"]
    return out


def _exact_norm(grads, p):
    if p == math.inf:
        return max(v.double().abs().max() for v in grads)
    return sum((v.double().abs() ** p).sum() for v in grads) ** (1 / p)


def _exact_clip(c, s):
    total = _exact_norm([p.grad for p in s["params"]], c["p"])
    coef = min(1.0, 0.9995 * s["max_norm"] / (float(total) + 1e-6))
    # what lies between the views stays as it is: the clipped values are put in their places
    held = [v.double() for v in s["held"]]
    of = {v.untyped_storage().data_ptr(): k for k, v in enumerate(s["held"])}
    for p in s["params"]:
        k = of[p.grad.untyped_storage().data_ptr()]
        flat = held[k].view(-1)
        at = p.grad.storage_offset()
        flat[at:at + p.grad.numel()] *= coef
    return {"norm": total, "grads": held}


def _exact_adam(c, s):
    b1, b2 = 0.9, 0.999
    t, p1, p2 = s["clock"].tolist()
    t, p1, p2 = t + 1, p1 * b1, p2 * b2
    total, coef = None, 1.0
    if s["max_norm"] is not None:
        total = _exact_norm(s["grads"], 2.0)
        coef = min(1.0, s["max_norm"] / (float(total) + 1e-6))
    held = {k: [v.double() for v in s[k]] for k in ("held", "held_m", "held_v", "held_w") if k in s}
    for i, g in enumerate(s["grads"]):
        def at(name, kept):
            v = s[name][i]
            k = next(k for k, f in enumerate(s[kept]) if f.untyped_storage().data_ptr() == v.untyped_storage().data_ptr())
            return held[kept][k].view(-1)[v.storage_offset():v.storage_offset() + v.numel()]
        gc = g.double().reshape(-1) * coef
        m, v, p = at("exp_avgs", "held_m"), at("exp_avg_sqs", "held_v"), at("params", "held")
        w = at("masters", "held_w") if "masters" in s else p
        m.copy_(b1 * m + (1 - b1) * gc)
        v.copy_(b2 * v + (1 - b2) * gc**2)
        w.copy_(w * (1 - _LR * c["decay"]) - _LR / (1 - p1) * m / (torch.sqrt(v / (1 - p2)) + _EPS_ADAM))
        p.copy_(w)
    return {"norm": total, "params": held["held"], "masters": held.get("held_w"), "exp_avg": held["held_m"], "exp_avg_sq": held["held_v"],
            "clock": torch.tensor([t, p1, p2], dtype=torch.float64)}
