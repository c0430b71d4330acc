"""The norms around a residual block in 64 bits, from their definition, with torch's autograd for the formula's gradient; and how far 32-bit
arithmetic with one rounding to the outputs' type may be from it."""
import torch

NAMES = ("x", "branch", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


def forward(t, kind, gate_act, a, eps):
    """(y, h) of a dict of fp64 tensors (y is None without a branch, h without "pre")."""
    def norm(v, w, b):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
        v = v if w is None else v * w
        return v if b is None else v + b

    y = t["x"]
    if t.get("branch") is not None:
        u = t["branch"]
        if t["post"]:
            u = norm(u, t.get("post_weight"), t.get("post_bias"))
        if t.get("gate") is not None:
            u = u * {"identity": lambda g: g, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[gate_act](t["gate"])
        if t.get("scale") is not None:
            u = u * t["scale"]
        y = y + a * u
    return (y if t.get("branch") is not None else None), (norm(y, t.get("pre_weight"), t.get("pre_bias")) if t["pre"] else None)


def reference(t, kind, gate_act, a, eps, dy=None, dh=None):
    """Outputs and (with dy / dh) the gradients of sum(dy * y) + sum(dh * h), all in 64 bits on the CPU."""
    d = {k: (v.detach().cpu().double().requires_grad_(dy is not None or dh is not None) if isinstance(v, torch.Tensor) else v) for k, v in t.items()}
    y, h = forward(d, kind, gate_act, a, eps)
    out = {"y": y, "h": h}
    if dy is not None or dh is not None:
        names = [n for n in NAMES if d.get(n) is not None]
        loss = sum((o * g.detach().cpu().double()).sum() for o, g in ((y, dy), (h, dh)) if o is not None and g is not None)
        out.update({"d_" + n: g for n, g in zip(names, torch.autograd.grad(loss, [d[n] for n in names], allow_unused=True))})
    return {k: None if v is None else v.detach() for k, v in out.items()}


def tolerance(t, kind, gate_act, a, eps, dy=None, dh=None):
    """For every output and gradient a bound of its error, element by element, without the last rounding (half a step of its type, added by
    `check`).  A 32-bit result is off by at most n * 2^-24 of the sum of the magnitudes it was added up from, n the operations on its longest
    path: for a value of a row at most 16 elements of a lane, 6 + 16 steps across lanes and waves, and some 30 elementwise ones, 80 in
    all; where a mean is taken off, the magnitudes are those before.  Through a normalised value v_hat = (v - mean) r the error grows by
    (1 + r max |v|) and once more through the product with mean(t v_hat).  A sum over n rows adds n more."""
    d = {k: (v.detach().cpu().double() if isinstance(v, torch.Tensor) else v) for k, v in t.items()}
    one = torch.ones((), dtype=torch.float64)
    get = lambda n: one if d.get(n) is None else d[n].abs()  # noqa: E731
    bias = lambda n: 0 * one if d.get(n) is None else d[n].abs()  # noqa: E731
    big = lambda v: v.amax(-1, keepdim=True)  # noqa: E731
    u24 = 80 * 2.0 ** -24
    x = d["x"]

    def stat(v):
        c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        return c * r, r
    U = sp = torch.zeros_like(x)
    o_hat, r_o, grow_o = torch.zeros_like(x), one, one
    if d.get("branch") is not None:
        o = d["branch"]
        g = one if d.get("gate") is None else {"identity": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[gate_act](d["gate"])
        if d["post"]:
            o_hat, r_o = stat(o)
            grow_o = 1 + r_o * big(o.abs())
            U = (o_hat.abs() + 1) * get("post_weight") * grow_o + bias("post_bias")
        else:
            o_hat, U = o, o.abs()
        sp = abs(a) * get("scale") * g.abs()
    Y = x.abs() + sp * U
    tol = {"y": u24 * Y}
    y, h = forward({k: v for k, v in d.items()}, kind, gate_act, a, eps)
    yv = x if y is None else y
    y_hat, r_y = stat(yv)
    grow = 1 + r_y * big(Y)
    tol["h"] = u24 * ((y_hat.abs() + 1) * get("pre_weight") * grow + bias("pre_bias"))
    if dy is None and dh is None:
        return tol
    n = x.numel() // x.shape[-1]
    D = 0 * x if dy is None or d.get("branch") is None else dy.detach().cpu().double().abs()
    if dh is not None:
        H = dh.detach().cpu().double().abs()
        T = H * get("pre_weight")
        D = D + r_y * (T + big(T) * (1 + y_hat.abs())) * grow * grow
        row = H * (y_hat.abs() + 1) * grow
        lead = tuple(range(x.ndim - 1))
        tol["d_pre_weight"], tol["d_pre_bias"] = (80 + n) * 2.0 ** -24 * row.sum(lead), (80 + n) * 2.0 ** -24 * H.sum(lead)
    tol["d_x"] = u24 * D
    if d.get("branch") is not None:
        E, lead, c = abs(a) * D, tuple(range(x.ndim - 1)), (80 + n) * 2.0 ** -24
        gm = one if d.get("gate") is None else g.abs()
        tol["d_scale"] = c * (E * gm * U).sum(lead)
        if d.get("gate") is not None:
            m = (E * get("scale") * U).expand(x.shape)
            while m.ndim > d["gate"].ndim:
                m = m.sum(0)
            for k in range(m.ndim):
                if d["gate"].shape[k] == 1:
                    m = m.sum(k, keepdim=True)
            tol["d_gate"] = (c + u24 * x.shape[-1] ** 0.5) * m
        du = D * sp
        tol["d_post_weight"], tol["d_post_bias"] = c * (du * (o_hat.abs() + 1) * grow_o).sum(lead), c * du.sum(lead)
        if d["post"]:
            q = du * get("post_weight")
            tol["d_branch"] = u24 * r_o * (q + big(q) * (1 + o_hat.abs())) * grow_o * grow_o
        else:
            tol["d_branch"] = u24 * du
    return tol


def check(got, want, tol, what):
    """got (a GPU tensor of its type) against want (64 bits): tol and half a step of the type, of the value, or of the smallest normal number."""
    f = torch.finfo(got.dtype)
    w = want.double()
    bound = tol + f.eps / 2 * (w.abs() + tol) + f.tiny
    err = (got.detach().cpu().double() - w).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).max()):.3g} of the bound at {float(err.max()):.3g}"
