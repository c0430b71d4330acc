"""The gates' activations and their slopes by themselves, over all of their range: with x = 0, one branch element of 1 per gate value and no
norm, y is act(g) and the gradient of the gate is act'(g), without any sum or product that rounds."""
import math

import pytest
import torch

from fluidnet_amd.models.block_norm import gated_residual

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# In steps of 2^-24: e = exp(-|g|) is off by three (two for the power, one for the product with the exponent's remainder), 1 + e by one, the
# reciprocal by one, a product by one.  A slope has 1 + e twice in its square, and the square rounds once.
VALUE = {"sigmoid": 6 * 2.0 ** -24, "tanh": 5 * 2.0 ** -23}       # tanh: five units, what OpenCL asks of the function
SLOPE = 8 * 2.0 ** -24
# below the smallest normal number the power is 0; a tanh slope is four times that
TINY = 4 * torch.finfo(F32).tiny


def _gates():
    g = torch.cat([torch.linspace(-100, 100, 4001), torch.linspace(-1, 1, 257), -2.0 ** torch.arange(-20, 6.0), torch.tensor([0.0, -8.0, -16.0, -25.5, 88.0])])
    return g.to(F32)


def _exact(act, g):
    g = g.double()
    e = torch.exp(-g.abs())
    if act == "sigmoid":
        return torch.where(g < 0, e / (1 + e), 1 / (1 + e)), e / (1 + e) ** 2
    return torch.tanh(g), 4 * e * e / (1 + e * e) ** 2


def _place(kind, g, width):
    """(shape of x, gate, where in x each gate value's one element lies)."""
    n = g.numel()
    if kind == "element":
        return (n, width), g[:, None].expand(n, width).contiguous(), lambda t: t[:, 0]
    if kind == "token":
        return (n, width), g[:, None].clone(), lambda t: t[:, 0]
    if kind == "channel":
        return (1, n), g.clone(), lambda t: t[0]
    return (n, 3, width), g[:, None, None].expand(n, 1, width).contiguous(), lambda t: t[:, 1, 0]


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("kind,width", [("element", 9), ("element", 600), ("token", 9), ("token", 2100), ("sample", 40), ("sample", 520), ("channel", 0)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_fp32_gates_are_taken_in_32_bits(act, kind, width, dtype):
    """Also next to 16-bit operands: the gate's gradient is fp32 there, and ones stay ones."""
    g = _gates()
    shape, gate, at = _place(kind, g, width)
    x, one = torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)
    at(one).fill_(1.0)
    gate = gate.cuda().requires_grad_()
    y, h = gated_residual(x.cuda(), one.cuda(), gate, post=False, pre=False, gate_act=act)
    d, = torch.autograd.grad(y, gate, one.cuda())
    value, slope = _exact(act, g)
    if dtype is F32:
        err = (at(y.detach().cpu()).double() - value).abs()
        assert (err <= VALUE[act] * value.abs() + TINY).all(), float((err / value.abs()).nan_to_num(0).max())
    d = d.cpu().double()
    d = d.reshape(g.numel(), -1)[:, 0] if kind != "channel" else d
    err = (d - slope).abs()
    assert (err <= SLOPE * slope + TINY).all(), (float((err / slope).nan_to_num(0).max()), float(g[(err / slope).nan_to_num(0).argmax()]))


@pytest.mark.parametrize("kind", ["element", "token", "sample", "channel"])
def test_gates_that_are_not_finite(kind):
    g = torch.tensor([math.inf, -math.inf, math.nan])
    for act, ends in (("sigmoid", (1.0, 0.0)), ("tanh", (1.0, -1.0))):
        for dtype in (F32, BF16):
            shape, gate, at = _place(kind, g, 12)
            one = torch.zeros(shape, dtype=dtype)
            at(one).fill_(1.0)
            gate = gate.cuda().requires_grad_()
            y, _ = gated_residual(torch.zeros(shape, dtype=dtype).cuda(), one.cuda(), gate, post=False, pre=False, gate_act=act)
            d = torch.autograd.grad(y, gate, one.cuda())[0].cpu().reshape(3, -1)[:, 0]
            y = at(y.detach().cpu()).float()
            assert (y[0], y[1]) == ends and torch.isnan(y[2]) and d[0] == 0 and d[1] == 0 and torch.isnan(d[2]), (act, dtype)


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_16_bit_gates(act, dtype):
    """The product -g log2(e) of a 16-bit gate is rounded before the power is taken: off by 2^-24 of itself (at most 150 here, and its own
    power changes by that times ln 2), 2^-23 each for the power and the reciprocal twice: below 3e-5, and half a step of the result's type."""
    g = _gates().to(dtype)
    shape, gate, at = _place("element", g, 9)
    one = torch.zeros(shape, dtype=dtype)
    at(one).fill_(1.0)
    gate = gate.cuda().requires_grad_()
    y, _ = gated_residual(torch.zeros(shape, dtype=dtype).cuda(), one.cuda(), gate, post=False, pre=False, gate_act=act)
    d, = torch.autograd.grad(y, gate, one.cuda())
    f = torch.finfo(dtype)
    least = max(f.tiny, TINY)
    for got, want in zip((at(y.detach().cpu()), d.cpu()[:, 0]), _exact(act, g)):
        assert ((got.double() - want).abs() <= (f.eps / 2 + 3e-5) * want.abs() + least).all()
