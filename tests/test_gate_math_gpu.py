"""The gated block's activations and their derivatives, one value at a time, through matrices
that pass a value on unchanged: relative accuracy in the tails, saturation at the far ends.

A value and its derivative are a few fp32 operations on an exponential of an argument e (silu
|g|, gelu_tanh 2 w, gelu_erf g^2 / 2), whose three roundings cost the exponential 3 |e| 2^-24 of
itself; the rest costs 16 units of 2^-24 of the terms' magnitudes, generously counted.  Then one
rounding to 16 bits."""
import math

import pytest
import torch

from block_util import U, act64, within

from icpp_tuning_b200 import block

pytestmark = pytest.mark.gpu
ACTS = ["silu", "gelu_tanh", "gelu_erf", "relu"]
D = 8


def exponent(act, g):
    if act == "silu":
        return g.abs()
    if act == "gelu_tanh":
        return (2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)).abs()
    return g * g / 2 if act == "gelu_erf" else torch.zeros_like(g)


def one(r, c):
    m = torch.zeros(D, D, dtype=torch.float64)
    m[r, c] = 1
    return m


def tail_values():
    g = torch.cat([torch.linspace(-6, 8, 1991, dtype=torch.float64), torch.tensor([0.0, -0.0, 1e-3, -1e-3, 20.0, 300.0, 60000.0])])
    return g.half().double()


@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("act", ACTS)
def test_values(act, short):
    """y = act(g) u with u a power of two that brings the tail back to ordinary sizes; the
    short-token form has act(g) u in two fp16 parts, whose low one ends at 2^-25."""
    dtype = torch.float16
    g = tail_values()
    a, _ = act64(act, g)
    u = torch.exp2(torch.round(-torch.log2(a.abs() + 2.0 ** -40)).clamp(0, 15))
    x = torch.zeros(len(g), D, dtype=torch.float64)
    x[:, 0], x[:, 1] = g, u
    w = [m.to(dtype).cuda() for m in (one(0, 0), one(0, 1), one(0, 0))]
    parts = x.to(dtype).cuda().split(32 if short else len(g))
    y = torch.cat([block.gated_ffn(p.contiguous(), *w, act=act, b_layout="nk")[:, 0] for p in parts])
    ref = a * u
    within(y, ref, U[dtype] * ref.abs() * 1.01 + (16 + 4 * exponent(act, g)).clamp(max=2.0 ** 20) * 2.0 ** -24 * ref.abs() + 2.0 ** -25, act)


@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("act", ACTS)
def test_derivatives(act, short):
    """dh = 1, so that dx holds dg = u act'(g) in one column and du = act(g) in another."""
    dtype = torch.float16
    g = tail_values()
    if act == "relu":
        g = g[g != 0]
    a, da = act64(act, g)
    n = len(g)
    e, U1 = exponent(act, g), U[dtype] * 1.01
    unit = (16 + 4 * e) * 2.0 ** -24
    terms = {"silu": da.abs() + 2 * a.abs(), "gelu_tanh": 1 + a.abs() * 1.6 * (1 + 0.135 * g * g), "gelu_erf": 1 + g.abs(), "relu": da}[act]
    # the far ends are exact: the exponential is nothing there
    terms, unit = torch.where(g.abs() > 15, da.abs(), terms), torch.where(g.abs() > 15, 16 * 2.0 ** -24, unit)
    G = torch.zeros(n, D, dtype=dtype)
    Up = torch.zeros(n, D, dtype=dtype)
    G[:, 0], Up[:, 0] = g.to(dtype), 1
    x = torch.zeros(n, D, dtype=dtype)
    dy = torch.zeros(n, D, dtype=dtype)
    dy[:, 0] = 1
    w = [m.to(dtype).cuda() for m in (one(0, 0), one(0, 1), one(0, 0))]
    size = 64 if short else n
    dx = torch.cat([block.gated_ffn_backward(*(t[i:i + size].contiguous().cuda() for t in (dy, x)), *w,
                                             *(t[i:i + size].contiguous().cuda() for t in (G, Up)), act=act, b_layout="nk")[0]
                    for i in range(0, n, size)])
    within(dx[:, 0], da, U1 * da.abs() + unit * terms, "act'")
    within(dx[:, 1], a, U1 * a.abs() + (unit * a.abs()).clamp(max=1.0) + 2.0 ** -25, "act")


@pytest.mark.parametrize("short", [True, False])
@pytest.mark.parametrize("act", ACTS)
def test_saturation_of_bfloat16(act, short):
    """Finite g of any size: act' is 1 or 0 there, act is g or 0."""
    dtype = torch.bfloat16
    g = torch.tensor([1e9, 1e14, 1e19, 1e20, 1e30, 3e38], dtype=torch.float64).to(dtype)
    g = torch.cat([g, -g]).repeat(1 if short else 20)
    n = len(g)
    G, Up, x, dy = (torch.zeros(n, D, dtype=dtype) for _ in range(4))
    G[:, 0], Up[:, 0], dy[:, 0] = g, 1, 1
    w = [m.to(dtype).cuda() for m in (one(0, 0), one(0, 1), one(0, 0))]
    dx = block.gated_ffn_backward(dy.cuda(), x.cuda(), *w, G.cuda(), Up.cuda(), act=act, b_layout="nk")[0].cpu()
    assert torch.equal(dx[:, 0].float(), (g > 0).float())
    assert torch.equal(dx[:, 1].float(), g.float().clamp(min=0))
    x[:, 0], x[:, 1] = g, 1
    y = block.gated_ffn(x.cuda(), *w, act=act, b_layout="nk")[:, 0].cpu()
    assert torch.equal(y.float(), g.float().clamp(min=0))
