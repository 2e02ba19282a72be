"""The gated feed-forward block against its 64-bit form, with derived bounds (block_util)."""
import pytest
import torch

from block_util import ACC, U, ffn_backward, ffn_forward, within
from gpu_util import gen, status_clean

from icpp_tuning_b200 import block
from icpp_tuning_b200.graphs import CapturedStep

pytestmark = pytest.mark.gpu


def make(T, D, F, Nn, dtype, layout, seed=0, pad=0):
    """x and the weights; pad > 0: as columns of wider matrices (row strides longer than rows)."""
    g = gen(seed)

    def t(r, c, std):
        m = (torch.randn(r, (c + 7) // 8 * 8 + pad, generator=g) * std).to(dtype)
        return m[:, :c] if pad or c % 8 else m

    kn = layout == "kn"
    up, down = ((D, F), (F, Nn)) if kn else ((F, D), (Nn, F))
    return t(T, D, 1.0), t(*up, D ** -0.5), t(*up, D ** -0.5), t(*down, F ** -0.5)


def cuda(t):
    """On the GPU with the same strides and the same memory around it."""
    return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda").copy_(t)


def as_kn(w, layout):
    return [m.double() if layout == "kn" else m.double().t() for m in w]


CASES = [  # T, D, F, N: the short-token kernels, tile edges, cut products, odd widths in padded rows
    (1, 64, 128, 64), (1, 8, 8, 8), (2, 200, 136, 72), (8, 512, 384, 128), (9, 1032, 264, 520), (16, 64, 2048, 64), (17, 100, 300, 52),
    (31, 72, 1000, 136), (32, 256, 640, 1024), (33, 64, 128, 64), (64, 136, 520, 264), (65, 1024, 264, 128), (129, 40, 2056, 264),
    (255, 200, 136, 8), (256, 256, 256, 256), (257, 257, 129, 33), (300, 64, 1288, 520), (511, 24, 40, 1032),
]


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("T,D,F,Nn", CASES)
def test_forward(T, D, F, Nn, layout):
    dtype = torch.bfloat16 if (T + D) % 2 else torch.float16
    act = ["silu", "gelu_tanh", "gelu_erf", "relu"][(T + F) % 4]
    x, *w = make(T, D, F, Nn, dtype, layout, seed=T)
    ref, bound = ffn_forward(x.double(), *as_kn(w, layout), act, U[dtype])
    y, g, u = block.gated_ffn(cuda(x), *map(cuda, w), act=act, b_layout=layout, save=True)
    for o, r, b, name in zip((y, g, u), ref, bound, "ygu"):
        within(o, r, b, name)
    assert torch.equal(y, block.gated_ffn(cuda(x), *map(cuda, w), act=act, b_layout=layout))  # saving changes nothing, and no run differs
    status_clean()


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("T,D,F,Nn", CASES)
def test_backward(T, D, F, Nn, layout):
    dtype = torch.float16 if (T + D) % 2 else torch.bfloat16
    act = ["relu", "silu", "gelu_tanh", "gelu_erf"][(T + F) % 4]
    x, *w = make(T, D, F, Nn, dtype, layout, seed=T + 1)
    g_ = gen(T + 2)
    kn = as_kn(w, layout)
    g, u = (cuda(_strided((x.double() @ m).to(dtype))) for m in kn[:2])
    dy = _strided((torch.randn(T, Nn, generator=g_) * 0.1).to(dtype))
    ref, bound = ffn_backward(dy.double(), x.double(), *kn, g.double().cpu(), u.double().cpu(), act, U[dtype])
    out = block.gated_ffn_backward(cuda(dy), cuda(x), *map(cuda, w), g, u, act=act, b_layout=layout)
    for i, (o, r, b, name) in enumerate(zip(out, ref, bound, ("dx", "dw_gate", "dw_up", "dw_down"))):
        within(o, r if layout == "kn" or i == 0 else r.t(), b if layout == "kn" or i == 0 else b.t(), name)
    again = block.gated_ffn_backward(cuda(dy), cuda(x), *map(cuda, w), g, u, act=act, b_layout=layout)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    status_clean()


@pytest.mark.parametrize("T,D,F,Nn", [(70, 7304, 2048, 520), (300, 7304, 2048, 520), (600, 4104, 2040, 2080)])
def test_backward_of_many_units(T, D, F, Nn):
    """More output tiles than are spread by name, those of dx longer or shorter than the rest."""
    test_backward(T, D, F, Nn, "kn")


def _strided(t):
    """Rows that start every multiple of 8 elements."""
    c = t.shape[1]
    if c % 8 == 0:
        return t
    wide = torch.zeros(t.shape[0], (c + 7) // 8 * 8, dtype=t.dtype)
    wide[:, :c] = t
    return wide[:, :c]


@pytest.mark.parametrize("T", [3, 40, 260])
def test_strided_rows(T):
    x, *w = make(T, 72, 136, 40, torch.bfloat16, "nk", seed=5, pad=24)
    ref, bound = ffn_forward(x.double(), *as_kn(w, "nk"), "silu", U[torch.bfloat16])
    for o, r, b in zip(block.gated_ffn(cuda(x), *map(cuda, w), b_layout="nk", save=True), ref, bound):
        within(o, r, b)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu_erf", "relu"])
def test_gradient_against_differences(act):
    """Along random directions of every input: <grad, v> against (L(+) - L(-)) / 2 eps of the
    64-bit forward pass, L = sum(dy * y).  The gradient's error is within its bound; the
    difference's own is O(eps^2)."""
    T, D, F, Nn, dtype, eps = 40, 64, 96, 56, torch.float16, 1e-4
    x, *w = make(T, D, F, Nn, dtype, "kn", seed=9)
    kn = as_kn(w, "kn")
    dy = (torch.randn(T, Nn, generator=gen(10)) * 0.1).to(dtype)
    g, u = ((x.double() @ m).to(dtype) for m in kn[:2])
    got = block.gated_ffn_backward(cuda(dy), cuda(x), *map(cuda, w), cuda(g), cuda(u), act=act)
    _, bound = ffn_backward(dy.double(), x.double(), *kn, g.double(), u.double(), act, U[dtype])

    def loss(args):
        return (dy.double() * ffn_forward(*args, act, 0.0)[0][0]).sum()

    args = [x.double(), *kn]
    # g and u reach the backward pass rounded: its exact gradient differs from the forward
    # pass's by that of their roundings, at most u (|g| |d grad / dg| + ..): 4 u of the sums
    for i in range(4):
        v = torch.randn(args[i].shape, generator=gen(20 + i), dtype=torch.float64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + eps * v, args[i] - eps * v
        num = (loss(up) - loss(down)) / (2 * eps)
        grad = got[i].double().cpu()
        slack = (bound[i] * v.abs()).sum() + 4 * U[dtype] * (grad.abs() * v.abs()).sum() + 1e-4 * (grad.abs() * v.abs()).sum()
        assert (num - (grad * v).sum()).abs() <= slack


def test_not_a_number_stays_in_its_token():
    for T in (4, 200):
        x, *w = make(T, 64, 128, 64, torch.bfloat16, "nk", seed=3)
        clean = block.gated_ffn(cuda(x), *map(cuda, w), b_layout="nk")
        x[1, 5] = float("nan")
        x[2, 7] = float("inf")
        y = block.gated_ffn(cuda(x), *map(cuda, w), b_layout="nk")
        assert y[1].isnan().all() and not y[2].isfinite().any()
        rest = [i for i in range(T) if i not in (1, 2)]
        assert torch.equal(y[rest], clean[rest])


def test_empty():
    _, *w = map(cuda, make(1, 64, 128, 64, torch.bfloat16, "nk"))
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    y, g, u = block.gated_ffn(x, *w, b_layout="nk", save=True)
    assert y.shape == (0, 64) and g.shape == u.shape == (0, 128)
    dx, *dw = block.gated_ffn_backward(y, x, *w, g, u, b_layout="nk")
    assert dx.shape == (0, 64) and all((m == 0).all() for m in dw)


def test_streams_and_graphs():
    for T in (2, 300):
        x, *w = map(cuda, make(T, 256, 512, 256, torch.bfloat16, "nk", seed=1))
        y = block.gated_ffn(x, *w, b_layout="nk")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        y2 = block.gated_ffn(x, *w, b_layout="nk", stream=s)
        s.synchronize()
        assert torch.equal(y, y2)
        step = CapturedStep(lambda t: block.gated_ffn(t, *w, b_layout="nk"), [torch.zeros_like(x)])
        assert torch.equal(step(x), y)
    status_clean()


def test_refusals():
    x, *w = map(cuda, make(4, 64, 128, 64, torch.bfloat16, "nk"))
    with pytest.raises(ValueError, match="act"):
        block.gated_ffn(x, *w, act="tanh", b_layout="nk")
    with pytest.raises(ValueError, match="b_layout"):
        block.gated_ffn(x, *w, b_layout="tt")
    with pytest.raises(ValueError, match="w_gate"):
        block.gated_ffn(x, *w, b_layout="kn")
    with pytest.raises(ValueError, match="dtype"):
        block.gated_ffn(x, w[0].half(), *w[1:], b_layout="nk")
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        block.gated_ffn(x.float(), *(m.float() for m in w), b_layout="nk")
    with pytest.raises(ValueError, match="unit column stride"):
        block.gated_ffn(x.t().contiguous().t(), *w, b_layout="nk")
    with pytest.raises(block.N.FoError, match="row stride"):
        block.gated_ffn(x[:, :60].contiguous(), *(m[:, :60].contiguous() for m in w[:2]), w[2][:60].contiguous(), b_layout="nk")
    y, g, u = block.gated_ffn(x, *w, b_layout="nk", save=True)
    with pytest.raises(ValueError, match="dy"):
        block.gated_ffn_backward(y[:2], x, *w, g, u, b_layout="nk")
    assert ACC < 2.0 ** -12  # the bounds above are those of the 16-bit roundings, not of the sums
