"""Products with 4-bit weights against their 64-bit form, with derived bounds (block_util)."""
import pytest
import torch

from block_util import ACC, U, act64, within
from gpu_util import gen, status_clean

from icpp_tuning_b200 import block
from icpp_tuning_b200.gated_block import GatedStack, make_weights, train_step
from icpp_tuning_b200.graphs import CapturedStep

pytestmark = pytest.mark.gpu


def weight(Nn, K, group, dtype, zeros, seed, pad=0):
    g = gen(seed)
    G = -(-K // group)
    q = torch.randint(0, 256, (Nn, K // 2 + 16 * pad), generator=g, dtype=torch.uint8)[:, :K // 2]
    s = ((0.5 + torch.rand(Nn, G + pad, generator=g)) * K ** -0.5 / 4).to(dtype)[:, :G]
    z = torch.randint(0, 16, (Nn, G + 3 * pad), generator=g, dtype=torch.uint8)[:, :G] if zeros else None
    return block.W4(q, s, z, group)


def opened(w):
    """(w, |scale| (q + zero + 128)) in float64: the values, and the sizes of what is summed."""
    Nn, K = w.q.shape[0], 2 * w.q.shape[1]
    v = torch.stack((w.q & 15, w.q >> 4), 2).reshape(Nn, K).double()
    at = torch.arange(K) // w.group
    s, z = w.scales.double()[:, at], 8.0 if w.zeros is None else w.zeros.double()[:, at]
    return (v - z) * s, s.abs() * (v + z + 128)


def gpu(w):
    def put(t):
        if t is None:
            return None
        room = torch.zeros(t.untyped_storage().nbytes() // t.element_size(), dtype=t.dtype, device="cuda")
        return room.as_strided(t.shape, t.stride(), t.storage_offset()).copy_(t)

    return block.W4(put(w.q), put(w.scales), put(w.zeros), w.group)


# T, N, K, group: one token to several chunks; N off the 32-row tiles; K off the 128-wide steps;
# groups shorter and longer than a step, not dividing it, longer than the row
CASES = [(1, 16, 32, 32), (1, 1, 64, 32), (2, 33, 96, 32), (3, 100, 160, 64), (5, 64, 128, 128), (8, 48, 256, 96), (9, 31, 416, 128),
         (16, 130, 1024, 256), (17, 512, 544, 64), (33, 20, 96, 4096), (64, 96, 2048, 32), (70, 40, 128, 32), (4, 5000, 384, 128),
         (1, 64, 16384, 32), (2, 48, 8224, 128), (40, 300, 640, 160)]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,Nn,K,group", CASES)
def test_matvec(T, Nn, K, group, zeros):
    dtype = torch.bfloat16 if (T + zeros) % 2 else torch.float16
    w = weight(Nn, K, group, dtype, zeros, seed=K + Nn, pad=T % 3)
    x = torch.randn(T, K, generator=gen(T)).to(dtype)
    bias = torch.randn(Nn, generator=gen(T + 1)).to(dtype) if Nn % 2 else None
    v, size = opened(w)
    ref, mag = x.double() @ v.t(), x.double().abs() @ size.t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    out = block.matvec_w4(x.cuda(), gpu(w), bias=None if bias is None else bias.cuda())
    within(out, ref, U[dtype] * ref.abs() * 1.01 + ACC * mag)
    assert torch.equal(out, block.matvec_w4(x.cuda(), gpu(w), bias=None if bias is None else bias.cuda()))
    status_clean()


@pytest.mark.parametrize("T,D,F,Nn,group", [(1, 64, 96, 40, 32), (2, 128, 160, 33, 64), (4, 416, 544, 100, 128), (5, 96, 64, 16, 96), (9, 1024, 256, 64, 32),
                                            (16, 64, 64, 8, 64), (17, 96, 128, 48, 32), (33, 160, 288, 24, 32)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu_erf", "relu"])
def test_gated(T, D, F, Nn, group, act):
    dtype = torch.float16 if (T + F) % 2 else torch.bfloat16
    zeros = D % 3 == 0
    wg, wu = (weight(F, D, group, dtype, zeros, seed=i + F) for i in range(2))
    wd = weight(Nn, F, 32, dtype, not zeros, seed=9)
    x = torch.randn(T, D, generator=gen(T)).to(dtype)
    (vg, sg), (vu, su), (vd, sd) = map(opened, (wg, wu, wd))
    X = x.double()
    g, p = X @ vg.t(), X @ vu.t()
    eg, ep = ACC * (X.abs() @ sg.t()), ACC * (X.abs() @ su.t())
    a, _ = act64(act, g)
    h = a * p
    # h travels as two 16-bit parts: 2 u^2 of it, or fp16's smallest step, is what is lost
    eh = 1.2 * eg * p.abs() + (a.abs() + 1.2 * eg) * ep + ACC * (h.abs() + p.abs()) + 2 * U[dtype] ** 2 * h.abs() + 2.0 ** -24
    ref = h @ vd.t()
    bound = U[dtype] * ref.abs() * 1.01 + eh @ vd.abs().t() + ACC * (h.abs() @ sd.t())
    out = block.gated_ffn_w4(x.cuda(), gpu(wg), gpu(wu), gpu(wd), act=act)
    within(out, ref, bound * 1.01)
    assert torch.equal(out, block.gated_ffn_w4(x.cuda(), gpu(wg), gpu(wu), gpu(wd), act=act))
    status_clean()


def step_most(x):
    """The largest magnitude of each value's 128 k's, which its fixed point is relative to."""
    T, K = x.shape
    pad = torch.nn.functional.pad(x.abs(), (0, -K % 128)).reshape(T, -1, 128)
    return pad.amax(2, keepdim=True).expand_as(pad).reshape(T, -1)[:, :K]


# large weights times a few tokens: x as digits; K off the steps, N off the tiles, every group
# size's path, the sums of a tile cut over warps and CTAs, values that span seven decades
LARGE = [(1, 8200, 2048, 32), (2, 16001, 1056, 64), (3, 4100, 4128, 128), (5, 1401, 12800, 256), (1, 129, 131072, 384), (4, 1070, 16000, 4096),
         (2, 540, 32032, 96), (1, 34000, 512, 128), (6, 2080, 8160, 128), (8, 4097, 4128, 512),
         (3, 8200, 4128, 128), (5, 2700, 12800, 256), (8, 12300, 4128, 512)]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("T,Nn,K,group", LARGE)
def test_matvec_of_large_weights(T, Nn, K, group, wide):
    dtype = torch.bfloat16 if (T + wide) % 2 else torch.float16
    w = weight(Nn, K, group, dtype, K % 3 == 0, seed=K + Nn, pad=T % 3)
    x = torch.randn(T, K, generator=gen(T)).to(dtype)
    if wide:
        x = (x * 10 ** (torch.rand(T, K, generator=gen(T + 2)) * 7 - 5)).to(dtype)
    bias = torch.randn(Nn, generator=gen(T + 1)).to(dtype) if Nn % 2 else None
    v, size = opened(w)
    X = x.double()
    ref, mag = X @ v.t(), X.abs() @ size.t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    wd, args = gpu(w), dict(bias=None if bias is None else bias.cuda())
    out = block.matvec_w4(x.cuda(), wd, **args)
    within(out, ref, U[dtype] * ref.abs() * 1.01 + ACC * mag + 2.0 ** -22 * step_most(X) @ v.abs().t())
    assert torch.equal(out, block.matvec_w4(x.cuda(), wd, **args))
    bad = x.repeat(2, 1)[:T + 1] if T == 1 else x.clone()
    bad[0, K - 1], bad[0, 0] = float("inf"), 0
    got = block.matvec_w4(bad.cuda(), wd, **args)
    assert not got[0].isfinite().any() and torch.equal(got[1:], out[:1] if T == 1 else out[1:])
    status_clean()


@pytest.mark.parametrize("T,D,F,Nn,group,down", [(1, 2048, 4160, 4100, 64, 32), (2, 1056, 8192, 2101, 32, 32), (4, 1024, 8224, 2100, 128, 128),
                                                 (5, 2080, 4128, 4100, 256, 128), (3, 2048, 4160, 4100, 128, 32),
                                                 (8, 1056, 8192, 2101, 128, 256), (4, 2080, 8224, 4104, 128, 128),
                                                 (8, 3104, 8192, 6200, 128, 256)])
def test_gated_of_large_weights(T, D, F, Nn, group, down):
    dtype = torch.float16 if T % 2 else torch.bfloat16
    wg, wu = (weight(F, D, group, dtype, T == 2, seed=i + F) for i in range(2))
    wd = weight(Nn, F, down, dtype, T != 2, seed=9)
    x = torch.randn(T, D, generator=gen(T)).to(dtype)
    (vg, sg), (vu, su), (vd, sd) = map(opened, (wg, wu, wd))
    X = x.double()
    g, p, most = X @ vg.t(), X @ vu.t(), 2.0 ** -22 * step_most(X)
    eg, ep = ACC * (X.abs() @ sg.t()) + most @ vg.abs().t(), ACC * (X.abs() @ su.t()) + most @ vu.abs().t()
    a, _ = act64("silu", g)
    h = a * p
    eh = 1.2 * eg * p.abs() + (a.abs() + 1.2 * eg) * ep + ACC * (h.abs() + p.abs()) + 2 * U[dtype] ** 2 * h.abs() + 2.0 ** -24
    eh = eh + 2.0 ** -22 * step_most(h.abs() + eh)
    ref = h @ vd.t()
    bound = U[dtype] * ref.abs() * 1.01 + eh @ vd.abs().t() + ACC * (h.abs() @ sd.t())
    args = [x.cuda(), gpu(wg), gpu(wu), gpu(wd)]
    out = block.gated_ffn_w4(*args)
    within(out, ref, bound * 1.01)
    assert torch.equal(out, block.gated_ffn_w4(*args))
    status_clean()


def test_every_nibble_is_exact():
    """x a unit vector, scale 1: the weights themselves, q - zero, in both types."""
    for dtype in (torch.float16, torch.bfloat16):
        K = 160
        w = weight(32, K, 32, dtype, True, seed=1)
        w = w._replace(scales=torch.ones_like(w.scales))
        out = block.matvec_w4(torch.eye(K, dtype=dtype).cuda(), gpu(w))
        assert torch.equal(out.double().cpu(), opened(w)[0].t())


def test_strided_x_and_not_a_number():
    w = gpu(weight(64, 128, 32, torch.float16, False, seed=2))
    wide = torch.randn(6, 200, generator=gen(3)).half().cuda()
    x = wide[:, 8:136]
    clean = block.matvec_w4(x, w)
    assert torch.equal(clean, block.matvec_w4(x.contiguous(), w))
    bad = x.clone()
    bad[2, 5] = float("nan")
    out = block.matvec_w4(bad, w)
    keep = [0, 1, 3, 4, 5]
    assert out[2].isnan().all() and torch.equal(out[keep], clean[keep])


def test_streams_graphs_and_empty():
    w = gpu(weight(96, 256, 64, torch.bfloat16, True, seed=4))
    x = torch.randn(3, 256, generator=gen(5)).bfloat16().cuda()
    want = block.matvec_w4(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = block.matvec_w4(x, w, stream=s)
    s.synchronize()
    step = CapturedStep(lambda t: block.matvec_w4(t, w), [torch.zeros_like(x)])
    assert torch.equal(want, got) and torch.equal(want, step(x))
    assert block.matvec_w4(x[:0], w).shape == (0, 96)


def test_refusals():
    w = gpu(weight(64, 128, 32, torch.float16, False, seed=6))
    x = torch.zeros(2, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="uint8"):
        block.matvec_w4(x[:, :64], w)
    with pytest.raises(ValueError, match="scales"):
        block.matvec_w4(x.bfloat16(), w)
    with pytest.raises(ValueError, match="scales must be"):
        block.matvec_w4(x, w._replace(group=64))
    with pytest.raises(ValueError, match="bias"):
        block.matvec_w4(x, w, bias=torch.zeros(64, device="cuda"))
    with pytest.raises(ValueError, match="act"):
        block.gated_ffn_w4(x, w, w, w, act="none")
    with pytest.raises(ValueError, match="w_down"):
        block.gated_ffn_w4(x, w, w, w)
    with pytest.raises(block.N.FoError, match="multiple of 32"):
        block.matvec_w4(x, block.W4(w.q, w.scales[:, :2].contiguous(), None, 80))


def test_stack_trains_and_serves():
    """The operators together: a few steps lower the loss; 4-bit serving stays near 16-bit."""
    weights = make_weights(2, 128, 256)
    stack = GatedStack(weights, torch.ones(128, dtype=torch.bfloat16, device="cuda"))
    for p in stack.parameters():
        p.requires_grad_()
    x, target = (torch.randn(96, 128, generator=gen(i)).bfloat16().cuda() for i in range(2))
    losses = [train_step(stack, x, target, 2.0).item() for _ in range(12)]
    assert losses[-1] < 0.97 * losses[0] and all(b < a * 1.02 for a, b in zip(losses, losses[1:]))
    want = stack(x[:3])
    assert torch.equal(want, CapturedStep(stack, [torch.zeros_like(x[:3])])(x[:3]))
    # rounding to 16 levels of a normal weight: about 1/10 of its deviation, in each of the
    # four products that a value passes; the residual stream carries the rest unchanged
    got = stack.quantize(32)(x[:3])
    assert (got - want).float().norm() < 0.4 * want.float().norm()
