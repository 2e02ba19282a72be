"""What the decoder-block operators accept beyond plain contiguous matrices."""
import pytest
import torch

from block_util import U, within
from gpu_util import gen, status_clean

from icpp_tuning_b200 import block
from test_block_norm_gpu import backward64, d64, gpu as norm_gpu, make as norm_inputs
from test_w4_gpu import gpu, weight

pytestmark = pytest.mark.gpu


def odd(t):
    """The one-row matrix `t` with a row stride of 1: contiguous, as PyTorch counts."""
    out = t.as_strided(t.shape, (1, 1))
    assert out.shape[0] == 1 and out.is_contiguous()
    return out


def test_one_row_of_any_stride():
    D, F, dt = 64, 128, torch.bfloat16
    x, y = (torch.randn(1, D, generator=gen(i)).to(dt).cuda() for i in range(2))
    w = [(torch.randn(*s, generator=gen(9)) * 0.1).to(dt).cuda() for s in ((F, D), (F, D), (D, F))]
    v = torch.ones(D, dtype=dt, device="cuda")
    saved = block.gated_ffn(x, *w, b_layout="nk", save=True)
    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
    assert same(saved, block.gated_ffn(odd(x), *w, b_layout="nk", save=True))
    back = block.gated_ffn_backward(y, x, *w, *saved[1:], b_layout="nk")
    assert same(back, block.gated_ffn_backward(odd(y), odd(x), *w, *map(odd, saved[1:]), b_layout="nk"))
    assert same(block.block_norm(y, x, v, v), block.block_norm(odd(y), odd(x), v, v))
    a, b = block.block_norm_backward(y, x, y, x, v, v), block.block_norm_backward(odd(y), odd(x), odd(y), odd(x), v, v)
    assert same(a.values(), b.values())
    q, one = gpu(weight(96, D, 32, dt, True, seed=1)), gpu(weight(1, D, 32, dt, True, seed=2))
    assert torch.equal(block.matvec_w4(x, q), block.matvec_w4(odd(x), q))
    assert torch.equal(block.matvec_w4(x, one), block.matvec_w4(x, one._replace(q=odd(one.q), scales=odd(one.scales), zeros=odd(one.zeros))))
    status_clean()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 5, 32, 40])
def test_an_infinity_between_the_products(T, dtype):
    """h = inf stays an infinity on its way through the second product, in parts or whole."""
    D, F = 64, 128
    x = torch.rand(T, D, generator=gen(T)).to(dtype).cuda() + 0.5
    x[0, 3] = float("inf")
    w = [(torch.rand(F, D, generator=gen(i)).to(dtype).cuda() + 0.25) / 8 for i in range(3)]
    y = block.gated_ffn(x, w[0], w[1], w[2].t().contiguous(), b_layout="nk")
    assert (y[0] == float("inf")).all()
    up = block.W4(torch.full((F, D // 2), 0x99, dtype=torch.uint8, device="cuda"), torch.full((F, 2), 2.0 ** -6, dtype=dtype, device="cuda"), None, 32)
    down = block.W4(torch.full((D, F // 2), 0x99, dtype=torch.uint8, device="cuda"), torch.full((D, 4), 2.0 ** -6, dtype=dtype, device="cuda"), None, 32)
    z = block.gated_ffn_w4(x, up, up, down)
    assert (z[0] == float("inf")).all()
    if T > 1:
        assert y[1:].isfinite().all() and z[1:].isfinite().all()
    status_clean()


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("T,D,rows", [(700, 129, 700), (900, 264, 300), (400, 1030, 200), (333, 64, 111)])
def test_norm_gradients_of_many_gate_rows(T, D, rows, layer):
    """A gate a token, and groups on both sides of one unit of work a gate row."""
    dtype, vec = torch.bfloat16, torch.float32
    v = norm_inputs(T, D, dtype, vec, layer, True, rows, seed=T)
    v["r"] = v.pop("x")
    dr, dz = ((torch.randn(T, D, generator=gen(i)) * 0.5).to(dtype) for i in range(2))
    w = d64(v)
    ref = backward64(w, dr.double(), dz.double(), w["r"], 0.5, layer, U[dtype], U[vec])
    c = {k: norm_gpu(t) for k, t in v.items()}
    out = block.block_norm_backward(dr.cuda(), dz.cuda(), c["y"], c["r"], c["w_post"], c["w_pre"], b_post=c["b_post"], b_pre=c["b_pre"],
                                    gate=c["gate"], residual_scale=0.5, norm="layer" if layer else "rms")
    assert set(out) == set(ref)
    for k, (r, b) in ref.items():
        within(out[k], r, b, k)
    status_clean()
