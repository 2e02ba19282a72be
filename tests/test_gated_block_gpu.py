"""The autograd functions of gated_block against the 64-bit gradients and their derived bounds."""
import pytest
import torch

from block_util import U, ffn_backward, within
from gpu_util import gen, status_clean
from test_block_norm_gpu import EPS, backward64, d64, gpu, make as norm_inputs
from test_gated_ffn_gpu import as_kn, cuda, make as ffn_inputs

from icpp_tuning_b200 import block, gated_block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("T,D,F,Nn", [(5, 72, 136, 100), (70, 264, 520, 33), (300, 64, 128, 520)])
def test_gated_ffn(T, D, F, Nn, layout):
    """Few and many tokens, output widths that are no multiple of 8."""
    dtype = torch.bfloat16
    x, *w = ffn_inputs(T, D, F, Nn, dtype, layout, seed=T)
    args = [cuda(t).requires_grad_() for t in (x, *w)]
    y = gated_block.GatedFFN.apply(*args, "silu", layout)
    dy = (torch.randn(T, Nn, generator=gen(2)) * 0.1).to(dtype)
    got = torch.autograd.grad(y, args, dy.cuda())
    _, g, u = block.gated_ffn(*(t.detach() for t in args), b_layout=layout, save=True)
    ref, bound = ffn_backward(dy.double(), x.double(), *as_kn(w, layout), g.double().cpu(), u.double().cpu(), "silu", U[dtype])
    for i, (o, r, b, name) in enumerate(zip(got, ref, bound, ("dx", "dw_gate", "dw_up", "dw_down"))):
        flip = layout == "nk" and i > 0
        within(o, r.t() if flip else r, b.t() if flip else b, name)
    status_clean()


@pytest.mark.parametrize("which", ["both", "r", "z"])
@pytest.mark.parametrize("layer", [False, True])
def test_block_norm(layer, which):
    """Gradients that come for both outputs or for one of them, in rows of any stride."""
    T, D, dtype = 24, 200, torch.float16
    v = norm_inputs(T, D, dtype, torch.float32, layer, True, 3, seed=3)
    names = [k for k in ("y", "x", "w_post", "w_pre", "b_post", "b_pre", "gate") if v[k] is not None]
    c = {k: None if t is None else gpu(t).requires_grad_() for k, t in v.items()}
    r, z = gated_block.BlockNorm.apply(c["y"], c["x"], c["w_post"], c["w_pre"], c["b_post"], c["b_pre"], c["gate"], 0.7,
                                       "layer" if layer else "rms", EPS)
    g = gen(4)
    dr, dz = ((torch.randn(D, T, generator=g) * 0.5).to(dtype).t() for _ in range(2))
    outs = {"both": ((r, z), (dr, dz)), "r": ((r,), (dr,)), "z": ((z,), (dz,))}[which]
    got = torch.autograd.grad(outs[0], [c[k] for k in names if which != "r" or k not in ("w_pre", "b_pre")], [t.cuda() for t in outs[1]])
    w = d64(v)
    w["r"] = r.detach().double().cpu()
    zero = torch.zeros(T, D, dtype=torch.float64)
    ref = backward64(w, dr.double() if which != "z" else zero, dz.double() if which != "r" else zero, w["r"], 0.7, layer, U[dtype], U[torch.float32])
    for k, o in zip([k for k in names if which != "r" or k not in ("w_pre", "b_pre")], got):
        within(o, *ref["d" + k], "d" + k)
    status_clean()
