"""Refusals of the decoder-block operators without a GPU: the C entries reject bad arguments
before touching a device, the Python calls refuse CPU tensors."""
import ctypes

import pytest
import torch

from icpp_tuning_b200 import _native as N
from icpp_tuning_b200 import block

A = 1 << 20  # an aligned fake address: validation never dereferences


def _ffn(**kw):
    d = N.FoGatedFfnDesc()
    d.T, d.D, d.F, d.N = 4, 64, 128, 64
    for n in ("x", "w_gate", "w_up", "w_down", "y", "dy", "dx", "dw_gate", "dw_up", "dw_down", "workspace"):
        setattr(d, n, A)
    d.ldx = d.ldy = d.lddy = d.lddx = 64
    d.ldwg = d.ldwu = d.lddwg = d.lddwu = 64
    d.ldwd = d.lddwd = 128
    d.ldg = d.ldu = 128
    d.dtype, d.b_layout, d.act, d.workspace_bytes = N.FO_DT_BF16, N.FO_B_NK, N.FO_GATE_SILU, 1 << 30
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=N.FO_DT_F32), "dtype"), (dict(b_layout=9), "b_layout"), (dict(act=0), "activation"), (dict(T=-1), "negative"),
    (dict(ldx=60), "x"), (dict(ldwg=32), "w_gate"), (dict(w_up=A + 8), "w_up"), (dict(w_down=None), "w_down"), (dict(y=None), "y"),
    (dict(g=A), "together"), (dict(workspace_bytes=16), "workspace"), (dict(D=0), "positive"),
])
def test_gated_ffn_rejects(kw, msg):
    assert N.lib().fo_gated_ffn(ctypes.byref(_ffn(**kw)), None) == N.FO_EINVAL
    assert msg in N.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(), "g must"), (dict(g=A, u=A, dy=None), "dy"), (dict(g=A, u=A, dw_down=None), "dw_down"),
    (dict(g=A, u=A, ldu=64), "u"), (dict(g=A, u=A, workspace=None), "workspace"),
])
def test_gated_ffn_backward_rejects(kw, msg):
    assert N.lib().fo_gated_ffn_backward(ctypes.byref(_ffn(**kw)), None) == N.FO_EINVAL
    assert msg in N.last_error()


def _norm(**kw):
    d = N.FoBlockNormDesc()
    d.T, d.D = 4, 64
    for n in ("y", "x", "r", "z", "dz", "dy", "dx", "w_pre", "dw_pre"):
        setattr(d, n, A)
    for n in ("ldy", "ldx", "ldr", "ldz", "lddz", "lddy", "lddx"):
        setattr(d, n, 64)
    d.dtype, d.vec_dtype, d.norm, d.residual_scale, d.eps = N.FO_DT_F16, N.FO_DT_F32, N.FO_NORM_RMS, 1.0, 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=N.FO_DT_F32), N.FO_EINVAL, "dtype"), (dict(vec_dtype=5), N.FO_EINVAL, "vec_dtype"),
    (dict(norm=2), N.FO_EINVAL, "norm"), (dict(eps=-1.0), N.FO_EINVAL, "eps"), (dict(b_pre=A), N.FO_EINVAL, "bias"),
    (dict(norm=N.FO_NORM_LAYER, b_post=A), N.FO_EINVAL, "w_post"), (dict(gate_rows=1), N.FO_EINVAL, "gate"),
    (dict(gate=A, gate_rows=3, ldgate=64), N.FO_EINVAL, "divide"), (dict(D=16385), N.FO_EUNSUPPORTED, "16384"),
    (dict(w_pre=None), N.FO_EINVAL, "w_pre"), (dict(T=-1), N.FO_EINVAL, "negative"),
])
def test_block_norm_rejects(kw, code, msg):
    assert N.lib().fo_block_norm(ctypes.byref(_norm(**kw)), None) == code
    assert msg in N.last_error()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(), N.FO_EINVAL, "workspace"), (dict(dz=None), N.FO_EINVAL, "dz"), (dict(w_post=A), N.FO_EINVAL, "dw_post"),
    (dict(gate=A, gate_rows=2, ldgate=64), N.FO_EINVAL, "dgate"), (dict(D=8193), N.FO_EUNSUPPORTED, "8192"),
])
def test_block_norm_backward_rejects(kw, code, msg):
    assert N.lib().fo_block_norm_backward(ctypes.byref(_norm(**kw)), None) == code
    assert msg in N.last_error()


def _w4(**kw):
    w = N.FoW4(A, A, None, 32, 2, 0, 32)
    for k, v in kw.items():
        setattr(w, k, v)
    return w


def _matvec(w=None, **kw):
    d = N.FoMatvecW4Desc()
    d.T, d.N, d.K, d.x, d.out, d.ldx, d.ldo, d.dtype = 1, 16, 64, A, A, 64, 16, N.FO_DT_F16
    d.w = w or _w4()
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("w,kw,msg", [
    (None, dict(K=48), "K = 48"), (None, dict(dtype=N.FO_DT_F32), "dtype"), (None, dict(ldx=60), "x"), (None, dict(x=None), "x must"),
    (None, dict(out=None), "out"), (None, dict(ldo=8), "out"), (_w4(group=48), {}, "group"), (_w4(group=0), {}, "group"),
    (_w4(ldq=24), {}, "ldq"), (_w4(q=A + 4), {}, "aligned"), (_w4(lds=1), {}, "scales"), (_w4(zeros=A), {}, "zeros"),
])
def test_matvec_w4_rejects(w, kw, msg):
    assert N.lib().fo_matvec_w4(ctypes.byref(_matvec(w, **kw)), None) == N.FO_EINVAL
    assert msg in N.last_error()


def test_matvec_w4_workspace():
    small, large = _matvec(), _matvec(_w4(ldq=2048, lds=128), N=8192, K=4096, ldx=4096, ldo=8192)
    need = N.lib().fo_matvec_w4_workspace_size
    assert need(ctypes.byref(small)) == 0 and need(ctypes.byref(large)) > 0 and need(None) == 0
    assert N.lib().fo_matvec_w4(ctypes.byref(large), None) == N.FO_EINVAL and "workspace" in N.last_error()


def test_gated_ffn_w4_rejects():
    d = N.FoGatedFfnW4Desc()
    d.T, d.D, d.F, d.N, d.x, d.out, d.ldx, d.ldo, d.dtype, d.act = 1, 64, 64, 16, A, A, 64, 16, N.FO_DT_F16, N.FO_GATE_SILU
    d.w_gate, d.w_up, d.w_down = _w4(), _w4(group=64, lds=1), _w4()
    call = lambda: N.lib().fo_gated_ffn_w4(ctypes.byref(d), None)  # noqa: E731
    assert call() == N.FO_EINVAL and "group size" in N.last_error()
    d.w_up = _w4()
    assert call() == N.FO_EINVAL and "workspace" in N.last_error()
    d.act = 7
    assert call() == N.FO_EINVAL and "activation" in N.last_error()


def test_empty_calls_are_no_ops():
    assert N.lib().fo_gated_ffn(ctypes.byref(_ffn(T=0)), None) == N.FO_OK
    assert N.lib().fo_block_norm(ctypes.byref(_norm(T=0)), None) == N.FO_OK
    assert N.lib().fo_matvec_w4(ctypes.byref(_matvec(T=0)), None) == N.FO_OK


def test_python_calls_refuse_cpu_tensors():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16)
    v = torch.ones(64, dtype=torch.bfloat16)
    q = block.W4(torch.zeros(64, 32, dtype=torch.uint8), torch.ones(64, 1, dtype=torch.bfloat16), None, 64)
    for call in (lambda: block.gated_ffn(x, w, w, w), lambda: block.gated_ffn_backward(x, x, w, w, w, x, x),
                 lambda: block.block_norm(x, x, v, v), lambda: block.block_norm_backward(x, x, x, x, v, v),
                 lambda: block.matvec_w4(x, q), lambda: block.gated_ffn_w4(x, q, q, q)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("K,group", [(96, 32), (160, 64), (64, 128)])
def test_quantize_w4_stays_within_half_a_step(symmetric, K, group):
    g = torch.Generator().manual_seed(3)
    w = torch.randn(5, K, generator=g)
    w[2] = 0
    q = block.quantize_w4(w, group, symmetric)
    assert q.q.shape == (5, K // 2) and q.scales.shape == (5, -(-K // group)) and (q.zeros is None) == symmetric
    v = torch.stack((q.q & 15, q.q >> 4), 2).reshape(5, K).double()
    at = torch.arange(K) // group
    s = q.scales.double()[:, at]
    back = (v - (8 if symmetric else q.zeros.double()[:, at])) * s
    # half a step; asymmetric zeros are rounded too, which costs the ends half a step more
    assert ((back - w.double()).abs() <= s * (0.5 if symmetric else 1.0) + 1e-6).all()
    assert (back[2] == 0).all()


def test_quantize_w4_refuses():
    for w, group in ((torch.zeros(4, 48), 32), (torch.zeros(64), 32), (torch.zeros(4, 64), 40), (torch.zeros(4, 64), 0)):
        with pytest.raises(ValueError):
            block.quantize_w4(w, group)
