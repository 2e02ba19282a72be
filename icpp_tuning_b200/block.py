"""Operators of a decoder block's feed-forward half over libb200fo.so, for torch CUDA tensors.

  gated_ffn, gated_ffn_backward     the gated feed-forward block (act(x Wg) * (x Wu)) Wd
  block_norm, block_norm_backward   the norms after and before a block, fused with its gate
                                    and the residual scale
  matvec_w4, gated_ffn_w4           products of a few tokens with 4-bit weights (W4), plain and
                                    as the whole gated feed-forward block; quantize_w4 lays
                                    such weights out

Functional calls like those of `fused`: PyTorch supplies device memory and the current
stream, every FLOP runs in the library's sm_100a kernels, CPU tensors are refused.  Outputs
are allocated on the stream the call runs on (`stream=` or the current one).
"""
from __future__ import annotations

import ctypes
from typing import Dict, NamedTuple, Optional, Tuple

import torch

from . import _native as N
from .fused import _require_cuda, _vec, dtype_code

GATE_ACTS = {"silu": N.FO_GATE_SILU, "gelu_tanh": N.FO_GATE_GELU_TANH, "gelu_erf": N.FO_GATE_GELU_ERF,
             "relu": N.FO_GATE_RELU}
NORMS = {"rms": N.FO_NORM_RMS, "layer": N.FO_NORM_LAYER}
MAX_NORM_BACKWARD = 8192  # columns of a row in block_norm_backward (block_norm: 16384)


def _run(dev: torch.device, fn, desc) -> None:
    """Calls a C entry on `dev`'s current stream."""
    stream = torch._C._cuda_getCurrentRawStream(dev.index)  # current_stream(dev).cuda_stream without the Stream object
    if torch.cuda.current_device() == dev.index:
        rc = fn(desc, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(desc, stream)
    if rc:
        N.check(rc)


def _cuda(*ts: Optional[torch.Tensor]) -> torch.device:
    """The one CUDA device of these tensors (None: not given)."""
    dev = ts[0].device
    for t in ts:
        if t is not None and t.device != dev:
            return _require_cuda(*ts)  # raises
    return dev if dev.type == "cuda" else _require_cuda(*ts)


def _ld(t: torch.Tensor, rows: int, cols: int, name: str) -> int:
    """Row stride of a 2-D operand that must be [rows, cols] with unit column stride.  A single
    row may carry any: it counts as one that every operator takes."""
    if t.shape != (rows, cols):
        raise ValueError(f"{name} must be [{rows}, {cols}], got {list(t.shape)}")
    st = t.stride()
    if st[1] != 1 and cols != 1:
        raise ValueError(f"{name} must be a 2-D tensor with unit column stride")
    return st[0] if rows != 1 else (cols + 15) // 16 * 16


def _shape2(t: torch.Tensor, name: str) -> Tuple[int, int]:
    if t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor with unit column stride")
    return t.shape


def _sixteen_bit(dt: torch.dtype, name: str) -> int:
    if dt is torch.bfloat16:
        return N.FO_DT_BF16
    if dt is torch.float16:
        return N.FO_DT_F16
    raise ValueError(f"{name} must be float16 or bfloat16, got {dt}")


def _new(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous [rows, cols] of like's type."""
    if like.shape == (rows, cols) and like.is_contiguous():
        return torch.empty_like(like, memory_format=torch.contiguous_format)  # the cheapest call
    return like.new_empty((rows, cols))


# ---------------------------------------------------------------------- gated feed-forward block
def _matrix(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """An uninitialised [rows, cols] whose row stride is a multiple of 8 elements."""
    if cols % 8 == 0:
        return _new(rows, cols, like)
    return like.new_empty((rows, (cols + 7) // 8 * 8))[:, :cols]


def aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """`t`, or a copy of it, as the gated block takes a matrix: unit column stride, rows that
    start on 16-byte boundaries (a row stride that is a multiple of 8 elements)."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return _matrix(*t.shape, t).copy_(t)


def _ffn_desc(x, w_gate, w_up, w_down, act, b_layout, others) -> N.FoGatedFfnDesc:
    code = GATE_ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(GATE_ACTS)}")
    if b_layout not in ("kn", "nk"):
        raise ValueError("b_layout must be 'kn' or 'nk'")
    kn = b_layout == "kn"
    dt = x.dtype
    for t in (w_gate, w_up, w_down, *others):
        if t.dtype is not dt:
            raise ValueError("every matrix of the block must share x's dtype")
    T, D = _shape2(x, "x")
    d = N.FoGatedFfnDesc()
    d.dtype, d.act, d.b_layout = _sixteen_bit(dt, "x"), code, N.FO_B_KN if kn else N.FO_B_NK
    if kn:
        F, Nn = _shape2(w_down, "w_down")
        d.ldwg, d.ldwu, d.ldwd = _ld(w_gate, D, F, "w_gate"), _ld(w_up, D, F, "w_up"), _ld(w_down, F, Nn, "w_down")
    else:
        Nn, F = _shape2(w_down, "w_down")
        d.ldwg, d.ldwu, d.ldwd = _ld(w_gate, F, D, "w_gate"), _ld(w_up, F, D, "w_up"), _ld(w_down, Nn, F, "w_down")
    d.T, d.D, d.F, d.N = T, D, F, Nn
    d.x, d.ldx = x.data_ptr(), _ld(x, T, D, "x")
    d.w_gate, d.w_up, d.w_down = w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr()
    return d


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *, act: str = "silu",
              b_layout: str = "kn", save: bool = False, stream=None):
    """y = (act(x Wg) * (x Wu)) Wd, the two products accumulated in fp32.

    x [T, D] float16 / bfloat16; w_gate, w_up [D, F] and w_down [F, N] when b_layout == "kn",
    [F, D] and [N, F] when "nk" (nn.Linear).  act: one of GATE_ACTS.  Returns y [T, N], or with
    save=True (y, g, u): the products before the activation, for gated_ffn_backward.  The
    intermediate act(g) * u is rounded to x's dtype; up to 32 tokens it is held in two parts of
    that dtype, its high and its low bits.  Row strides must be multiples of 8; results whose
    width is no multiple of 8 are views of such wider rows."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return gated_ffn(x, w_gate, w_up, w_down, act=act, b_layout=b_layout, save=save)
    dev = _cuda(x, w_gate, w_up, w_down)
    d = _ffn_desc(x, w_gate, w_up, w_down, act, b_layout, ())
    T, F, Nn = d.T, d.F, d.N
    y = _matrix(T, Nn, x)
    d.y, d.ldy = y.data_ptr(), y.stride(0)
    if save:
        g, u = _matrix(T, F, x), _matrix(T, F, x)
        d.g, d.ldg, d.u, d.ldu = g.data_ptr(), g.stride(0), u.data_ptr(), u.stride(0)
    lib = N.lib()
    ref = ctypes.byref(d)
    need = lib.fo_gated_ffn_workspace_size(ref, 0)
    ws = x.new_empty((need + 1) // 2)  # x's dtype has two bytes
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_gated_ffn, ref)
    return (y, g, u) if save else y


def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       g: torch.Tensor, u: torch.Tensor, *, act: str = "silu", b_layout: str = "kn",
                       stream=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw_gate, dw_up, dw_down) of gated_ffn from dy [T, N] and the g, u it saved, each laid
    out like its operand in rows whose stride is a multiple of 8.  `aligned_rows` brings a dy of
    any strides into that form."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return gated_ffn_backward(dy, x, w_gate, w_up, w_down, g, u, act=act, b_layout=b_layout)
    dev = _cuda(x, dy, w_gate, w_up, w_down, g, u)
    d = _ffn_desc(x, w_gate, w_up, w_down, act, b_layout, (dy, g, u))
    T, F = d.T, d.F
    d.dy, d.lddy = dy.data_ptr(), _ld(dy, T, d.N, "dy")
    d.g, d.ldg = g.data_ptr(), _ld(g, T, F, "g")
    d.u, d.ldu = u.data_ptr(), _ld(u, T, F, "u")
    dx, dwg, dwu, dwd = (_matrix(*t.shape, x) for t in (x, w_gate, w_up, w_down))
    d.dx, d.dw_gate, d.dw_up, d.dw_down = dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr(), dwd.data_ptr()
    d.lddx, d.lddwg, d.lddwu, d.lddwd = dx.stride(0), dwg.stride(0), dwu.stride(0), dwd.stride(0)
    lib = N.lib()
    ref = ctypes.byref(d)
    need = lib.fo_gated_ffn_workspace_size(ref, 1)
    ws = x.new_empty((need + 1) // 2)  # x's dtype has two bytes
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_gated_ffn_backward, ref)
    return dx, dwg, dwu, dwd


# ---------------------------------------------------------------------- norms around a block
def _param(v: Optional[torch.Tensor], D: int, dt: torch.dtype, name: str) -> Optional[int]:
    if v is None:
        return None
    if v.dtype is not dt:
        raise ValueError("the norms' parameters and the gate must share one dtype")
    if v.shape != (D,) or not v.is_contiguous():
        _vec(v, D, name)  # raises
    return v.data_ptr()



def _norm_desc(y, w_post, w_pre, b_post, b_pre, gate, residual_scale, norm, eps) -> N.FoBlockNormDesc:
    T, D = _shape2(y, "y")
    if norm not in NORMS:
        raise ValueError(f"norm must be one of {sorted(NORMS)}")
    if w_pre is None:
        raise ValueError("w_pre is required")
    dt = w_pre.dtype
    d = N.FoBlockNormDesc()
    d.T, d.D, d.dtype, d.norm, d.vec_dtype = T, D, _sixteen_bit(y.dtype, "y"), NORMS[norm], dtype_code(dt)
    d.residual_scale, d.eps = residual_scale, eps
    d.y, d.ldy = y.data_ptr(), _ld(y, T, D, "y")
    d.w_pre = _param(w_pre, D, dt, "w_pre")
    if w_post is not None:
        d.w_post = _param(w_post, D, dt, "w_post")
    if b_pre is not None:
        d.b_pre = _param(b_pre, D, dt, "b_pre")
    if b_post is not None:
        d.b_post = _param(b_post, D, dt, "b_post")
    if gate is not None:
        if gate.dim() == 1:
            d.gate, d.gate_rows, d.ldgate = _param(gate, D, dt, "gate"), 1, D
        else:
            G = gate.shape[0]
            if gate.dtype is not dt:
                raise ValueError("the norms' parameters and the gate must share one dtype")
            if gate.dim() != 2 or gate.shape[1] != D or G == 0 or T % G:
                raise ValueError(f"gate must be [{D}] or [G, {D}] with G dividing T = {T}, got {list(gate.shape)}")
            d.gate, d.gate_rows, d.ldgate = gate.data_ptr(), G, _ld(gate, G, D, "gate")
    return d


def block_norm(y: torch.Tensor, x: torch.Tensor, w_post: Optional[torch.Tensor], w_pre: torch.Tensor, *,
               b_post: Optional[torch.Tensor] = None, b_pre: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, norm: str = "rms", eps: float = 1e-5,
               stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(r, z): r = residual_scale * x + gate * norm_post(y), z = norm_pre(r).

    y: the block's output, x: the residual stream, [T, D] float16 / bfloat16.  norm "rms"
    (v * rsqrt(mean v^2 + eps) * w) or "layer" (with mean and optional biases).  w_post None:
    no norm after the block.  gate: None, [D], or [G, D], each row for T / G consecutive rows.
    z is computed from the unrounded r."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return block_norm(y, x, w_post, w_pre, b_post=b_post, b_pre=b_pre, gate=gate, residual_scale=residual_scale,
                              norm=norm, eps=eps)
    dev = _cuda(y, x, w_post, w_pre, b_post, b_pre, gate)
    d = _norm_desc(y, w_post, w_pre, b_post, b_pre, gate, residual_scale, norm, eps)
    if x.dtype is not y.dtype:
        raise ValueError("x and y must share one dtype")
    T, D = y.shape
    d.x, d.ldx = x.data_ptr(), _ld(x, T, D, "x")
    r, z = _new(T, D, y), _new(T, D, y)
    d.r, d.z, d.ldr, d.ldz = r.data_ptr(), z.data_ptr(), D, D
    _run(dev, N.lib().fo_block_norm, ctypes.byref(d))
    return r, z


def block_norm_backward(dr: Optional[torch.Tensor], dz: torch.Tensor, y: torch.Tensor, r: torch.Tensor,
                        w_post: Optional[torch.Tensor], w_pre: torch.Tensor, *, b_post: Optional[torch.Tensor] = None,
                        b_pre: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        residual_scale: float = 1.0, norm: str = "rms", eps: float = 1e-5,
                        stream=None) -> Dict[str, torch.Tensor]:
    """Gradients of block_norm's inputs from those of r (`dr`; None: zero) and z (`dz`), its
    input y and its output r: {"dy", "dx", "dw_pre"} and, for the parameters that are given,
    "dw_post", "db_post", "db_pre" and "dgate".  The statistics are recomputed from y and r."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return block_norm_backward(dr, dz, y, r, w_post, w_pre, b_post=b_post, b_pre=b_pre, gate=gate,
                                       residual_scale=residual_scale, norm=norm, eps=eps)
    dev = _cuda(y, dr, dz, r, w_post, w_pre, b_post, b_pre, gate)
    d = _norm_desc(y, w_post, w_pre, b_post, b_pre, gate, residual_scale, norm, eps)
    T, D = y.shape
    for t, name in ((dr, "dr"), (dz, "dz"), (r, "r")):
        if t is not None and t.dtype is not y.dtype:
            raise ValueError(f"{name} and y must share one dtype")
    if dr is not None:
        d.dr, d.lddr = dr.data_ptr(), _ld(dr, T, D, "dr")
    d.dz, d.lddz = dz.data_ptr(), _ld(dz, T, D, "dz")
    d.r, d.ldr = r.data_ptr(), _ld(r, T, D, "r")
    out = {"dy": _new(T, D, y), "dx": _new(T, D, y)}
    d.lddy = d.lddx = D
    # the parameters' gradients share one allocation, gate rows last
    names = [n for n, p in (("dw_pre", w_pre), ("dw_post", w_post), ("db_pre", b_pre), ("db_post", b_post)) if p is not None]
    rows = len(names)
    flat = w_pre.new_empty((rows + d.gate_rows, D))
    at, step = flat.data_ptr(), D * flat.element_size()
    out.update(zip(names, flat.unbind(0)))
    for i, name in enumerate(names):
        setattr(d, name, at + i * step)
    if gate is not None:
        out["dgate"] = out_gate = flat[rows] if gate.dim() == 1 else flat[rows:]
        d.dgate = out_gate.data_ptr()
    d.dy, d.dx = out["dy"].data_ptr(), out["dx"].data_ptr()
    lib = N.lib()
    ref = ctypes.byref(d)
    need = lib.fo_block_norm_backward_workspace_size(ref)
    ws = y.new_empty((max(16, need) + 1) // 2)  # y's dtype has two bytes
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_block_norm_backward, ref)
    return out


# ---------------------------------------------------------------------- 4-bit weights
class W4(NamedTuple):
    """A weight matrix [N, K] in 4 bits: w[n, k] = scales[n, k // group] * (q - zeros[n, k // group]).

    q: uint8 [N, K / 2], two weights to a byte, the lower nibble the even k; scales: [N,
    ceil(K / group)] of the activations' dtype; zeros: uint8 of the same shape, or None
    (every zero is 8).  K and group are multiples of 32."""
    q: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor]
    group: int


def quantize_w4(w: torch.Tensor, group: int = 128, symmetric: bool = True) -> W4:
    """Rounds w [N, K] to 4 bits, each group of `group` weights of a row with its own scale
    (and zero, if not symmetric).  Done once per weight, in plain PyTorch on w's device."""
    if w.dim() != 2 or group <= 0 or group % 32 or w.shape[1] % 32:
        raise ValueError("quantize_w4 takes [N, K] with K and group multiples of 32")
    Nn, K = w.shape
    G = -(-K // group)
    v = torch.nn.functional.pad(w.float(), (0, G * group - K)).reshape(Nn, G, group)
    if symmetric:
        scale = (v.abs().amax(2) / 7).clamp_min(1e-12).to(w.dtype)
        zero = torch.full((Nn, G), 8.0, device=w.device)
    else:
        lo, hi = v.amin(2).clamp_max(0), v.amax(2).clamp_min(0)
        scale = ((hi - lo) / 15).clamp_min(1e-12).to(w.dtype)
        zero = (-lo / scale.float().clamp_min(1e-12)).round().clamp(0, 15)
    s = scale.float().unsqueeze(2)
    q = torch.where(s > 0, v / s.clamp_min(1e-30), torch.zeros((), device=w.device)) + zero.unsqueeze(2)
    q = q.round().clamp(0, 15).to(torch.uint8).reshape(Nn, -1)[:, :K]
    return W4(q[:, 0::2] | (q[:, 1::2] << 4), scale, None if symmetric else zero.to(torch.uint8), group)


def _w4(w: W4, K: int, dtype: torch.dtype, name: str) -> Tuple[N.FoW4, int]:
    """The C form of a weight and its number of rows."""
    q, scales, zeros, group = w
    if q.dim() != 2 or q.dtype is not torch.uint8 or 2 * q.shape[1] != K:
        raise ValueError(f"{name}.q must be uint8 [N, {K // 2}], got {q.dtype} {list(q.shape)}")
    if group <= 0:
        raise ValueError(f"{name}.group must be a positive multiple of 32, got {group}")
    n, G = q.shape[0], -(-K // group)
    if scales.dtype is not dtype:
        raise ValueError(f"{name}.scales must be {dtype}, the activations' dtype")
    if zeros is None:
        return N.FoW4(q.data_ptr(), scales.data_ptr(), None, _ld(q, n, K // 2, name + ".q"),
                      _ld(scales, n, G, name + ".scales"), 0, group), n
    if zeros.dtype is not torch.uint8:
        raise ValueError(f"{name}.zeros must be uint8")
    return N.FoW4(q.data_ptr(), scales.data_ptr(), zeros.data_ptr(), _ld(q, n, K // 2, name + ".q"),
                  _ld(scales, n, G, name + ".scales"), _ld(zeros, n, G, name + ".zeros"), group), n


def matvec_w4(x: torch.Tensor, w: W4, *, bias: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """x [T, K] @ w^T (+ bias) for a few tokens, w in 4 bits: [T, N] of x's dtype.

    Sums are fp32.  One token, or a few, times large weights takes x as fixed point of 23 bits
    relative to the largest of its 128 values: an infinity in x then gives NaN in its row."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return matvec_w4(x, w, bias=bias)
    dev = _cuda(x, w.q, w.scales, w.zeros, bias)
    T, K = _shape2(x, "x")
    dt = x.dtype
    d = N.FoMatvecW4Desc()
    d.dtype, d.ldx = _sixteen_bit(dt, "x"), _ld(x, T, K, "x")
    d.w, n = _w4(w, K, dt, "w")
    d.T, d.K, d.N = T, K, n
    if bias is not None:
        if bias.dtype is not dt:
            raise ValueError("bias must have the activations' dtype")
        d.bias = _vec(bias, n, "bias").data_ptr()
    out = _new(T, n, x)
    d.x, d.out, d.ldo = x.data_ptr(), out.data_ptr(), n
    lib = N.lib()
    ref = ctypes.byref(d)
    need = lib.fo_matvec_w4_workspace_size(ref)
    if need:
        ws = x.new_empty((need + 1) // 2)  # x's dtype has two bytes
        d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_matvec_w4, ref)
    return out


def gated_ffn_w4(x: torch.Tensor, w_gate: W4, w_up: W4, w_down: W4, *, act: str = "silu", stream=None) -> torch.Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T for a few tokens, all weights in 4 bits: [T, N]
    of x's dtype.  w_gate and w_up share one group size."""
    code = GATE_ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(GATE_ACTS)}")
    if stream is not None:
        with torch.cuda.stream(stream):
            return gated_ffn_w4(x, w_gate, w_up, w_down, act=act)
    dev = _cuda(x, *w_gate[:3], *w_up[:3], *w_down[:3])
    T, D = _shape2(x, "x")
    dt = x.dtype
    d = N.FoGatedFfnW4Desc()
    d.dtype, d.act, d.ldx = _sixteen_bit(dt, "x"), code, _ld(x, T, D, "x")
    d.w_gate, F = _w4(w_gate, D, dt, "w_gate")
    d.w_up, F_up = _w4(w_up, D, dt, "w_up")
    if F_up != F:
        raise ValueError(f"w_gate has {F} rows, w_up {F_up}")
    d.w_down, n = _w4(w_down, F, dt, "w_down")
    d.T, d.D, d.F, d.N = T, D, F, n
    out = _new(T, n, x)
    d.x, d.out, d.ldo = x.data_ptr(), out.data_ptr(), n
    lib = N.lib()
    ref = ctypes.byref(d)
    need = lib.fo_gated_ffn_w4_workspace_size(ref)
    ws = x.new_empty((need + 1) // 2)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_gated_ffn_w4, ref)
    return out
