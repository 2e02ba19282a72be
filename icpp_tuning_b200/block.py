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
from .fused import _require_cuda, _rows, _vec, dtype_code

GATE_ACTS = {"silu": N.FO_GATE_SILU, "gelu_tanh": N.FO_GATE_GELU_TANH, "gelu_erf": N.FO_GATE_GELU_ERF,
             "relu": N.FO_GATE_RELU}
NORMS = {"rms": N.FO_NORM_RMS, "layer": N.FO_NORM_LAYER}


def _run(dev: torch.device, fn, *args) -> None:
    """Calls a C entry on `dev`'s current stream."""
    s = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        N.check(fn(*args, s))
    else:
        with torch.cuda.device(dev):
            N.check(fn(*args, s))


def _like(t: torch.Tensor, shape: Tuple[int, int], name: str) -> int:
    """Row stride of a 2-D operand that must have this shape."""
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return _rows(t, name)


def _sixteen_bit(dt: torch.dtype, name: str) -> int:
    if dt not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{name} must be float16 or bfloat16, got {dt}")
    return dtype_code(dt)


# ---------------------------------------------------------------------- gated feed-forward block
def _matrix(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """An uninitialised [rows, cols] whose row stride is a multiple of 8 elements."""
    t = torch.empty((rows, (cols + 7) // 8 * 8), dtype=like.dtype, device=like.device)
    return t if cols % 8 == 0 else t[:, :cols]


def _ffn_desc(x, w_gate, w_up, w_down, act, b_layout, others) -> N.FoGatedFfnDesc:
    if act not in GATE_ACTS:
        raise ValueError(f"act must be one of {sorted(GATE_ACTS)}")
    if b_layout not in ("kn", "nk"):
        raise ValueError("b_layout must be 'kn' or 'nk'")
    kn = b_layout == "kn"
    d = N.FoGatedFfnDesc()
    d.dtype, d.act, d.b_layout = _sixteen_bit(x.dtype, "x"), GATE_ACTS[act], N.FO_B_KN if kn else N.FO_B_NK
    for t in (w_gate, w_up, w_down, *others):
        if t.dtype != x.dtype:
            raise ValueError("every matrix of the block must share x's dtype")
    d.x, d.ldx = x.data_ptr(), _rows(x, "x")
    d.T, d.D = x.shape
    d.ldwd = _rows(w_down, "w_down")
    d.F, d.N = w_down.shape if kn else reversed(w_down.shape)
    up = (d.D, d.F) if kn else (d.F, d.D)
    d.ldwg, d.ldwu = _like(w_gate, up, "w_gate"), _like(w_up, up, "w_up")
    d.w_gate, d.w_up, d.w_down = w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr()
    return d


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *, act: str = "silu",
              b_layout: str = "kn", save: bool = False, stream=None):
    """y = (act(x Wg) * (x Wu)) Wd, the two products accumulated in fp32.

    x [T, D] float16 / bfloat16; w_gate, w_up [D, F] and w_down [F, N] when b_layout == "kn",
    [F, D] and [N, F] when "nk" (nn.Linear).  act: one of GATE_ACTS.  Returns y [T, N], or with
    save=True (y, g, u): the products before the activation, for gated_ffn_backward.  The
    intermediate act(g) * u is rounded to x's dtype.  Row strides must be multiples of 8."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return gated_ffn(x, w_gate, w_up, w_down, act=act, b_layout=b_layout, save=save)
    dev = _require_cuda(x, w_gate, w_up, w_down)
    d = _ffn_desc(x, w_gate, w_up, w_down, act, b_layout, ())
    y = _matrix(d.T, d.N, x)
    d.y, d.ldy = y.data_ptr(), y.stride(0)
    if save:
        g, u = _matrix(d.T, d.F, x), _matrix(d.T, d.F, x)
        d.g, d.ldg, d.u, d.ldu = g.data_ptr(), g.stride(0), u.data_ptr(), u.stride(0)
    lib = N.lib()
    need = lib.fo_gated_ffn_workspace_size(ctypes.byref(d), 0)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_gated_ffn, ctypes.byref(d))
    return (y, g, u) if save else y


def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       g: torch.Tensor, u: torch.Tensor, *, act: str = "silu", b_layout: str = "kn",
                       stream=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw_gate, dw_up, dw_down) of gated_ffn from dy [T, N] and the g, u it saved."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return gated_ffn_backward(dy, x, w_gate, w_up, w_down, g, u, act=act, b_layout=b_layout)
    dev = _require_cuda(x, dy, w_gate, w_up, w_down, g, u)
    d = _ffn_desc(x, w_gate, w_up, w_down, act, b_layout, (dy, g, u))
    d.dy, d.lddy = dy.data_ptr(), _like(dy, (d.T, d.N), "dy")
    d.g, d.ldg = g.data_ptr(), _like(g, (d.T, d.F), "g")
    d.u, d.ldu = u.data_ptr(), _like(u, (d.T, d.F), "u")
    dx, dwg, dwu, dwd = (_matrix(*t.shape, x) for t in (x, w_gate, w_up, w_down))
    d.dx, d.dw_gate, d.dw_up, d.dw_down = dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr(), dwd.data_ptr()
    d.lddx, d.lddwg, d.lddwu, d.lddwd = dx.stride(0), dwg.stride(0), dwu.stride(0), dwd.stride(0)
    lib = N.lib()
    need = lib.fo_gated_ffn_workspace_size(ctypes.byref(d), 1)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_gated_ffn_backward, ctypes.byref(d))
    return dx, dwg, dwu, dwd


# ---------------------------------------------------------------------- norms around a block
def _norm_desc(y, w_post, w_pre, b_post, b_pre, gate, residual_scale, norm, eps) -> N.FoBlockNormDesc:
    if y.dim() != 2:
        raise ValueError("y must be a 2-D tensor with unit column stride")
    T, D = y.shape
    if norm not in NORMS:
        raise ValueError(f"norm must be one of {sorted(NORMS)}")
    vecs = [(_vec(v, D, name), name) for v, name in ((w_pre, "w_pre"), (w_post, "w_post"), (b_pre, "b_pre"), (b_post, "b_post"))]
    if w_pre is None:
        raise ValueError("w_pre is required")
    d = N.FoBlockNormDesc()
    d.T, d.D, d.dtype, d.norm = T, D, _sixteen_bit(y.dtype, "y"), NORMS[norm]
    d.vec_dtype = dtype_code(w_pre.dtype)
    d.residual_scale, d.eps = residual_scale, eps
    for v, name in vecs:
        if v is not None:
            if v.dtype != w_pre.dtype:
                raise ValueError("the norms' parameters and the gate must share one dtype")
            setattr(d, name, v.data_ptr())
    if gate is not None:
        g2 = gate.unsqueeze(0) if gate.dim() == 1 else gate
        if gate.dtype != w_pre.dtype:
            raise ValueError("the norms' parameters and the gate must share one dtype")
        if g2.dim() != 2 or g2.shape[1] != D or g2.shape[0] == 0 or T % g2.shape[0]:
            raise ValueError(f"gate must be [{D}] or [G, {D}] with G dividing T = {T}, got {list(gate.shape)}")
        d.gate, d.gate_rows, d.ldgate = g2.data_ptr(), g2.shape[0], _rows(g2, "gate")
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
    dev = _require_cuda(y, x, w_post, w_pre, b_post, b_pre, gate)
    d = _norm_desc(y, w_post, w_pre, b_post, b_pre, gate, residual_scale, norm, eps)
    shape = (d.T, d.D)
    if x.dtype != y.dtype:
        raise ValueError("x and y must share one dtype")
    d.y, d.ldy, d.x, d.ldx = y.data_ptr(), _rows(y, "y"), x.data_ptr(), _like(x, shape, "x")
    r, z = (torch.empty(shape, dtype=y.dtype, device=dev) for _ in range(2))
    d.r, d.z, d.ldr, d.ldz = r.data_ptr(), z.data_ptr(), d.D, d.D
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
    dev = _require_cuda(y, dr, dz, r, w_post, w_pre, b_post, b_pre, gate)
    d = _norm_desc(y, w_post, w_pre, b_post, b_pre, gate, residual_scale, norm, eps)
    shape = (d.T, d.D)
    for t, name in ((dr, "dr"), (dz, "dz"), (r, "r")):
        if t is not None:
            if t.dtype != y.dtype:
                raise ValueError(f"{name} and y must share one dtype")
            setattr(d, name, t.data_ptr())
            setattr(d, "ld" + name, _like(t, shape, name))
    d.y, d.ldy = y.data_ptr(), _rows(y, "y")
    out = {k: torch.empty(shape, dtype=y.dtype, device=dev) for k in ("dy", "dx")}
    d.lddy = d.lddx = d.D
    for p, name in ((w_pre, "dw_pre"), (w_post, "dw_post"), (b_pre, "db_pre"), (b_post, "db_post"), (gate, "dgate")):
        if p is not None:
            out[name] = torch.empty(p.shape, dtype=p.dtype, device=dev)
    for name, t in out.items():
        setattr(d, name, t.data_ptr())
    lib = N.lib()
    need = lib.fo_block_norm_backward_workspace_size(ctypes.byref(d))
    ws = torch.empty(max(16, need), dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _run(dev, lib.fo_block_norm_backward, ctypes.byref(d))
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
    if w.q.dim() != 2 or w.q.dtype != torch.uint8 or 2 * w.q.shape[1] != K:
        raise ValueError(f"{name}.q must be uint8 [N, {K // 2}], got {w.q.dtype} {list(w.q.shape)}")
    if w.group <= 0:
        raise ValueError(f"{name}.group must be a positive multiple of 32, got {w.group}")
    n, G = w.q.shape[0], -(-K // w.group)
    if w.scales.dtype != dtype:
        raise ValueError(f"{name}.scales must be {dtype}, the activations' dtype")
    if w.zeros is not None and w.zeros.dtype != torch.uint8:
        raise ValueError(f"{name}.zeros must be uint8")
    return N.FoW4(w.q.data_ptr(), w.scales.data_ptr(), None if w.zeros is None else w.zeros.data_ptr(),
                  _rows(w.q, name + ".q"), _like(w.scales, (n, G), name + ".scales"),
                  0 if w.zeros is None else _like(w.zeros, (n, G), name + ".zeros"), w.group), n


def _matvec_w4(x, w, w_up, bias, act):
    dev = _require_cuda(x, w.q, w.scales, w.zeros, bias, *(w_up[:3] if w_up is not None else ()))
    d = N.FoMatvecW4Desc()
    d.dtype, d.ldx = _sixteen_bit(x.dtype, "x"), _rows(x, "x")
    d.T, d.K = x.shape
    d.w, d.N = _w4(w, d.K, x.dtype, "w")
    if w_up is not None:
        d.w_up, n = _w4(w_up, d.K, x.dtype, "w_up")
        if n != d.N:
            raise ValueError(f"w_gate has {d.N} rows, w_up {n}")
    if bias is not None:
        if bias.dtype != x.dtype:
            raise ValueError("bias must have the activations' dtype")
        d.bias = _vec(bias, d.N, "bias").data_ptr()
    out = torch.empty((d.T, d.N), dtype=x.dtype, device=dev)
    d.x, d.out, d.ldo, d.act = x.data_ptr(), out.data_ptr(), d.N, act
    _run(dev, N.lib().fo_matvec_w4, ctypes.byref(d))
    return out


def matvec_w4(x: torch.Tensor, w: W4, *, bias: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """x [T, K] @ w^T (+ bias) for a few tokens, w in 4 bits: [T, N] of x's dtype."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _matvec_w4(x, w, None, bias, N.FO_GATE_NONE)
    return _matvec_w4(x, w, None, bias, N.FO_GATE_NONE)


def gated_ffn_w4(x: torch.Tensor, w_gate: W4, w_up: W4, w_down: W4, *, act: str = "silu", stream=None) -> torch.Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T for a few tokens, all weights in 4 bits.  The
    product is rounded to x's dtype between the two kernels."""
    if act not in GATE_ACTS:
        raise ValueError(f"act must be one of {sorted(GATE_ACTS)}")
    if stream is not None:
        with torch.cuda.stream(stream):
            return gated_ffn_w4(x, w_gate, w_up, w_down, act=act)
    return _matvec_w4(_matvec_w4(x, w_gate, w_up, None, GATE_ACTS[act]), w_down, None, None, N.FO_GATE_NONE)
