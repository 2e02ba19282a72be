"""A stack of gated feed-forward blocks on the `block` operators: trained with autograd, and
served token by token with 4-bit weights.

Each layer is  y = (act(z Wg) * (z Wu)) Wd,  r' = scale r + gate * norm_post(y),  z' = norm_pre'(r'):
one `gated_ffn` and one `block_norm`, which also computes the next layer's input.

    python -m icpp_tuning_b200.gated_block --mode train --tokens 4096 --dim 1024 --inner 4096 --layers 4
    python -m icpp_tuning_b200.gated_block --mode decode --tokens 1 --dim 4096 --inner 16384 --layers 4
"""
from __future__ import annotations

import argparse
from typing import Dict, List, Optional, Tuple

import torch

from . import block


def _wants_gradients(*args) -> bool:
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args)


class _FirstDerivatives(torch.autograd.Function):
    """Runs a backward pass.  Under create_graph its results depend on every tensor that it
    was given, and differentiating them raises: the operators have no second derivatives."""

    @staticmethod
    def forward(ctx, run, *tensors):
        return run(*tensors)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the decoder-block operators have first derivatives only")


class GatedFFN(torch.autograd.Function):
    """y = (act(x Wg) * (x Wu)) Wd with its first derivatives; keeps x and the two products
    where a gradient is wanted."""

    @classmethod
    def apply(cls, x, w_gate, w_up, w_down, act, b_layout):
        if not _wants_gradients(x, w_gate, w_up, w_down):
            return block.gated_ffn(x, w_gate, w_up, w_down, act=act, b_layout=b_layout)
        return super().apply(x, w_gate, w_up, w_down, act, b_layout)

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act, b_layout):
        y, g, u = block.gated_ffn(x, w_gate, w_up, w_down, act=act, b_layout=b_layout, save=True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, g, u)
        ctx.act, ctx.b_layout = act, b_layout
        return y

    @staticmethod
    def backward(ctx, dy):
        def run(dy, *saved):
            return block.gated_ffn_backward(block.aligned_rows(dy), *saved, act=ctx.act, b_layout=ctx.b_layout)

        return (*_FirstDerivatives.apply(run, dy, *ctx.saved_tensors), None, None)


class BlockNorm(torch.autograd.Function):
    """(r, z) of `block.block_norm` with their first derivatives; keeps y and r."""

    @classmethod
    def apply(cls, y, *rest):
        if y.shape[-1] > block.MAX_NORM_BACKWARD and _wants_gradients(y, *rest):
            raise ValueError(f"the norms' backward pass takes rows of at most {block.MAX_NORM_BACKWARD} columns, got {y.shape[-1]}")
        return super().apply(y, *rest)

    @staticmethod
    def forward(ctx, y, x, w_post, w_pre, b_post, b_pre, gate, residual_scale, norm, eps):
        ctx.kw = dict(residual_scale=residual_scale, norm=norm, eps=eps)
        r, z = block.block_norm(y, x, w_post, w_pre, b_post=b_post, b_pre=b_pre, gate=gate, **ctx.kw)
        ctx.save_for_backward(y, r, w_post, w_pre, b_post, b_pre, gate)
        ctx.set_materialize_grads(False)
        return r, z

    @staticmethod
    def backward(ctx, dr, dz):
        def run(dr, dz, y, r, w_post, w_pre, b_post, b_pre, gate):
            dz = torch.zeros_like(r) if dz is None else dz.contiguous()
            d = block.block_norm_backward(None if dr is None else dr.contiguous(), dz, y, r, w_post, w_pre, b_post=b_post, b_pre=b_pre,
                                          gate=gate, **ctx.kw)
            return tuple(d.get(k) for k in ("dy", "dx", "dw_post", "dw_pre", "db_post", "db_pre", "dgate"))

        return (*_FirstDerivatives.apply(run, dr, dz, *ctx.saved_tensors), None, None, None)


def make_weights(layers: int, dim: int, inner: int, dtype=torch.bfloat16, device="cuda", seed: int = 0) -> List[Dict[str, torch.Tensor]]:
    """Random weights, nn.Linear layout: per layer w_gate, w_up [inner, dim], w_down [dim, inner],
    norm weights w_pre (before the block), w_post, and a gate."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(*shape, generator=gen, device=device) * std).to(dtype)

    return [dict(w_gate=normal(inner, dim, std=dim ** -0.5), w_up=normal(inner, dim, std=dim ** -0.5),
                 w_down=normal(dim, inner, std=inner ** -0.5), w_pre=torch.ones(dim, dtype=dtype, device=device),
                 w_post=torch.ones(dim, dtype=dtype, device=device), gate=torch.full((dim,), 0.5, dtype=dtype, device=device))
            for _ in range(layers)]


class GatedStack:
    """The stack; `w_final` is the norm after the last layer.  `quantize` replaces the
    projections by 4-bit ones (`block.W4`) for serving."""

    def __init__(self, weights: List[Dict[str, torch.Tensor]], w_final: torch.Tensor, act: str = "silu", residual_scale: float = 1.0,
                 norm: str = "rms", eps: float = 1e-5):
        self.layers, self.w_final, self.act = weights, w_final, act
        self.kw = dict(residual_scale=residual_scale, norm=norm, eps=eps)

    def parameters(self) -> List[torch.Tensor]:
        return [w for layer in self.layers for w in layer.values()] + [self.w_final]

    def quantize(self, group: int = 128, symmetric: bool = True) -> "GatedStack":
        q = [{**{k: w.detach() for k, w in layer.items()},
              **{k: block.quantize_w4(layer[k].detach(), group, symmetric) for k in ("w_gate", "w_up", "w_down")}} for layer in self.layers]
        return GatedStack(q, self.w_final.detach(), self.act, self.kw["residual_scale"], self.kw["norm"], self.kw["eps"])

    def _start(self, x: torch.Tensor, norm) -> Tuple[torch.Tensor, torch.Tensor]:
        """The first layer's input norm: r = x, z = norm_pre(x)."""
        return norm(x, x, None, self.layers[0]["w_pre"], None, None, None, 0.0, self.kw["norm"], self.kw["eps"])

    def train_forward(self, x: torch.Tensor) -> torch.Tensor:
        """[T, dim] -> [T, dim] with gradients through every weight."""
        r, z = self._start(x, BlockNorm.apply)
        for i, layer in enumerate(self.layers):
            y = GatedFFN.apply(z, layer["w_gate"], layer["w_up"], layer["w_down"], self.act, "nk")
            after = self.layers[i + 1]["w_pre"] if i + 1 < len(self.layers) else self.w_final
            r, z = BlockNorm.apply(y, r, layer["w_post"], after, None, None, layer["gate"], *self.kw.values())
        return z

    @torch.no_grad()
    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """Inference on 16-bit or 4-bit projections."""
        r, z = self._start(x, lambda y, x_, wp, w, bp, b, g, s, n, e: block.block_norm(y, x_, wp, w, residual_scale=s, norm=n, eps=e))
        for i, layer in enumerate(self.layers):
            if isinstance(layer["w_gate"], block.W4):
                y = block.gated_ffn_w4(z, layer["w_gate"], layer["w_up"], layer["w_down"], act=self.act)
            else:
                y = block.gated_ffn(z, layer["w_gate"], layer["w_up"], layer["w_down"], act=self.act, b_layout="nk")
            after = self.layers[i + 1]["w_pre"] if i + 1 < len(self.layers) else self.w_final
            r, z = block.block_norm(y, r, layer["w_post"], after, gate=layer["gate"], **self.kw)
        return z


def train_step(stack: GatedStack, x: torch.Tensor, target: torch.Tensor, lr: float) -> torch.Tensor:
    """One plain gradient step on the mean squared error; returns the loss (fp32, on the GPU)."""
    loss = (stack.train_forward(x).float() - target.float()).square().mean()
    grads = torch.autograd.grad(loss, stack.parameters())
    with torch.no_grad():
        for w, g in zip(stack.parameters(), grads):
            w.add_(g, alpha=-lr)
    return loss.detach()


def _timed(fn, steps: int = 20) -> float:
    for _ in range(5):
        fn()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    a.record()
    for _ in range(steps):
        fn()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / steps


def main(argv: Optional[List[str]] = None) -> None:
    ap = argparse.ArgumentParser(description="gated feed-forward blocks with B200 operators")
    ap.add_argument("--mode", default="train", choices=["train", "decode"])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--dim", type=int, default=1024)
    ap.add_argument("--inner", type=int, default=4096)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--group", type=int, default=128, help="decode: weights that share a scale")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    weights = make_weights(a.layers, a.dim, a.inner)
    stack = GatedStack(weights, torch.ones(a.dim, dtype=torch.bfloat16, device="cuda"))
    x = torch.randn(a.tokens, a.dim, device="cuda").bfloat16()
    if a.mode == "train":
        for w in stack.parameters():
            w.requires_grad_()
        target = torch.randn_like(x)
        first = train_step(stack, x, target, 0.0).item()
        ms = _timed(lambda: train_step(stack, x, target, 0.05))
        flops = 18.0 * a.layers * a.tokens * a.dim * a.inner
        print(f"train {a.tokens} x {a.dim} x {a.inner}, {a.layers} layers: {ms:.3f} ms a step ({flops / ms / 1e9:.0f} TFLOP/s), "
              f"loss {first:.4f} -> {train_step(stack, x, target, 0.0).item():.4f}")
    else:
        from .graphs import CapturedStep

        small = stack.quantize(a.group)
        for name, s in (("16-bit weights", stack), (f"4-bit weights, groups of {a.group}", small)):
            step = CapturedStep(s, [x])
            print(f"decode {a.tokens} x {a.dim} x {a.inner}, {a.layers} layers, {name}: {_timed(lambda: step(x)) * 1e3:.1f} us a step (CUDA graph)")


if __name__ == "__main__":
    main()
