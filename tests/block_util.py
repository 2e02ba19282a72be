"""64-bit restatements of the decoder-block operators with error bounds, for their GPU tests.

Every bound is derived from what the kernels may round, elementwise:
  u      the unit roundoff of the 16-bit type, half its epsilon (2^-8 bf16, 2^-11 fp16), for the
         result and for every intermediate that is held in 16 bits;
  ACC    2^-18 of the sum of magnitudes for an fp32 sum of products (64 units of 2^-24: a sum
         of up to 4096 terms whose roundings add like a random walk), and for the activations'
         approximations, whose error is below 2^-18 of their arguments' products;
  tiny   the type's smallest normal number, for results that underflow."""
import torch

ACC = 2.0 ** -18
U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {t: torch.finfo(t).tiny for t in U}


def act64(name, g):
    """(act(g), act'(g)) in float64, relu'(0) = 0."""
    g = g.detach().requires_grad_()
    nn = torch.nn.functional
    a = {"silu": nn.silu, "relu": nn.relu, "gelu_erf": nn.gelu, "gelu_tanh": lambda t: nn.gelu(t, approximate="tanh")}[name](g)
    (d,) = torch.autograd.grad(a.sum(), g)
    return a.detach(), d


def within(out, ref, bound, what=""):
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    o = out.double().cpu()
    bad = ~((o - ref).abs() <= bound + 2 * TINY[out.dtype])
    if bad.any():
        i = int(((o - ref).abs() / (bound + 1e-300)).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {o.numel()} outside; worst {o.flatten()[i]} for {ref.flatten()[i]}, "
                             f"bound {bound.flatten()[i]}")


def ffn_forward(x, wg, wu, wd, act, u):
    """(y, g, u) and their bounds; weights as [D, F], [D, F], [F, N], all float64."""
    g, p = x @ wg, x @ wu
    eg, ep = ACC * (x.abs() @ wg.abs()), ACC * (x.abs() @ wu.abs())
    a, _ = act64(act, g)
    h = a * p
    eh = 1.2 * eg * p.abs() + (a.abs() + 1.2 * eg) * ep + (ACC + u) * h.abs() + ACC * p.abs()  # |act'| < 1.2
    y = h @ wd
    ey = u * y.abs() + eh @ wd.abs() + ACC * (h.abs() @ wd.abs())
    return (y, g, p), (ey * (1 + u), eg + u * g.abs() * (1 + u), ep + u * p.abs() * (1 + u))


def ffn_backward(dy, x, wg, wu, wd, g, p, act, u):
    """(dx, dwg, dwu, dwd) and their bounds."""
    dh = dy @ wd.t()
    edh = ACC * (dy.abs() @ wd.abs().t())
    a, da = act64(act, g)
    dg, dp, h = dh * p * da, dh * a, a * p
    edg = edh * (p * da).abs() + ACC * (dh * p).abs() * (1 + g.abs()) + u * dg.abs()
    edp = edh * a.abs() + ACC * dh.abs() * (1 + g.abs()) + u * dp.abs()
    eh = ACC * p.abs() * (1 + g.abs()) + u * h.abs()

    def product(ma, ea, mb, eb):
        return ea @ mb.abs() + ma.abs() @ eb + ACC * (ma.abs() @ mb.abs())

    none = torch.zeros((), dtype=torch.float64)
    outs = (dg @ wg.t() + dp @ wu.t(), x.t() @ dg, x.t() @ dp, h.t() @ dy)
    errs = (product(dg, edg, wg.t(), none.expand_as(wg.t())) + product(dp, edp, wu.t(), none.expand_as(wu.t())),
            product(x.t(), none.expand_as(x.t()), dg, edg), product(x.t(), none.expand_as(x.t()), dp, edp),
            product(h.t(), eh.t(), dy, none.expand_as(dy)))
    return outs, tuple(e * 1.05 + u * o.abs() for o, e in zip(outs, errs))


def rows_of_gate(gate, T):
    return gate if gate.dim() == 1 else gate.repeat_interleave(T // gate.shape[0], 0)


def hat(v, layer, eps):
    if layer:
        v = v - v.mean(1, keepdim=True)
    rho = 1 / torch.sqrt(v.square().mean(1, keepdim=True) + eps)
    return v * rho, rho


def norm_forward(y, x, w_post, w_pre, b_post, b_pre, gate, scale, layer, eps, u):
    """(r, z) and their bounds, float64 in."""
    T = y.shape[0]
    n, m = y, torch.zeros_like(y)
    if w_post is not None:
        yh, rho = hat(y, layer, eps)
        n = yh * w_post
        m = w_post.abs() * (yh.abs() + rho * y.abs().mean(1, keepdim=True))  # the mean is as exact as its terms
        if b_post is not None:
            n, m = n + b_post, m + b_post.abs()
    g = torch.ones(()) if gate is None else rows_of_gate(gate, T)
    r = scale * x + g * n
    er = ACC * ((scale * x).abs() + g.abs() * (n.abs() + m))
    rh, rho = hat(r, layer, eps)
    z = rh * w_pre
    ez = w_pre.abs() * rho * (er + er.mean(1, keepdim=True) + (er * rh.abs()).mean(1, keepdim=True) * rh.abs()) + ACC * (
        z.abs() + w_pre.abs() * rho * r.abs().mean(1, keepdim=True))
    if b_pre is not None:
        z, ez = z + b_pre, ez + ACC * b_pre.abs()
    return (r, z), (er + u * r.abs() * 1.01, ez * 1.1 + u * z.abs() * 1.01)
