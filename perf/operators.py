"""The decoder-block operators of icpp_tuning_b200.block as measurable cases.

A case is one call of one operator at one size:

  ffn_fwd   y = (act(x Wg) * (x Wu)) Wd, with the two products before the activation saved
            for the backward pass where "save" is set
  ffn_bwd   the gradients of x, Wg, Wu and Wd from dy and the saved products
  norm_fwd  r = scale x + gate * norm_post(y), z = norm_pre(r)
  norm_bwd  the gradients of y, x, the norms' weights and the gate from those of r and z
  w4        x W^T (+ bias) with W held in 4 bits and scaled by groups
  w4_ffn    the gated block with all three weights held in 4 bits

With `own` false, `run` computes in elementary float32 torch operations; with `own` true it
calls the framework.  `exact` restates every operator in float64.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ffn(kind, name, T, D, F, dtype="bf16", act="silu", layout="kn", save=False):
    return {"name": name, "kind": kind, "T": T, "D": D, "F": F, "dtype": dtype, "act": act, "layout": layout, "save": save}


def _norm(kind, name, T, D, dtype="bf16", vec="bf16", norm="rms", post=True, gate=0, scale=1.0):
    return {"name": name, "kind": kind, "T": T, "D": D, "dtype": dtype, "vec": vec, "norm": norm, "post": post,
            "gate": gate, "scale": scale}


def listed():
    return [
        # One token through the gated block at the wider encoder's hidden size: latency of serving.
        _ffn("ffn_fwd", "ffn_fwd 1x1024x4096", 1, 1024, 4096, layout="nk"),
        # A few requests decoded together, at the up-projection workload's widths: weight bytes.
        _ffn("ffn_fwd", "ffn_fwd 24x4096x16384", 24, 4096, 16384, layout="nk"),
        # A ragged prompt at an inner width that is no multiple of a tile.
        _ffn("ffn_fwd", "ffn_fwd 1999x1024x2744", 1999, 1024, 2744, dtype="fp16", act="gelu_tanh"),
        # The up-projection workload's 8192 tokens in training: the saved products are written too.
        _ffn("ffn_fwd", "ffn_fwd 8192x4096x16384", 8192, 4096, 16384, save=True),
        # Fine-tuning on a short ragged batch.
        _ffn("ffn_bwd", "ffn_bwd 1999x1024x4096", 1999, 1024, 4096, dtype="fp16", act="gelu_erf", layout="nk"),
        # A training step's micro-batch.
        _ffn("ffn_bwd", "ffn_bwd 4096x4096x8192", 4096, 4096, 8192),
        # One decoded token between two blocks.
        _norm("norm_fwd", "norm_fwd 1x4096", 1, 4096, post=False),
        # The LayerNorm workload's 16384 rows, both norms, a gate and a residual scale.
        _norm("norm_fwd", "norm_fwd 16384x4096", 16384, 4096, gate=1, scale=0.5),
        # An odd width, a gate per sequence, LayerNorm with biases.
        _norm("norm_bwd", "norm_bwd 4680x1001", 4680, 1001, dtype="fp16", vec="fp32", norm="layer", gate=8, scale=0.7),
        # The same training rows backwards.
        _norm("norm_bwd", "norm_bwd 16384x4096", 16384, 4096, gate=1, scale=0.5),
        # One token through a 4-bit output projection.
        {"name": "w4 1x4096x4096", "kind": "w4", "T": 1, "N": 4096, "K": 4096, "group": 128, "dtype": "bf16", "zeros": False, "bias": False},
        # A few tokens through the 4-bit gated block, asymmetric groups of 32.
        {"name": "w4_ffn 5x4096x16384", "kind": "w4_ffn", "T": 5, "D": 4096, "F": 16384, "group": 32, "dtype": "fp16", "zeros": True, "act": "silu"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["ffn_fwd", "ffn_bwd", "norm_fwd", "norm_bwd", "w4", "w4_ffn"])
    if kind in ("ffn_fwd", "ffn_bwd"):
        D, F = _log_int(rng, 256, 4096, 8), _log_int(rng, 256, 16384, 8)
        T = _log_int(rng, 1, 8192) if kind == "ffn_fwd" else _log_int(rng, 16, 8192)
        c = _ffn(kind, "", T, D, F, rng.choice(["bf16", "fp16"]), rng.choice(["silu", "gelu_tanh", "gelu_erf", "relu"]),
                 rng.choice(["kn", "nk"]), kind == "ffn_fwd" and T > 64 and rng.random() < 0.5)
        top = 3 * 2 * 8192 * 4096 * 16384
        while work(c)["flops"] > top:
            c["T"] = c["T"] * 3 // 4
    elif kind in ("norm_fwd", "norm_bwd"):
        D = _log_int(rng, 64, 8192, rng.choice([1, 8]))
        rows = _log_int(rng, 1, min(16384, 16384 * 4096 // D))
        gate = rng.choice([0, 1, 1, 3])
        c = _norm(kind, "", max(gate, 1) * max(1, rows // max(gate, 1)), D, rng.choice(["bf16", "fp16"]),
                  rng.choice(["same", "fp32"]), rng.choice(["rms", "layer"]), rng.random() < 0.7, gate,
                  rng.choice([1.0, 0.5, 1.25]))
        if c["vec"] == "same":
            c["vec"] = c["dtype"]
    elif kind == "w4":
        c = {"kind": kind, "T": _log_int(rng, 1, 64), "N": _log_int(rng, 128, 16384), "K": _log_int(rng, 256, 16384, 32),
             "group": rng.choice([32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"]), "zeros": rng.random() < 0.5,
             "bias": rng.random() < 0.5}
    else:
        c = {"kind": kind, "T": _log_int(rng, 1, 64), "D": _log_int(rng, 256, 4096, 32), "F": _log_int(rng, 256, 16384, 32),
             "group": rng.choice([32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"]), "zeros": rng.random() < 0.5,
             "act": rng.choice(["silu", "gelu_tanh", "gelu_erf"])}
    c.pop("name", None)
    return c


def _w4_data(gen, N, K, group, dtype, zeros):
    """4-bit weights as they come from a checkpoint: two to a byte, low nibble first."""
    dev, G = gen.device, -(-K // group)
    q = torch.randint(0, 256, (N, K // 2), generator=gen, device=dev, dtype=torch.uint8)
    # groups of a normal weight matrix spread over 16 levels: about +-2.5 deviations, each group its own range
    s = ((0.8 + 0.4 * torch.rand(N, G, generator=gen, device=dev)) * (K ** -0.5) / 4.6).to(dtype)
    z = torch.randint(5, 11, (N, G), generator=gen, device=dev, dtype=torch.uint8) if zeros else None
    return q, s, z


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dt = case["kind"], _DT[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)

    s = {"case": case}
    if kind in ("ffn_fwd", "ffn_bwd"):
        T, D, F = case["T"], case["D"], case["F"]
        up, down = ((D, F), (F, D)) if case["layout"] == "kn" else ((F, D), (D, F))
        s["x"] = normal(T, D)
        s["w_gate"], s["w_up"] = normal(*up, std=D ** -0.5), normal(*up, std=D ** -0.5)
        s["w_down"] = normal(*down, std=F ** -0.5)
        if kind == "ffn_bwd":
            kn = case["layout"] == "kn"
            s["g"] = s["x"] @ (s["w_gate"] if kn else s["w_gate"].t())  # what the forward pass saved
            s["u"] = s["x"] @ (s["w_up"] if kn else s["w_up"].t())
            s["dy"] = normal(T, D, std=0.1)
    elif kind in ("norm_fwd", "norm_bwd"):
        T, D, vec = case["T"], case["D"], _DT[case["vec"]]
        loud = 1.0 + 7.0 * (torch.rand(D, generator=gen, device="cuda") < 0.01).float()  # a few loud channels
        s["y"] = (torch.randn(T, D, generator=gen, device="cuda") * loud).to(dt)
        s["y"][T - T // 16:] = 0  # padding rows of a ragged batch: zeros from the block
        for k, on, mean in (("w_post", case["post"], 1.0), ("w_pre", True, 1.0), ("b_post", case["post"] and case["norm"] == "layer", 0.0),
                            ("b_pre", case["norm"] == "layer", 0.0)):
            s[k] = normal(D, std=0.1, mean=mean, dtype=vec) if on else None
        G = case["gate"]
        s["gate"] = None if G == 0 else normal(*((D,) if G == 1 else (G, D)), std=0.2, mean=0.5, dtype=vec)
        s["x" if kind == "norm_fwd" else "r"] = (torch.randn(T, D, generator=gen, device="cuda") * 2.0 * loud).to(dt)
        if kind == "norm_bwd":
            s["dr"], s["dz"] = normal(T, D, std=0.1), normal(T, D, std=0.1)
    elif kind == "w4":
        T, N, K = case["T"], case["N"], case["K"]
        s["x"] = normal(T, K)
        s["w"] = _w4_data(gen, N, K, case["group"], dt, case["zeros"])
        s["bias"] = normal(N, std=0.1) if case["bias"] else None
    else:
        T, D, F = case["T"], case["D"], case["F"]
        s["x"] = normal(T, D)
        s["gate"], s["up"] = (_w4_data(gen, F, D, case["group"], dt, case["zeros"]) for _ in range(2))
        s["down"] = _w4_data(gen, D, F, case["group"], dt, case["zeros"])
    return s


# ------------------------------------------------------------------ plain forms, float32
def _act(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    if name == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    if name == "gelu_erf":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return torch.clamp(g, min=0)


def _dact(name, g):
    if name == "silu":
        p = 1 / (1 + torch.exp(-g))
        return p * (1 + g * (1 - p))
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    if name == "gelu_erf":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    return (g > 0).float()


def _ffn_weights(s):
    w = [s[k].float() for k in ("w_gate", "w_up", "w_down")]
    return w if s["case"]["layout"] == "kn" else [m.t() for m in w]


def _plain_ffn_fwd(s):
    c, dt = s["case"], s["x"].dtype
    wg, wu, wd = _ffn_weights(s)
    x = s["x"].float()
    g, u = x @ wg, x @ wu
    y = ((_act(c["act"], g) * u) @ wd).to(dt)
    return (y, g.to(dt), u.to(dt)) if c["save"] else y


def _plain_ffn_bwd(s):
    c, dt = s["case"], s["x"].dtype
    wg, wu, wd = _ffn_weights(s)
    x, dy, g, u = (s[k].float() for k in ("x", "dy", "g", "u"))
    dh = dy @ wd.t()
    a = _act(c["act"], g)
    dg, du, h = dh * u * _dact(c["act"], g), dh * a, a * u
    dx = dg @ wg.t() + du @ wu.t()
    dw = [x.t() @ dg, x.t() @ du, h.t() @ dy]
    if c["layout"] == "nk":
        dw = [m.t() for m in dw]
    return (dx.to(dt), *(m.to(dt) for m in dw))


def _f(t):
    return None if t is None else t.float()


def _hat(v, case):
    """The normalised rows and the rows' reciprocal deviations."""
    if case["norm"] == "layer":
        v = v - v.mean(1, keepdim=True)
    rho = torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5)
    return v * rho, rho


def _rows_of_gate(gate, T):
    return gate if gate.dim() == 1 else gate.repeat_interleave(T // gate.shape[0], 0)


def _post(y, s):
    if s["w_post"] is None:
        return y, None, None
    h, rho = _hat(y, s["case"])
    n = h * s["w_post"].float()
    return (n if s["b_post"] is None else n + s["b_post"].float()), h, rho


def _plain_norm_fwd(s):
    c, dt = s["case"], s["y"].dtype
    n, _, _ = _post(s["y"].float(), s)
    if s["gate"] is not None:
        n = n * _rows_of_gate(s["gate"].float(), c["T"])
    r = c["scale"] * s["x"].float() + n
    z = _hat(r, c)[0] * s["w_pre"].float()
    if s["b_pre"] is not None:
        z = z + s["b_pre"].float()
    return r.to(dt), z.to(dt)


def _through(c, hat, rho, case):
    """The gradient of the rows whose normalised form `hat` has the gradient `c`."""
    t = c - hat * (c * hat).mean(1, keepdim=True)
    return rho * (t - c.mean(1, keepdim=True) if case["norm"] == "layer" else t)


def _plain_norm_bwd(s):
    c, dt, vec = s["case"], s["y"].dtype, s["w_pre"].dtype
    dr, dz = s["dr"].float(), s["dz"].float()
    n, yhat, yrho = _post(s["y"].float(), s)
    rhat, rrho = _hat(s["r"].float(), c)
    t = dr + _through(dz * s["w_pre"].float(), rhat, rrho, c)
    dn = t if s["gate"] is None else t * _rows_of_gate(s["gate"].float(), c["T"])
    out = {"dx": (c["scale"] * t).to(dt), "dw_pre": (dz * rhat).sum(0).to(vec)}
    if s["b_pre"] is not None:
        out["db_pre"] = dz.sum(0).to(vec)
    if s["gate"] is not None:
        out["dgate"] = (t * n).reshape(c["gate"], -1, c["D"]).sum(1).reshape(s["gate"].shape).to(vec)
    if s["w_post"] is None:
        out["dy"] = dn.to(dt)
    else:
        out["dw_post"] = (dn * yhat).sum(0).to(vec)
        if s["b_post"] is not None:
            out["db_post"] = dn.sum(0).to(vec)
        out["dy"] = _through(dn * s["w_post"].float(), yhat, yrho, c).to(dt)
    return out


def _open_w4(w, group):
    q, scale, zero = w
    v = torch.stack((q & 15, q >> 4), 2).reshape(q.shape[0], -1).float()
    K = v.shape[1]
    at = torch.arange(K, device=q.device) // group
    return (v - (8.0 if zero is None else zero.float()[:, at])) * scale.float()[:, at]


def _plain_w4(s):
    y = s["x"].float() @ _open_w4(s["w"], s["case"]["group"]).t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def _plain_w4_ffn(s):
    G, x = s["case"]["group"], s["x"].float()
    h = _act(s["case"]["act"], x @ _open_w4(s["gate"], G).t()) * (x @ _open_w4(s["up"], G).t())
    return (h @ _open_w4(s["down"], G).t()).to(s["x"].dtype)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from icpp_tuning_b200 import block

    c, kind = s["case"], s["case"]["kind"]
    if kind == "ffn_fwd":
        return block.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], act=c["act"], b_layout=c["layout"], save=c["save"])
    if kind == "ffn_bwd":
        return block.gated_ffn_backward(s["dy"], s["x"], s["w_gate"], s["w_up"], s["w_down"], s["g"], s["u"], act=c["act"],
                                        b_layout=c["layout"])
    if kind == "norm_fwd":
        return block.block_norm(s["y"], s["x"], s["w_post"], s["w_pre"], b_post=s["b_post"], b_pre=s["b_pre"], gate=s["gate"],
                                residual_scale=c["scale"], norm=c["norm"], eps=1e-5)
    if kind == "norm_bwd":
        return block.block_norm_backward(s["dr"], s["dz"], s["y"], s["r"], s["w_post"], s["w_pre"], b_post=s["b_post"],
                                         b_pre=s["b_pre"], gate=s["gate"], residual_scale=c["scale"], norm=c["norm"], eps=1e-5)
    if kind == "w4":
        return block.matvec_w4(s["x"], block.W4(*s["w"], c["group"]), bias=s["bias"])
    return block.gated_ffn_w4(s["x"], *(block.W4(*s[k], c["group"]) for k in ("gate", "up", "down")), act=c["act"])


_PLAIN = {"ffn_fwd": _plain_ffn_fwd, "ffn_bwd": _plain_ffn_bwd, "norm_fwd": _plain_norm_fwd, "norm_bwd": _plain_norm_bwd,
          "w4": _plain_w4, "w4_ffn": _plain_w4_ffn}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["kind"]](state)


def _w4_bytes(N, K, case):
    return N * K // 2 + N * -(-K // case["group"]) * (2 + case["zeros"])


def work(case):
    kind, T = case["kind"], case["T"]
    if kind in ("ffn_fwd", "ffn_bwd"):
        D, F = case["D"], case["F"]
        if kind == "ffn_fwd":  # x, the weights, y; and g, u
            return {"bytes": 2 * (2 * T * D + 3 * D * F + (2 * T * F if case["save"] else 0)), "flops": 6 * T * D * F}
        return {"bytes": 2 * (3 * T * D + 6 * D * F + 2 * T * F), "flops": 12 * T * D * F}
    if kind in ("norm_fwd", "norm_bwd"):
        D, v = case["D"], 4 if case["vec"] == "fp32" else 2
        vecs = (1 + case["post"]) * (1 + (case["norm"] == "layer")) + case["gate"]
        if kind == "norm_fwd":
            return {"bytes": 8 * T * D + v * vecs * D, "flops": 14 * T * D}
        return {"bytes": 12 * T * D + 2 * v * vecs * D, "flops": 30 * T * D}
    if kind == "w4":
        N, K = case["N"], case["K"]
        return {"bytes": _w4_bytes(N, K, case) + 2 * T * (N + K), "flops": 2 * T * N * K}
    D, F = case["D"], case["F"]
    return {"bytes": 2 * _w4_bytes(F, D, case) + _w4_bytes(D, F, case) + 4 * T * D, "flops": 6 * T * D * F}


# ------------------------------------------------------------------ the definitions, float64
def _act64(name):
    nn = torch.nn.functional
    return {"silu": nn.silu, "relu": nn.relu, "gelu_erf": nn.gelu, "gelu_tanh": lambda g: nn.gelu(g, approximate="tanh")}[name]


def _exact_ffn(s):
    c = s["case"]
    d = {k: v.double() for k, v in s.items() if k != "case"}
    e = "ij,jk->ik" if c["layout"] == "kn" else "ij,kj->ik"
    if c["kind"] == "ffn_fwd":
        g, u = torch.einsum(e, d["x"], d["w_gate"]), torch.einsum(e, d["x"], d["w_up"])
        y = torch.einsum(e, _act64(c["act"])(g) * u, d["w_down"])
        return (y, g, u) if c["save"] else y
    for k in ("g", "u", "w_down"):
        d[k].requires_grad_()
    y = torch.einsum(e, _act64(c["act"])(d["g"]) * d["u"], d["w_down"])
    dg, du, dwd = torch.autograd.grad(y, (d["g"], d["u"], d["w_down"]), d["dy"])
    for k in ("x", "w_gate", "w_up"):
        d[k].requires_grad_()
    both = torch.cat((torch.einsum(e, d["x"], d["w_gate"]), torch.einsum(e, d["x"], d["w_up"])), 1)
    dx, dwg, dwu = torch.autograd.grad(both, (d["x"], d["w_gate"], d["w_up"]), torch.cat((dg, du), 1))
    return dx, dwg, dwu, dwd


def _exact_norm(s):
    c = s["case"]
    d = {k: None if v is None else v.double() for k, v in s.items() if k != "case"}

    def norm(v, w, b):
        if c["norm"] == "layer":
            return torch.nn.functional.layer_norm(v, (c["D"],), w, b, 1e-5)
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w

    def before(y, w, b, gate):
        n = y if w is None else norm(y, w, b)
        if gate is None:
            return n
        return (n.reshape(max(1, c["gate"]), -1, c["D"]) * gate.reshape(-1, 1, c["D"])).reshape(n.shape)

    if c["kind"] == "norm_fwd":
        r = c["scale"] * d["x"] + before(d["y"], d["w_post"], d["b_post"], d["gate"])
        return r, norm(r, d["w_pre"], d["b_pre"])
    names = [k for k in ("y", "w_post", "w_pre", "b_post", "b_pre", "gate", "r") if d[k] is not None]
    for k in names:
        d[k].requires_grad_()
    first = [k for k in ("r", "w_pre", "b_pre") if k in names]
    got = dict(zip(first, torch.autograd.grad(norm(d["r"], d["w_pre"], d["b_pre"]), [d[k] for k in first], d["dz"])))
    t = d["dr"] + got.pop("r")
    rest = [k for k in ("y", "w_post", "b_post", "gate") if k in names]
    got.update(zip(rest, torch.autograd.grad(before(d["y"], d["w_post"], d["b_post"], d["gate"]), [d[k] for k in rest], t)))
    return {"dx": c["scale"] * t, **{"d" + k: v for k, v in got.items()}}


def _exact_w4(s):
    c = s["case"]

    def weight(w):
        q, scale, zero = w
        out = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=q.device)
        out[:, 0::2], out[:, 1::2] = q % 16, q // 16
        K = out.shape[1]
        wide = lambda t: t.double().repeat_interleave(c["group"], 1)[:, :K]  # noqa: E731
        return (out - (8 if zero is None else wide(zero))) * wide(scale)

    x = s["x"].double()
    if c["kind"] == "w4":
        y = torch.einsum("tk,nk->tn", x, weight(s["w"]))
        return y if s["bias"] is None else y + s["bias"].double()
    h = _act64(c["act"])(torch.einsum("tk,nk->tn", x, weight(s["gate"]))) * torch.einsum("tk,nk->tn", x, weight(s["up"]))
    return torch.einsum("tk,nk->tn", h, weight(s["down"]))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("ffn_fwd", "ffn_bwd"):
        return _exact_ffn(s)
    return _exact_norm(s) if case["kind"] in ("norm_fwd", "norm_bwd") else _exact_w4(s)
