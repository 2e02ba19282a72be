"""The norms around a block against their 64-bit form, with derived bounds (block_util)."""
import pytest
import torch

from block_util import ACC, U, hat, norm_forward, rows_of_gate, within
from gpu_util import gen, status_clean

from icpp_tuning_b200 import block
from icpp_tuning_b200.graphs import CapturedStep

pytestmark = pytest.mark.gpu
EPS = 1e-5


def make(T, D, dtype, vec, layer, post, gate, seed=0, ld=0, shift=0):
    """Inputs on the CPU; ld > 0: rows that far apart, starting `shift` elements into the memory."""
    g = gen(seed)

    def rows(std):
        wide = (torch.randn(T, max(ld, D), generator=g) * std).to(dtype)
        return wide[:, shift:shift + D] if ld else wide

    def p(mean, std=0.2, shape=(D,)):
        return (torch.randn(*shape, generator=g) * std + mean).to(vec)

    v = dict(y=rows(1.0), x=rows(2.0), w_pre=p(1.0), w_post=p(1.0) if post else None, b_pre=p(0.0) if layer else None,
             b_post=p(0.0) if layer and post else None, gate=None if gate == 0 else p(0.5, 0.3, (D,) if gate == 1 else (gate, D)))
    if T > 2:
        v["y"][1] = 0  # a padding row: rho is 1 / sqrt(eps)
    return v


def gpu(t):
    """On the GPU with the same strides and the same offset into its memory."""
    if t is None:
        return None
    room = torch.zeros(t.untyped_storage().nbytes() // t.element_size(), dtype=t.dtype, device="cuda")
    return room.as_strided(t.shape, t.stride(), t.storage_offset()).copy_(t)


def d64(v):
    return {k: None if t is None else t.double() for k, t in v.items()}


SHAPES = [(1, 1), (1, 4096), (2, 8), (3, 100), (5, 256), (7, 257), (33, 64), (4, 512), (6, 520), (9, 1001), (3, 1024), (5, 2047), (2, 2048),
          (3, 4095), (3, 4096), (2, 4104), (2, 6001), (2, 8192), (300, 40), (1300, 264), (700, 129)]
GATES = [0, 1, "rows", "two"]


def _gate(kind, T):
    return {"rows": T, "two": 2 if T % 2 == 0 else 1}.get(kind, kind)


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("T,D", SHAPES + [(2, 8200), (3, 16384), (2, 12001)])
def test_forward(T, D, layer):
    dtype = torch.bfloat16 if (T + D) % 2 else torch.float16
    vec = [torch.float32, dtype][T % 2]
    post, gate = D % 3 != 0, _gate(GATES[(T + D) % 4], T)
    v = make(T, D, dtype, vec, layer, post, gate, seed=D)
    scale = [1.0, 0.5, -1.25][T % 3]
    w = d64(v)
    ref, bound = norm_forward(w["y"], w["x"], w["w_post"], w["w_pre"], w["b_post"], w["b_pre"], w["gate"], scale, layer, EPS, U[dtype])
    c = {k: gpu(t) for k, t in v.items()}
    kw = dict(b_post=c["b_post"], b_pre=c["b_pre"], gate=c["gate"], residual_scale=scale, norm="layer" if layer else "rms", eps=EPS)
    out = block.block_norm(c["y"], c["x"], c["w_post"], c["w_pre"], **kw)
    for o, r, b, name in zip(out, ref, bound, "rz"):
        within(o, r, b, name)
    assert all(torch.equal(a, b) for a, b in zip(out, block.block_norm(c["y"], c["x"], c["w_post"], c["w_pre"], **kw)))
    status_clean()


def backward64(w, dr, dz, r, scale, layer, u, uv):
    """Every gradient and its bound.  Each is a few fp32 operations on values of the sizes that
    are summed up beside it (M), plus the final rounding; a mean over a row is as exact as its
    terms, a sum over rows gets ACC of its terms' magnitudes."""
    T = dr.shape[0]
    post = w["w_post"] is not None
    rh, rr = hat(r, layer, EPS)
    c = dz * w["w_pre"]
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    t = dr + rr * (c - rh * mean(c * rh) - (mean(c) if layer else 0))
    # the centring of r loses ACC of its row's size, which rho scales
    off = rr * mean(r.abs()) if layer else torch.zeros(T, 1)
    rha = rh.abs() + off
    Mt = dr.abs() + rr * (c.abs() + rha * mean(c.abs() * rha) + (mean(c.abs()) if layer else 0))
    g = torch.ones(()) if w["gate"] is None else rows_of_gate(w["gate"], T)
    out = {"dx": (scale * t, abs(scale) * Mt, u), "dw_pre": ((dz * rh).sum(0), (dz.abs() * rha).sum(0), uv)}
    if w["b_pre"] is not None:
        out["db_pre"] = dz.sum(0), dz.abs().sum(0), uv
    dn, Mn = g * t, g.abs() * Mt
    if post:
        yh, ry = hat(w["y"], layer, EPS)
        yha = yh.abs() + (ry * mean(w["y"].abs()) if layer else 0)
        n, Ma = yh * w["w_post"], yha * w["w_post"].abs()
        out["dw_post"] = (dn * yh).sum(0), (Mn * yha).sum(0), uv
        if w["b_post"] is not None:
            n, Ma = n + w["b_post"], Ma + w["b_post"].abs()
            out["db_post"] = dn.sum(0), Mn.sum(0), uv
        e, Me = dn * w["w_post"], Mn * w["w_post"].abs()
        out["dy"] = (ry * (e - yh * mean(e * yh) - (mean(e) if layer else 0)),
                     ry * (Me + yha * mean(Me * yha) + (mean(Me) if layer else 0)), u)
    else:
        n, Ma = w["y"], w["y"].abs()
        out["dy"] = dn, Mn, u
    if w["gate"] is not None:
        G = 1 if w["gate"].dim() == 1 else w["gate"].shape[0]
        per = lambda q: q.reshape(G, T // G, -1).sum(1).reshape(w["gate"].shape)  # noqa: E731
        out["dgate"] = per(t * n), per(Mt * Ma), uv
    return {k: (v, 4 * ACC * M + 1.01 * r_ * v.abs()) for k, (v, M, r_) in out.items()}


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("T,D", SHAPES)
def test_backward(T, D, layer):
    dtype = torch.float16 if (T + D) % 2 else torch.bfloat16
    vec = [dtype, torch.float32][T % 2]
    post, gate = D % 5 != 0, _gate(GATES[(T + D + 1) % 4], T)
    v = make(T, D, dtype, vec, layer, post, gate, seed=D + 1)
    g = gen(D + 2)
    v["r"] = v.pop("x")
    v["dr"], v["dz"] = ((torch.randn(T, D, generator=g) * 0.5).to(dtype) for _ in range(2))
    scale = [0.7, 1.0][T % 2]
    w = d64(v)
    with_dr = T % 4 != 3
    dr = w["dr"] if with_dr else torch.zeros_like(w["dr"])
    ref = backward64(w, dr, w["dz"], w["r"], scale, layer, U[dtype], U[vec])
    c = {k: gpu(t) for k, t in v.items()}
    call = lambda: block.block_norm_backward(c["dr"] if with_dr else None, c["dz"], c["y"], c["r"], c["w_post"], c["w_pre"],  # noqa: E731
                                             b_post=c["b_post"], b_pre=c["b_pre"], gate=c["gate"], residual_scale=scale,
                                             norm="layer" if layer else "rms", eps=EPS)
    out = call()
    assert set(out) == set(ref)
    for k, (r, b) in ref.items():
        within(out[k], r, b, k)
        assert out[k].dtype == (dtype if k in ("dx", "dy") else vec)
    again = call()
    assert all(torch.equal(out[k], again[k]) for k in out)
    status_clean()


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("ld,shift,D", [(72, 8, 64), (72, 1, 64), (71, 0, 64), (200, 3, 129), (1040, 5, 1001), (1048, 8, 1032), (603, 2, 600)])
def test_strides_and_alignments(ld, shift, D, layer):
    """Rows that start anywhere: padded, odd strides, memory that starts off a 16-byte block."""
    T, dtype = 9, torch.bfloat16
    v = make(T, D, dtype, dtype, layer, True, 3, seed=ld + D, ld=ld, shift=shift)
    w = d64(v)
    c = {k: gpu(t) for k, t in v.items()}
    kw = dict(b_post=c["b_post"], b_pre=c["b_pre"], gate=c["gate"], residual_scale=0.5, norm="layer" if layer else "rms")
    ref, bound = norm_forward(w["y"], w["x"], w["w_post"], w["w_pre"], w["b_post"], w["b_pre"], w["gate"], 0.5, layer, EPS, U[dtype])
    out = block.block_norm(c["y"], c["x"], c["w_post"], c["w_pre"], **kw)
    for o, r, b in zip(out, ref, bound):
        within(o, r, b)
    # x stands in for r, y for dr, x for dz: all of them oddly placed
    got = block.block_norm_backward(c["y"], c["x"], c["y"], c["x"], c["w_post"], c["w_pre"], **kw)
    for k, (r, b) in backward64(w, w["y"], w["x"], w["x"], 0.5, layer, U[dtype], U[dtype]).items():
        within(got[k], r, b, k)


def test_broadcast_rows():
    """A row stride of zero: every token reads the same row."""
    for D in (64, 65):
        one = torch.randn(1, D, generator=gen(1)).bfloat16()
        y, x, w = one.cuda().expand(5, D), torch.randn(5, D, generator=gen(2)).bfloat16().cuda(), torch.ones(D, dtype=torch.bfloat16, device="cuda")
        a, b = block.block_norm(y, x, w, w), block.block_norm(y.contiguous(), x, w, w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("layer", [False, True])
def test_gradient_against_differences(layer):
    """<grad, v> against differences of the 64-bit forward pass, L = sum(dr r + dz z)."""
    T, D, h = 6, 48, 1e-5
    v = make(T, D, torch.float16, torch.float32, layer, True, 3, seed=4)
    v["y"][1] = torch.randn(D, generator=gen(5)).half()
    w = d64(v)
    g = gen(6)
    dr, dz = ((torch.randn(T, D, generator=g) * 0.5).half() for _ in range(2))
    names = [k for k in ("y", "x", "w_post", "w_pre", "b_post", "b_pre", "gate") if w[k] is not None]

    def run(q):
        return norm_forward(q["y"], q["x"], q["w_post"], q["w_pre"], q["b_post"], q["b_pre"], q["gate"], 0.5, layer, EPS, 0.0)[0]

    def loss(q):
        r, z = run(q)
        return (dr.double() * r + dz.double() * z).sum()

    r16 = run(w)[0].half()
    c = {k: gpu(t) for k, t in v.items()}
    got = block.block_norm_backward(dr.cuda(), dz.cuda(), c["y"], r16.cuda(), c["w_post"], c["w_pre"], b_post=c["b_post"], b_pre=c["b_pre"],
                                    gate=c["gate"], residual_scale=0.5, norm="layer" if layer else "rms", eps=EPS)
    for i, k in enumerate(names):
        vdir = torch.randn(w[k].shape, generator=gen(30 + i), dtype=torch.float64)
        num = (loss({**w, k: w[k] + h * vdir}) - loss({**w, k: w[k] - h * vdir})) / (2 * h)
        grad = got["d" + k].double().cpu()
        # the gradient is rounded to 11 bits, and so is the r it reads: a few unit roundoffs of
        # the terms (each term of t has r's rounding once in rhat and once in the row's means)
        assert (num - (grad * vdir).sum()).abs() <= 8 * U[torch.float16] * (grad.abs() * vdir.abs()).sum() + 1e-3


def test_not_a_number_stays_in_its_row():
    for D in (64, 1001):
        v = {k: gpu(t) for k, t in make(5, D, torch.bfloat16, torch.float32, True, True, 0, seed=7).items()}
        args = dict(b_post=v["b_post"], b_pre=v["b_pre"], norm="layer")
        clean = block.block_norm(v["y"], v["x"], v["w_post"], v["w_pre"], **args)
        v["y"][2, 3] = float("nan")
        v["y"][4, 1] = float("inf")
        out = block.block_norm(v["y"], v["x"], v["w_post"], v["w_pre"], **args)
        keep = [0, 1, 3]
        for a, b in zip(out, clean):
            assert torch.equal(a[keep], b[keep]) and a[[2, 4]].isnan().all()
        back = block.block_norm_backward(None, v["x"], v["y"], v["x"], v["w_post"], v["w_pre"], **args)
        assert back["dy"][keep].isfinite().all() and back["dy"][2].isnan().all()


def test_empty_streams_and_graphs():
    e = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    r, z = block.block_norm(e, e, w, w)
    assert r.shape == z.shape == (0, 64)
    back = block.block_norm_backward(e, e, e, e, w, w, gate=w)
    assert back["dx"].shape == (0, 64) and all((back[k] == 0).all() for k in ("dw_pre", "dw_post", "dgate"))
    y, x = (torch.randn(70, 64, generator=gen(i)).bfloat16().cuda() for i in range(2))
    want = block.block_norm(y, x, w, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = block.block_norm(y, x, w, w, stream=s)
    s.synchronize()
    step = CapturedStep(lambda a, b: block.block_norm(a, b, w, w), [torch.zeros_like(y), torch.zeros_like(x)])
    for a, b, c in zip(want, got, step(y, x)):
        assert torch.equal(a, b) and torch.equal(a, c)
    status_clean()


def test_refusals():
    y = torch.zeros(6, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for kw, msg in ((dict(norm="batch"), "norm"), (dict(gate=w[:32]), "gate"), (dict(gate=torch.ones(4, 64, dtype=w.dtype, device="cuda")), "dividing"),
                    (dict(gate=w.float()), "dtype"), (dict(b_pre=w[::2]), "b_pre")):
        with pytest.raises(ValueError, match=msg):
            block.block_norm(y, y, w, w, **kw)
    with pytest.raises(ValueError, match="x must be"):
        block.block_norm(y, y[:3], w, w)
    with pytest.raises(ValueError, match="w_pre"):
        block.block_norm(y, y, w, None)
    with pytest.raises(block.N.FoError, match="bias"):
        block.block_norm(y, y, w, w, b_pre=w)
    wide = torch.zeros(2, 16392, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(block.N.FoError, match="16384"):
        block.block_norm(wide, wide, None, wide[0])
    assert ACC > 0
