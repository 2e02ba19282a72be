"""The decoder-block operators at training sizes, and with offsets past 32 bits."""
import pytest
import torch

from block_util import ACC, U, act64
from gpu_util import status_clean

from icpp_tuning_b200 import block

pytestmark = pytest.mark.gpu


def normal(*shape, std=1.0, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def inside(out, ref, bound, what):
    bad = ~((out.double() - ref).abs() <= bound + 2.0 ** -120)
    assert not bad.any(), (what, int(bad.sum()), float(((out.double() - ref).abs() / bound).max()))


def test_gated_block_of_a_training_step():
    """8192 tokens, 1024 x 4096, both directions, in float64 on the GPU; bounds as in block_util."""
    T, D, F, u = 8192, 1024, 4096, U[torch.bfloat16]
    x, wg, wu, wd = normal(T, D, seed=1), normal(F, D, std=D ** -0.5, seed=2), normal(F, D, std=D ** -0.5, seed=3), normal(D, F, std=F ** -0.5, seed=4)
    y, g, p = block.gated_ffn(x, wg, wu, wd, b_layout="nk", save=True)
    X, WG, WU, WD = (t.double() for t in (x, wg, wu, wd))
    rg, rp = X @ WG.t(), X @ WU.t()
    eg, ep = ACC * (X.abs() @ WG.abs().t()), ACC * (X.abs() @ WU.abs().t())
    inside(g, rg, eg + u * rg.abs() * (1 + u), "g")
    inside(p, rp, ep + u * rp.abs() * (1 + u), "u")
    a, _ = act64("silu", rg)
    h = a * rp
    eh = 1.2 * eg * rp.abs() + (a.abs() + 1.2 * eg) * ep + (ACC + u) * h.abs() + ACC * rp.abs()
    ry = h @ WD.t()
    inside(y, ry, (u * ry.abs() + eh @ WD.abs().t() + ACC * (h.abs() @ WD.abs().t())) * (1 + u), "y")
    del eg, ep, eh, h, ry, rg, rp, a
    dy = normal(T, D, std=0.1, seed=5)
    dx, dwg, dwu, dwd = block.gated_ffn_backward(dy, x, wg, wu, wd, g, p, b_layout="nk")
    G, P, DY = g.double(), p.double(), dy.double()
    dh, edh = DY @ WD, ACC * (DY.abs() @ WD.abs())
    a, da = act64("silu", G)
    dg, dp, h = dh * P * da, dh * a, a * P
    edg = edh * (P * da).abs() + ACC * (dh * P).abs() * (1 + G.abs()) + u * dg.abs()
    edp = edh * a.abs() + ACC * dh.abs() * (1 + G.abs()) + u * dp.abs()
    eh = ACC * P.abs() * (1 + G.abs()) + u * h.abs()

    def check(out, ma, ea, mb, what):
        ref = ma @ mb
        inside(out, ref, (ea @ mb.abs() + 2 * ACC * (ma.abs() @ mb.abs())) * 1.05 + u * ref.abs(), what)  # 8192 terms: twice ACC

    inside(dx, dg @ WG + dp @ WU, (edg @ WG.abs() + edp @ WU.abs() + 2 * ACC * (dg.abs() @ WG.abs() + dp.abs() @ WU.abs())) * 1.05
           + u * (dg @ WG + dp @ WU).abs(), "dx")
    check(dwg, dg.t(), edg.t(), X, "dw_gate")
    check(dwu, dp.t(), edp.t(), X, "dw_up")
    check(dwd.t(), h.t(), eh.t(), DY, "dw_down")
    status_clean()


@pytest.mark.parametrize("layer", [False, True])
def test_norms_of_a_training_step(layer):
    """16384 x 4096 in float64 on the GPU, a gate for each of four sequences."""
    T, D, u, eps, scale = 16384, 4096, U[torch.bfloat16], 1e-5, 0.5
    y, x = normal(T, D, seed=1), normal(T, D, std=2.0, seed=2)
    wq, wp, gate = normal(D, std=0.1, seed=3) + 1, normal(D, std=0.1, seed=4) + 1, normal(4, D, std=0.2, seed=5) + 0.5
    bq, bp = (normal(D, std=0.1, seed=6), normal(D, std=0.1, seed=7)) if layer else (None, None)
    kw = dict(b_post=bq, b_pre=bp, gate=gate, residual_scale=scale, norm="layer" if layer else "rms", eps=eps)
    r, z = block.block_norm(y, x, wq, wp, **kw)
    dr, dz = normal(T, D, std=0.1, seed=8), normal(T, D, std=0.1, seed=9)
    d = block.block_norm_backward(dr, dz, y, r, wq, wp, **kw)
    sums = {k: torch.zeros_like(v, dtype=torch.float64) for k, v in d.items() if k not in ("dx", "dy")}
    sizes = {k: torch.zeros_like(v) for k, v in sums.items()}
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731

    def hat(v):
        v = v - mean(v) if layer else v
        rho = 1 / torch.sqrt(mean(v * v) + eps)
        return v * rho, rho

    WQ, WP, BQ, BP = (None if t is None else t.double() for t in (wq, wp, bq, bp))
    for i in range(0, T, 2048):  # rows are their own: a slice at a time
        s, gi = slice(i, i + 2048), i * 4 // T
        Y, X, DR, DZ, R, G = y[s].double(), x[s].double(), dr[s].double(), dz[s].double(), r[s].double(), gate[gi].double()
        yh, ry = hat(Y)
        n = yh * WQ + (BQ if layer else 0)
        rr = scale * X + G * n
        size = (scale * X).abs() + G.abs() * (n.abs() + (WQ * (yh.abs() + ry * mean(Y.abs()))).abs())
        inside(r[s], rr, 2 * ACC * size + u * rr.abs() * 1.01, "r")
        rh, rho = hat(rr)
        zz = rh * WP + (BP if layer else 0)
        inside(z[s], zz, 8 * ACC * (zz.abs() + WP.abs() * rho * (size + mean(size) * (1 + rh.abs())) + (BP.abs() if layer else 0)) + u * zz.abs() * 1.01, "z")
        rh, rho = hat(R)  # the backward pass reads the rounded r
        c = DZ * WP
        t = DR + rho * (c - rh * mean(c * rh) - (mean(c) if layer else 0))
        off = rho * mean(R.abs()) if layer else 0
        rha = rh.abs() + off
        Mt = DR.abs() + rho * (c.abs() + rha * mean(c.abs() * rha) + (mean(c.abs()) if layer else 0))
        inside(d["dx"][s], scale * t, 4 * ACC * scale * Mt + 1.01 * u * (scale * t).abs(), "dx")
        yha = yh.abs() + (ry * mean(Y.abs()) if layer else 0)
        dn, Mn = G * t, G.abs() * Mt
        e, Me = dn * WQ, Mn * WQ.abs()
        dyy = ry * (e - yh * mean(e * yh) - (mean(e) if layer else 0))
        inside(d["dy"][s], dyy, 4 * ACC * ry * (Me + yha * mean(Me * yha) + (mean(Me) if layer else 0)) + 1.01 * u * dyy.abs(), "dy")
        for k, v, m in (("dw_pre", DZ * rh, DZ.abs() * rha), ("dw_post", dn * yh, Mn * yha), ("db_pre", DZ, DZ.abs()), ("db_post", dn, Mn)):
            if k in sums:
                sums[k] += v.sum(0)
                sizes[k] += m.sum(0)
        sums["dgate"][gi] += (t * n).sum(0)
        sizes["dgate"][gi] += (Mt * (yha * WQ.abs() + (BQ.abs() if layer else 0))).sum(0)
    for k in sums:
        inside(d[k], sums[k], 4 * ACC * sizes[k] + 1.01 * u * sums[k].abs(), k)
    status_clean()


def far(t, ld):
    """`t` as rows ld elements apart, the last of them more than 2^31 elements from the first."""
    assert (t.shape[0] - 1) * ld >= 2 ** 31
    out = torch.empty((t.shape[0] - 1) * ld + t.shape[1], dtype=t.dtype, device="cuda").as_strided(t.shape, (ld, 1))
    return out.copy_(t)


def test_offsets_past_32_bits():
    """Every operand in rows that lie 4 to 5 GB apart: the results of plain ones, bit for bit."""
    T, D, F = 70, 264, 328
    ld = 2 ** 31 // (T - 1) // 8 * 8 + 8
    x, dy = normal(T, D, seed=1), normal(T, D, std=0.1, seed=2)
    w = [normal(F, D, std=0.06, seed=3), normal(F, D, std=0.06, seed=4), normal(D, F, std=0.06, seed=5)]
    one, two = far(x, ld), far(dy, ld)
    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
    for n in (T, 33, 5):  # pairs of CTAs, and the short-token kernels' two sizes
        saved = block.gated_ffn(x[:n], *w, b_layout="nk", save=True)
        if n == T:
            assert same(saved, block.gated_ffn(one, *w, b_layout="nk", save=True))
        back = block.gated_ffn_backward(dy[:n], x[:n], *w, *saved[1:], b_layout="nk")
        if n == T:
            g, u = (far(t, ld) for t in saved[1:])
            assert same(back, block.gated_ffn_backward(two, one, *w, g, u, b_layout="nk"))
            del g, u
    v = normal(D, std=0.1, seed=6) + 1
    for shift in (0, 1):  # rows on 16-byte boundaries, and not
        cols = slice(shift, D)
        assert same(block.block_norm(dy[:, cols], x[:, cols], v[cols], v[cols]), block.block_norm(two[:, cols], one[:, cols], v[cols], v[cols]))
        a = block.block_norm_backward(dy[:, cols], x[:, cols], dy[:, cols], x[:, cols], v[cols], v[cols])
        b = block.block_norm_backward(two[:, cols], one[:, cols], two[:, cols], one[:, cols], v[cols], v[cols])
        assert same(a.values(), b.values())
    del two
    wf = far(w[0], 2 ** 31 // (F - 1) // 8 * 8 + 8)
    for n in (T, 5):
        assert torch.equal(block.gated_ffn(x[:n], *w, b_layout="nk"), block.gated_ffn(x[:n], wf, *w[1:], b_layout="nk"))
    del wf, one
    q = block.quantize_w4(normal(300, 256, std=0.06, seed=7), 32, symmetric=False)
    xs = normal(T, 256, seed=8)
    far_q = q._replace(q=far(q.q, 2 ** 31 // 299 // 16 * 16 + 16), scales=far(q.scales, 2 ** 31 // 299 // 8 * 8 + 8),
                       zeros=far(q.zeros, 2 ** 31 // 299 // 8 * 8 + 8))
    for n in (1, 9, T):
        assert torch.equal(block.matvec_w4(xs[:n], q), block.matvec_w4(xs[:n], far_q))
    assert torch.equal(block.matvec_w4(xs, q), block.matvec_w4(far(xs, ld), q))
    status_clean()
