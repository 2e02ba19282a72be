"""The autograd functions of gated_block without a GPU: the operators are stand-ins on CPU
tensors that hold their callers to the real ones' argument rules."""
import pytest
import torch

from icpp_tuning_b200 import block, gated_block


def _rows(*ts):
    for t in ts:
        assert t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0, (t.shape, t.stride())


def _ffn(x, w_gate, w_up, w_down, *, act, b_layout, save):
    assert act == "relu" and b_layout == "nk" and save
    _rows(x, w_gate, w_up, w_down)
    y, g, u = (block._matrix(x.shape[0], n, x) for n in (w_down.shape[0], w_gate.shape[0], w_gate.shape[0]))
    g.copy_(x @ w_gate.t()), u.copy_(x @ w_up.t())
    y.copy_((g.relu() * u) @ w_down.t())
    return y, g, u


def _ffn_backward(dy, x, w_gate, w_up, w_down, g, u, *, act, b_layout):
    _rows(dy, x, w_gate, w_up, w_down, g, u)
    dh, a = dy @ w_down, g.relu()
    dg, du = dh * u * (g > 0), dh * a
    return dg @ w_gate + du @ w_up, dg.t() @ x, du.t() @ x, dy.t() @ (a * u)


@pytest.fixture
def operators(monkeypatch):
    monkeypatch.setattr(block, "gated_ffn", _ffn)
    monkeypatch.setattr(block, "gated_ffn_backward", _ffn_backward)


def _ffn_inputs(T=5, D=16, F=24, N=64):
    g = torch.Generator().manual_seed(N)
    return [(torch.randn(*s, generator=g) * 0.5).requires_grad_() for s in ((T, D), (F, D), (F, D), (N, F))]


@pytest.mark.parametrize("N", [8, 64, 100, 3])
@pytest.mark.parametrize("how", ["plain", "rows", "transposed", "broadcast", "sliced"])
def test_gated_ffn_passes_any_gradient_on(operators, N, how):
    """dy as autograd may bring it, at output widths that are no multiple of 8 too."""
    args = _ffn_inputs(N=N)
    y = gated_block.GatedFFN.apply(*args, "relu", "nk")
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(1))
    if how == "rows":  # as y lies
        dy = block._matrix(*y.shape, y).copy_(dy)
    if how == "transposed":
        dy = dy.t().contiguous().t()
    if how == "broadcast":
        dy = torch.ones(()).expand(y.shape)
    if how == "sliced":
        dy = torch.cat((dy, dy), 1)[:, 1:N + 1]
    got = torch.autograd.grad(y, args, dy)
    ref = [t.detach().clone().requires_grad_() for t in args]
    want = torch.autograd.grad(((ref[0] @ ref[1].t()).relu() * (ref[0] @ ref[2].t())) @ ref[3].t(), ref, dy)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)


def _norm(y, x, w_post, w_pre, *, b_post, b_pre, gate, residual_scale, norm, eps):
    assert w_post is None and gate is None and b_pre is None and norm == "rms"
    r = residual_scale * x + y
    return r, r * torch.rsqrt((r * r).mean(1, keepdim=True) + eps) * w_pre


def _norm_backward(dr, dz, y, r, w_post, w_pre, *, b_post, b_pre, gate, residual_scale, norm, eps):
    rho = torch.rsqrt((r * r).mean(1, keepdim=True) + eps)
    c = dz * w_pre
    t = rho * (c - r * rho * (c * r * rho).mean(1, keepdim=True)) + (0 if dr is None else dr)
    return {"dy": t, "dx": residual_scale * t, "dw_pre": (dz * r * rho).sum(0)}


@pytest.mark.parametrize("into", [0, 1, 3])
def test_second_derivatives_raise(operators, monkeypatch, into):
    """The operators have none: a loss with a gradient in it is an error, whatever it is
    differentiated by, not a sum that lacks that term."""
    monkeypatch.setattr(block, "block_norm", _norm)
    monkeypatch.setattr(block, "block_norm_backward", _norm_backward)
    args = _ffn_inputs()
    y = gated_block.GatedFFN.apply(*args, "relu", "nk")
    (dx,) = torch.autograd.grad(y.sum(), args[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(y.square().sum() + dx.square().sum(), args[into])
    x, w = torch.randn(4, 8).requires_grad_(), torch.ones(8).requires_grad_()
    r, z = gated_block.BlockNorm.apply(x, x, None, w, None, None, None, 0.5, "rms", 1e-5)
    (dx,) = torch.autograd.grad(z.square().sum() + r.sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(r.sum() + dx.square().sum(), w if into else x)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        (r.sum() + dx.square().sum()).backward()


def test_gradients_without_a_graph_carry_none(operators):
    args = _ffn_inputs()
    got = torch.autograd.grad(gated_block.GatedFFN.apply(*args, "relu", "nk").square().sum(), args)
    assert not any(t.requires_grad for t in got)


def test_widths_without_a_backward_pass_are_refused_forward(monkeypatch):
    """The backward kernels hold rows of at most 8192 columns, the forward ones 16384."""
    monkeypatch.setattr(block, "block_norm", _norm)
    x, w = torch.randn(2, 8193), torch.ones(8193)
    call = lambda: gated_block.BlockNorm.apply(x, x, None, w, None, None, None, 0.5, "rms", 1e-5)  # noqa: E731
    want = call()
    w.requires_grad_()
    with pytest.raises(ValueError, match="8192"):
        call()
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(call(), want))


def test_nothing_is_saved_without_gradients(monkeypatch):
    saves = []

    def ffn(x, w_gate, w_up, w_down, *, act, b_layout, save=False):
        saves.append(save)
        out = _ffn(x, w_gate, w_up, w_down, act=act, b_layout=b_layout, save=True)
        return out if save else out[0]

    monkeypatch.setattr(block, "gated_ffn", ffn)
    args = _ffn_inputs()
    y = gated_block.GatedFFN.apply(*args, "relu", "nk")
    with torch.no_grad():
        z = gated_block.GatedFFN.apply(*args, "relu", "nk")
    w = gated_block.GatedFFN.apply(*(t.detach() for t in args), "relu", "nk")
    assert saves == [True, False, False] and torch.equal(y, z) and torch.equal(y, w)
    assert y.requires_grad and not z.requires_grad and not w.requires_grad
