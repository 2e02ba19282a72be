"""Products with 4-bit weights at the ends of their types' ranges, and where only the last of
the bits that travel through them is left in the result."""
import pytest
import torch

from block_util import ACC, U, within
from gpu_util import gen, status_clean
from test_w4_gpu import CASES, LARGE, gpu, opened, step_most, weight

from icpp_tuning_b200 import block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,Nn,K,group", [(1, 8200, 2048, 32), (2, 16001, 1056, 64), (4, 8200, 4128, 128), (8, 12300, 4128, 512)])
def test_large_finite_values_as_digits(T, Nn, K, group):
    """bf16 values of one sign up to 2^125: every product with a weight and every sum of them
    stays far below fp32's end, the plain sum of a group's x does not."""
    dtype = torch.bfloat16
    w = weight(Nn, K, group, dtype, True, seed=K)
    w = w._replace(scales=w.scales / 64)
    x = ((1 + torch.rand(T, K, generator=gen(T))) * 2.0 ** 124).to(dtype)
    v, _ = opened(w)
    X = x.double()
    out = block.matvec_w4(x.cuda(), gpu(w))
    ref = X @ v.t()
    assert ref.abs().max() < 2.0 ** 127
    within(out, ref, U[dtype] * ref.abs() * 1.01 + ACC * X @ v.abs().t() + 2.0 ** -22 * step_most(X) @ v.abs().t())
    status_clean()


def products(x, v):
    """x v^T in float64, term by term: an infinity times nothing is NaN here as in the kernel."""
    return torch.stack([(row * v).sum(1) for row in x])


# the 16-bit form: one block of tokens to several, groups of each path
SMALL = [(1, 64, 160, 32), (3, 33, 256, 64), (8, 100, 544, 128), (9, 31, 416, 96), (16, 130, 1024, 256), (33, 20, 96, 4096), (40, 300, 640, 160)]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,Nn,K,group", SMALL)
def test_infinities_as_defined(T, Nn, K, group, zeros):
    """+-inf times the sign of each weight, NaN where the weight is zero; other tokens untouched."""
    dtype = torch.bfloat16 if (T + zeros) % 2 else torch.float16
    w = weight(Nn, K, group, dtype, zeros, seed=K, pad=T % 2)
    w.q[0, -1] = (w.q[0, -1] & 0xF0) | (8 if w.zeros is None else w.zeros[0, -1])  # one weight of nothing
    v, _ = opened(w)
    x = torch.randn(T, K, generator=gen(T)).to(dtype)
    clean = block.matvec_w4(x.cuda(), gpu(w))
    x[0, K - 2] = float("-inf")
    if T > 2:
        x[2, 3], x[2, 40] = float("inf"), float("inf")
    ref = products(x.double(), v)
    out = block.matvec_w4(x.cuda(), gpu(w)).double().cpu()
    odd = [0, 2] if T > 2 else [0]
    assert not ref[odd].isfinite().any() and ref[0].isinf().any() and ref[0].isnan().any()
    assert torch.equal(out[odd].nan_to_num(7.0), ref[odd].nan_to_num(7.0))
    rest = [i for i in range(T) if i not in odd]
    assert torch.equal(out[rest], clean.double().cpu()[rest])
    status_clean()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,Nn,K,group", SMALL)
def test_large_finite_values(T, Nn, K, group, zeros):
    """bf16 values up to 2^125: only what is inside the type's range may enter a sum."""
    dtype = torch.bfloat16
    w = weight(Nn, K, group, dtype, zeros, seed=K)
    w = w._replace(scales=w.scales / 64)
    x = ((1 + torch.rand(T, K, generator=gen(T))) * 2.0 ** 124).to(dtype)
    v, _ = opened(w)
    X = x.double()
    ref = X @ v.t()
    assert ref.abs().max() < 2.0 ** 127
    within(block.matvec_w4(x.cuda(), gpu(w)), ref, U[dtype] * ref.abs() * 1.01 + ACC * X @ v.abs().t())
    status_clean()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_any_zero_of_eight_bits(dtype):
    """Zeros past the nibbles' range are what the definition says too."""
    K = 256
    q = torch.arange(256 * K // 2, dtype=torch.int64).mul(37).remainder(256).to(torch.uint8).reshape(256, K // 2)
    w = block.W4(q, torch.ones(256, K // 32, dtype=dtype), torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, K // 32), 32)
    out = block.matvec_w4(torch.eye(K, dtype=dtype)[:64].cuda(), gpu(w))
    assert torch.equal(out.double().cpu(), opened(w)[0].t()[:64])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,Nn,K,group", CASES)
def test_bounds_without_an_offset(T, Nn, K, group, zeros):
    """What is summed is x (q - zero): the bound has its magnitudes alone, in both types."""
    dtype = torch.bfloat16 if (T + zeros) % 2 else torch.float16
    w = weight(Nn, K, group, dtype, zeros, seed=K + Nn + 1)
    x = (torch.randn(T, K, generator=gen(T)) + 3.0).to(dtype)
    v, _ = opened(w)
    X = x.double()
    ref = X @ v.t()
    within(block.matvec_w4(x.cuda(), gpu(w)), ref, U[dtype] * ref.abs() * 1.01 + ACC * X.abs() @ v.abs().t())


@pytest.mark.parametrize("T,Nn,K,group", LARGE)
def test_bounds_without_an_offset_as_digits(T, Nn, K, group):
    """The same for the digits, whose own rounding is half a unit, 2^-22 of the step's largest."""
    dtype = torch.bfloat16 if T % 2 else torch.float16
    w = weight(Nn, K, group, dtype, K % 3 == 0, seed=K + Nn + 1)
    x = (torch.randn(T, K, generator=gen(T)) + 3.0).to(dtype)
    v, _ = opened(w)
    X = x.double()
    ref = X @ v.t()
    out = block.matvec_w4(x.cuda(), gpu(w))
    within(out, ref, U[dtype] * ref.abs() * 1.01 + ACC * X.abs() @ v.abs().t() + 2.0 ** -22 * step_most(X) @ v.abs().t())


@pytest.mark.parametrize("T,Nn,K,group", [(1, 8200, 2048, 32), (2, 16001, 1056, 64), (8, 12300, 4128, 512)])
def test_any_zero_of_eight_bits_as_digits(T, Nn, K, group):
    dtype = torch.float16 if T % 2 else torch.bfloat16
    w = weight(Nn, K, group, dtype, True, seed=K)
    w = w._replace(zeros=torch.randint(0, 256, w.zeros.shape, generator=gen(K), dtype=torch.uint8))
    x = torch.randn(T, K, generator=gen(T)).to(dtype)
    v, _ = opened(w)
    X = x.double()
    ref = X @ v.t()
    within(block.matvec_w4(x.cuda(), gpu(w)), ref, U[dtype] * ref.abs() * 1.01 + ACC * X.abs() @ v.abs().t() + 2.0 ** -22 * step_most(X) @ v.abs().t())
    status_clean()
