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
