"""The bits that the rounded results of ordinary inputs hide: values whose high parts cancel, so
that a product's result is what its lowest part carried.  Everything here is exact in fp32, and
the results have to be equal."""
import pytest
import torch

from gpu_util import gen, status_clean

from icpp_tuning_b200 import block

pytestmark = pytest.mark.gpu


def low_parts(T, n, dtype):
    """u [T, 2 n] = 1 + m x1 for even features, 1 for odd ones, and x1: a part of u that rounding
    to dtype takes away whole."""
    step = 2.0 ** -11 if dtype is torch.bfloat16 else 2.0 ** -14
    m = torch.randint(1, 4, (n,), generator=gen(n)).double()
    x1 = step * torch.randint(1, 3, (T,), generator=gen(T)).double()
    u = torch.ones(T, 2 * n, dtype=torch.float64)
    u[:, 0::2] += x1[:, None] * m
    assert (u.to(dtype) == 1).all()  # the high parts alone would cancel to nothing
    return m, x1, u


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,D,n", [(1, 64, 64), (3, 512, 40), (16, 72, 500), (17, 64, 64), (32, 1024, 260)])
def test_low_part_between_the_products(T, D, n, dtype):
    """h = relu(1) u = 1 + m x1 and 1 by w_down's 1 and -1: y = m x1."""
    m, x1, _ = low_parts(T, n, dtype)
    F = 2 * n
    x = torch.zeros(T, D, dtype=torch.float64)
    x[:, 0], x[:, 1] = 1, x1
    wg, wu, wd = torch.zeros(F, D), torch.zeros(F, D), torch.zeros(n, F)
    wg[:, 0] = wu[:, 0] = 1
    wu[0::2, 1] = m.float()
    wd[range(n), range(0, F, 2)], wd[range(n), range(1, F, 2)] = 1, -1
    pad = torch.zeros(n, (F + 7) // 8 * 8, dtype=dtype, device="cuda")
    pad[:, :F] = wd
    y = block.gated_ffn(x.to(dtype).cuda(), wg.to(dtype).cuda(), wu.to(dtype).cuda(), pad[:, :F], act="relu", b_layout="nk")
    assert torch.equal(y.double().cpu(), x1[:, None] * m)
    status_clean()


def four_bits(w, group, dtype):
    """Whole numbers of -8 .. 7 as W4 of scale 1."""
    q = (w + 8).to(torch.uint8)
    return block.W4((q[:, 0::2] | (q[:, 1::2] << 4)).cuda(), torch.ones(w.shape[0], -(-w.shape[1] // group), dtype=dtype, device="cuda"), None, group)


# 16-bit operands with one and two blocks of tokens, then digits (large weights)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,D,n,group", [(1, 64, 32, 32), (3, 256, 48, 128), (8, 96, 64, 32), (9, 128, 32, 64), (33, 64, 32, 32),
                                         (1, 2048, 4112, 64), (4, 4160, 4128, 128)])
def test_low_part_between_4_bit_products(T, D, n, group, dtype):
    m, x1, _ = low_parts(T, n, dtype)
    F = 2 * n
    x = torch.zeros(T, D, dtype=torch.float64)
    x[:, 0], x[:, 1] = 1, x1
    wg, wu, wd = torch.zeros(F, D), torch.zeros(F, D), torch.zeros(n, F)
    wg[:, 0] = wu[:, 0] = 1
    wu[0::2, 1] = m.float()
    wd[range(n), range(0, F, 2)], wd[range(n), range(1, F, 2)] = 1, -1
    y = block.gated_ffn_w4(x.to(dtype).cuda(), *(four_bits(w, group, dtype) for w in (wg, wu, wd)), act="relu")
    assert torch.equal(y.double().cpu(), x1[:, None] * m)
    status_clean()


def digit_inputs(T, Nn, K, dtype):
    """x with a pair of 1024's in each 32 k's and else m 2^-11, |m| <= 100, which only the last of
    three digits holds (units 2^-11 of 1024's fixed point of 23 bits); rows whose weights for a
    pair cancel.  -> x, w (whole numbers), the exact products in units of 2^-11."""
    g = gen(Nn + K)
    m = torch.randint(-100, 101, (T, K), generator=g).double()
    w = torch.randint(-8, 8, (Nn, K), generator=g).double()
    w[:, 0::32] = torch.randint(1, 8, (Nn, K // 32), generator=g).double()
    w[:, 1::32] = -w[:, 0::32]
    big = torch.zeros(K, dtype=torch.bool)
    big[0::32] = big[1::32] = True
    m[:, big] = 0
    x = m * 2.0 ** -11
    x[:, big] = 1024
    assert torch.equal(x.to(dtype).double(), x)
    return x, w, m @ w.t()


def last_digit(x):
    """The lowest of the three digits of x in units of 2^-11 (|x| <= 1024), as an oracle takes it."""
    v = torch.round(x * 2.0 ** 11).long()
    return (v + 128) % 256 - 128


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,Nn,K,group", [(1, 8200, 2048, 32), (2, 16001, 1056, 64), (4, 8200, 4128, 128), (8, 12300, 4128, 512)])
def test_last_digit(T, Nn, K, group, dtype):
    x, w, units = digit_inputs(T, Nn, K, dtype)
    d = last_digit(x).double()
    dropped = ((torch.round(x * 2.0 ** 11) - d) @ w.t())
    assert not dropped.any() and units.any()  # an oracle without the last digit has nothing left
    out = block.matvec_w4(x.to(dtype).cuda(), four_bits(w, group, dtype))
    assert torch.equal(out.cpu(), (units * 2.0 ** -11).to(dtype))  # one rounding of the exact sum
    status_clean()
