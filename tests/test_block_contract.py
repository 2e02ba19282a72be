"""What the decoder-block operators promise at their C entries and in their autograd functions,
without a GPU."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from icpp_tuning_b200 import _native as N
from icpp_tuning_b200 import block
from test_block_abi import A, _matvec, _norm, _w4

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("T", [0, 4])
@pytest.mark.parametrize("kw,msg", [
    (dict(db_pre=A), "bias"), (dict(db_post=A, w_post=A, dw_post=A), "bias"),  # rms: nothing would be summed for them
    (dict(norm=N.FO_NORM_LAYER, db_post=A), "w_post"),
])
def test_norm_backward_refuses_gradients_of_absent_biases(kw, msg, T):
    d = _norm(T=T, workspace=A, workspace_bytes=1 << 30, **kw)
    assert N.lib().fo_block_norm_backward(ctypes.byref(d), None) == N.FO_EINVAL
    assert msg in N.last_error()


SIZE_QUERY = """
import ctypes
from icpp_tuning_b200 import _native as N
d = N.FoBlockNormDesc()
d.T, d.D, d.gate_rows, d.norm = {T}, 64, {rows}, N.FO_NORM_LAYER
print(N.lib().fo_block_norm_backward_workspace_size(ctypes.byref(d)))
"""


@pytest.mark.parametrize("T,rows", [(1 << 32, 1 << 32), (4, 1 << 32), (4, 3), (4, 8), (1 << 31, 1), (4, -1), (0, 0)])
def test_norm_workspace_size_of_what_the_entry_refuses_is_zero(T, rows):
    # in a process of its own: a division by zero would end it
    r = subprocess.run([sys.executable, "-c", SIZE_QUERY.format(T=T, rows=rows)], capture_output=True, text=True, cwd=ROOT, timeout=120)
    assert r.returncode == 0, r.stderr
    assert int(r.stdout) == 0


@pytest.mark.parametrize("cols", [1, 8, 60, 64])
def test_the_row_stride_of_a_single_row_does_not_count(cols):
    """A matrix of one row may carry any row stride (PyTorch calls it contiguous all the same)."""
    for one in (torch.zeros(cols, 1).t(), torch.zeros(3 * cols)[None, :cols], torch.zeros(1, cols)):
        ld = block._ld(one, 1, cols, "x")
        assert ld % 16 == 0 and ld >= cols
        assert block._matrix(1, cols, one).stride(0) % 8 == 0 and block._new(1, cols, one).stride(0) == cols
    two = torch.zeros(2, cols + 3)[:, :cols]
    assert block._ld(two, 2, cols, "x") == cols + 3


def test_w4_groups_longer_than_the_index_division_holds_are_refused():
    """A step's group is found by a product with a 32-bit reciprocal, exact while steps x steps
    a group stay within 2^32; one group for the whole row needs none."""
    def call(K, group):
        d = _matvec(_w4(ldq=K // 2, lds=K // 32, group=group), K=K, ldx=K, out=None)  # nothing can run
        return N.lib().fo_matvec_w4(ctypes.byref(d), None)

    K = 1 << 25
    assert call(K, (1 << 21) + 128) == N.FO_EUNSUPPORTED and "group" in N.last_error()
    for fine in (1 << 21, 128, K, 2 * K):
        assert call(K, fine) == N.FO_EINVAL and "out" in N.last_error()
    # the bound itself, on the integers of the kernel: the worst reciprocals of 2^32 / per
    for per in (3, 7, 641, 6700417 % 65536, 40503, 65535, 16385):
        rcp = -(-(1 << 32) // per)
        last = (1 << 32) // per
        at = sorted({i for q in (1, 2, 3, last // per, last // per - 1) for i in (q * per - 1, q * per, q * per + 1) if 0 <= i <= last})
        assert all((i * rcp) >> 32 == i // per for i in at), per
    per = (1 << 18) - 5  # and past it
    rcp = -(-(1 << 32) // per)
    assert any((i * rcp) >> 32 != i // per for i in range(per - 1, 1 << 20, per))


@pytest.mark.parametrize("T,D,rows", [(16384, 4096, 16384), (4096, 1001, 4), (7, 64, 0)])
def test_norm_workspace_holds_the_sums_that_the_form_has(T, D, rows):
    """Per unit of rows, fp32: two sums a column in the rms form, four in the other."""
    d = _norm(T=T, D=D, gate_rows=rows, gate=A if rows else None)
    need = N.lib().fo_block_norm_backward_workspace_size
    rms = need(ctypes.byref(d))
    units, odd = divmod(rms, 2 * 4 * ((D + 3) // 4 * 4))
    assert odd == 0 and units >= max(1, rows)
    if rows == T:
        assert units == rows  # one row a unit
    d.norm = N.FO_NORM_LAYER
    assert need(ctypes.byref(d)) == 2 * rms


@pytest.mark.parametrize("D,layer,units", [(4096, False, 296), (4096, True, 148), (2049, False, 148), (2048, True, 296), (8192, False, 148)])
def test_norm_backward_plans_the_units_that_run_at_once(D, layer, units):
    """Two CTAs a SM, one where the kernel has 512 threads of 128 registers."""
    d = _norm(T=16384, D=D, norm=N.FO_NORM_LAYER if layer else N.FO_NORM_RMS)
    need = N.lib().fo_block_norm_backward_workspace_size(ctypes.byref(d))
    assert need == units * (4 if layer else 2) * 4 * ((D + 3) // 4 * 4)
