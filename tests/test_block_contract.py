"""What the decoder-block operators promise at their C entries and in their autograd functions,
without a GPU."""
import ctypes

import pytest

from icpp_tuning_b200 import _native as N
from test_block_abi import A, _norm


@pytest.mark.parametrize("T", [0, 4])
@pytest.mark.parametrize("kw,msg", [
    (dict(db_pre=A), "bias"), (dict(db_post=A, w_post=A, dw_post=A), "bias"),  # rms: nothing would be summed for them
    (dict(norm=N.FO_NORM_LAYER, db_post=A), "w_post"),
])
def test_norm_backward_refuses_gradients_of_absent_biases(kw, msg, T):
    d = _norm(T=T, workspace=A, workspace_bytes=1 << 30, **kw)
    assert N.lib().fo_block_norm_backward(ctypes.byref(d), None) == N.FO_EINVAL
    assert msg in N.last_error()
