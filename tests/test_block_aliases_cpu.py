"""Results that share their storage are refused before anything runs."""
import ctypes

import pytest

from ginn_b200 import binding as B
from test_block_cpu import BAD, P, described, drop


@pytest.mark.parametrize("cols", [4, 0])
def test_one_tensor_for_both_weight_gradients(cols):
    L = B.lib()
    for accumulate in (0, 1):
        assert L.ginn_b200_layer_norm_backward(0, None, 0, 8, cols, P, 8, None, P, P, P, 8, 2 * P, 8, 3 * P, 3 * P, accumulate) == BAD
        assert L.ginn_b200_residual_norm_backward(0, None, 0, 8, cols, P, 8, None, P, P, P, 8, None, 0, drop(), 2 * P, 8, None, 0, 3 * P, 3 * P,
                                                  accumulate) == BAD
        assert b"dgain" in L.ginn_b200_last_error()


@pytest.mark.parametrize("change,dtable", [({}, 4 * P), ({}, 5 * P), ({}, 6 * P), ({}, P), ({}, 2 * P), ({}, 3 * P), (dict(tq=0), 5 * P), (dict(tk=0), P)])
def test_table_gradient_over_another_tensor(change, dtable):
    """dq, dk, dv, the table (and q, k, v), o, d_o; without queries dk, without keys the table."""
    g = dict(d_o=3 * P, lddo=8, stride_do_head=40, stride_do_batch=160, dq=4 * P, lddq=8, stride_dq_head=40, stride_dq_batch=160, dk=5 * P, lddk=8,
             stride_dk_head=48, stride_dk_batch=96, dv=6 * P, lddv=8, stride_dv_head=48, stride_dv_batch=96, dtable=dtable, lddt=32)
    call = B.lib().ginn_b200_relative_attention_backward
    assert call(0, None, 0, ctypes.byref(described(**change)), ctypes.byref(B._RelativeAttentionGrad(**g))) == BAD
    assert b"dtable" in B.lib().ginn_b200_last_error()
