"""Results that share their storage are refused before anything runs."""
import pytest

from ginn_b200 import binding as B
from test_block_cpu import BAD, P, drop


@pytest.mark.parametrize("cols", [4, 0])
def test_one_tensor_for_both_weight_gradients(cols):
    L = B.lib()
    for accumulate in (0, 1):
        assert L.ginn_b200_layer_norm_backward(0, None, 0, 8, cols, P, 8, None, P, P, P, 8, 2 * P, 8, 3 * P, 3 * P, accumulate) == BAD
        assert L.ginn_b200_residual_norm_backward(0, None, 0, 8, cols, P, 8, None, P, P, P, 8, None, 0, drop(), 2 * P, 8, None, 0, 3 * P, 3 * P,
                                                  accumulate) == BAD
        assert b"dgain" in L.ginn_b200_last_error()
