"""Normalisation gradients where a call is legal and rare: matrices without columns at every layout of the backward
pass, and columns whose mean is far larger than their spread."""
import numpy as np
import pytest
import torch

from ginn_b200 import binding as B

pytestmark = pytest.mark.gpu
DT = [np.float32, np.float16]


def torch_type(dt):
    return torch.float32 if dt == np.float32 else torch.float16


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows", [1, 40, 8192, 8193, 9000, 16391, 65536, 65544, 70000])
@pytest.mark.parametrize("residual", [False, True])
def test_weight_gradients_of_no_columns(gpu, dt, rows, residual):
    """Sums of nothing: zero when they are assigned, unchanged when they are added to."""
    X = torch.empty((0, rows), dtype=torch_type(dt), device="cuda").t()
    M = torch.empty(0, device="cuda")
    for accumulate, want in ((True, 2.0), (False, 0.0)):
        DG, DB = (torch.full((rows,), 2.0, dtype=X.dtype, device="cuda") for _ in range(2))
        if residual:
            gpu.residual_norm_backward(X, None, M, M, X, X, X, X.clone(), DG, DB, p=0.5, accumulate=accumulate)
        else:
            gpu.layer_norm_backward(X, None, M, M, X, X, DG, DB, accumulate=accumulate)
        assert (DG == want).all() and (DB == want).all()
