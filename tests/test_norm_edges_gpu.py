"""Normalisation gradients where a call is legal and rare: matrices without columns at every layout of the backward
pass, and columns whose mean is far larger than their spread."""
import numpy as np
import pytest
import torch

from ginn_b200 import binding as B
from test_norm_gpu import check_backward, host

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


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows", [8, 120, 256, 512])
def test_columns_of_one_warp_refill_their_stages_many_times(gpu, dt, rows):
    """Up to 512 rows a warp has a column to itself and meets no barrier: the gradient from elsewhere, which the
    column sums do not depend on, has to be read before its place is filled again."""
    cols = 30000
    rng = np.random.default_rng(rows)
    x, dy, dh, old = (rng.standard_normal((rows, cols)).astype(dt) for _ in range(4))
    mean, rstd = x.astype(np.float64).mean(0).astype(np.float32), (1 / x.astype(np.float64).std(0)).astype(np.float32)
    X, DY, DH = (B.from_host(a) for a in (x, dy, dh))
    M, R = torch.from_numpy(mean).cuda(), torch.from_numpy(rstd).cuda()
    seen = []
    for _ in range(2):
        DX, DG, DB = B.from_host(old), torch.empty(rows, dtype=X.dtype, device="cuda"), torch.empty(rows, dtype=X.dtype, device="cuda")
        gpu.residual_norm_backward(X, None, M, R, DY, DH, None, DX, DG, DB, accumulate=False)
        seen.append([host(t) for t in (DX, DG, DB)])
    check_backward(x, None, mean, rstd, dy, dict(dres=seen[0][0], dgain=seen[0][1], dbias=seen[0][2]), dt, dh=dh.astype(np.float64))
    assert all((a == b).all() for a, b in zip(*seen))
