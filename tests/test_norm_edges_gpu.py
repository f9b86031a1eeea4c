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


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows", [64, 384, 640, 641, 4096, 8200, 8193])
def test_gradients_of_columns_far_from_zero(gpu, dt, rows):
    """A constant column gives no weight gradient and xh = 0 exactly, on the 16-byte grid and off it; columns whose mean is
    a thousand times their spread keep it.  x - mean is exact for values close to the mean, so xh is off by two
    roundings, 2^-23, and what is summed by the additions in a row, below 256."""
    rng = np.random.default_rng(rows)
    cols = 300
    # multiples of 2^-6: of up to 16 bits, exact in fp32 and, from 64 to 128 in steps of 2^-4, in Half
    step = 2.0 ** -6 if dt == np.float32 else 2.0 ** -4
    x = 100.0 + step * rng.integers(-20, 21, (rows, cols))
    x[:, ::3] = 100.0 + step * rng.integers(-20, 21, cols)[::3]
    x = x.astype(dt)
    dy = rng.standard_normal((rows, cols)).astype(dt)
    mean = x.astype(np.float64).mean(0).astype(np.float32)
    rstd = (1 / np.sqrt(x.astype(np.float64).var(0) + 1e-5)).astype(np.float32)
    X, DX = B.from_host(x), B.from_host(np.zeros_like(x))
    DG, DB = (torch.empty(rows, dtype=X.dtype, device="cuda") for _ in range(2))
    gpu.layer_norm_backward(X, None, torch.from_numpy(mean).cuda(), torch.from_numpy(rstd).cuda(), B.from_host(dy), DX, DG, DB, accumulate=False)
    m, r = mean.astype(np.float64), rstd.astype(np.float64)
    xh, g = (x.astype(np.float64) - m) * r, dy.astype(np.float64)
    assert (xh[:, ::3] == 0).all() and np.abs(xh).max() > 1
    u, half = 2.0 ** -24, np.finfo(dt).eps / 2
    dg = (g * xh).sum(1)
    assert (np.abs(host(DG) - dg) <= 256 * u * np.abs(g * xh).sum(1) + half * np.abs(dg) + 2.0 ** -25).all()
    inner = g - g.mean(0) - xh * (g * xh).mean(0)
    size = np.abs(g) + np.abs(g).mean(0) + np.abs(xh) * np.abs(g * xh).mean(0)
    assert (np.abs(host(DX) - r * inner) <= r * (256 * u * size + half * np.abs(inner)) + 2.0 ** -25).all()
    # constant columns alone
    X0 = B.from_host(np.ascontiguousarray(x[:, ::3]))
    gpu.layer_norm_backward(X0, None, torch.from_numpy(mean[::3].copy()).cuda(), torch.from_numpy(rstd[::3].copy()).cuda(),
                            B.from_host(np.ascontiguousarray(dy[:, ::3])), None, DG, DB, accumulate=False)
    assert (DG == 0).all()
