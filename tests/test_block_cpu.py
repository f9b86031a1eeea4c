"""What the transformer-block operators (layer norm, dropout, residual norm) promise without a GPU: the
oracle's formulas against differences and published numbers, and the refusals of the C ABI, which
come before any GPU call."""
import numpy as np
import pytest

from ginn_b200 import binding as B
from oracle import oracle as orc

BAD, UNSUPPORTED = 1, 2
P = 0x1000  # stands for a device pointer: a refused call does not touch it


def words(*hexes):
    return [int(h, 16) for h in hexes]


def test_philox_published_answers():
    """Known answers that come with the generator's publication (philox4x32, 10 rounds)."""
    for ctr, key, out in [
        (["0"] * 4, ["0"] * 2, ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]),
        (["ffffffff"] * 4, ["ffffffff"] * 2, ["408f276d", "41c83b0e", "a20bc7c6", "6d5451fd"]),
        (["243f6a88", "85a308d3", "13198a2e", "03707344"], ["a4093822", "299f31d0"], ["d16cfe09", "94fdcceb", "5001e420", "24126ea1"]),
    ]:
        got = orc.philox4x32(np.array(words(*ctr), np.uint64)[:, None], words(*key))
        assert [int(v) for v in got[:, 0]] == words(*out)


def test_mask_is_a_function_of_the_element_number():
    """A matrix and its transpose-shaped view share the numbers; the kept share is the probability's."""
    a = orc.dropout_mask(40, 25, 0.3, 7, 8).T.reshape(-1)
    b = orc.dropout_mask(8, 125, 0.3, 7, 8).T.reshape(-1)
    np.testing.assert_array_equal(a, b)
    big = orc.dropout_mask(1000, 1000, 0.3, 7, 8)
    # mean 1, standard deviation sqrt(p / (1 - p)) / 1000 = 0.00065: six of them
    assert abs(big.mean() - 1) < 0.004
    assert (orc.dropout_mask(30, 30, 0.0, 1, 1) == 1).all()


def test_layer_norm_gradient_against_differences():
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((9, 4)), rng.standard_normal((9, 4))
    gain, bias = rng.standard_normal(9), rng.standard_normal(9)
    _, m, r = orc.layer_norm_forward(x, gain, bias)
    dx, dg, db = orc.layer_norm_backward(x, gain, m, r, dy)
    loss = lambda x, g, b: (orc.layer_norm_forward(x, g, b)[0] * dy).sum()  # noqa: E731
    e = 1e-6

    def diff(at, which):
        out = np.zeros_like(at)
        for i in np.ndindex(at.shape):
            hi, lo = at.copy(), at.copy()
            hi[i] += e
            lo[i] -= e
            args = [[x, gain, bias], [x, gain, bias]]
            args[0][which], args[1][which] = hi, lo
            out[i] = (loss(*args[0]) - loss(*args[1])) / (2 * e)
        return out

    # central differences: truncation e^2, rounding 2^-52 / e relative to a loss of order 10
    for got, ref in ((dx, diff(x, 0)), (dg, diff(gain, 1)), (db, diff(bias, 2))):
        np.testing.assert_allclose(got, ref, rtol=1e-6, atol=1e-7)


def norm_fwd(dtype=0, rows=8, cols=4, x=P, ldx=8, eps=1e-5, y=P, ldy=8):
    return B.lib().ginn_b200_layer_norm_forward(0, None, dtype, rows, cols, x, ldx, None, None, eps, y, ldy, None, None)


def norm_bwd(dtype=0, rows=8, cols=4, x=P, ldx=8, mean=P, rstd=P, dy=P, lddy=8, dx=P, lddx=8):
    return B.lib().ginn_b200_layer_norm_backward(0, None, dtype, rows, cols, x, ldx, None, mean, rstd, dy, lddy, dx, lddx, None, None, 0)


def drop(p=0.1):
    import ctypes
    return ctypes.byref(B._Dropout(p, 1, 2, None))


@pytest.mark.parametrize("call,status", [
    (lambda: norm_fwd(dtype=7), UNSUPPORTED), (lambda: norm_fwd(rows=-1), BAD), (lambda: norm_fwd(cols=1 << 31), BAD),
    (lambda: norm_fwd(x=None), BAD), (lambda: norm_fwd(y=None), BAD), (lambda: norm_fwd(ldx=7), BAD), (lambda: norm_fwd(ldy=7), BAD),
    (lambda: norm_fwd(eps=0.0), BAD), (lambda: norm_fwd(eps=float("nan")), BAD),
    (lambda: norm_bwd(mean=None), BAD), (lambda: norm_bwd(rstd=None), BAD), (lambda: norm_bwd(dy=None), BAD), (lambda: norm_bwd(lddx=7), BAD),
    (lambda: B.lib().ginn_b200_dropout_forward(0, None, 0, 8, 4, P, 8, None, 0, None, P, 8), BAD),
    (lambda: B.lib().ginn_b200_dropout_forward(0, None, 0, 8, 4, P, 8, P, 7, drop(), P, 8), BAD),
    (lambda: B.lib().ginn_b200_dropout_backward(0, None, 0, 8, 4, P, 8, drop(), None, 8, 0), BAD),
    (lambda: B.lib().ginn_b200_residual_norm_forward(0, None, 0, 8, 4, P, 8, P + 64, 8, drop(), None, None, 1e-5, P, 8, P, 8, None, None), BAD),
    (lambda: B.lib().ginn_b200_residual_norm_backward(0, None, 0, 8, 4, P, 8, None, P, P, P, 8, None, 0, drop(), P, 8, P, 8, None, None, 0), BAD),
])
def test_refusals(call, status):
    assert call() == status
    assert B.lib().ginn_b200_last_error()


@pytest.mark.parametrize("p", [-0.1, 1.0, 1.5, float("nan"), 1 - 2.0 ** -18])
def test_refused_probabilities(p):
    assert B.lib().ginn_b200_dropout_forward(0, None, 0, 8, 4, P, 8, None, 0, drop(p), P, 8) == BAD


def test_empty_matrices_need_no_gpu():
    assert norm_fwd(rows=0) == 0 and norm_fwd(cols=0) == 0 and norm_bwd(cols=0) == 0
    assert B.lib().ginn_b200_dropout_forward(0, None, 0, 0, 4, None, 8, None, 0, drop(), None, 8) == 0
