"""What the transformer-block operators (layer norm, dropout, residual norm,
attention with a relative position bias) promise without a GPU: the
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
    (lambda: norm_fwd(ldx=9), BAD), (lambda: norm_bwd(x=P + 64, lddy=9), BAD),  # in place with another leading dimension
    (lambda: B.lib().ginn_b200_dropout_forward(0, None, 0, 8, 4, P, 9, None, 0, drop(), P, 8), BAD),
    (lambda: B.lib().ginn_b200_dropout_forward(0, None, 0, 8, 4, P, 8, 2 * P, 9, drop(), 2 * P, 8), BAD),
    (lambda: B.lib().ginn_b200_dropout_backward(0, None, 0, 8, 4, P, 9, drop(), P, 8, 0), BAD),
    (lambda: B.lib().ginn_b200_residual_norm_forward(0, None, 0, 8, 4, P, 8, 2 * P, 9, drop(), None, None, 1e-5, 2 * P, 8, 3 * P, 8, None, None), BAD),
    (lambda: B.lib().ginn_b200_residual_norm_backward(0, None, 0, 8, 4, P, 8, None, P, P, 2 * P, 8, 3 * P, 9, drop(), 4 * P, 8, 3 * P, 8, None, None, 0), BAD),
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


# ---- attention with a relative position bias ----

@pytest.mark.parametrize("causal,lengths", [(False, None), (True, None), (True, ([3, 0, 5], [2, 4, 6]))])
def test_relative_attention_gradient_against_differences(causal, lengths):
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((4, 5, 4, 3)), rng.standard_normal((4, 6, 2, 3)), rng.standard_normal((4, 6, 2, 3))
    table, d_o = rng.standard_normal((6, 4)), rng.standard_normal(q.shape)
    bmap = [orc.relative_bucket(d, 6, 4, True) for d in range(-4, 5)]
    kw = dict(scale=0.7, causal=causal, offsets=[1, -2, 0])
    if lengths:
        kw |= dict(q_lengths=lengths[0], k_lengths=lengths[1])
    got = orc.relative_attention(q, k, v, table, bmap, d_o=d_o, **kw)
    at = {"dq": q, "dk": k, "dv": v, "dtable": table}
    e = 1e-6
    for name, x in at.items():
        for i in list(np.ndindex(x.shape))[::7]:
            old, x[i] = x[i], x[i] + e
            hi = (orc.relative_attention(q, k, v, table, bmap, **kw)["o"] * d_o).sum()
            x[i] = old - e
            lo = (orc.relative_attention(q, k, v, table, bmap, **kw)["o"] * d_o).sum()
            x[i] = old
            # central difference: truncation of order e^2, rounding 2^-52 * |loss| / e
            assert abs(got[name][i] - (hi - lo) / (2 * e)) < 1e-7, (name, i)


@pytest.mark.parametrize("buckets,max_distance,both,reach", [
    (32, 128, True, 300), (32, 128, False, 300), (2, 1, False, 5), (4, 7, True, 20), (65, 32, True, 40), (65, 32, False, 40),
    (16, 3, True, 30), (40, 1000, False, 1200), (64, 4096, True, 5000), (12, 729, False, 800), (32, 128, True, 0), (512, 1 << 20, False, 3000),
])
def test_relative_buckets(buckets, max_distance, both, reach):
    """Against the definition in Python's whole numbers; (12, 729) has borders that are distances
    exactly, where a logarithm in floating point may fall on either side."""
    got = B.relative_buckets(buckets, max_distance, both, reach).tolist()
    step = 1 if buckets < 512 else 97
    for at in range(0, 2 * reach + 1, step):
        assert got[at] == orc.relative_bucket(at - reach, buckets, max_distance, both), at - reach


@pytest.mark.parametrize("args", [(1, 8, 0, 4), (3, 8, 1, 4), (513, 8, 0, 4), (8, 0, 0, 4), (8, (1 << 20) + 1, 0, 4), (8, 8, 0, -1), (8, 8, 0, (1 << 24) + 1)])
def test_refused_bucket_maps(args):
    out = np.zeros(16, np.int32)
    assert B.lib().ginn_b200_relative_buckets(*args, out.ctypes.data) == BAD
    assert (out == 0).all()


def described(**change):
    """A valid description of 3 sequences, 4 heads over 2, 5 queries, 6 keys of size 8, changed."""
    d = dict(tq=5, tk=6, head_size=8, heads=4, kv_heads=2, batch=3, q=P, ldq=8, stride_q_head=40, stride_q_batch=160, k=P, ldk=8,
             stride_k_head=48, stride_k_batch=96, v=P, ldv=8, stride_v_head=48, stride_v_batch=96, table=P, ldt=32, buckets=32, map=P,
             reach=16, scale=1.0, causal=0, q_offset=0, o=2 * P, ldo=8, stride_o_head=40, stride_o_batch=160, lse=P)
    return B._RelativeAttention(**{**d, **change})


def forward(dtype=0, **change):
    import ctypes
    return B.lib().ginn_b200_relative_attention_forward(0, None, dtype, ctypes.byref(described(**change)))


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), UNSUPPORTED), (dict(tq=-1), BAD), (dict(tk=1 << 29), BAD), (dict(heads=65536), BAD), (dict(head_size=0), UNSUPPORTED),
    (dict(head_size=257), UNSUPPORTED), (dict(kv_heads=3), BAD), (dict(kv_heads=0), BAD), (dict(scale=float("inf")), BAD),
    (dict(scale=float("nan")), BAD), (dict(q_offset=1 << 31), BAD), (dict(buckets=0), BAD), (dict(ldt=31), BAD), (dict(map=None), BAD),
    (dict(reach=-1), BAD), (dict(q=None), BAD), (dict(k=None), BAD), (dict(v=None), BAD), (dict(o=None), BAD), (dict(lse=None), BAD),
    (dict(ldq=-8), BAD), (dict(ldo=7), BAD), (dict(stride_o_head=39), BAD), (dict(stride_o_batch=0), BAD), (dict(o=P), BAD), (dict(batch=1 << 20, heads=1 << 12, kv_heads=1), BAD),
])
def test_refused_attention(change, status):
    assert forward(**change) == status
    assert B.lib().ginn_b200_last_error()


@pytest.mark.parametrize("change,grad", [
    ({}, dict(d_o=None)), (dict(table=None), dict(dtable=P, lddt=32)), ({}, dict(dtable=P, lddt=31)), ({}, dict(dk=P, lddk=8, stride_dk_head=47)),
    ({}, dict(lddo=-1)), ({}, dict(dq=P)), ({}, dict(dq=2 * P)), ({}, dict(dq=3 * P)), ({}, dict(dk=4 * P, lddk=8, stride_dk_head=48, stride_dk_batch=96)),
])
def test_refused_attention_gradient(change, grad):
    import ctypes
    g = dict(d_o=3 * P, lddo=8, stride_do_head=40, stride_do_batch=160, dq=4 * P, lddq=8, stride_dq_head=40, stride_dq_batch=160)
    call = lambda g: B.lib().ginn_b200_relative_attention_backward(  # noqa: E731
        0, None, 0, ctypes.byref(described(**change)), None if g is None else ctypes.byref(B._RelativeAttentionGrad(**g)))
    assert call({**g, **grad}) == BAD
    assert call(None) == BAD


def test_attention_without_queries_needs_no_gpu():
    assert forward(tq=0) == 0 and forward(batch=0) == 0
