"""GPU parity of attention with a relative position bias against the fp64 oracle, through the C ABI.

Bounds, element by element.  u: half a unit in the last place of the storage type (a result's one
rounding, and for Half operands that of the probabilities and of the scores' gradient on their way
into the second products, and of the stored output in delta).  E = 2^-17: what a product may be off
relative to the product of the magnitudes (fp32 accumulation of exact Half products, or three
TF32 products per term), which also covers the exponentials and the statistics.

Floors of the Half operands inside the backward products, where a relative bound ends: below a Half's
normal range a rounding is off by half a subnormal step, 2^-25, whatever the value.  P is formed times
2^12: 2^-37 each.  dS is formed times 2^floor(14 - log2 B) with B = 2 max|d_o row| max|v row| per
sequence and key head, which is more than 2^13 / B: less than 2^-38 B each.  A key that no query
attends to (p < 1e-8) has a gradient of that size, 3e-8 in the peaked case with B = 2^8, so there the
floor and not u decides whether the result rounds to 0 or to the smallest Half.
"""
import numpy as np
import pytest
import torch

from ginn_b200 import binding as B
from oracle import oracle as orc

pytestmark = pytest.mark.gpu
E = 2.0 ** -17


def spread(a, dt, pad=0, order=(3, 2, 1)):
    """Host (hs, t, heads, batch) array on the GPU; `order`: outer to inner dimension order in memory."""
    t = torch.from_numpy(np.ascontiguousarray(a.astype(dt)))
    outer = list(order) + [0]
    m = t.permute(*outer).contiguous()
    if pad:
        m = torch.nn.functional.pad(m, (0, pad))
    back = [outer.index(i) for i in range(4)]
    return m.cuda().permute(*back)[:a.shape[0]]


def host(t):
    return t.detach().cpu().numpy().astype(np.float64)


class Case:
    def __init__(self, dt, hs, tq, tk, heads=2, kv=None, batch=2, causal=False, q_lengths=None, k_lengths=None, offsets=None, table=True,
                 buckets=32, reach=20, pad=0, order=(3, 2, 1), scale=None, spread_scores=1.0, seed=0):
        rng = np.random.default_rng(seed + hs * 131 + tq * 17 + tk)
        kv = heads if kv is None else kv
        self.dt, self.causal, self.scale = dt, causal, scale or spread_scores / np.sqrt(hs)
        self.scale = float(np.float32(self.scale))
        mk = lambda *s: rng.standard_normal(s).astype(dt)  # noqa: E731
        self.q, self.k, self.v, self.d_o = mk(hs, tq, heads, batch), mk(hs, tk, kv, batch), mk(hs, tk, kv, batch), mk(hs, tq, heads, batch)
        self.table = mk(buckets, heads) if table else None
        self.map = B.relative_buckets(buckets, max(reach, 1), not causal, reach) if table else None
        self.q_lengths, self.k_lengths, self.offsets = q_lengths, k_lengths, offsets
        self.pad, self.order = pad, order

    def ints(self, x):
        return None if x is None or isinstance(x, int) else torch.tensor(x, dtype=torch.int32, device="cuda")

    def upload(self):
        sp = lambda a: spread(a, self.dt, self.pad, self.order)  # noqa: E731
        self.Q, self.K, self.V, self.DO = (sp(a) for a in (self.q, self.k, self.v, self.d_o))
        self.T = None if self.table is None else B.from_host(self.table)
        self.M = None if self.map is None else self.map.cuda()
        self.O = sp(np.full(self.q.shape, 9.0))
        self.L = torch.full((self.q.shape[3], self.q.shape[2], self.q.shape[1]), 9.0, device="cuda")
        self.kw = dict(scale=self.scale, causal=self.causal, q_lengths=self.ints(self.q_lengths), k_lengths=self.ints(self.k_lengths),
                       q_offsets=self.ints(self.offsets), q_offset=self.offsets if isinstance(self.offsets, int) else 0)
        self.DQ, self.DK, self.DV = sp(self.q), sp(self.k), sp(self.v)  # old gradients: the operands themselves
        self.DT = None if self.table is None else B.from_host(self.table)
        return self

    def forward(self, gb):
        gb.relative_attention_forward(self.Q, self.K, self.V, self.T, self.M, self.O, self.L, **self.kw)

    def backward(self, gb, accumulate=False):
        gb.relative_attention_backward(self.Q, self.K, self.V, self.T, self.M, self.O, self.L, self.DO, dq=self.DQ, dk=self.DK, dv=self.DV,
                                       dtable=self.DT, accumulate=accumulate, **self.kw)

    def reference(self):
        """Results and their bounds, from the definition."""
        u = np.finfo(self.dt).eps / 2
        ui = u if self.dt == np.float16 else 0.0  # roundings inside: Half only
        batch, heads, group = self.q.shape[3], self.q.shape[2], self.q.shape[2] // self.k.shape[2]
        offsets = [self.offsets or 0] * batch if self.offsets is None or isinstance(self.offsets, int) else self.offsets
        kw = dict(causal=self.causal, offsets=offsets, q_lengths=self.q_lengths, k_lengths=self.k_lengths)
        clean = lambda a: np.where(np.isfinite(a), a, 0).astype(np.float64)  # noqa: E731
        q, k, v, g = (clean(a) for a in (self.q, self.k, self.v, self.d_o))
        bmap = np.zeros(1, int) if self.map is None else self.map.numpy()
        ref = orc.relative_attention(q, k, v, self.table, bmap, self.scale, d_o=g, **kw)
        tol = {n: np.zeros(np.shape(x)) for n, x in ref.items() if x is not None}
        tol["lse"] = np.full(ref["lse"].shape, 0.0)
        for b in range(batch):
            nq = q.shape[1] if self.q_lengths is None else max(0, min(q.shape[1], self.q_lengths[b]))
            nk = k.shape[1] if self.k_lengths is None else max(0, min(k.shape[1], self.k_lengths[b]))
            d = np.arange(nk)[:, None] - (np.arange(nq)[None] + offsets[b])
            reach = len(bmap) // 2
            kind = bmap[np.clip(d, -reach, reach) + reach]
            for h in range(heads if nq and nk else 0):
                Q, K, V, G = q[:, :nq, h, b], k[:, :nk, h // group, b], v[:, :nk, h // group, b], g[:, :nq, h, b]
                s = self.scale * (K.T @ Q) + (0 if self.table is None else self.table.astype(np.float64)[kind, h])
                if self.causal:
                    s = np.where(d <= 0, s, -np.inf)
                lse = ref["lse"][b, h, :nq]
                p = np.exp(s - np.where(np.isfinite(lse), lse, np.inf))
                es = E * (self.scale * (np.abs(K).T @ np.abs(Q)) + 1)  # error of a score, relative error of p
                seen = np.isfinite(s)
                top = np.where(seen, es, 0).max(0)
                ep = p * (es + top)
                tol["lse"][b, h, :nq] = top + E * np.abs(np.where(np.isfinite(lse), lse, 0))
                o = ref["o"][:, :nq, h, b]
                eo = np.abs(V) @ (ep + (ui + E) * p) + (len(V.T) * 2.0 ** -24 * np.abs(V).max() if ui else 0)
                tol["o"][:, :nq, h, b] = eo + u * np.abs(o)
                dp = V.T @ G
                delta = (p * dp).sum(0)
                ds = p * (dp - delta)
                edelta = (np.abs(G) * (eo + u * np.abs(o))).sum(0)
                exact = ep * np.abs(dp - delta) + p * (E * (np.abs(V).T @ np.abs(G)) + edelta) + E * np.abs(ds)  # of ds before it is rounded
                bound = 2 * np.sqrt((G ** 2).sum(0).max() * (V ** 2).sum(0).max()) if group == 1 else \
                    2 * np.sqrt((g[:, :nq, h // group * group:(h // group + 1) * group, b] ** 2).sum(0).max() * (V ** 2).sum(0).max())
                eds = exact + ui * np.abs(ds) + (2.0 ** -38 * bound if ui else 0)
                a = abs(self.scale)
                tol["dq"][:, :nq, h, b] += a * (np.abs(K) @ (eds + E * np.abs(ds)))
                tol["dk"][:, :nk, h // group, b] += a * (np.abs(Q) @ (eds + E * np.abs(ds)).T)
                tol["dv"][:, :nk, h // group, b] += np.abs(G) @ (ep + (ui + E) * p + (2.0 ** -37 if ui else 0)).T
                if self.table is not None:
                    np.add.at(tol["dtable"][:, h], kind, exact + E * np.abs(ds))
        for n in ("dq", "dk", "dv", "dtable"):
            if n in tol:
                tol[n] = tol[n] + u * np.abs(ref[n]) + 2.0 ** -25
        tol["o"] = tol["o"] + 2.0 ** -25
        return ref, tol


def compare(what, got, ref, tol):
    got = host(got)
    assert got.shape == ref.shape
    np.testing.assert_array_equal(np.isneginf(got), np.isneginf(ref), err_msg=what)
    fine = np.isfinite(ref)
    bad = ~(np.abs(got[fine] - ref[fine]) <= tol[fine] + 1e-30)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(np.abs(got[fine] - ref[fine]) / (tol[fine] + 1e-30)):.2f} x the bound"


def check(gb, c, accumulate=False):
    c.upload()
    c.forward(gb)
    ref, tol = c.reference()
    compare("o", c.O, ref["o"], tol["o"])
    compare("lse", c.L, ref["lse"], tol["lse"])
    c.backward(gb, accumulate)
    u = np.finfo(c.dt).eps / 2
    for n, got, old in (("dq", c.DQ, c.q), ("dk", c.DK, c.k), ("dv", c.DV, c.v), ("dtable", c.DT, c.table)):
        if got is None:
            continue
        r, t = ref[n], tol[n]
        if accumulate:
            r = r + old.astype(np.float64)
            t = t + u * np.abs(r) + u * np.abs(old)
        compare(n, got, r, t)
    return c


DT = [np.float32, np.float16]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hs,tq,tk", [(64, 1, 1), (64, 1, 200), (64, 5, 300), (64, 64, 64), (64, 128, 128), (64, 129, 127), (64, 300, 300), (64, 513, 130),
                                      (128, 128, 256), (128, 257, 257), (32, 100, 100), (16, 40, 70), (80, 150, 150), (96, 130, 140), (40, 200, 99),
                                      (57, 65, 66), (1, 9, 9), (192, 33, 140), (256, 20, 20), (64, 1, 2500), (128, 1100, 1100),
                                      (64, 300, 1500), (128, 700, 600), (120, 3, 3000), (72, 16, 900), (17, 2, 777), (64, 1300, 2100)])
def test_shapes(gpu, dt, causal, hs, tq, tk):
    check(gpu, Case(dt, hs, tq, tk, causal=causal, offsets=max(tk - tq, 0) if causal else 0))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads,kv", [(4, 1), (4, 2), (6, 3), (1, 1)])
def test_shared_heads(gpu, dt, heads, kv):
    check(gpu, Case(dt, 64, 150, 170, heads=heads, kv=kv, causal=True, offsets=20))
    check(gpu, Case(dt, 64, 1, 170, heads=heads, kv=kv, causal=True, offsets=169))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_and_offsets(gpu, dt, causal):
    """Ragged sequences, one of them empty, one full, lengths past the tensor; offsets per sequence,
    some so far ahead of the keys that rows stay empty."""
    check(gpu, Case(dt, 64, 200, 200, batch=5, causal=causal, q_lengths=[200, 0, 131, 1, 500], k_lengths=[200, 0, 131, 1, 128]))
    check(gpu, Case(dt, 64, 60, 300, batch=5, causal=causal, k_lengths=[300, 60, 0, 129, 7], offsets=[240, 0, -30, 69, -53]))
    check(gpu, Case(dt, 128, 1, 700, batch=4, heads=4, kv=2, causal=causal, k_lengths=[700, 1, 0, 513], offsets=[699, 0, -1, 512]))
    check(gpu, Case(dt, 64, 40, 40, causal=causal, offsets=-25))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hs", [64, 128])
def test_one_sequence_against_a_long_cache(gpu, dt, hs):
    """More parts of the cache than one round of the join's threads, most of them behind the sequence's end in the
    second case."""
    check(gpu, Case(dt, hs, 1, 20000, heads=2, kv=1, batch=1, causal=True, offsets=19999))
    check(gpu, Case(dt, hs, 2, 9000, heads=4, kv=1, batch=1, k_lengths=[100]))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("pad,order", [(0, (3, 1, 2)), (8, (3, 2, 1)), (0, (2, 3, 1)), (3, (3, 2, 1)), (1, (1, 2, 3))])
def test_orders_and_strides(gpu, dt, pad, order):
    """Heads side by side within a token, padded tokens (aligned and not), batch inside the heads, time
    outermost."""
    check(gpu, Case(dt, 64, 140, 150, heads=3, batch=3, pad=pad, order=order), accumulate=True)
    check(gpu, Case(dt, 64, 140, 140, heads=3, batch=2, pad=pad, order=order, q_lengths=[140, 100], k_lengths=[130, 100], causal=True))


@pytest.mark.parametrize("dt", DT)
def test_accumulation_and_partial_results(gpu, dt):
    check(gpu, Case(dt, 64, 200, 140, heads=4, kv=2), accumulate=True)
    c = check(gpu, Case(dt, 64, 200, 140))
    full = [x.clone() for x in (c.DQ, c.DK, c.DV, c.DT)]
    for i, name in enumerate(("dq", "dk", "dv", "dtable")):
        out = torch.empty_like(full[i])
        gpu.relative_attention_backward(c.Q, c.K, c.V, c.T, c.M, c.O, c.L, c.DO, accumulate=False, **{name: out}, **c.kw)
        assert torch.equal(out, full[i]), name


@pytest.mark.parametrize("dt", DT)
def test_bias_of_other_kinds(gpu, dt):
    """No table; a bucket for every distance; reach of zero; a map with buckets that do not exist; entries of
    the type's lowest value and of -inf."""
    check(gpu, Case(dt, 64, 150, 150, table=False, causal=True))
    check(gpu, Case(dt, 64, 150, 150, buckets=64, reach=500))
    check(gpu, Case(dt, 64, 150, 150, buckets=4, reach=0))
    c = Case(dt, 64, 300, 300, reach=200)
    c.map = c.map.clone()
    c.map[150:170] = -1
    c.map[230:240] = 32
    c.upload()
    c.forward(gpu)
    table = c.table
    wide = np.concatenate([table, np.zeros((1, table.shape[1]), table.dtype)])
    m = c.map.numpy().copy()
    m[(m < 0) | (m > 31)] = 32
    ref = Case(dt, 64, 300, 300, reach=200)
    ref.table, ref.map = wide, torch.from_numpy(m)
    r, t = ref.reference()
    compare("o", c.O, r["o"], t["o"])
    c.backward(gpu)
    compare("dtable", c.DT, r["dtable"][:32], t["dtable"][:32])
    compare("dk", c.DK, r["dk"], t["dk"])
    for low in (np.finfo(dt).min, -np.inf):
        c = Case(dt, 64, 200, 200, heads=2, reach=40)
        c.table[5:9] = low  # some distances are as good as masked
        if np.isinf(low):
            c.upload()
            c.forward(gpu)
            r, t = orc.relative_attention(c.q, c.k, c.v, c.table, c.map.numpy(), c.scale, d_o=c.d_o), None
            c2 = Case(dt, 64, 200, 200, heads=2, reach=40)
            c2.table[5:9] = -60000  # what the bounds are taken from: as far from mattering
            _, t = c2.reference()
            compare("o", c.O, r["o"], t["o"])
            c.backward(gpu)
            for n, got in (("dq", c.DQ), ("dk", c.DK), ("dv", c.DV), ("dtable", c.DT)):
                compare(n, got, r[n], t[n])
        else:
            c.table = np.maximum(c.table, np.asarray(-60000, dt))  # scores stay finite in 32 bits
            check(gpu, c)


@pytest.mark.parametrize("dt", DT)
def test_what_lies_behind_the_lengths_is_not_looked_at(gpu, dt):
    """NaN and infinities in q, k, v and d_o behind the sequences' ends change nothing; o and the gradients are
    zero there."""
    c = Case(dt, 64, 200, 200, batch=3, heads=4, kv=2, q_lengths=[200, 77, 129], k_lengths=[150, 77, 1])
    for b, (nq, nk) in enumerate(zip(c.q_lengths, c.k_lengths)):
        c.q[:, nq:, :, b] = np.nan
        c.d_o[:, nq:, :, b] = np.inf
        c.k[:, nk:, :, b] = np.nan
        c.v[:, nk:, :, b] = -np.inf
    check(gpu, c)
    for b, (nq, nk) in enumerate(zip(c.q_lengths, c.k_lengths)):
        assert (c.O[:, nq:, :, b] == 0).all() and (c.DQ[:, nq:, :, b] == 0).all()
        assert (c.DK[:, nk:, :, b] == 0).all() and (c.DV[:, nk:, :, b] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hs,tq,tk,offsets", [(64, 40, 300, [100, 3, -20]), (128, 1, 700, [500, 0, -1]), (192, 20, 50, [10, 25, 0]),
                                              (128, 130, 200, 50)])
def test_keys_that_no_query_sees_yet_are_not_looked_at(gpu, dt, hs, tq, tk, offsets):
    """A causal pass over a cache that is filled so far: what lies behind the last query's position may be
    anything, and takes no gradient."""
    c = Case(dt, hs, tq, tk, batch=3, heads=4, kv=2, causal=True, offsets=offsets)
    last = [max(0, min(tk, o + tq)) for o in ([offsets] * 3 if isinstance(offsets, int) else offsets)]
    for b, n in enumerate(last):
        c.k[:, n:, :, b] = np.nan
        c.v[:, n:, :, b] = -np.inf
    check(gpu, c)
    for b, n in enumerate(last):
        assert (c.DK[:, n:, :, b] == 0).all() and (c.DV[:, n:, :, b] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hs,tq,tk", [(64, 200, 300), (128, 150, 150), (64, 1, 500), (160, 20, 30)])
def test_negative_and_zero_scale(gpu, dt, hs, tq, tk):
    """A negative scale is the positive one with q negated, which is exact; a scale of zero leaves the bias."""
    c = Case(dt, hs, tq, tk, causal=True, offsets=tk - tq)
    ref, tol = c.reference()
    c.q = -c.q
    c.upload()
    c.kw["scale"] = -c.scale
    c.forward(gpu)
    c.backward(gpu)
    compare("o", c.O, ref["o"], tol["o"])
    compare("dq", c.DQ, -ref["dq"], tol["dq"])
    for n, got in (("dk", c.DK), ("dv", c.DV), ("dtable", c.DT)):
        compare(n, got, ref[n], tol[n])
    c = Case(dt, hs, tq, tk, causal=True, offsets=tk - tq)
    c.scale = 0.0
    check(gpu, c)
    assert (c.DQ == 0).all() and (c.DK == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hs,tq,tk", [(64, 40, 300), (128, 1, 700), (192, 20, 50)])
def test_what_is_not_a_number_stays_one(gpu, dt, hs, tq, tk):
    """A key that is not a number reaches every query that sees it, in o, lse and dq; a query that is not one
    only its own.  Nothing is turned into zeros on the way."""
    c = Case(dt, hs, tq, tk, heads=2, kv=2, batch=2)
    c.k[:, tk // 3, 1, 0] = np.nan
    c.q[:, 0, 0, 1] = np.nan
    c.upload()
    c.forward(gpu)
    c.backward(gpu)
    ref, tol = c.reference()
    o, lse, dq = host(c.O), host(c.L), host(c.DQ)
    assert np.isnan(o[:, :, 1, 0]).all() and np.isnan(lse[0, 1]).all() and np.isnan(dq[:, :, 1, 0]).all()
    assert np.isnan(o[:, 0, 0, 1]).all() and np.isnan(lse[1, 0, 0]) and np.isnan(dq[:, 0, 0, 1]).all()
    compare("o", c.O[:, :, 0, 0], ref["o"][:, :, 0, 0], tol["o"][:, :, 0, 0])
    compare("o", c.O[:, 1:, 0, 1], ref["o"][:, 1:, 0, 1], tol["o"][:, 1:, 0, 1])
    compare("dq", c.DQ[:, :, 0, 0], ref["dq"][:, :, 0, 0], tol["dq"][:, :, 0, 0])


@pytest.mark.parametrize("dt", DT)
def test_no_keys_and_no_queries(gpu, dt):
    c = Case(dt, 64, 30, 30).upload()
    none_k, none_q = c.K[:, :0], c.Q[:, :0]
    gpu.relative_attention_forward(c.Q, none_k, none_k, c.T, c.M, c.O, c.L, scale=1.0)
    assert (c.O == 0).all() and torch.isneginf(c.L).all()
    for accumulate in (True, False):
        dq, dt_ = torch.ones_like(c.Q), torch.ones_like(c.T)
        gpu.relative_attention_backward(c.Q, none_k, none_k, c.T, c.M, c.O, c.L, c.DO, dq=dq, dtable=dt_, accumulate=accumulate)
        assert (dq == accumulate).all() and (dt_ == accumulate).all()
        dk = torch.ones_like(c.K)
        gpu.relative_attention_backward(none_q, c.K, c.V, c.T, c.M, none_q, c.L[:, :, :0].contiguous(), none_q, dk=dk, accumulate=accumulate)
        assert (dk == accumulate).all()


@pytest.mark.parametrize("dt", DT)
def test_peaked_and_large_scores(gpu, dt):
    """Scores of several tens: the running maximum moves, most probabilities vanish."""
    check(gpu, Case(dt, 64, 400, 700, spread_scores=20.0))
    c = Case(dt, 64, 300, 900, spread_scores=3.0, causal=True, offsets=600)
    c.k = np.sort(c.k, axis=1)  # scores grow along the keys for queries of one sign: a new maximum in every tile
    check(gpu, c)


@pytest.mark.parametrize("size", [2.0 ** -16, 2.0 ** 9])
def test_half_gradients_of_extreme_size(gpu, size):
    """Upstream gradients whose products with v leave a Half's normal range on either side."""
    c = Case(np.float16, 64, 300, 600)
    c.d_o = (c.d_o * np.float16(size)).astype(np.float16)
    c.upload()
    c.forward(gpu)
    c.backward(gpu)
    ref, tol = c.reference()
    for n, got in (("dq", c.DQ), ("dk", c.DK), ("dv", c.DV), ("dtable", c.DT)):
        compare(n, got, ref[n], tol[n])


@pytest.mark.parametrize("dt", DT)
def test_gradient_against_differences(gpu, dt):
    """The kernels' own forward pass, moved along the kernels' own gradient in a direction of each operand."""
    c = Case(np.float32, 32, 60, 70, causal=True, offsets=10, spread_scores=0.7) if dt == np.float32 else Case(np.float16, 64, 60, 70, spread_scores=0.7)
    c.upload()
    c.forward(gpu)
    c.backward(gpu)
    rng = np.random.default_rng(1)
    loss = lambda: float((c.O.double() * c.DO.double()).sum())  # noqa: E731
    # step and bound: truncation ~ step^2; rounding of o (u per element, 2 x 60 x 64 independent ones) / step
    step, tol = (0.02, 2e-3) if dt == np.float32 else (0.1, 2e-2)
    for X, G in ((c.Q, c.DQ), (c.K, c.DK), (c.V, c.DV), (c.T, c.DT)):
        way = torch.from_numpy(rng.standard_normal(tuple(X.shape))).cuda()
        way = (way / way.norm() * step * X.numel() ** 0.5 / 4).to(X.dtype)
        old = X.clone()
        X.copy_(old + way)
        up = X.double() - old.double()
        c.forward(gpu)
        hi = loss()
        X.copy_(old - way)
        down = old.double() - X.double()
        c.forward(gpu)
        lo = loss()
        X.copy_(old)
        want = float((G.double() * (up + down)).sum())
        scale = float(G.double().norm() * (up + down).norm())
        assert abs((hi - lo) - want) < tol * scale + (0 if dt == np.float32 else 0.3), (hi - lo, want, scale)


@pytest.mark.parametrize("dt", DT)
def test_results_do_not_depend_on_the_run(gpu, dt):
    c = Case(dt, 64, 260, 300, heads=4, kv=2, batch=3, causal=True).upload()
    seen = []
    for _ in range(4):
        c.forward(gpu)
        c.backward(gpu)
        seen.append([x.clone() for x in (c.O, c.L, c.DQ, c.DK, c.DV, c.DT)])
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


@pytest.mark.parametrize("dt", DT)
def test_captured_pass_and_two_streams(gpu, dt):
    """Forward and backward in a CUDA graph, two graphs replayed side by side, new inputs in place."""
    cases, graphs, streams = [Case(dt, 64, 200, 200, seed=s, causal=True) for s in (1, 2)], [], [torch.cuda.Stream() for _ in range(2)]
    for c in cases:
        c.upload()
        c.forward(gpu)
        c.backward(gpu)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.forward(gpu)
            c.backward(gpu)
        graphs.append(g)
    for turn in range(2):
        for c in cases:
            other = Case(dt, 64, 200, 200, seed=10 + turn, causal=True)
            c.q, c.k, c.d_o = other.q, other.k, other.d_o
            for X, x in ((c.Q, c.q), (c.K, c.k), (c.DO, c.d_o)):
                X.copy_(torch.from_numpy(x))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for c in cases:
            ref, tol = c.reference()
            for n, got in (("o", c.O), ("dq", c.DQ), ("dk", c.DK), ("dv", c.DV), ("dtable", c.DT)):
                compare(n, got, ref[n], tol[n])


def test_cache_past_32_bits(gpu):
    """One token against a Half cache of 4.4e9 elements: the last head of the last sequence lies behind element
    2^32."""
    hs, tk, kv, batch = 128, 1 << 15, 8, 131
    k = torch.zeros((batch, kv, tk, hs), dtype=torch.float16, device="cuda")
    v = torch.zeros((batch, kv, tk, hs), dtype=torch.float16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for b in (0, batch - 1):
        k[b].normal_(generator=gen)
        v[b].normal_(generator=gen)
    K, V = k.permute(3, 2, 1, 0), v.permute(3, 2, 1, 0)
    Q = torch.randn((batch, kv, 1, hs), generator=gen, device="cuda").half().permute(3, 2, 1, 0)
    O, L = torch.empty_like(Q), torch.empty(batch * kv, device="cuda")
    gpu.relative_attention_forward(Q, K, V, None, None, O, L, scale=hs ** -0.5, causal=True, q_offset=tk - 1)
    for b in (0, batch - 1):
        s = (k[b].double() @ Q[:, 0, :, b].t().double()[:, :, None]).squeeze(2) * float(np.float32(hs ** -0.5))
        p = torch.softmax(s, 1)
        o = (p[:, None] @ v[b].double()).squeeze(1)
        tol = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -13) * (p[:, None] @ v[b].double().abs()).squeeze(1) + tk * 2.0 ** -24
        assert ((O[:, 0, :, b].t().double() - o).abs() <= tol).all(), b
    assert (O[:, :, :, 1] == 0).all()


def test_a_transformer_block_end_to_end(gpu):
    """residual -> norm -> attention -> residual norm, forward and backward, as they are used together:
    x1 = norm(x); a = attention(x1 as q, k, v); h = x + drop(a); y = norm(h); the gradient of sum(y * w) with
    respect to x, the gains and the table against differences of the fp64 oracle's loss."""
    hs, t, heads, batch = 16, 20, 2, 2
    rows, cols = hs * heads, t * batch
    rng = np.random.default_rng(2)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    g1, g2, b1, b2 = (rng.standard_normal(rows).astype(np.float32) for _ in range(4))
    table, w = rng.standard_normal((8, heads)).astype(np.float32), rng.standard_normal((rows, cols)).astype(np.float32)
    bmap = B.relative_buckets(8, 16, False, 16)
    rnd = dict(p=0.25, seed=11, offset=4)
    mask = orc.dropout_mask(rows, cols, **rnd)
    four = lambda m: m.reshape(hs, heads, t, batch, order="F").transpose(0, 2, 1, 3)  # noqa: E731
    flat = lambda a: a.transpose(0, 2, 1, 3).reshape(rows, cols, order="F")  # noqa: E731

    def loss(x, g1, g2, table):
        x1 = four(orc.layer_norm_forward(x, g1, b1)[0])
        a = flat(orc.relative_attention(x1, x1, x1, table, bmap.numpy(), 0.25, causal=True)["o"])
        return float((orc.layer_norm_forward(x + a * mask, g2, b2)[0] * w).sum())

    X, G1, G2, B1, B2, W = (B.from_host(a) for a in (x, g1, g2, b1, b2, w))
    T, M = B.from_host(table), bmap.cuda()
    new = lambda: B.colmajor(rows, cols, torch.float32)  # noqa: E731
    view = lambda m: torch.as_strided(m, (hs, t, heads, batch), (1, rows, hs, rows * t))  # noqa: E731
    X1, A, H, Y, DA, DX, DX1 = (new() for _ in range(7))
    M1, R1, M2, R2 = (torch.empty(cols, device="cuda") for _ in range(4))
    L = torch.empty(t * heads * batch, device="cuda")
    gpu.layer_norm_forward(X, G1, B1, X1, M1, R1)
    gpu.relative_attention_forward(view(X1), view(X1), view(X1), T, M, view(A), L, scale=0.25, causal=True)
    gpu.residual_norm_forward(A, X, G2, B2, H, Y, M2, R2, **rnd)
    DG1, DB1, DG2, DB2 = (torch.zeros(rows, device="cuda") for _ in range(4))
    DT = torch.zeros_like(T)
    gpu.residual_norm_backward(H, G2, M2, R2, W, None, DA, DX, DG2, DB2, accumulate=False, **rnd)
    DX1.zero_()
    for name in ("dq", "dk", "dv"):  # q, k and v are one tensor: their gradients add up in it
        gpu.relative_attention_backward(view(X1), view(X1), view(X1), T, M, view(A), L, view(DA), scale=0.25, causal=True,
                                        dtable=DT if name == "dq" else None, **{name: view(DX1)})
    gpu.layer_norm_backward(X, G1, M1, R1, DX1, DX, DG1, DB1)
    args = [x.astype(np.float64), g1.astype(np.float64), g2.astype(np.float64), table.astype(np.float64)]
    for at, got in ((0, DX), (1, DG1), (2, DG2), (3, DT)):
        got = host(got)
        for i in list(np.ndindex(args[at].shape))[::max(1, args[at].size // 40)]:
            e, side = 1e-5, []
            for sign in (1, -1):
                moved = [a.copy() for a in args]
                moved[at][i] += sign * e
                side.append(loss(*moved))
            want = (side[0] - side[1]) / (2 * e)
            # fp32 through four operators: 2^-17 of the gradient's size each; differences: 1e-7
            assert abs(got[i] - want) < 8 * E * (np.abs(got).max() + 1) + 1e-6, (at, i, got[i], want)
