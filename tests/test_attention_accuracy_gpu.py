"""Attention with operands whose sums do not cancel: values of one sign, and queries, keys, values and gradients with
a mean of their own.  Sums of such terms show a bias in how they are added, and gradients what is left of scores'
gradients that should add up to nothing; operands with mean zero hide both.

Bounds.  Products: 2^-17 of the product of the magnitudes, the bound of the other attention tests (22 bits of each
fp32 operand, fp32 accumulation).  Gradients behind the softmax, as a whole (Frobenius): 1e-5 for fp32, what every
fp32 product of this library keeps; 4 u for Half, u = 2^-11: the roundings of the probabilities, of the scores'
gradient and of the result, the second one enlarged by |k| / |k - mean|, which is sqrt(2) here."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -17


def heads_of(x):
    """(batch, heads, t, hs) in memory as the calls' (hs, t, heads, batch)."""
    return x.permute(3, 2, 1, 0)


def randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


@pytest.mark.parametrize("tk,batch", [(4096, 1184), (1000, 1184), (16384, 400)])
def test_fp32_tokens_of_many_sequences(gpu, tk, batch):
    """So many sequences that the caches need no parts to fill the device: the sums of a long cache are cut all the
    same.  Scores are so small (|q| |k| scale < 1/2) that their errors are below 2^-22, an exponential's is 2^-22
    and its argument's rounding 2^-24: a probability and their sum are off by 2^-20 each at most, 2^-19 in all."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    hs = 16
    q, k, v = 0.05 * randn(gen, batch, 1, 1, hs), randn(gen, batch, 1, tk, hs), randn(gen, batch, 1, tk, hs).abs_() + 0.5
    o, lse = torch.empty_like(q), torch.empty(batch, device="cuda")
    gpu.relative_attention_forward(heads_of(q), heads_of(k), heads_of(v), None, None, heads_of(o), lse, scale=0.125)
    for b in (0, batch // 2, batch - 1):
        s = 0.125 * (k[b, 0].double() @ q[b, 0, 0].double())
        ref = torch.softmax(s, 0) @ v[b, 0].double()
        off = (o[b, 0, 0].double() - ref).abs() / ref
        assert (off <= E + 2.0 ** -19).all(), float(off.max())
        assert abs(float(lse[b]) - float(torch.logsumexp(s, 0))) <= E * math.log(tk)


class Operands:
    """Heads of hs elements with a mean of `shift`, and what the definition makes of them in 64 bits."""

    def __init__(self, dtype, hs, tq, tk, heads=2, kv=2, batch=1, causal=False, shift=1.0, small=1.0, pad=0, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed + hs + tq + tk)
        new = lambda n, t, s: (s * (randn(gen, batch, n, t, hs + pad) + shift)).to(dtype)[..., :hs]  # noqa: E731
        self.q, self.k, self.v, self.d_o = new(heads, tq, small), new(kv, tk, 1), new(kv, tk, 1), new(heads, tq, 1)
        self.o, self.dq = torch.empty_like(self.q), torch.empty_like(self.q)
        self.dk, self.dv = torch.empty_like(self.k), torch.empty_like(self.v)
        self.lse = torch.empty(batch, heads, tq, device="cuda")
        self.scale = float(torch.tensor(hs ** -0.5))
        self.causal, self.offset = causal, tk - tq if causal else 0

    def forward(self, gb):
        gb.relative_attention_forward(heads_of(self.q), heads_of(self.k), heads_of(self.v), None, None, heads_of(self.o), self.lse, scale=self.scale,
                                      causal=self.causal, q_offset=self.offset)

    def backward(self, gb, accumulate=False):
        gb.relative_attention_backward(heads_of(self.q), heads_of(self.k), heads_of(self.v), None, None, heads_of(self.o), self.lse, heads_of(self.d_o),
                                       heads_of(self.dq), heads_of(self.dk), heads_of(self.dv), scale=self.scale, causal=self.causal,
                                       q_offset=self.offset, accumulate=accumulate)

    def reference(self):
        """(results, products of the magnitudes); the probabilities are taken as they are."""
        q, k, v, g = (x.double() for x in (self.q, self.k, self.v, self.d_o))
        n = q.shape[1] // k.shape[1]
        K, V = k.repeat_interleave(n, 1), v.repeat_interleave(n, 1)
        s = self.scale * (q @ K.transpose(2, 3))
        if self.causal:
            i, j = torch.arange(q.shape[2], device="cuda")[:, None], torch.arange(k.shape[2], device="cuda")
            s = s.masked_fill(j > i + self.offset, -math.inf)
        p = torch.softmax(s, 3)
        dp = g @ V.transpose(2, 3)
        ds = p * (dp - (p * dp).sum(3, keepdim=True))
        shared = lambda x: x.unflatten(1, (k.shape[1], n)).sum(2)  # noqa: E731
        return (dict(o=p @ V, dq=self.scale * ds @ K, dk=self.scale * shared(ds.transpose(2, 3) @ q), dv=shared(p.transpose(2, 3) @ g)),
                dict(o=p @ V.abs(), dv=shared(p.transpose(2, 3) @ g.abs())))


def elementwise(name, got, ref, size, bound):
    off = ((got.double() - ref).abs() / size).max()
    assert off <= bound, (name, float(off), bound)


# scores below 1/2 as above: 2^-19 for the probabilities
SMALL = E + 2.0 ** -19


@pytest.mark.parametrize("hs,tq,tk,heads,kv,causal,pad", [
    (64, 100, 512, 2, 2, False, 0), (64, 40, 513, 2, 2, False, 0), (64, 300, 1024, 4, 2, True, 0), (57, 20, 1537, 2, 1, True, 0), (64, 130, 4096, 2, 2, False, 4),
    (61, 33, 2050, 1, 1, False, 1), (128, 200, 3000, 2, 2, False, 0), (128, 140, 1100, 2, 1, True, 0), (16, 1500, 1500, 1, 1, True, 0)])
def test_fp32_sums_of_values_of_one_sign(gpu, hs, tq, tk, heads, kv, causal, pad):
    c = Operands(torch.float32, hs, tq, tk, heads, kv, causal=causal, shift=0.0, small=0.05, pad=pad)
    c.v.abs_().add_(0.5)
    c.forward(gpu)
    ref, size = c.reference()
    elementwise("o", c.o, ref["o"], size["o"], SMALL)


@pytest.mark.parametrize("hs,tq,tk", [(64, 70, 1500), (128, 40, 2100), (40, 200, 1024)])
def test_fp32_rows_that_see_little_of_the_first_keys(gpu, hs, tq, tk):
    """A bias of -inf behind a distance: whole chains of keys in which a row sees nothing, then some, its maximum
    moving in every tile; rows that see nothing at all."""
    c = Operands(torch.float32, hs, tq, tk, shift=0.0)
    c.v.abs_().add_(0.5)
    reach, near = 1200, 300
    d = torch.arange(-reach, reach + 1, device="cuda")
    bucket = torch.where(d < -near, 1, 0).to(torch.int32)
    table = torch.tensor([[0.25, 0.5], [-math.inf, -math.inf]], device="cuda").t().contiguous().t()
    ramp = torch.linspace(0, 30, tk, device="cuda")[None, None, :, None]
    c.k = c.k + ramp * 0.2 * c.q[:, :, :1].sign()
    for offset in (tk - tq, tk + near - tq // 2):
        gpu.relative_attention_forward(heads_of(c.q), heads_of(c.k), heads_of(c.v), table, bucket, heads_of(c.o), c.lse, scale=c.scale, q_offset=offset)
        s = c.scale * (c.q.double() @ c.k.double().transpose(2, 3))
        size = c.scale * (c.q.double().abs() @ c.k.double().abs().transpose(2, 3))
        far = torch.arange(tk, device="cuda")[None, :] - torch.arange(tq, device="cuda")[:, None] - offset < -near
        s = torch.where(far, -math.inf, s + table[0].double()[None, :, None, None])
        seen = ~far.all(1)
        assert bool(seen.any()) and bool(seen.all()) == (offset == tk - tq)
        p = torch.softmax(s[:, :, seen], 3)
        es = E * (size.max() + 1)  # of a score, relative of a probability; its sum's error as much again
        elementwise("o", c.o[:, :, seen], p @ c.v.double(), p @ c.v.double(), 2 * es + E)
        assert (c.o[:, :, ~seen] == 0).all() and torch.isneginf(c.lse[:, :, ~seen]).all()


def frobenius(name, got, ref, bound):
    off = float((got.double() - ref).norm() / ref.norm())
    assert off <= bound, (name, off, bound)


@pytest.mark.parametrize("hs,tq,tk,heads,kv,causal,pad", [
    (64, 1024, 200, 1, 1, False, 0), (64, 1025, 200, 2, 2, False, 0), (64, 300, 300, 8, 2, True, 0), (57, 2100, 130, 1, 1, True, 0), (64, 4096, 150, 1, 1, False, 4),
    (64, 130, 2500, 2, 1, False, 0), (61, 700, 1100, 3, 1, True, 1), (128, 1500, 300, 2, 2, False, 0), (128, 150, 2049, 2, 1, True, 0), (128, 500, 500, 4, 1, False, 0)])
def test_fp32_sums_of_gradients_of_one_sign(gpu, hs, tq, tk, heads, kv, causal, pad):
    """d_o of one sign against dv, and random ones over more terms than a chain holds, the results taken anew and added
    to."""
    c = Operands(torch.float32, hs, tq, tk, heads, kv, causal=causal, shift=0.0, small=0.05, pad=pad)
    if causal:  # a first row that sees one key, rather than the last ones only
        c.offset = 0 if tk <= tq else c.offset
    c.d_o.abs_().add_(0.5)
    c.forward(gpu)
    c.backward(gpu)
    ref, size = c.reference()
    elementwise("dv", c.dv, ref["dv"], size["dv"] + 1e-30, SMALL)
    c.d_o.copy_(randn(torch.Generator(device="cuda").manual_seed(2), *c.d_o.shape))
    ref, _ = c.reference()
    old = {}
    for accumulate in (False, True):
        c.backward(gpu, accumulate)
        for n in ("dq", "dk", "dv"):
            got = getattr(c, n)
            frobenius(n, got - old[n] if accumulate else got, ref[n], 1e-5)
            old[n] = got.clone()


@pytest.mark.parametrize("hs,tq,tk,heads,kv,causal", [
    (64, 64, 64, 2, 2, False), (64, 128, 128, 2, 2, False), (64, 256, 256, 8, 8, True), (64, 300, 512, 4, 2, False), (128, 256, 256, 2, 2, False),
    (128, 500, 500, 2, 1, True), (57, 90, 200, 3, 3, False), (16, 40, 1024, 2, 2, True)])
def test_fp32_gradients_of_operands_with_a_mean(gpu, hs, tq, tk, heads, kv, causal):
    """A row's score gradients add up to zero; keys with a mean show what is left of that."""
    c = Operands(torch.float32, hs, tq, tk, heads, kv, causal=causal, shift=1.0)
    c.forward(gpu)
    c.backward(gpu)
    ref, _ = c.reference()
    for n in ("o", "dq", "dk", "dv"):
        frobenius(n, getattr(c, n), ref[n], 1e-5)


@pytest.mark.parametrize("hs,tq,tk,heads,kv,causal", [
    (64, 64, 64, 2, 2, False), (64, 300, 300, 4, 2, False), (64, 200, 600, 4, 4, True), (128, 512, 512, 2, 1, True), (57, 90, 900, 3, 3, False),
    (64, 2048, 2048, 2, 2, False), (128, 300, 4096, 1, 1, False)])
def test_half_gradients_of_operands_with_a_mean(gpu, hs, tq, tk, heads, kv, causal):
    c = Operands(torch.float16, hs, tq, tk, heads, kv, causal=causal, shift=1.0)
    c.forward(gpu)
    c.backward(gpu)
    ref, _ = c.reference()
    for n in ("o", "dq", "dk", "dv"):
        frobenius(n, getattr(c, n), ref[n], 4 * 2.0 ** -11)
    dq, dk = c.dq.clone(), c.dk.clone()
    for out in ("dq", "dk"):  # a result does not depend on which others are wanted
        new = torch.empty_like(getattr(c, out))
        gpu.relative_attention_backward(heads_of(c.q), heads_of(c.k), heads_of(c.v), None, None, heads_of(c.o), c.lse, heads_of(c.d_o), scale=c.scale,
                                        causal=c.causal, q_offset=c.offset, accumulate=False, **{out: heads_of(new)})
        assert torch.equal(new, dq if out == "dq" else dk)


@pytest.mark.parametrize("hs,t,heads", [(64, 900, 2), (64, 2100, 1), (128, 1500, 1)])
def test_fp32_sums_that_begin_with_their_largest_terms(gpu, hs, t, heads):
    """The first keys of a causal sequence get 1, 1/2, 1/3 .. of its rows' gradients: nearly every addition of a chain is
    made to a sum of its full size."""
    c = Operands(torch.float32, hs, t, t, heads, heads, causal=True, shift=0.0, small=0.05)
    c.d_o.abs_().add_(0.5)
    c.forward(gpu)
    c.backward(gpu)
    ref, size = c.reference()
    elementwise("dv", c.dv, ref["dv"], size["dv"], SMALL)


@pytest.mark.parametrize("hs,tq,tk,heads,kv,causal", [(64, 100, 8192, 2, 1, False), (128, 40, 5000, 1, 1, True), (64, 4097, 100, 1, 1, False),
                                                      (57, 2100, 150, 4, 2, True), (128, 4500, 4500, 1, 1, True)])
def test_fp32_sums_of_long_sequences(gpu, hs, tq, tk, heads, kv, causal):
    c = Operands(torch.float32, hs, tq, tk, heads, kv, causal=causal, shift=0.0, small=0.05)
    c.offset = 0 if tk <= tq else c.offset
    c.v.abs_().add_(0.5)
    c.d_o.abs_().add_(0.5)
    c.forward(gpu)
    c.backward(gpu)
    ref, size = c.reference()
    elementwise("o", c.o, ref["o"], size["o"], SMALL)
    elementwise("dv", c.dv, ref["dv"], size["dv"] + 1e-30, SMALL)
    for x in (c.v, c.d_o):
        x.copy_(randn(torch.Generator(device="cuda").manual_seed(3), *x.shape))
    c.forward(gpu)
    c.backward(gpu)
    ref, _ = c.reference()
    for n in ("o", "dq", "dk", "dv"):
        frobenius(n, getattr(c, n), ref[n], 1e-5)


@pytest.mark.parametrize("hs,t,tk,heads,kv,causal,span", [(64, 40, 40, 2, 2, True, 30), (64, 200, 200, 4, 2, True, 24), (128, 130, 300, 2, 2, False, 24),
                                                          (57, 70, 70, 1, 1, True, 40)])
def test_fp32_tokens_of_very_different_size(gpu, hs, t, tk, heads, kv, causal, span):
    """Values and gradients of sizes over 2^span, in random order.  What the header promises: an element keeps 2^-39 of
    the largest of its sequence and key head at least, a probability 2^-32 of its row's largest, P in the backward pass 2^-38 and
    a score's gradient 2^-38 of 2 max|d_o row| max|v row|; above that 2^-17 of the terms' magnitudes."""
    c = Operands(torch.float32, hs, t, tk, heads, kv, causal=causal, shift=0.0, small=0.5)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for x in (c.v, c.d_o):
        x.mul_(2.0 ** torch.randint(0, span + 1, x.shape[:3] + (1,), generator=gen, device="cuda"))
    c.forward(gpu)
    c.backward(gpu)
    ref, size = c.reference()
    q, k, v, g = (x.double() for x in (c.q, c.k, c.v, c.d_o))
    n = heads // kv
    K, V = k.repeat_interleave(n, 1), v.repeat_interleave(n, 1)
    s = c.scale * (q @ K.transpose(2, 3))
    if causal:
        seen = torch.arange(tk, device="cuda") <= torch.arange(t, device="cuda")[:, None] + c.offset
        s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, 3)
    see = (p > 0).double()
    es = E * (c.scale * (q.abs() @ K.abs().transpose(2, 3)) + 1)
    ep = p * 2 * (es * see).amax(3, keepdim=True)  # the exponential and the sum it is divided by
    top = lambda x: x.abs().amax((2, 3), keepdim=True)  # noqa: E731
    shared = lambda x: x.unflatten(1, (kv, n)).sum(2)  # noqa: E731
    most_v, most_g = top(V), top(g).unflatten(1, (kv, n)).amax(2, keepdim=True).expand(-1, -1, n, -1, -1).flatten(1, 2)
    eo = (ep + E * p + 2.0 ** -32 * p.amax(3, keepdim=True) * see) @ V.abs() + 2.0 ** -39 * most_v
    assert ((c.o.double() - ref["o"]).abs() <= eo).all()
    dp = g @ V.transpose(2, 3)
    delta = (p * dp).sum(3, keepdim=True)
    ey = E * (g.abs() @ V.abs().transpose(2, 3)) + 2.0 ** -39 * (most_v * g.abs().sum(3, keepdim=True) + (most_g * V.abs().sum(3, keepdim=True)).transpose(2, 3))
    norm = lambda x: (x ** 2).sum(3).amax(2)[..., None, None].sqrt()  # noqa: E731
    bound = 2 * norm(g).unflatten(1, (kv, n)).amax(2, keepdim=True).expand(-1, -1, n, -1, -1).flatten(1, 2) * norm(V)
    eds = ep * (dp - delta).abs() + p * (ey + (p * ey + ep * dp.abs()).sum(3, keepdim=True)) + 2.0 ** -38 * bound * see
    eds = eds + E * (p * (dp - delta)).abs()
    ds = (p * (dp - delta)).abs()
    for name, ref_, tol in (("dq", ref["dq"], c.scale * (eds + E * ds) @ K.abs()), ("dk", ref["dk"], shared(c.scale * (eds + E * ds).transpose(2, 3) @ q.abs())),
                            ("dv", ref["dv"], shared((ep + E * p + 2.0 ** -38 * see).transpose(2, 3) @ g.abs() + 2.0 ** -39 * most_g * p.sum(2)[..., None]))):
        got = getattr(c, name).double()
        bad = ~((got - ref_).abs() <= tol)
        assert not bad.any(), (name, int(bad.sum()), float(((got - ref_).abs() / tol).max()))


@pytest.mark.parametrize("hs,t,heads,kv,causal", [(64, 40000, 2, 1, False), (128, 36000, 1, 1, False), (64, 33000, 1, 1, True), (57, 20000, 4, 2, False)])
def test_half_sums_of_one_sign_have_no_bias(gpu, hs, t, heads, kv, causal):
    """Roundings average out, truncation does not: 512 additions to a chain of 8192 terms truncate less than 2^-22 of its
    sum each, 2^-13 in all.  150 queries over t keys for o, 150 keys under t queries for dv.  Element by element three
    roundings of 2^-11 (P, the result and a margin) and, for results below a Half's normal range, 2^-14, half of the
    step of 2^-24 that they are rounded to: a key that one query among 33000 keys sees has a dv of 3e-5."""
    for tq, tk in ((150, t), (t, 150)):
        c = Operands(torch.float16, hs, tq, tk, heads, kv, causal=causal and tk > tq, shift=0.0, small=0.05)
        c.v.abs_().add_(0.5)
        c.d_o.abs_().add_(0.5)
        c.forward(gpu)
        c.backward(gpu)
        ref, size = c.reference()
        for n in ("o", "dv"):
            off = (getattr(c, n).double() - ref[n]) / size[n]
            assert abs(float(off.mean())) <= 2.0 ** -13, (n, float(off.mean()))
            left = (getattr(c, n).double() - ref[n]).abs() - 3 * 2.0 ** -11 * size[n]
            assert float(left.max()) <= 2.0 ** -25, (n, float(left.max()))
        for n in ("dq", "dk"):
            frobenius(n, getattr(c, n), ref[n], 4 * 2.0 ** -11)


def test_half_tokens_of_many_long_sequences_have_no_bias(gpu):
    """1184 caches of 131072 keys: parts of 32768 keys, 8192 to a warp."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    batch, tk, hs = 1184, 131072, 8
    q = (0.05 * randn(gen, batch, 1, 1, hs)).half()
    k, v = (torch.empty(batch, 1, tk, hs, dtype=torch.float16, device="cuda").normal_(generator=gen) for _ in "kv")
    v.abs_().add_(0.5)
    o, lse = torch.empty_like(q), torch.empty(batch, device="cuda")
    gpu.relative_attention_forward(heads_of(q), heads_of(k), heads_of(v), None, None, heads_of(o), lse, scale=0.25)
    off = []
    for b in range(0, batch, 9):
        ref = torch.softmax(0.25 * (k[b, 0].double() @ q[b, 0, 0].double()), 0) @ v[b, 0].double()
        off.append((o[b, 0, 0].double() - ref) / ref)
    off = torch.stack(off)  # 1056 results, rounded by 2^-11 at most: their mean by 2^-11 / sqrt(1056) = 2^-16
    assert abs(float(off.mean())) <= 2.0 ** -13 + 2.0 ** -15, float(off.mean())
    assert float(off.abs().max()) <= 3 * 2.0 ** -11
