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


def heads(x):
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
    gpu.relative_attention_forward(heads(q), heads(k), heads(v), None, None, heads(o), lse, scale=0.125)
    for b in (0, batch // 2, batch - 1):
        s = 0.125 * (k[b, 0].double() @ q[b, 0, 0].double())
        ref = torch.softmax(s, 0) @ v[b, 0].double()
        off = (o[b, 0, 0].double() - ref).abs() / ref
        assert (off <= E + 2.0 ** -19).all(), float(off.max())
        assert abs(float(lse[b]) - float(torch.logsumexp(s, 0))) <= E * math.log(tk)
