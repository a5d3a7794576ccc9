"""The bound that attention of few rows is held to on a GPU tells 16 bits of a probability from 8: seen on the host, with probabilities cut off or rounded in the oracle's place."""
import math

import pytest
import torch

import paged_bits
import paged_oracle as O


def _cut(p):
    return (p.float().view(torch.int32) & -65536).view(torch.float32).to(O.F64)


def _rounded(p):
    return p.bfloat16().to(O.F64)


def _both(p):
    return _cut(p) + _rounded(p - _cut(p))


def _attention(c, weights):
    """The oracle's attention with probabilities, relative to the largest, as ``weights`` leaves them in front of the product; the divisor adds them up as they are."""
    K, V = c.pool(c.kpages), c.pool(c.vpages)
    q = c.q.to(O.F64).view(c.N, c.NH, c.HS)
    out, at = torch.zeros_like(q), 0
    for b, n in enumerate(c.new):
        for i in range(n):
            seen = c.flat[b][:c.keys[b] - n + i + 1]
            k, v = (x[seen].repeat_interleave(c.NH // c.NKV, 1) for x in (K, V))
            z = torch.einsum("hd,khd->hk", q[at + i], k) / math.sqrt(c.HS)
            p = torch.exp(z - z.amax(1, keepdim=True))
            out[at + i] = torch.einsum("hk,khd->hd", weights(p), v) / p.sum(1)[:, None]
        at += n
    return out.view(c.N, -1).bfloat16().to(O.F64)


@pytest.mark.parametrize("args", paged_bits.CASES)
def test_the_bound_sees_half_of_a_probability_missing(args):
    c = paged_bits.case(*args)
    exact, size = O.attention(c)
    bound = paged_bits.bound(c, exact, size)
    outside = lambda weights: int(((_attention(c, weights) - exact).abs() > bound).sum())
    assert outside(lambda p: p) == 0 and outside(_both) == 0
    assert outside(_cut) > 0 and outside(_rounded) > 0
