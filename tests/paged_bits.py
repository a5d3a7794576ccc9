"""How far attention of few query rows over a cache in pages may be from 64 bits, and calls that its kernel takes (at most 16 rows of a sequence and cached head on average)."""
import math

import torch

import paged_oracle as O

# keys and new tokens of the sequences, query and cached heads, channels: groups of 8 rows by blocks and by warps, of 16 rows by blocks and by warps; tables of at most 256 keys, whose pieces are not cut
CASES = [((161,), (1,), 32, 8, 64), ((1500,), (1,), 8, 2, 128), ((33, 700, 256), (1, 1, 1), 6, 2, 96), (tuple(300 - i % 60 for i in range(100)), (1,) * 100, 8, 8, 128),
         (tuple(400 - 17 * i for i in range(20)), (1,) * 20, 12, 12, 64), ((900,), (3,), 8, 2, 128), ((250, 40), (7, 2), 4, 2, 64), (tuple(500 - 20 * i for i in range(20)), (12,) * 20, 12, 12, 64)]


def case(keys, new, NH, NKV, HS, device="cpu"):
    assert sum(new) * (NH // NKV) <= 16 * len(keys)
    c = O.Case(keys, new, NH, NKV, HS, 16, seed=len(keys) + HS, device=device, pad=0)
    c.q *= 2                                             # a few keys of a row have most of the weight, so that roundings of probabilities do not average out
    return c


def bound(c, exact, size):
    """The result's rounding; sum |p v| times what a probability and the sums are off by, relative to themselves:
    a score, in units of the exponent, is added up in HS / 16 steps and scaled, each of which rounds by at most 2^-23 of sum |q k| / sqrt(HS), and its exponential is off by 2^-22: twice, in the
    sum and in its divisor; the upper 8 bits of a probability leave less than 2^-7 of it, of which the lower 8 leave half a step, 2^-9: 2^-16;
    sums of 32 bits over the tiles of 16 keys, their parts and their divisor, 2^-23 a step."""
    q, K = c.q.to("cpu", O.F64).view(c.N, c.NH, c.HS).abs(), c.pool(c.kpages).nan_to_num(0.0).abs()
    most = 0.0
    at = 0
    for f, n in zip(c.flat, c.new):
        k = K[f].repeat_interleave(c.NH // c.NKV, 1)
        most = max(most, float(torch.einsum("nhd,khd->nhk", q[at:at + n], k).max()) / math.sqrt(c.HS))
        at += n
    score = (c.HS / 16 + 3) * 2.0 ** -23 * most + 2.0 ** -22
    steps = max(c.keys) / 16 + 16
    return 2.0 ** -8 * exact.abs() + (2 * score + 2.0 ** -16 + 2 * steps * 2.0 ** -23) * size
