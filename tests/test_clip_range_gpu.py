"""Clipping of finite gradients whose squares fp32 does not hold (csrc/clip.cu) against 64 bits.

Bounds: as for other gradients; sums that leave fp32's range are formed in 64 bits, so they are off by less.  The norm: 20 * 2^-24 of its size; a result: 24 * 2^-24 and its own rounding
(2^-8 in bf16, 2^-24 in fp32)."""
import math

import pytest
import torch

from llmc_b200 import ops

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size,rest", [(1e20, 1.0), (1e20, 0.0), (1e37, 1e-30), (1.5e19, 1.5e19), (1e-25, 0.0), (1e-21, 1e-23), (1e-30, 1e-30), (3e-13, 0.0)])
def test_squares_out_of_range(dtype, size, rest):
    g = [torch.full((n,), rest, device="cuda").to(dtype) for n in (1, 70_001, 9, 4096)]
    g[1][123], g[2][8] = size, -size
    g[3][::7] = size
    want = math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in g))
    norm, out = torch.zeros(1, device="cuda"), [torch.zeros_like(t) for t in g]
    limit = 0.3 * want
    ops.clip_grad_norm(norm, ops.clip_plan(out, g), limit)
    assert abs(float(norm) - want) <= 20 * EPS * want
    tol = (24 * EPS + (2.0 ** -8 if dtype == torch.bfloat16 else EPS)) * 1.01
    for o, t in zip(out, g):
        assert ((o.double() - t.double() * 0.3).abs() <= tol * (t.double() * 0.3).abs() + 1e-40).all()


def test_zeros_and_signed_zeros():
    g = [torch.zeros(70_001, device="cuda"), -torch.zeros(5000, device="cuda").to(torch.bfloat16)]
    norm = torch.ones(1, device="cuda")
    ops.clip_grad_norm(norm, ops.clip_plan(None, g), 1.0)
    assert float(norm) == 0.0 and not g[0].any() and not g[1].any()
