"""Clipping by a plan that was made in another stream."""
import math

import pytest
import torch

from llmc_b200 import ops

pytestmark = pytest.mark.gpu


def test_a_plan_that_was_made_in_a_busy_stream():
    """The stream of the plan's making has work in front of it and behind it; a call in another stream does not wait for it.  Norm: 20 roundings of 2^-24 at most (fp32 sums of 32 squares)."""
    g = [torch.full((70_001,), 2.0, device="cuda"), torch.full((3,), 1.0, device="cuda")]
    out = [torch.zeros_like(t) for t in g]
    norm = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(1_000_000)
        plan = ops.clip_plan(out, g)
        torch.cuda._sleep(50_000_000)
    with torch.cuda.stream(b):
        for _ in range(3):
            ops.clip_grad_norm(norm, plan, 1.0)
    b.synchronize()
    want = math.sqrt(4.0 * 70_001 + 3)
    assert abs(float(norm) - want) <= 20 * 2.0 ** -24 * want
    assert all(((o.double() - t.double() / want).abs() <= 26 * 2.0 ** -24 * t.double() / want).all() for o, t in zip(out, g))
    a.synchronize()
