"""Rows that are left out of the head's gradients may hold anything, on the host."""
import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("accumulate", [False, True])
def test_rows_that_are_left_out(value, accumulate):
    N, C, V = 9, 16, 40
    x, w, t = O.make(N, C, V, dtype=torch.float32)
    t[2], t[5] = -1, V
    lse = torch.logsumexp(x @ w.t(), 1)
    out = [torch.zeros_like(x), torch.full_like(w, 0.5)]
    ops.linear_cross_entropy_backward(*out, x, w, t, lse, 0.3, V, accumulate=accumulate)
    y, spoiled = x.clone(), lse.clone()
    y[2], y[5, 3] = value, value
    spoiled[[2, 5]] = value
    weights = torch.full((N,), 0.3)
    weights[[2, 5]] = value
    for dloss in (0.3, weights):
        got = [torch.full_like(x, 7.0), torch.full_like(w, 0.5)]
        ops.linear_cross_entropy_backward(*got, y, w, t, spoiled, dloss, V, accumulate=accumulate)
        assert all(torch.equal(a, b) for a, b in zip(got, out))
