"""Rows that are left out of the head's gradients may hold anything (csrc/linear_ce.cu): the same bits as with finite inputs there, at sizes of every kernel that forms them."""
import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops
from llmc_b200.ops import kernels as KN

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("N,C,V,piece", [(7, 72, 63, None), (77, 264, 20001, None), (100, 136, 700, 256), (200, 264, 20001, None), (256, 1544, 300, None), (300, 264, 20001, None), (700, 264, 3001, 1024),
                                         (1500, 72, 700, None), (40, 4104, 300, None)])
@pytest.mark.parametrize("moved", [False, True])
@pytest.mark.parametrize("accumulate", [False, True])
def test_rows_that_are_left_out(N, C, V, piece, moved, accumulate, monkeypatch):
    if moved:
        monkeypatch.setattr(KN, "HEAD_KEPT_WORK", 0)
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N))
    out = torch.zeros(N, dtype=torch.bool, device=DEV)
    out[[1, N // 2, N - 1]] = True
    t[out] = torch.tensor([-1, V, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    lse = torch.zeros(N, device=DEV)
    ops.linear_cross_entropy_forward(torch.zeros(N, device=DEV), lse, x, w, t, V)
    old = torch.randn(V, C, generator=torch.Generator().manual_seed(1)).mul_(1e-3).to(torch.bfloat16).to(DEV)
    wide = torch.zeros(N, C + 8, dtype=torch.bfloat16, device=DEV)
    weights = torch.rand(N, generator=torch.Generator().manual_seed(2)).to(DEV)
    for by_row in (False, True):
        want = [torch.full_like(x, 7.0), old.clone()]
        ops.linear_cross_entropy_backward(*want, x, w, t, lse, weights if by_row else 0.3, V, accumulate=accumulate, piece=piece)
        assert not want[0][out].any()
        for value in (float("nan"), float("inf")):
            wide[:, :C] = x
            wide[1, :C], wide[N // 2, 3], wide[N - 1, C - 1] = value, -value, value
            spoiled, factor = lse.clone(), weights.clone()
            spoiled[out], factor[out] = value, value
            got = [torch.full_like(x, 7.0), old.clone()]
            ops.linear_cross_entropy_backward(*got, wide[:, :C], w, t, spoiled, factor if by_row else 0.3, V, accumulate=accumulate, piece=piece)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            alone = old.clone()
            ops.linear_cross_entropy_backward(None, alone, wide[:, :C], w, t, spoiled, factor if by_row else 0.3, V, accumulate=accumulate, piece=piece)
            assert torch.isfinite(alone).all()


@pytest.mark.parametrize("N", [20, 200, 300])
def test_a_row_that_is_left_out_has_no_gradient_under_infinite_weights(N):
    """0 times an infinite weight is no part of it."""
    C, V = 72, 500
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N))
    w[17, 5] = float("inf")
    t[3] = -1
    dinp = torch.full_like(x, 7.0)
    ops.linear_cross_entropy_backward(dinp, None, x, w, t, torch.zeros(N, device=DEV), 0.3, V)
    assert not dinp[3].any()
