"""Loss of a linear layer without logits and its gradients at sizes that reach every form of their kernels (csrc/linear_ce.cu, linear_ce_few.cu, gemm2.cu), against 64 bits; bounds in
linear_ce_oracle.py.  The gradients start from an lse of 64 bits."""
import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _loss(x, w, t, V):
    losses, lse = torch.full((x.shape[0],), 7.0, device=DEV), torch.full((x.shape[0],), 7.0, device=DEV)
    ops.linear_cross_entropy_forward(losses, lse, x, w, t, V)
    want, want_lse, e, e_lse = O.forward(x, w, t, V)
    O.within(lse, want_lse, e_lse)
    O.within(losses, want, e)
    return want_lse.float().to(DEV)


def _gradients(x, w, t, V, lse, accumulate, N, C):
    old = torch.randn(V, C, generator=torch.Generator().manual_seed(1)).mul_(1e-3).to(torch.bfloat16).to(DEV)
    for dloss in (0.9 / N, torch.linspace(0.1, 1.0, N, device=DEV) / N):
        dinp, dw = torch.full_like(x, 7.0), old.clone()
        ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, dloss, V, accumulate=accumulate)
        want, want_w, e, e_w = O.gradient(x, w, t, V, lse, dloss if torch.is_tensor(dloss) else torch.full((N,), dloss), old if accumulate else None)
        O.within(dinp, want, e)
        O.within(dw, want_w, e_w)


@pytest.mark.parametrize("N,C,V", [(129, 1032, 3001), (256, 768, 5003), (200, 2056, 20001), (700, 2056, 3001), (300, 520, 257), (2100, 1544, 1000), (128, 4104, 700), (40, 264, 1000)])
def test_logits_that_are_summed_in_parts(N, C, V):
    """More channels than one part of the sum in tensor memory: whole and ragged last parts, one row tile and several."""
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N, left_out=0.1))
    _loss(x, w, t, V)


@pytest.mark.parametrize("N,C,V", [(129, 264, 20001), (200, 72, 50257), (256, 520, 20001), (256, 768, 20001)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_both_gradients_of_129_to_256_rows(N, C, V, accumulate):
    """In one launch, panels for the weight gradient, whole tiles of rows for the input gradient."""
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N, left_out=0.1))
    t[N // 2:N // 2 + 3] = int(t[0])                         # shared targets
    _gradients(x, w, t, V, _loss(x, w, t, V), accumulate, N, C)


@pytest.mark.parametrize("N", [1, 33, 40, 64, 100, 128])
@pytest.mark.parametrize("C,V", [(72, 50257), (264, 38001), (16, 80003)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_more_tiles_than_ctas(N, C, V, accumulate):
    """At most 128 rows, several tiles of the vocabulary for each CTA, targets in the first and in the last of them."""
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N + V, left_out=0.1))
    t[0], t[N - 1], t[N // 2] = V - 1, 0, V - 2
    _gradients(x, w, t, V, _loss(x, w, t, V), accumulate, N, C)
