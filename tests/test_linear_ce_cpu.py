"""Loss of a linear layer without logits, its gradients and clipping by the global norm on host tensors, against autograd in 64 bits."""
import math

import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops
from llmc_b200.ops import kernels as KN
from llmc_b200.ops import reference as RF


@pytest.mark.parametrize("N,C,V,left_out", [(1, 8, 1, 0.0), (5, 24, 63, 0.0), (33, 16, 300, 0.3), (16, 40, 129, 1.0)])
@pytest.mark.parametrize("piece", [None, 64, 7])
@pytest.mark.parametrize("accumulate", [False, True])
def test_head_against_autograd(N, C, V, left_out, piece, accumulate, monkeypatch):
    if piece is not None:
        monkeypatch.setattr(RF, "HEAD_PIECE", piece)
    x, w, t = O.make(N, C, V, seed=V, rows=V + 2, left_out=left_out, dtype=torch.float32)
    losses, lse = torch.full((N,), 2.0), torch.zeros(N)
    ops.linear_cross_entropy_forward(losses, lse, x, w, t, V, accumulate_loss=accumulate)
    weights = torch.rand(N, generator=torch.Generator().manual_seed(1))
    xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
    z = xd @ wd[:V].t()
    each = torch.nn.functional.cross_entropy(z, t.long(), ignore_index=-1, reduction="none")
    # sums of C products and of V exponentials in fp32: at most (C + V) eps of their magnitudes, which are below 40 and 1 here
    tol = (C + V) * O.EPS * 40
    assert ((losses.double() - each - (2.0 if accumulate else 0.0)).abs() <= tol).all()
    assert ((lse.double() - torch.logsumexp(z, 1)).abs() <= tol).all()
    for dloss in (0.25, weights):
        xd.grad = wd.grad = None
        (each * (dloss.double() if torch.is_tensor(dloss) else dloss)).sum().backward(retain_graph=True)
        old = torch.randn(w.shape, generator=torch.Generator().manual_seed(2))
        dinp, dw = torch.full_like(x, 3.0), old.clone()
        ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        assert ((dinp.double() - xd.grad).abs() <= 4 * tol).all()
        want = wd.grad + (old.double() if accumulate else 0.0)
        assert ((dw.double() - want).abs() <= 4 * tol * N).all()
        only = old.clone()
        ops.linear_cross_entropy_backward(None, only, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        assert torch.equal(only, dw)


def test_pieces_of_the_vocabulary():
    for N in (1, 77, 2667, 2668, 16384, 65536, 10 ** 6):
        for V in (1, 300, 50257, 128256):
            cols = KN.head_piece(N, V)
            assert cols == V or (cols % 256 == 0 and cols < V and (2 * N * cols <= KN.HEAD_PIECE_BYTES or cols == 256))
            if cols < V and cols > 256:          # even pieces: the last is no sliver
                pieces = -(-V // cols)
                assert V - (pieces - 1) * cols > cols - 256 * pieces


@pytest.mark.parametrize("in_place", [False, True])
def test_clip(in_place):
    g = torch.Generator().manual_seed(3)
    grads = [torch.randn(n, generator=g).to(dt) for n, dt in [(1, torch.float32), (0, torch.float32), (1000, torch.bfloat16), (33, torch.float32)]]
    before = [t.clone() for t in grads]
    outs = None if in_place else [torch.zeros_like(t) for t in grads]
    norm = torch.zeros(1)
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in before))
    ops.clip_grad_norm(norm, ops.clip_plan(outs, grads), 0.5)
    assert abs(float(norm) - want) <= 4 * O.EPS * want
    for o, b in zip(grads if in_place else outs, before):
        assert ((o.double() - b.double() * 0.5 / want).abs() <= (O.B + 8 * O.EPS) * b.double().abs()).all()
    kept = [t.clone() for t in before]
    ops.clip_grad_norm(norm, ops.clip_plan(None, kept), 2 * want)
    assert all(torch.equal(a, b) for a, b in zip(kept, before))
    ops.clip_grad_norm(norm, ops.clip_plan([], []), 1.0)
    assert float(norm) == 0.0


def test_refusals():
    x, w, t = O.make(4, 16, 20, dtype=torch.float32)
    losses = torch.zeros(4)
    for bad in [lambda: ops.linear_cross_entropy_forward(losses, losses, x, w, t, 21), lambda: ops.linear_cross_entropy_forward(losses, losses, x, w, t.long(), 20),
                lambda: ops.linear_cross_entropy_forward(losses[:2], losses, x, w, t, 20), lambda: ops.linear_cross_entropy_forward(losses, losses, x, w[:, :8], t, 20),
                lambda: ops.linear_cross_entropy_backward(x[:2].clone(), None, x, w, t, losses, 1.0, 20),
                lambda: ops.linear_cross_entropy_backward(x.clone(), None, x, w, t, losses, 1.0, 20, piece=-1),
                lambda: ops.linear_cross_entropy_backward(None, w.bfloat16(), x, w, t, losses, 1.0, 20),
                lambda: ops.clip_plan([losses], [losses, x]), lambda: ops.clip_plan(None, [losses.half()]), lambda: ops.clip_plan(None, [x[:, :3]]),
                lambda: ops.clip_grad_norm(torch.zeros(1), ops.clip_plan(None, [losses]), 0.0)]:
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("N,V", [(1, 700), (100, 5003)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_of_a_nearly_certain_target(N, V, dtype):
    x, w, t, want, e = O.certain(N, V, dtype)
    losses = torch.zeros(N)
    ops.linear_cross_entropy_forward(losses, None, x, w, t, V)
    O.within(losses, want, e)
