"""Outputs that share memory with what is still read are refused, before anything is written; those that lie between the rows of an input are not."""
import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops


def test_clipping_refuses_tensors_that_overlap():
    a, b = torch.ones(64), torch.ones(64)
    for outs, grads in [(None, [a, a]), (None, [a, a[10:20]]), ([a[8:40], b[:32]], [a[:32], a[32:]]), ([b, b], [a, a.clone()]), ([b[:32], b[31:63]], [a[:32], a[32:]])]:
        with pytest.raises(ValueError, match="overlap"):
            ops.clip_plan(outs, grads)
    ops.clip_plan([a[:32], b[:32]], [a[:32], a[32:]])            # one in place, one not
    ops.clip_plan(None, [a[:0], a, a[5:5]])                      # empty ones overlap nothing


N, C, V = 12, 16, 20


def _args():
    x, w, t = O.make(N, C, V, dtype=torch.float32)
    lse = torch.logsumexp(x @ w.t(), 1)
    return x, w, t, lse


def test_the_loss_refuses_outputs_over_inputs():
    x, w, t, _ = _args()
    both = torch.zeros(2 * N - 1)
    for losses, lse in [(both[:N], both[:N]), (both[:N], both[N - 1:]), (t.view(torch.float32), None), (both[:N], t.view(torch.float32)),
                        (x.view(-1)[5:5 + N], None), (both[:N], w.view(-1)[-N:])]:
        kept = [a.clone() for a in (x, w, t, both)]
        with pytest.raises(ValueError, match="memory"):
            ops.linear_cross_entropy_forward(losses, lse, x, w, t, V)
        assert all(torch.equal(a, b) for a, b in zip(kept, (x, w, t, both)))
    space = torch.zeros(2 * N)
    ops.linear_cross_entropy_forward(space[:N], space[N:], x, w, t, V)


def test_the_gradients_refuse_outputs_over_inputs_and_over_each_other():
    x, w, t, lse = _args()
    pool = torch.zeros(N + V + 4, C)
    for name, a in (("x", x), ("w", w)):
        pool[{"x": 0, "w": N}[name]:][:len(a)] = a
    px, pw = pool[:N], pool[N:N + V]
    row = torch.zeros(N, C)
    dloss = torch.ones(N)
    for dinp, dw, inp, weight, l, d in [(pool[1:N + 1], None, px, pw, lse, 1.0), (pool[N - 1:2 * N - 1], None, x, pw, lse, 1.0), (None, pool[N + 4:], x, pw, lse, 1.0), (None, pool[:V], px, w, lse, 1.0),
                                        (pool[:N], pool[N - 1:N - 1 + V], x, w, lse, 1.0), (row, None, x, w, row.view(-1)[40:40 + N], 1.0), (row, None, x, w, lse, row.view(-1)[:N]),
                                        (row, None, x, w, lse, row.view(-1)[N * C - N:]), (x, None, x, w, lse, 1.0), (None, w, x, w, lse, 1.0)]:
        kept = pool.clone()
        with pytest.raises(ValueError, match="memory"):
            ops.linear_cross_entropy_backward(dinp, dw, inp, weight, t, l, d, V)
        assert torch.equal(pool, kept)
    with pytest.raises(ValueError, match="memory"):
        as_rows = torch.zeros(N, C)
        ops.linear_cross_entropy_backward(as_rows, None, x, w, as_rows.view(torch.int32).view(-1)[3:3 + N], lse, 1.0, V)


def test_gradients_between_the_rows_of_an_input():
    """Columns of one buffer of wider rows: side by side, they share no element."""
    x, w, t, lse = _args()
    want = torch.zeros_like(x), torch.zeros_like(w)
    ops.linear_cross_entropy_backward(*want, x, w, t, lse, 1.0, V)
    rows, weights = torch.zeros(N, 2 * C + 8), torch.zeros(V + 3, 3 * C)
    rows[:, C + 8:], weights[:V, C:2 * C] = x, w
    dinp, dw = rows[:, :C], weights[:V, 2 * C:]
    ops.linear_cross_entropy_backward(dinp, dw, rows[:, C + 8:], weights[:, C:2 * C], t, lse, 1.0, V)
    assert torch.equal(dinp, want[0]) and torch.equal(dw, want[1]) and torch.equal(rows[:, C + 8:], x)
    ops.linear_cross_entropy_backward(weights[:N, :C], weights[:V, 2 * C:], x, weights[:, C:2 * C], t, lse, 1.0, V, accumulate=False)
    assert torch.equal(weights[:N, :C], want[0])
    with pytest.raises(ValueError, match="memory"):                     # one column too far
        ops.linear_cross_entropy_backward(rows[:, 9:C + 9], None, rows[:, C + 8:], w, t, lse, 1.0, V)
