"""The head's operators called by several threads on one stream: a call's launches may have another thread's between them."""
import threading

import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("sizes", [[(24, 72, 5003), (100, 136, 3001)], [(300, 264, 5003), (700, 264, 3001)], [(24, 72, 5003), (700, 264, 9001), (200, 72, 20001)]])
def test_threads(sizes):
    def passes(args, V, turns):
        x, w, t = args
        N = x.shape[0]
        losses, lse, dinp, dw = torch.zeros(N, device=DEV), torch.zeros(N, device=DEV), torch.zeros_like(x), torch.zeros_like(w)
        for _ in range(turns):
            ops.linear_cross_entropy_forward(losses, lse, x, w, t, V)
            ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, 0.3, V, accumulate=False)
        return losses, lse, dinp, dw

    inputs = [tuple(a.to(DEV) for a in O.make(N, C, V, seed=N)) for N, C, V in sizes]
    want = [passes(a, s[2], 1) for a, s in zip(inputs, sizes)]
    got, failed = [None] * len(sizes), []

    def work(i):
        try:
            got[i] = passes(inputs[i], sizes[i][2], 40)
        except Exception as e:                      # shown by the main thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed, failed
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
