"""Loss of a linear layer without logits and its gradients (csrc/linear_ce.cu) against 64 bits; bounds in linear_ce_oracle.py."""
import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops
from llmc_b200.ops import kernels as KN

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _forward(x, w, t, V):
    losses, lse = torch.full((x.shape[0],), 7.0, device=DEV), torch.full((x.shape[0],), 7.0, device=DEV)
    ops.linear_cross_entropy_forward(losses, lse, x, w, t, V)
    return losses, lse


@pytest.mark.parametrize("N,C,V", [(1, 8, 1), (1, 64, 2), (7, 72, 63), (24, 768, 5003), (77, 136, 64), (128, 64, 65), (129, 64, 255), (256, 200, 256),
                                   (257, 64, 257), (700, 264, 1000), (2100, 64, 3001), (33, 4096, 1500), (5, 768, 50257)])
def test_loss(N, C, V):
    x, w, t = O.make(N, C, V, seed=N + V, rows=V + 5, left_out=0.2 if N > 20 else 0.0)
    w[V:] = float("nan")                       # rows past the vocabulary belong to nobody
    x, w, t = x.to(DEV), w.to(DEV), t.to(DEV)
    losses, lse = _forward(x, w, t, V)
    want, want_lse, e, e_lse = O.forward(x, w, t, V)
    O.within(lse, want_lse, e_lse)
    O.within(losses, want, e)
    ops.linear_cross_entropy_forward(losses, None, x, w, t, V, accumulate_loss=True)
    O.within(losses, 2 * want, 2 * e + 4 * O.EPS * want.abs())


@pytest.mark.parametrize("N,C,V,piece,left_out", [(1, 8, 1, None, 0.0), (1, 768, 5003, None, 0.0), (7, 72, 63, None, 0.0), (77, 136, 1003, None, 0.5), (128, 64, 65, 64, 0.0),
                                                  (129, 64, 255, 256, 0.1), (257, 72, 257, 256, 0.0), (300, 264, 9001, 4096, 0.1), (700, 264, 9001, None, 0.0),
                                                  (1300, 64, 1501, 512, 1.0), (2100, 520, 3001, 1024, 0.1), (40, 2048, 2000, 256, 0.0)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(N, C, V, piece, left_out, accumulate):
    x, w, t = O.make(N, C, V, seed=N + V, rows=V + 3, left_out=left_out)
    w[V:] = float("nan")
    x, w, t = x.to(DEV), w.to(DEV), t.to(DEV)
    _, lse = _forward(x, w, t, V)
    g = torch.Generator().manual_seed(1)
    for dloss in (1.0 / N, (torch.rand(N, generator=g) / N).to(DEV)):
        old = torch.randn(V + 3, C, generator=g).mul_(1e-3).to(torch.bfloat16).to(DEV)
        dinp, dw = torch.full_like(x, 7.0), old.clone()
        ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        factor = dloss if torch.is_tensor(dloss) else torch.full((N,), dloss)
        want, want_w, e, e_w = O.gradient(x, w, t, V, lse, factor, old if accumulate else None, pieces=V // 256 + 1)
        O.within(dinp, want, e)
        O.within(dw[:V], want_w, e_w)
        assert torch.equal(dw[V:], old[V:] if accumulate else torch.zeros_like(old[V:]))
        # either gradient alone, the same bits
        d1, d2 = torch.zeros_like(dinp), old.clone()
        ops.linear_cross_entropy_backward(d1, None, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        ops.linear_cross_entropy_backward(None, d2, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        assert torch.equal(d1, dinp) and torch.equal(d2, dw)


def test_gradient_against_differences():
    """The change of the summed loss along a direction, in the loss's own fp32 arithmetic: the step is a power of two that bf16 weights hold exactly."""
    N, C, V = 96, 64, 500
    x, w, t = O.make(N, C, V, seed=3)
    w = (w.float() * 8).round().div(8).to(torch.bfloat16)            # multiples of 1/8 below 8: a step of 1/16 is exact
    d = torch.randint(-1, 2, (V, C), generator=torch.Generator().manual_seed(4)).float()
    h = 1.0 / 16
    up, down = (w.float() + h * d).to(torch.bfloat16), (w.float() - h * d).to(torch.bfloat16)
    assert torch.equal(up.float() - down.float(), 2 * h * d)
    x, w, t, up, down, d = (a.to(DEV) for a in (x, w, t, up, down, d))
    _, lse = _forward(x, w, t, V)
    dw = torch.zeros_like(w)
    ops.linear_cross_entropy_backward(None, dw, x, w, t, lse, 1.0, V, accumulate=False)
    slope = float((dw.double() * d.double()).sum())
    diff = float((_forward(x, up, t, V)[0].double() - _forward(x, down, t, V)[0].double()).sum()) / (2 * h)
    # central differences: h^2 / 6 times the third derivative along the direction, which in 64 bits is the difference's own distance from the slope
    exact = lambda a: O.forward(x, a, t, V)[0].sum()
    truncation = abs(float(exact(up) - exact(down)) / (2 * h) - float((O.gradient(x, w, t, V, lse, torch.ones(N))[1] * d.cpu().double()).sum()))
    _, want_w, _, e_w = O.gradient(x, w, t, V, lse, torch.ones(N))
    e_loss = sum(float(O.forward(x, a, t, V)[2].sum()) for a in (up, down)) / (2 * h)
    assert abs(slope - diff) <= truncation + float(e_w.sum()) + e_loss
    assert abs(slope) > 3 * truncation                                # the test says something


def test_rows_do_not_touch_one_another():
    N, C, V = 300, 64, 1000
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=5))
    losses, lse = _forward(x, w, t, V)
    y = x.clone()
    y[17, 3], y[200, 0], y[299, 5] = float("nan"), float("inf"), -float("inf")
    t2 = t.clone()
    t2[40] = -100
    t2[41] = V
    l2, lse2 = _forward(y, w, t2, V)
    other = torch.ones(N, dtype=torch.bool)
    other[[17, 200, 299, 40, 41]] = False
    assert torch.equal(l2[other.to(DEV)], losses[other.to(DEV)]) and torch.equal(lse2[40:42], lse[40:42])
    assert torch.isnan(lse2[17]) and float(l2[40]) == 0.0 and float(l2[41]) == 0.0
    assert not torch.isfinite(lse2[[200, 299]]).any()
    d1, d2 = torch.zeros_like(x), torch.zeros_like(x)
    ops.linear_cross_entropy_backward(d1, None, x, w, t, lse, 1.0, V)
    ops.linear_cross_entropy_backward(d2, None, y, w, t2, lse2, 1.0, V)
    assert torch.equal(d1[other.to(DEV)], d2[other.to(DEV)]) and not d2[40:42].any()


def test_logits_far_apart():
    """Rows with very large, very small and infinite logits."""
    C, V = 8, 700
    w = torch.zeros(V, C)
    w[:, 0] = torch.linspace(-100.0, 100.0, V)
    w[:, 1] = 1.0
    w[5, 2] = float("inf")
    w[6:, 3] = -float("inf")
    w = w.to(torch.bfloat16)
    x = torch.zeros(5, C)
    x[0, 0], x[1, 0], x[2, 1] = 100.0, -100.0, -30000.0
    x = x.to(torch.bfloat16)
    t = torch.tensor([V - 1, 0, 3, 0, 0], dtype=torch.int32)
    finite = w.clone()
    finite[~torch.isfinite(finite)] = 0
    losses, lse = _forward(x.to(DEV), finite.to(DEV), t.to(DEV), V)
    want, want_lse, e, e_lse = O.forward(x, finite, t, V)
    O.within(lse, want_lse, e_lse)
    O.within(losses, want, e)
    # 0 * inf is NaN in a product: rows that meet the infinite weights need inputs that are not 0 there
    x = torch.zeros(2, C)
    x[:, 1:4] = torch.tensor([[1.0, 1.0, 0.0], [1.0, 0.0, 1.0]])
    up, down = finite.clone(), finite.clone()
    up[5, 1], down[6:, 1] = float("inf"), -float("inf")
    x = x.to(torch.bfloat16).to(DEV)
    l1, s1 = _forward(x, up.to(DEV), torch.tensor([0, 5], dtype=torch.int32, device=DEV), V)
    assert torch.isinf(s1).all() and (s1 > 0).all() and float(l1[0]) == float("inf") and torch.isnan(l1[1])
    l2, s2 = _forward(x, down.to(DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV), V)
    want = torch.logsumexp(x.double().cpu() @ down[:6].double().t(), 1)
    assert torch.allclose(s2.double().cpu(), want, rtol=1e-5, atol=0)
    every = down.clone()
    every[:, 1] = -float("inf")
    _, s3 = _forward(x, every.to(DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV), V)
    assert (s3 == -float("inf")).all()


def test_strides_streams_and_repeats():
    N, C, V = 300, 264, 2001
    big_x, big_w = torch.randn(N, 2 * C + 16, device=DEV).to(torch.bfloat16), (torch.randn(V, C + 40, device=DEV) / 16).to(torch.bfloat16)
    x, w = big_x[:, 8:8 + C], big_w[:, 32:32 + C]
    t = torch.randint(0, V, (N,), device=DEV, dtype=torch.int32)
    a = _forward(x.contiguous(), w.contiguous(), t, V)
    dense = torch.zeros(N, C, device=DEV, dtype=torch.bfloat16), torch.zeros(V, C, device=DEV, dtype=torch.bfloat16)
    ops.linear_cross_entropy_backward(*dense, x.contiguous(), w.contiguous(), t, a[1], 0.5, V, accumulate=False)
    wide_in, wide_w = torch.full((N, C + 24), 3.0, device=DEV, dtype=torch.bfloat16), torch.full((V, C + 8), 3.0, device=DEV, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        b = _forward(x, w, t, V)
        ops.linear_cross_entropy_backward(wide_in[:, 16:16 + C], wide_w[:, :C], x, w, t, b[1], 0.5, V, accumulate=False)
    other.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(wide_in[:, 16:16 + C], dense[0]) and torch.equal(wide_w[:, :C], dense[1])
    assert (wide_in[:, :16] == 3).all() and (wide_in[:, 16 + C:] == 3).all() and (wide_w[:, C:] == 3).all()


def test_no_rows():
    w = torch.randn(100, 64, device=DEV).to(torch.bfloat16)
    none = torch.zeros(0, device=DEV)
    x, t = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(0, device=DEV, dtype=torch.int32)
    ops.linear_cross_entropy_forward(none, none, x, w, t, 100)
    dw = torch.ones_like(w)
    ops.linear_cross_entropy_backward(x.clone(), dw, x, w, t, none, 1.0, 100)
    assert (dw == 1).all()
    ops.linear_cross_entropy_backward(x.clone(), dw, x, w, t, none, 1.0, 100, accumulate=False)
    assert not dw.any()


def test_memory_stays_bounded(monkeypatch):
    """The gradient of the logits is held in pieces, and so is the pieces' size chosen."""
    monkeypatch.setattr(KN, "HEAD_PIECE_BYTES", 1 << 20)
    N, C, V = 1000, 64, 5003
    assert KN.head_piece(N, V) == 512 and KN.head_piece(10, V) == V and KN.head_piece(10 ** 7, V) == 256
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=8))
    _, lse = _forward(x, w, t, V)
    a, b = (torch.zeros_like(x), torch.zeros_like(w)), (torch.zeros_like(x), torch.zeros_like(w))
    ops.linear_cross_entropy_backward(*a, x, w, t, lse, 1.0 / N, V, accumulate=False)
    ops.linear_cross_entropy_backward(*b, x, w, t, lse, 1.0 / N, V, accumulate=False, piece=512)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    want, want_w, e, e_w = O.gradient(x, w, t, V, lse, torch.full((N,), 1.0 / N), pieces=20)
    O.within(a[0], want, e)
    O.within(a[1], want_w, e_w)


def test_fp32_tensors():
    """fp32 tensors on the device take the operators' plain form, as the other operators without an fp32 kernel do."""
    N, C, V = 40, 64, 300
    x, w, t = O.make(N, C, V, seed=9, dtype=torch.float32, left_out=0.2)
    x, w, t = x.to(DEV), w.to(DEV), t.to(DEV)
    losses, lse = _forward(x, w, t, V)
    want, want_lse, e, e_lse = O.forward(x, w, t, V)
    O.within(losses, want, 4 * e + 1e-5)
    dinp, dw = torch.zeros_like(x), torch.zeros_like(w)
    ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, 0.1, V, accumulate=False)
    want, want_w, e, e_w = O.gradient(x, w, t, V, lse, torch.full((N,), 0.1), b=2 * O.EPS)
    O.within(dinp, want, 4 * e + 1e-6)
    O.within(dw, want_w, 4 * e_w + 1e-6)


def test_refusals():
    N, C, V = 16, 64, 100
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=9))
    losses = torch.zeros(N, device=DEV)
    f = lambda *a, **k: ops.linear_cross_entropy_forward(*a, **k)
    wide = torch.zeros(N + 1, C + 12, device=DEV, dtype=torch.bfloat16)
    for bad in [lambda: f(losses, losses, x, w, t, V + 1), lambda: f(losses, losses, x, w, t, 0), lambda: f(losses, losses, x, w[:, :56], t, V),
                lambda: f(losses, losses, x, w, t.long(), V), lambda: f(losses, losses, x, w, t[:8], V), lambda: f(losses[:8], losses, x, w, t, V),
                lambda: f(losses, losses.double(), x, w, t, V), lambda: f(losses, losses, x.half(), w.half(), t, V), lambda: f(losses, losses, x, w.cpu(), t, V),
                lambda: f(losses, losses, wide[:N, :C], w, t, V), lambda: f(losses, losses, wide[:N, 4:4 + C], w, t, V), lambda: f(losses, losses, x[:, :60], w[:, :60], t, V),
                lambda: f(losses, losses, x, w.t().contiguous().t(), t, V)]:
        with pytest.raises(ValueError):
            bad()
    b = lambda dinp, dw, dloss, **k: ops.linear_cross_entropy_backward(dinp, dw, x, w, t, losses, dloss, V, **k)
    for bad in [lambda: b(x[:8].clone(), None, 1.0), lambda: b(None, w[:50].clone(), 1.0), lambda: b(x.float(), None, 1.0), lambda: b(x.clone(), None, losses[:3]),
                lambda: b(x.clone(), None, 1.0, piece=0), lambda: b(None, w.clone()[:, :56], 1.0), lambda: b(x, None, 1.0), lambda: b(None, w, 1.0),
                lambda: f(losses, losses, x[0], w, t[:1], V), lambda: f(losses, losses, x, w.view(-1), t, V)]:
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("N", [24, 300])
def test_captured(N):
    """A pass that is captured before any other call, replayed on changing inputs."""
    C, V = 64, 1003
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=11))
    losses, lse, dinp, dw = torch.zeros(N, device=DEV), torch.zeros(N, device=DEV), torch.zeros_like(x), torch.zeros_like(w)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.linear_cross_entropy_forward(losses, lse, x, w, t, V)
            ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, 0.5, V, accumulate=False)
    for seed, graph in ((12, graphs[1]), (13, graphs[0]), (14, graphs[1])):
        y = O.make(N, C, V, seed=seed)[0].to(DEV)
        x.copy_(y)
        for out in (losses, dinp, dw):
            out.zero_()
        graph.replay()
        got = [losses.clone(), lse.clone(), dinp.clone(), dw.clone()]
        want = [torch.zeros_like(a) for a in got]
        ops.linear_cross_entropy_forward(want[0], want[1], y, w, t, V)
        ops.linear_cross_entropy_backward(want[2], want[3], y, w, t, want[1], 0.5, V, accumulate=False)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_after_a_graph_has_gone():
    """A graph's scratch lives as long as the graph, whatever became of the memory of graphs before it and of the calls that follow in the same capture."""
    C, V = 64, 1003
    small, large = [tuple(a.to(DEV) for a in O.make(n, C, V, seed=n)) for n in (200, 900)]
    make = lambda a: (torch.zeros(a[0].shape[0], device=DEV), torch.zeros(a[0].shape[0], device=DEV), torch.zeros_like(a[0]), torch.zeros_like(a[1]))

    def both(args, outs):
        ops.linear_cross_entropy_forward(outs[0], outs[1], *args, V)
        ops.linear_cross_entropy_backward(outs[2], outs[3], *args, outs[1], 0.5, V, accumulate=False)

    gone, outs = torch.cuda.CUDAGraph(), make(small)
    with torch.cuda.graph(gone):
        both(small, outs)
    del gone
    graph, outs = torch.cuda.CUDAGraph(), make(large)
    with torch.cuda.graph(graph):
        both(large, outs)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    other, more = torch.cuda.CUDAGraph(), make(small)
    with torch.cuda.graph(other):
        both(small, more)
    want, want_small = make(large), make(small)
    both(large, want)
    both(small, want_small)
    for _ in range(2):
        for o in outs + more:
            o.zero_()
        graph.replay()
        other.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs + more, want + want_small))


@pytest.mark.parametrize("N,C,V,left_out,accumulate", [(1, 264, 20001, 0.0, False), (77, 264, 20001, 0.3, True), (128, 520, 14000, 0.0, False), (300, 520, 14000, 0.1, True),
                                                       (1100, 264, 19999, 0.9, False)])
def test_gradients_of_a_large_vocabulary(N, C, V, left_out, accumulate):
    """Enough tiles for both gradients in one launch."""
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N, left_out=left_out))
    t[N // 2:N // 2 + 3] = int(t[0])                         # shared targets
    _, lse = _forward(x, w, t, V)
    old = torch.randn(V, C, generator=torch.Generator().manual_seed(1)).mul_(1e-3).to(torch.bfloat16).to(DEV)
    dinp, dw = torch.full_like(x, 7.0), old.clone()
    dloss = torch.linspace(0.1, 1.0, N, device=DEV) / N
    ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, dloss, V, accumulate=accumulate)
    want, want_w, e, e_w = O.gradient(x, w, t, V, lse, dloss, old if accumulate else None)
    O.within(dinp, want, e)
    O.within(dw, want_w, e_w)


@pytest.mark.parametrize("N,kept", [(1, 1), (40, 1), (3000, 1), (500, 64), (500, 65), (500, 256), (300, 5)])
def test_few_rows_that_count(N, kept):
    """Where few rows count, the target's entry of each is not left at its bf16 rounding: gradients as near as two roundings of the result allow, in the 2-norm.
    A rounding to bf16 is off by 2^-8 / sqrt(12) to 2^-8 / sqrt(3) of an element, rms over a binade 0.0017; two independent ones 0.0024, and 0.0003 for the other entries of g."""
    C, V = 768, 2000
    x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N + kept))
    x += 3 * w[t.long()] / w[t.long()].float().norm(dim=1, keepdim=True).to(w.dtype)
    keep = torch.randperm(N, generator=torch.Generator().manual_seed(2))[:kept].to(DEV)
    t2 = torch.full_like(t, -1)
    t2[keep] = t[keep]
    if kept == 5:
        t2[keep] = t[keep[0]]                                # all of the same target
    _, lse = _forward(x, w, t2, V)
    dinp, dw = torch.zeros_like(x), torch.zeros_like(w)
    ops.linear_cross_entropy_backward(dinp, dw, x, w, t2, lse, 0.37, V, accumulate=False)
    want, want_w, _, _ = O.gradient(x, w, t2, V, lse, torch.full((N,), 0.37))
    rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())
    assert rel(dinp, want) <= 0.0027 and rel(dw, want_w) <= 0.0027


def test_an_infinite_weight_of_the_target():
    """It decides the gradient of its channel; what is put back of the target's entry leaves it alone."""
    C, V = 72, 500
    x, w, t = (a.to(DEV) for a in O.make(1, C, V, seed=3))
    x[0, 5], w[int(t[0]), 5] = 1.0, float("-inf")            # the target's logit is -inf, its softmax 0, its entry of g -dloss
    lse = torch.logsumexp((x.double() @ w.double().T)[0], 0).float().reshape(1)
    dinp, dw = torch.zeros_like(x), torch.zeros_like(w)
    ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, 0.3, V, accumulate=False)
    assert dinp[0, 5].item() == float("inf") and torch.isfinite(dinp[0, :5]).all() and torch.isfinite(dinp[0, 6:]).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("N,V", [(1, 700), (100, 5003), (300, 5003)])
def test_loss_of_a_nearly_certain_target(N, V):
    x, w, t, want, e = O.certain(N, V)
    losses, _ = _forward(x.to(DEV), w.to(DEV), t.to(DEV), V)
    O.within(losses, want, e)


def test_rows_of_weights_past_32_bits():
    """Rows of the weights and of their gradient 2^20 elements apart: the last ones lie past 2^31 elements."""
    N, C, V, ld = 70, 72, 2100, 1 << 20
    x, w, t = O.make(N, C, V, seed=9)
    t[:3] = torch.tensor([V - 1, 0, V - 2])
    space = [torch.empty(V * ld, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    wide, dwide = (s.view(V, ld)[:, 64:64 + C] for s in space)
    wide.copy_(w)
    xd, td = x.to(DEV), t.to(DEV)
    losses, lse = _forward(xd, wide, td, V)
    want, _, e, _ = O.forward(x, w, t, V)
    O.within(losses, want, e)
    dinp = torch.zeros_like(xd)
    ops.linear_cross_entropy_backward(dinp, dwide, xd, wide, td, lse, 0.1, V, accumulate=False)
    want, want_w, e, e_w = O.gradient(x, w, t, V, lse, torch.full((N,), 0.1))
    O.within(dinp, want, e)
    O.within(dwide.contiguous(), want_w, e_w)


def test_gradient_of_the_logits_past_32_bits():
    """70000 rows over 32000 columns at once, 2.2 G entries, of which the last 64 rows count."""
    N, C, V, k = 70000, 16, 32000, 64
    x, w, t = O.make(N, C, V, seed=10)
    t[:-k] = -1
    xd, wd, td = x.to(DEV), w.to(DEV), t.to(DEV)
    losses, lse = _forward(xd, wd, td, V)
    want, _, e, _ = O.forward(x[-k:], w, t[-k:], V)
    O.within(losses[-k:], want, e)
    assert not losses[:-k].any()
    dinp, dw = torch.full_like(xd, 7.0), torch.full_like(wd, 7.0)
    ops.linear_cross_entropy_backward(dinp, dw, xd, wd, td, lse, 0.1, V, accumulate=False, piece=V)
    want, want_w, e, e_w = O.gradient(x[-k:], w, t[-k:], V, lse[-k:], torch.full((k,), 0.1))
    O.within(dinp[-k:], want, e)
    O.within(dw, want_w, e_w)
    assert not dinp[:-k].any()


@pytest.mark.parametrize("seed", [0, 1, 2])
@pytest.mark.parametrize("piece", [None, 256])
def test_gradient_of_a_nearly_certain_target(seed, piece):
    """A softmax of 1 - d, d about 1e-4, at a logit z of about 16: what z is off by stands over d in the target's entry of the logits' gradient.  A dot product of 1024 terms in
    32 lanes that is as far off as 32 additions near z / 32 in each lane and 5 near z with errors of any sign: sqrt(32 * 32) / 32 + sqrt(5) halves of 2 eps z, 3.3 eps z, about 1 % of d.
    Everything else is two roundings to bf16, as for few rows."""
    C, V = 1024, 700
    x, w, t = O.make(1, C, V, seed=seed)
    to = w[t.long()].float()
    x = (0.3 * x.float() + 8.0 * to / to.norm(dim=1, keepdim=True)).to(torch.bfloat16)
    z = (x.double() @ w.double().T)[0]
    lse = torch.logsumexp(z, 0).float()
    zt = float(z[int(t)])
    d = float(-torch.expm1(zt - lse.double()))
    assert 5e-5 < d < 5e-4 and 14 < zt < 18
    x, w, t, lse = (a.to(DEV) for a in (x, w, t, lse.reshape(1)))
    dinp, dw = torch.zeros_like(x), torch.zeros_like(w)
    ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, 0.37, V, accumulate=False, piece=piece)
    want, want_w, _, _ = O.gradient(x, w, t, V, lse, torch.full((1,), 0.37))
    rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())
    assert rel(dinp, want) <= 3.3 * O.EPS * zt / d + 0.0027
    if piece is None:
        assert rel(dw, want_w) <= 3.3 * O.EPS * zt / d + 0.0027


@pytest.mark.parametrize("N,C,V,piece,left_out", [(257, 64, 300, None, 0.5), (300, 264, 20001, None, 0.5), (1100, 264, 20001, None, 0.97), (1300, 64, 1501, 512, 0.9), (2100, 520, 3001, None, 0.3),
                                                  (2100, 264, 700, None, 0.99), (3000, 72, 1000, 256, 0.0), (9000, 40, 900, None, 0.6), (700, 136, 5000, None, 2.0), (513, 2048, 600, None, 0.999)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_of_rows_that_count(N, C, V, piece, left_out, accumulate, monkeypatch):
    """The rows that count moved together, as for large products: the rest of x and of dinp is not read and 0."""
    monkeypatch.setattr(KN, "HEAD_KEPT_WORK", 0)
    x, w, t = O.make(N, C, V, seed=N + V, rows=V + 3, left_out=left_out)
    if left_out < 2:
        t[N // 3], t[N - 1], t[0] = 5, V - 1, V            # at least two count, the first does not
    w[V:] = float("nan")
    x, w, t = x.to(DEV), w.to(DEV), t.to(DEV)
    _, lse = _forward(x, w, t, V)
    g = torch.Generator().manual_seed(1)
    for dloss in (0.7 / N, (torch.rand(N, generator=g) / N).to(DEV)):
        old = torch.randn(V + 3, C, generator=g).mul_(1e-3).to(torch.bfloat16).to(DEV)
        dinp, dw = torch.full_like(x, 7.0), old.clone()
        ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        factor = dloss if torch.is_tensor(dloss) else torch.full((N,), dloss)
        want, want_w, e, e_w = O.gradient(x, w, t, V, lse, factor, old if accumulate else None, pieces=V // 256 + 1)
        O.within(dinp, want, e)
        O.within(dw[:V], want_w, e_w)
        assert not dinp[(t < 0) | (t >= V)].any()
        assert torch.equal(dw[V:], old[V:] if accumulate else torch.zeros_like(old[V:]))
        d1, d2 = torch.zeros_like(dinp), old.clone()
        ops.linear_cross_entropy_backward(d1, None, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        ops.linear_cross_entropy_backward(None, d2, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        again, more = torch.zeros_like(dinp), old.clone()
        ops.linear_cross_entropy_backward(again, more, x, w, t, lse, dloss, V, accumulate=accumulate, piece=piece)
        assert torch.equal(again, dinp) and torch.equal(more, dw)
        O.within(d1, want, e)
        O.within(d2[:V], want_w, e_w)
