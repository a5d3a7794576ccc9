"""Global norm of a list of gradients and clipping (csrc/clip.cu) against 64 bits.

Bounds: a thread's chunk sums at most 32 squares in fp32 (each product and each addition 2^-24), everything else is 64-bit and the root is rounded once: the norm is
off by at most 20 * 2^-24 of its size; the factor by 2^-23 more, and a result by that and its own rounding (2^-8 in bf16, 2^-24 in fp32)."""
import math

import pytest
import torch

from llmc_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def _norm64(grads):
    return math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in grads))


def _check(outs, norm, grads, before, max_norm):
    want = _norm64(before)
    assert abs(float(norm) - want) <= 20 * EPS * want
    s = min(1.0, max_norm / want) if want > 0 else 1.0
    for o, g in zip(outs, before):
        tol = (24 * EPS + (2.0 ** -8 if g.dtype == BF16 else EPS)) * 1.01
        assert ((o.double() - g.double() * s).abs() <= tol * (g.double() * s).abs() + 1e-40).all()


def _tensors(sizes, seed, dtypes=(BF16, F32)):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(n, generator=g, device=DEV).mul_(0.01 * (1 + i % 5)).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


@pytest.mark.parametrize("sizes", [[1], [0], [3, 0, 1], [8191, 8192, 8193, 4096, 4095, 4097], [100_003] * 9, [7] * 1500, [5_000_001, 12, 300_000]])
@pytest.mark.parametrize("in_place", [False, True])
def test_clip(sizes, in_place):
    grads = _tensors(sizes, 1)
    before = [g.clone() for g in grads]
    outs = None if in_place else [torch.full_like(g, 7.0) for g in grads]
    plan = ops.clip_plan(outs, grads)
    norm = torch.zeros(1, device=DEV)
    limit = 0.37 * _norm64(before) or 1.0
    ops.clip_grad_norm(norm, plan, limit)
    _check(grads if in_place else outs, norm, grads, before, limit)
    if not in_place:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        again = [o.clone() for o in outs]
        first = norm.clone()
        ops.clip_grad_norm(norm, plan, limit)                 # the same plan again, and the same bits
        assert torch.equal(first, norm) and all(torch.equal(a, b) for a, b in zip(outs, again))
        ops.clip_grad_norm(norm, plan, 10 * _norm64(before) + 1)
        assert all(torch.equal(a, b) for a, b in zip(outs, before))          # below the limit nothing changes
    else:
        now = [g.clone() for g in grads]
        ops.clip_grad_norm(norm, plan, float("inf"))
        assert all(torch.equal(a, b) for a, b in zip(grads, now))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_pieces_on_any_element(dtype, shift):
    """Views of a flat buffer; outputs that lie on the same and on another element of a 16-byte unit.  What lies between is not touched."""
    flat, to = _tensors([70_000], 2, (dtype,))[0], torch.full((70_000,), 7.0, device=DEV, dtype=dtype)
    spans = [(1, 2), (3, 3), (5, 4_103), (4_104, 20_000), (20_001, 20_009), (20_016, 69_990)]
    grads, outs = [flat[a:b] for a, b in spans], [to[a + shift:b + shift] for a, b in spans]
    plan, norm = ops.clip_plan(outs, grads), torch.zeros(1, device=DEV)
    limit = 0.5 * _norm64(grads)
    ops.clip_grad_norm(norm, plan, limit)
    _check(outs, norm, grads, grads, limit)
    gap = torch.ones(70_000, dtype=torch.bool, device=DEV)
    for a, b in spans:
        gap[a + shift:b + shift] = False
    assert (to[gap] == 7.0).all()


def test_matrices_in_another_order_and_another_stream():
    g = torch.randn(300, 200, device=DEV).t()
    out = torch.zeros(300, 200, device=DEV).t()
    plan, norm = ops.clip_plan([out], [g]), torch.zeros(1, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.clip_grad_norm(norm, plan, 1.0)
    s.synchronize()
    _check([out], norm, [g], [g], 1.0)


def test_values_that_are_not_finite():
    norm = torch.zeros(1, device=DEV)
    g = [torch.ones(100, device=DEV), torch.ones(50, device=DEV)]
    g[1][7] = float("inf")
    ops.clip_grad_norm(norm, ops.clip_plan(None, g), 1.0)
    assert float(norm) == float("inf") and not g[0].any() and torch.isnan(g[1][7])
    g = [torch.ones(100, device=DEV), torch.full((50,), float("nan"), device=DEV)]
    ops.clip_grad_norm(norm, ops.clip_plan(None, g), 1.0)
    assert torch.isnan(norm).all() and (g[0] == 1).all()


def test_refusals():
    norm = torch.zeros(1, device=DEV)
    a, b = torch.ones(64, device=DEV), torch.ones(64, device=DEV)
    for outs, grads in [([a], [a, b]), ([a.to(BF16)], [a]), ([a[:32]], [a]), (None, [a.half()]), (None, [a.double()]), (None, [a[::2]]), ([a.cpu()], [a]),
                        (None, [a, a]), (None, [a, a[10:20]]), ([a[8:40], b[:32]], [a[:32], a[32:]]), ([b, b], [a, a.clone()])]:
        with pytest.raises(ValueError):
            ops.clip_plan(outs, grads)
    plan = ops.clip_plan([b], [a])
    for call in [lambda: ops.clip_grad_norm(norm, plan, 0.0), lambda: ops.clip_grad_norm(norm, plan, float("nan")), lambda: ops.clip_grad_norm(norm, plan, -1.0),
                 lambda: ops.clip_grad_norm(norm.double(), plan, 1.0), lambda: ops.clip_grad_norm(norm.cpu(), plan, 1.0), lambda: ops.clip_grad_norm(norm[:0], plan, 1.0)]:
        with pytest.raises(ValueError):
            call()


def test_captured():
    """A captured call on gradients that change between replays."""
    grads = _tensors([70_001, 3, 5_000], 4)
    outs = [torch.zeros_like(g) for g in grads]
    plan, norm = ops.clip_plan(outs, grads), torch.zeros(1, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.clip_grad_norm(norm, plan, 0.25)
    for seed in (5, 6):
        for g, new in zip(grads, _tensors([70_001, 3, 5_000], seed)):
            g.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        _check(outs, norm, grads, grads, 0.25)


def test_large_sums():
    """Sums of squares beyond what fp32 counts exactly: 2^25 equal elements, whose norm is 2^12.5 times the element."""
    g = [torch.full((1 << 25,), 1.0, device=DEV)]
    norm = torch.zeros(1, device=DEV)
    ops.clip_grad_norm(norm, ops.clip_plan(None, g), 1e9)
    assert abs(float(norm) - 2.0 ** 12.5) <= 20 * EPS * 2.0 ** 12.5
