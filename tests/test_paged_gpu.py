"""Operators on a key / value cache in pages against 64 bits: lengths, heads, pages and layouts where a kernel can go wrong; captured calls; entries that name nothing."""
import pytest
import torch

from llmc_b200 import _lib, ops

import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(c, tree=None, layer=0):
    """Half a step of bf16 for the result, and as much of sum |p v| for probabilities rounded to bf16; 32-bit sums and exponentials over at most some thousand keys are far below
    the last term."""
    exact, size = O.attention(c, tree, layer)
    got = c.out.cpu().double()
    off = (got[:c.N] - exact).abs() - (2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -12) * size)
    assert bool((off <= 0).all()), "row %d, %g too far" % (int(off.max(1).values.argmax()), float(off.max()))
    assert bool((got[c.N:] == 7).all())


# single tokens: one key, pages that begin and end, nothing, several lengths in one batch; every kind of head
@pytest.mark.parametrize("keys,NH,NKV,HS,rows", [
    ((1,), 2, 2, 64, 16), ((16,), 4, 1, 64, 16), ((17, 15, 1, 64), 4, 1, 128, 16), ((700,), 32, 8, 128, 16), ((3, 0, 511, 64, 65, 127, 128, 129), 8, 2, 64, 8),
    ((1300, 40), 6, 2, 96, 32), ((33, 290), 5, 1, 40, 16), ((100, 257), 7, 1, 128, 256), ((64, 63), 8, 1, 16, 64), ((200, 90), 16, 1, 128, 16), ((260, 31), 12, 12, 64, 16),
    ((90, 500), 24, 2, 72, 64), (tuple(range(1, 60, 3)), 4, 2, 128, 16), ((5000,), 8, 2, 64, 16), ((3001, 2, 900), 2, 1, 128, 128)])
@pytest.mark.parametrize("layout", ["rows", "heads", "both"])
def test_single_tokens(keys, NH, NKV, HS, rows, layout):
    new = [min(1, k) for k in keys]
    c = O.Case(keys, new, NH, NKV, HS, rows, seed=sum(keys), device=DEV, layout=layout, layers=2, std=1.5)
    ops.paged_attention(c.out, c.q, c.cache(ops), NH, layer=1)
    _check(c, layer=1)


# prompts and parts of them: from the first slot and behind a context, edges of 32, 64 and 128 rows and keys, next to single tokens and to sequences with nothing new
@pytest.mark.parametrize("keys,new,NH,NKV,HS,rows", [
    ((2,), (2,), 2, 2, 64, 16), ((128,), (128,), 2, 2, 64, 16), ((129,), (129,), 4, 1, 128, 16), ((300,), (300,), 4, 2, 128, 16), ((257, 40, 1), (255, 3, 1), 2, 1, 64, 16),
    ((500, 0, 130, 64), (2, 0, 129, 0), 3, 1, 128, 32), ((200, 77), (64, 77), 5, 1, 96, 8), ((300, 9), (33, 9), 7, 1, 64, 64), ((260,), (130,), 16, 2, 128, 16), ((140, 150), (20, 150), 12, 12, 64, 16),
    ((90, 33), (90, 32), 4, 2, 40, 16), ((385,), (257,), 1, 1, 128, 512), ((1100,), (5,), 8, 1, 128, 16), ((700, 20, 20, 20), (9, 1, 1, 1), 8, 2, 64, 16), ((66,), (66,), 32, 1, 16, 16)])
@pytest.mark.parametrize("layout", ["rows", "both"])
def test_ragged(keys, new, NH, NKV, HS, rows, layout):
    c = O.Case(keys, new, NH, NKV, HS, rows, seed=sum(new), device=DEV, layout=layout, width=2)
    ops.paged_attention(c.out, c.q, c.cache(ops), NH)
    _check(c)


@pytest.mark.parametrize("keys,new,NH,NKV,HS,rows", [
    ((1,), (1,), 2, 2, 64, 16), ((100,), (7,), 4, 1, 128, 16), ((64, 200), (64, 64), 8, 2, 128, 16), ((30, 1000, 5), (12, 3, 5), 4, 4, 64, 8), ((129, 500), (2, 33), 16, 2, 96, 32),
    ((127, 128, 129, 191), (63, 64, 64, 63), 2, 1, 64, 64), ((70,), (64,), 6, 1, 40, 16)])
def test_trees(keys, new, NH, NKV, HS, rows):
    c = O.Case(keys, new, NH, NKV, HS, rows, seed=sum(keys), device=DEV)
    tree = ops.tree_masks([O.random_tree(n, n) for n in new])
    ops.paged_tree_attention(c.out, c.q, c.cache(ops), torch.cat([tree, torch.full((3,), -1)]).to(DEV), NH)
    _check(c, tree)


def test_rows_that_see_nothing_are_zero():
    for n in (1, 5, 40):
        c = O.Case((n, n), (n, n), 8, 2, 128, 16, device=DEV, pad=0)
        tree = torch.cat([torch.zeros(n, dtype=torch.int64), ops.tree_masks([O.random_tree(n, n)])])
        ops.paged_tree_attention(c.out, c.q, c.cache(ops), tree.to(DEV), 8)
        _check(c, tree)
        assert bool((c.out[:n] == 0).all())
        # more new tokens than keys: the first of them have no slot
        c = O.Case((n, 3), (n, 3), 8, 2, 128, 16, device=DEV, pad=0)
        c.lengths[0] = n // 2
        ops.paged_attention(c.out, c.q, c.cache(ops), 8)
        c.keys[0] = n // 2
        _check(c)
        assert bool((c.out[:n - n // 2] == 0).all())


def test_masks_of_any_form():
    g = torch.Generator().manual_seed(5)
    c = O.Case((90, 64), (20, 64), 4, 2, 64, 16, device=DEV)
    tree = torch.randint(-2 ** 63, 2 ** 63 - 1, (84,), generator=g)
    tree[:20] &= (1 << 20) - 1
    ops.paged_tree_attention(c.out, c.q, c.cache(ops), torch.cat([tree, tree[:3]]).to(DEV), 4)
    _check(c, tree)


@pytest.mark.parametrize("new", [1, 9, 200])
def test_scores_far_apart_and_all_alike(new):
    c = O.Case((400,), (new,), 4, 2, 64, 16, device=DEV, pad=0, std=30.0)
    ops.paged_attention(c.out, c.q, c.cache(ops), 4)
    # scores of some hundreds: their 32-bit sums of 64 products are off by up to 64 * 2^-24 * sum |q k| / 8, below 2^-10 here, and with it each probability
    exact, size = O.attention(c)
    assert bool(((c.out.cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -9) * size).all())
    c = O.Case((400,), (new,), 4, 2, 64, 16, device=DEV, pad=0)
    c.q.zero_()
    ops.paged_attention(c.out, c.q, c.cache(ops), 4)
    _check(c)


def test_rows_of_wider_buffers():
    c = O.Case((150, 20), (140, 1), 4, 2, 64, 16, device=DEV, pad=0)
    wide_q, wide_out = torch.randn(141, 1024, device=DEV).bfloat16(), torch.full((141, 640), 7.0, device=DEV).bfloat16()
    wide_q[:, 64:320] = c.q
    ops.paged_attention(wide_out[:, 128:384], wide_q[:, 64:320], c.cache(ops), 4)
    ops.paged_attention(c.out, c.q, c.cache(ops), 4)
    assert torch.equal(wide_out[:, 128:384], c.out) and bool((wide_out[:, :128] == 7).all()) and bool((wide_out[:, 384:] == 7).all())


@pytest.mark.parametrize("new", [1, 3, 100])
def test_same_bits_again_and_captured(new):
    """A captured call follows lengths, table and queries that change between replays; two graphs and an eager call do not disturb one another."""
    c = O.Case((800, 333, 120), (new,) * 3, 8, 2, 128, 16, device=DEV)
    cache = c.cache(ops)
    ops.paged_attention(c.out, c.q, cache, 8)
    first = c.out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [torch.zeros_like(c.out) for _ in range(2)], []
    with torch.cuda.stream(side):
        for o in outs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                ops.paged_attention(o, c.q, cache, 8)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    other = torch.cuda.Stream()
    for _ in range(5):
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graphs[1].replay()
        graphs[0].replay()
        ops.paged_attention(c.out, c.q, cache, 8)
        torch.cuda.current_stream().wait_stream(other)
        assert torch.equal(c.out, first) and all(torch.equal(o[:c.N], first[:c.N]) for o in outs)
    # shorter sequences, the first two of them exchanged
    keys = [333, 700, 110]
    c.table[:2] = c.table[:2].flip(0)
    c.flat = [c.flat[1], c.flat[0][:700], c.flat[2][:110]]
    c.keys = keys
    c.lengths.copy_(torch.tensor(keys, dtype=torch.int32))
    graphs[0].replay()
    c.out = outs[0]
    c.out[c.N:] = 7
    _check(c)


@pytest.mark.parametrize("new", [1, 2, 70])
def test_entries_that_name_nothing_are_reported(new):
    """The status word says so, sequences next to the wrong one are right, and nothing else is written."""
    def wrong(name, at, value):
        c = O.Case((100, 90, 80), (new,) * 3, 4, 2, 64, 16, device=DEV)
        getattr(c, name)[at] = value
        ops.paged_attention(c.out, c.q, c.cache(ops), 4)
        assert _lib.read_status() >> 24 == 3
        _check_only(c, 0)
        assert bool((c.out[c.N:] == 7).all())
        return c

    def _check_only(c, b):
        exact, size = O.attention(O.Case((100, 90, 80), (new,) * 3, 4, 2, 64, 16))
        rows = slice(b * new, (b + 1) * new)
        assert bool(((c.out[rows].cpu().double() - exact[rows]).abs() <= 2.0 ** -8 * exact[rows].abs() + (2.0 ** -8 + 2.0 ** -12) * size[rows]).all())

    for value in (-1, 1 << 20, -2 ** 31, 2 ** 31 - 1):
        wrong("table", (1, 2), value)
    for value in (-1, 2 ** 31 - 1, 10 ** 6):
        wrong("lengths", 1, value)
    for value in (-1, new - 1 if new > 1 else -5, 2 ** 31 - 1):
        wrong("starts", 2, value)


def test_too_many_drafted_tokens_are_reported():
    c = O.Case((100, 90), (65, 3), 4, 2, 64, 16, device=DEV)
    tree = torch.full((c.q.shape[0],), -1, dtype=torch.int64, device=DEV)
    ops.paged_tree_attention(c.out, c.q, c.cache(ops), tree, 4)
    assert _lib.read_status() >> 24 == 3


@pytest.mark.parametrize("keys,new,NH,NKV,HS,R,rows", [
    ((1,), (1,), 2, 2, 64, 64, 16), ((9, 0, 40, 16), (9, 0, 5, 1), 4, 2, 16, 8, 8), ((300, 1, 65), (300, 1, 64), 32, 8, 128, 128, 16), ((100, 40), (3, 40), 5, 1, 96, 48, 32),
    ((70,) * 40, (1,) * 40, 8, 8, 72, 2, 64), ((33, 290), (33, 2), 3, 1, 40, 40, 16), ((50, 90), (1, 7), 12, 12, 64, 20, 16)])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("layout", ["rows", "heads", "both"])
def test_append(keys, new, NH, NKV, HS, R, rows, halves, layout):
    c = O.Case(keys, new, NH, NKV, HS, rows, layers=2, device=DEV, layout=layout)
    f = O.angles(max(keys), R, DEV)
    old = c.kpages.clone(), c.vpages.clone()
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, f, NH, layer=1, halves=halves)
    pos = torch.cat([torch.arange(k - n, k) for k, n in zip(keys, new)])
    x = c.raw[:c.N].cpu().double().view(c.N, NH + 2 * NKV, HS)
    y = O.rotated(x[:, :NH + NKV], f.cpu()[pos].double(), halves)
    # the result's rounding, and two operations in 32 bits on products of at most |x|
    near = lambda a, b: bool(((a.cpu().double() - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -22 * x.abs().max()).all())
    assert near(c.out[:c.N].view(c.N, NH, HS), y[:, :NH]) and bool((c.out[c.N:] == 7).all())
    at = torch.cat([s[k - n:] for s, k, n in zip(c.flat, keys, new)])
    k, v = c.pool(c.kpages, 1), c.pool(c.vpages, 1)
    assert near(k[at], y[:, NH:]) and torch.equal(v[at], x[:, NH + NKV:])
    rest = torch.ones(k.shape[0], dtype=torch.bool)
    rest[at] = False
    for now, then in ((c.kpages, old[0]), (c.vpages, old[1])):
        assert torch.equal(c.pool(now, 1)[rest].nan_to_num(9.0), c.pool(then, 1)[rest].nan_to_num(9.0))
        assert torch.equal(now[0].nan_to_num(9.0), then[0].nan_to_num(9.0))


def test_append_gives_the_bits_of_the_rectangular_cache():
    B, Tq, start, NH, NKV, HS = 3, 5, 11, 8, 2, 64
    c = O.Case((16,) * B, (Tq,) * B, NH, NKV, HS, 16, device=DEV, pad=0)
    f = O.angles(64, HS, DEV)
    kc, vc = torch.zeros(B, 32, NKV, HS, device=DEV).bfloat16(), torch.zeros(B, 32, NKV, HS, device=DEV).bfloat16()
    q = torch.zeros_like(c.out)
    ops.rope_cache(q, kc, vc, c.raw, f, Tq, start, NH, NKV)
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, f, NH)
    assert torch.equal(q, c.out)
    for mine, other in ((c.kpages, kc), (c.vpages, vc)):
        assert torch.equal(torch.stack([mine[0].reshape(-1, NKV, HS)[s.to(DEV)][start:] for s in c.flat]), other[:, start:16])
    # at positions of one's own: the angles of those
    positions = torch.arange(B * Tq, dtype=torch.int32, device=DEV) * 3 % 17
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, f, NH, positions=positions)
    x = c.raw.cpu().double().view(B * Tq, -1, HS)[:, :NH]
    y = O.rotated(x, f.cpu()[positions.cpu().long()].double(), False).view(B * Tq, -1)
    assert bool(((c.out.cpu().double() - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -22 * x.abs().max()).all())


def test_append_reports_what_has_no_place():
    for name, at, value in (("table", (1, 0), -1), ("table", (1, 0), 1 << 20), ("lengths", 1, 2), ("lengths", 1, -1), ("lengths", 1, 10 ** 6), ("starts", 3, 2 ** 31 - 1)):
        c = O.Case((16, 9, 20), (3, 4, 2), 4, 2, 16, 16, device=DEV)
        getattr(c, name)[at] = value
        old = c.kpages.clone()
        ops.paged_rope_cache(c.out, c.cache(ops), c.raw, O.angles(64, 16, DEV), 4)
        assert _lib.read_status() >> 24 == 3
        changed = (c.pool(c.kpages).nan_to_num(9.0) != c.pool(old).nan_to_num(9.0)).any(-1).any(-1).nonzero().view(-1).tolist()
        allowed = torch.cat([s[k - n:] for s, k, n in zip(c.flat, c.keys, c.new)]).tolist()
        assert set(changed) <= set(allowed) and set(c.flat[0][-3:].tolist()) <= set(changed)
    for positions in ([0] * 8 + [64], [0] * 8 + [-1]):
        c = O.Case((16, 9, 20), (3, 4, 2), 4, 2, 16, 16, device=DEV, pad=0)
        ops.paged_rope_cache(c.out, c.cache(ops), c.raw, O.angles(64, 16, DEV), 4, positions=torch.tensor(positions, dtype=torch.int32, device=DEV))
        assert _lib.read_status() >> 24 == 3


@pytest.mark.parametrize("NKV,HS,rows,L,layout", [(2, 16, 8, 3, "rows"), (8, 128, 16, 2, "both"), (5, 72, 64, 1, "heads")])
def test_keep(NKV, HS, rows, L, layout):
    keys, new = (9, 33, 20, 12, 300, 64), (4, 33, 7, 0, 256, 64)
    c = O.Case(keys, new, NKV, NKV, HS, rows, layers=L, device=DEV, layout=layout)
    lists = [[1, 3], list(range(0, 33, 2)), [6, 6, 6], [], list(range(1, 256)), [0, 1, 2, 40, 41, 63]]
    kept = torch.zeros(6, 256, dtype=torch.int32)
    for b, l in enumerate(lists):
        kept[b, :len(l)] = torch.tensor(l, dtype=torch.int32)
    old = c.kpages.clone(), c.vpages.clone()
    ops.paged_keep(c.cache(ops), kept.to(DEV), torch.tensor([len(l) for l in lists], dtype=torch.int32, device=DEV))
    for then, now in zip(old, (c.kpages, c.vpages)):
        for layer in range(L):
            source = c.pool(then, layer)
            want = source.clone()
            for f, n, l in zip(c.flat, c.new, lists):
                base = len(f) - n
                for j, s in enumerate(l):
                    want[f[base + j]] = source[f[base + s]]
            assert torch.equal(c.pool(now, layer).nan_to_num(9.0), want.nan_to_num(9.0))


def test_keep_reports_lists_that_make_no_sense():
    for kept, counts in (([[1, 0], [1, 2]], [2, 2]), ([[1, 4], [1, 2]], [2, 2]), ([[1, 2], [1, 2]], [3, 2]), ([[1, 2], [1, 2]], [-1, 2]), ([[-1, 2], [1, 2]], [2, 2])):
        c = O.Case((20, 19), (4, 4), 2, 2, 16, 8, device=DEV)
        old = c.kpages.clone()
        ops.paged_keep(c.cache(ops), torch.tensor(kept, dtype=torch.int32, device=DEV), torch.tensor(counts, dtype=torch.int32, device=DEV))
        assert _lib.read_status() >> 24 == 3
        now, then = c.pool(c.kpages), c.pool(old)
        assert torch.equal(now[c.flat[0]], then[c.flat[0]])
        assert torch.equal(now[c.flat[1][15:17]], then[c.flat[1][16:18]])


def test_a_run_of_them():
    """Prompts enter, a tree of drafts is checked, part of it accepted, a single token follows; after each step against the oracle on what the pages hold."""
    NH, NKV, HS, f = 8, 2, 64, O.angles(400, 64, DEV)
    c = O.Case((150, 61, 230), (150, 61, 230), NH, NKV, HS, 16, device=DEV, layers=2)
    g = torch.Generator().manual_seed(3)

    def step(new, tree=None, positions=None):
        c.new, c.N = new, sum(new)
        c.keys = [k for k in keys]
        c.lengths.copy_(torch.tensor(keys, dtype=torch.int32))
        c.starts.copy_(torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32))
        c.raw = torch.randn(c.N + 2, (NH + 2 * NKV) * HS, generator=g).bfloat16().to(DEV)
        c.q, c.out = torch.zeros(c.N + 2, NH * HS, device=DEV).bfloat16(), torch.full((c.N + 2, NH * HS), 7.0, device=DEV).bfloat16()
        c.flat = [full[:k] for full, k in zip(slots, keys)]
        ops.paged_rope_cache(c.q, cache, c.raw, f, NH, layer=1, positions=positions)
        if tree is None:
            ops.paged_attention(c.out, c.q, cache, NH, layer=1)
        else:
            ops.paged_tree_attention(c.out, c.q, cache, tree.to(DEV), NH, layer=1)
        _check(c, tree, layer=1)

    slots, cache = c.flat, c.cache(ops)
    keys = [100, 40, 200]
    step([100, 40, 200])
    parents = [[-1, 0, 0, 1, 2], [-1], [-1, -1, 1, 2, 3, 0, 5]]
    keys = [k + len(p) for k, p in zip(keys, parents)]
    masks = ops.tree_masks(parents)
    depth = [bin(m & (1 << 64) - 1).count("1") - 1 for m in masks.tolist()] + [0, 0]
    context = [100] * 5 + [40] + [200] * 7 + [0, 0]
    step([5, 1, 7], torch.cat([masks, masks[:2]]), torch.tensor([d + k for d, k in zip(depth, context)], dtype=torch.int32, device=DEV))
    before = c.pool(c.kpages, 1)
    lists = [[0, 2, 4], [], [1, 2, 3]]
    kept = torch.tensor([l + [0] * (3 - len(l)) for l in lists], dtype=torch.int32, device=DEV)
    ops.paged_keep(cache, kept, torch.tensor([3, 0, 3], dtype=torch.int32, device=DEV))
    after = c.pool(c.kpages, 1)
    for b, l in enumerate(lists):
        for j, s in enumerate(l):
            assert torch.equal(after[slots[b][[100, 40, 200][b] + j]], before[slots[b][[100, 40, 200][b] + s]])
    keys = [104, 41, 204]
    step([1, 1, 1])
