"""Operators on a key / value cache in pages, at the ends of their ranges: many sequences, many heads, offsets that pass 32 bits, tables that are a part of a wider one, batches with rows behind
the last sequence, streams and graphs."""
import pytest
import torch

from llmc_b200 import _lib, ops
from llmc_b200.ops import kernels as KN

import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _near(got, exact, size):
    """Half a step of bf16 for the result, and as much of sum |p v| for probabilities rounded to bf16; 32-bit sums are far below the last term."""
    return bool(((got.cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -12) * size).all())


def _check(c, tree=None):
    exact, size = O.attention(c, tree)
    assert _near(c.out[:c.N], exact, size) and bool((c.out[c.N:] == 7).all())


@pytest.mark.parametrize("B", [33, 70, 300])
@pytest.mark.parametrize("kind", ["one", "few", "many", "tree"])
def test_many_sequences(B, kind):
    keys = [(i * 37) % 90 if i % 11 else 0 for i in range(B)]
    most = {"one": 1, "few": 3, "many": 40, "tree": 20}[kind]
    new = [min(k, 1 + (i * 7) % most) for i, k in enumerate(keys)]
    c = O.Case(keys, new, 4, 2, 64, 16, seed=B, device=DEV)
    if kind == "tree":
        tree = ops.tree_masks([O.random_tree(n, n) for n in new])
        ops.paged_tree_attention(c.out, c.q, c.cache(ops), torch.cat([tree, tree[:3]]).to(DEV), 4)
        _check(c, tree)
    else:
        ops.paged_attention(c.out, c.q, c.cache(ops), 4)
        _check(c)


def test_append_to_many_sequences():
    keys = [(i * 37) % 90 if i % 11 else 0 for i in range(300)]
    new = [min(k, i % 4) for i, k in enumerate(keys)]
    c = O.Case(keys, new, 4, 2, 16, 8, device=DEV)
    f = O.angles(90, 16, DEV)
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, f, 4)
    pos = torch.cat([torch.arange(k - n, k) for k, n in zip(keys, new)])
    x = c.raw[:c.N].cpu().double().view(c.N, 8, 16)
    y = O.rotated(x[:, :6], f.cpu()[pos].double(), False)
    near = lambda a, b: bool(((a.cpu().double() - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -22 * x.abs().max()).all())
    at = torch.cat([s[k - n:] for s, k, n in zip(c.flat, keys, new)])
    assert near(c.out[:c.N].view(c.N, 4, 16), y[:, :4]) and near(c.pool(c.kpages)[at], y[:, 4:]) and torch.equal(c.pool(c.vpages)[at], x[:, 6:])
    assert bool((c.out[c.N:] == 7).all())


@pytest.mark.parametrize("NH,NKV,HS,new", [(128, 1, 64, 1), (128, 1, 64, 3), (130, 1, 64, 1), (260, 2, 16, 5), (96, 32, 128, 1), (64, 64, 64, 9)])
def test_many_heads(NH, NKV, HS, new):
    c = O.Case((50, 140), (min(new, 50), new), NH, NKV, HS, 16, device=DEV, pad=1)
    ops.paged_attention(c.out, c.q, c.cache(ops), NH)
    _check(c)


@pytest.mark.parametrize("tokens,NH,NKV,HS", [(2500, 1, 1, 16), (700, 2, 1, 24), (1300, 40, 20, 128), (600, 6, 2, 40)])
def test_append_of_many_tokens(tokens, NH, NKV, HS):
    """More tokens than a block looks up at once, several tokens side by side, heads that are split over blocks."""
    c = O.Case((tokens, 300), (tokens, 299), NH, NKV, HS, 32, device=DEV)
    f = O.angles(tokens, 8, DEV)
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, f, NH)
    pos = torch.cat([torch.arange(tokens), torch.arange(1, 300)])
    x = c.raw[:c.N].cpu().double().view(c.N, NH + 2 * NKV, HS)
    y = O.rotated(x[:, :NH + NKV], f.cpu()[pos].double(), False)
    near = lambda a, b: bool(((a.cpu().double() - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -22 * x.abs().max()).all())
    at = torch.cat([c.flat[0], c.flat[1][1:]])
    assert near(c.out[:c.N].view(c.N, NH, HS), y[:, :NH]) and near(c.pool(c.kpages)[at], y[:, NH:]) and torch.equal(c.pool(c.vpages)[at], x[:, NH + NKV:])


def test_heads_that_do_not_group_are_refused():
    c = O.Case((600, 300), (600, 299), 3, 2, 40, 32, device=DEV)
    with pytest.raises(ValueError):
        ops.paged_rope_cache(c.out, c.cache(ops), c.raw, O.angles(600, 8, DEV), 3)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements whose last pages are in use."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 20 GB")
    small = O.Case((200, 33), (70, 33), 4, 2, 128, 16, device=DEV, layers=1)
    pages = (1 << 32) // (16 * 2 * 128) + 40
    pools = [torch.empty(1, pages, 16, 2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    shift = pages - small.kpages.shape[1]
    for pool, mine in zip(pools, (small.kpages, small.vpages)):
        pool[:, shift:].copy_(mine)
    table = torch.where(small.table < 1 << 20, small.table + shift, small.table)
    cache = ops.paged_cache(*pools, table, small.lengths, small.starts)
    ops.paged_attention(small.out, small.q, cache, 4)
    _check(small)
    one = O.Case((200, 33), (1, 1), 4, 2, 128, 16, device=DEV)
    for pool, mine in zip(pools, (one.kpages, one.vpages)):
        pool[:, shift:].copy_(mine)
    cache = ops.paged_cache(*pools, torch.where(one.table < 1 << 20, one.table + shift, one.table), one.lengths, one.starts)
    ops.paged_attention(one.out, one.q, cache, 4)
    _check(one)
    ops.paged_rope_cache(one.out, cache, one.raw, O.angles(200, 128, DEV), 4)
    v = one.raw[:2].view(2, 8, 128)[:, 6:]
    flat = pools[1][0, shift:].reshape(-1, 2, 128)
    assert torch.equal(flat[[int(one.flat[0][-1]), int(one.flat[1][-1])]], v)
    cache = ops.paged_cache(*pools, torch.where(one.table < 1 << 20, one.table + shift, one.table), one.lengths, torch.tensor([0, 3, 5], dtype=torch.int32, device=DEV))
    before = flat.clone()
    ops.paged_keep(cache, torch.tensor([[1, 2], [1, 0]], dtype=torch.int32, device=DEV), torch.tensor([2, 1], dtype=torch.int32, device=DEV))
    assert torch.equal(flat[one.flat[0][-3:-1].to(DEV)], before[one.flat[0][-2:].to(DEV)]) and torch.equal(flat[one.flat[1][-2].to(DEV)], before[one.flat[1][-1].to(DEV)])


@pytest.mark.parametrize("new", [(1, 1, 1), (40, 2, 9)])
def test_a_part_of_a_wider_table(new):
    c = O.Case((100, 30, 9), new, 4, 2, 64, 8, device=DEV)
    wide = torch.full((5, 40), -3, dtype=torch.int32, device=DEV)
    wide[1:4, 7:7 + c.table.shape[1]] = c.table
    cache = ops.paged_cache(c.kpages, c.vpages, wide[1:4, 7:7 + c.table.shape[1]], c.lengths, c.starts)
    ops.paged_attention(c.out, c.q, cache, 4)
    _check(c)


@pytest.mark.parametrize("new", [1, 30])
def test_nothing_cached(new):
    """Sequences without keys: rows of zeros; a table of no columns."""
    c = O.Case((0, 0), (0, 0), 4, 2, 64, 16, device=DEV, pad=2 * new + 2)
    c.starts.copy_(torch.tensor([0, new, 2 * new]))
    c.q.zero_()
    for table in (c.table, c.table[:, :0]):
        c.out.fill_(7.0)
        ops.paged_attention(c.out, c.q, ops.paged_cache(c.kpages, c.vpages, table, c.lengths, c.starts), 4)
        assert bool((c.out[:2 * new] == 0).all()) and bool((c.out[2 * new:] == 7).all())


@pytest.mark.parametrize("new", [1, 5, 60])
def test_a_batch_padded_with_rows(new):
    c = O.Case((90, 200), (new, new), 8, 2, 128, 16, device=DEV, pad=500)
    ops.paged_attention(c.out, c.q, c.cache(ops), 8)
    _check(c)
    # rows that are missing: the sequence is reported and left out
    ops.paged_attention(c.out[:new + 1], c.q[:new + 1], c.cache(ops), 8)
    assert (_lib.read_status() >> 24 == 3) == (new > 1)


def test_the_same_page_in_two_sequences():
    """A common beginning that is cached once."""
    c = O.Case((64, 64), (1, 30), 4, 2, 64, 16, device=DEV)
    c.table[1, :2] = c.table[0, :2]
    c.flat[1] = torch.cat([c.flat[0][:32], c.flat[1][32:]])
    ops.paged_attention(c.out, c.q, c.cache(ops), 4)
    _check(c)


def test_streams_and_threads():
    import threading
    cases = [O.Case((500 + i, 77), (n, n), 8, 2, 128, 16, seed=i, device=DEV) for i, n in enumerate((1, 3, 64, 1))]
    want = []
    for c in cases:
        ops.paged_attention(c.out, c.q, c.cache(ops), 8)
        want.append(c.out.clone())
        c.out.fill_(7.0)
    torch.cuda.synchronize()
    wrong = []

    def work(c, w, own):
        stream = torch.cuda.Stream() if own else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            cache = c.cache(ops)
            for _ in range(50):
                c.out.fill_(7.0)
                ops.paged_attention(c.out, c.q, cache, 8)
                if not torch.equal(c.out, w):
                    wrong.append(c.new)

    for own in (True, False):
        threads = [threading.Thread(target=work, args=(c, w, own)) for c, w in zip(cases, want)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not wrong


def test_a_step_in_a_graph():
    """Append, attention, tree attention and keep of one captured step, replayed with other lengths, masks and kept tokens."""
    c = O.Case((60, 200), (6, 6), 8, 2, 64, 16, device=DEV, pad=0, layers=2)
    f = O.angles(256, 64, DEV)
    cache = c.cache(ops)
    tree = torch.zeros(12, dtype=torch.int64, device=DEV)
    positions = torch.zeros(12, dtype=torch.int32, device=DEV)
    kept, counts = torch.zeros(2, 6, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    q, plain, treed = (torch.zeros_like(c.q) for _ in range(3))

    def step():
        for layer in range(2):
            ops.paged_rope_cache(q, cache, c.raw, f, 8, layer=layer, positions=positions)
            ops.paged_attention(plain, q, cache, 8, layer=layer)
            ops.paged_tree_attention(treed, q, cache, tree, 8, layer=layer)
        ops.paged_keep(cache, kept, counts)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with KN.scratch_taken() as held, torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    start = c.kpages.clone(), c.vpages.clone()
    for lengths, lists in (([60, 200], [[0, 2], [1, 3, 5]]), ([40, 150], [[], [5]]), ([6, 199], [[0, 1, 2, 3, 4, 5], [2]])):
        c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        trees = [O.random_tree(6, lengths[0]), O.random_tree(6, lengths[1])]
        masks = ops.tree_masks(trees)
        tree.copy_(masks)
        positions.copy_(torch.tensor([lengths[i // 6] - 6 + bin(int(m)).count("1") - 1 for i, m in enumerate(masks)], dtype=torch.int32))
        counts.copy_(torch.tensor([len(l) for l in lists], dtype=torch.int32))
        kept.zero_()
        for b, l in enumerate(lists):
            kept[b, :len(l)] = torch.tensor(l, dtype=torch.int32)
        results = []
        for run in (step, graph.replay):
            c.kpages.copy_(start[0]), c.vpages.copy_(start[1])
            for t in (q, plain, treed):
                t.zero_()
            run()
            results.append([t.clone() for t in (q, plain, treed, c.kpages, c.vpages)])
        for a, b in zip(*results):
            assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))
    assert held is not None


def test_other_devices_and_streams_are_refused_or_followed():
    c = O.Case((20,), (1,), 2, 2, 64, 16, device=DEV)
    with pytest.raises(ValueError):
        ops.paged_attention(c.out, c.q.cpu(), c.cache(ops), 2)
    with pytest.raises(ValueError):
        ops.paged_cache(c.kpages, c.vpages, c.table.cpu(), c.lengths, c.starts)
    with pytest.raises(ValueError):
        ops.paged_rope_cache(c.out, c.cache(ops), c.raw, O.angles(64, 64), 2)
    with pytest.raises(ValueError):
        ops.paged_keep(c.cache(ops), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32, device=DEV))


def test_fp32_pages_on_a_device():
    c = O.Case((40, 17), (3, 17), 4, 2, 24, 8, device=DEV, dtype=torch.float32)
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, O.angles(64, 24, DEV), 4)
    ops.paged_attention(c.out, c.q, c.cache(ops), 4)
    exact, size = O.attention(c)
    assert bool(((c.out[:c.N].cpu().double() - exact).abs() <= 2.0 ** -23 * exact.abs() + 2.0 ** -14 * size).all())


@pytest.mark.parametrize("N,heads", [(1024, 1), (2048, 19)])
def test_starts_that_claim_rows_many_times(N, heads):
    """32 sequences that claim all rows, over 2^26 keys each (of one page): more units of work than 32-bit counts hold.  The call does nothing and says so."""
    B, rows, width = 96, 1024, 1 << 16
    pages = torch.zeros(2, 1, rows, heads, 16, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda").expand(B, width)
    lengths = torch.full((B,), rows * width, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0] + [0, N, 0] * 32, dtype=torch.int32, device="cuda")
    q = torch.zeros(N, heads * 16, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 7.0)
    ops.paged_attention(out, q, ops.paged_cache(pages[0], pages[1], table, lengths, starts), heads)
    torch.cuda.synchronize()
    assert _lib.read_status() >> 24 == 3
    assert bool((out == 7.0).all())
