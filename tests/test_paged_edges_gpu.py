"""Operators on a key / value cache in pages on a GPU, where a call is larger, or its numbers are less ordinary, than those that the other tests make."""
import pytest
import torch

from llmc_b200 import _lib, ops
from llmc_b200.ops import kernels as KN

import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("NH,sequences", [(128, 2100), (64, 4200)])
def test_many_rows_of_many_grouped_heads(NH, sequences):
    """More than 65536 pairs of row tiles in one call, of short sequences: the limit on units is what counts."""
    new, HS, rows, cached = 64, 16, 16, 10
    N = sequences * new
    assert N * NH // 256 > 65536
    g = torch.Generator(device=DEV).manual_seed(NH)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.bfloat16)
    keys = [new + i % cached for i in range(sequences)]
    width = -(-(new + cached) // rows)
    table = torch.randperm(sequences * width, generator=g, device=DEV).to(torch.int32).view(sequences, width)
    kpages, vpages, q = normal(sequences * width, rows, 1, HS), normal(sequences * width, rows, 1, HS), normal(N, NH * HS)
    out = torch.full_like(q, 7.0)
    lengths, starts = torch.tensor(keys, dtype=torch.int32, device=DEV), torch.arange(0, N + 1, new, dtype=torch.int32, device=DEV)
    ops.paged_attention(out, q, ops.paged_cache(kpages, vpages, table, lengths, starts), NH)
    assert _lib.read_status() == 0
    # all sequences at once, a padded rectangle of keys; in 64 bits, some sequences at a time
    for b0 in range(0, sequences, 300):
        b1 = min(sequences, b0 + 300)
        K, V = (p[table[b0:b1].long()].view(b1 - b0, width * rows, HS).double() for p in (kpages, vpages))
        seen = torch.arange(width * rows, device=DEV) <= (lengths[b0:b1, None, None] - new + torch.arange(new, device=DEV)[None, :, None])
        for h0 in range(0, NH, 16):
            mine = slice(h0 * HS, (h0 + 16) * HS)
            z = torch.einsum("bnhd,bkd->bhnk", q[b0 * new:b1 * new, mine].double().view(b1 - b0, new, 16, HS), K) / HS ** 0.5
            p = torch.softmax(z.masked_fill(~seen[:, None], -float("inf")), -1)
            exact, size = torch.einsum("bhnk,bkd->bnhd", p, V), torch.einsum("bhnk,bkd->bnhd", p, V.abs())
            got = out[b0 * new:b1 * new, mine].double().view(exact.shape)
            # half a step of bf16 for the result and for the probabilities; sums of at most 80 products in 32 bits are far below the last term
            assert bool(((got - exact).abs() <= 2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -12) * size).all()), (b0, h0)


@pytest.mark.parametrize("new", [1, 6, 200])
def test_graphs_of_two_owners_at_the_same_time(new):
    cases = [O.Case((3000 + 500 * i, 700, 260), (new,) * 3, 8, 2, 128, 16, seed=i, device=DEV, pad=0) for i in range(2)]
    want, graphs, streams, held = [], [], [], []
    for c in cases:
        cache = c.cache(ops)
        ops.paged_attention(c.out, c.q, cache, 8)
        want.append(c.out.clone())
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), KN.scratch_taken() as taken, torch.cuda.graph(graph, stream=stream):
            for _ in range(20):
                ops.paged_attention(c.out, c.q, cache, 8)
        graphs.append(graph), streams.append(stream), held.append((taken, cache))
    for _ in range(20):
        for c in cases:
            c.out.fill_(7.0)
        for graph, stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        assert all(torch.equal(c.out, w) for c, w in zip(cases, want))
    # the graphs have the memory, not the list that owners keep
    assert not any(taken for taken, _ in held)


# (new tokens of a sequence: single tokens, groups of 16 rows, row tiles; cached keys: whole pieces, pieces that are cut and joined)
@pytest.mark.parametrize("HS", [64, 128])
@pytest.mark.parametrize("new,NH,NKV", [(1, 2, 2), (1, 8, 1), (3, 8, 2), (12, 2, 2), (50, 4, 1), (64, 2, 2)])
@pytest.mark.parametrize("cached", [0, 60, 3000])
@pytest.mark.parametrize("tree", [False, True])
def test_numbers_that_are_not_finite(new, NH, NKV, HS, cached, tree):
    """A query that is not a number, scores past 32 bits, and visible scores that are all minus infinity give no number, as a softmax does; a single score of minus infinity is a weight of 0; only a row
    without a key is 0.  The rows beside them are what they are."""
    c = O.Case((cached + new, 40 + new, new + 7), (new,) * 3, NH, NKV, HS, 16, seed=new, device=DEV, layers=1)
    heads = c.q[:c.N].view(c.N, NH, HS)
    heads[:, :, 0] = 0
    pages = c.kpages[0].view(-1, NKV, HS)
    first, second = (f.to(DEV) for f in c.flat[:2])
    pages[first, :, 0] = 1e38                            # every key of the first sequence, one of the second
    pages[second, :, 0] = 0
    pages[second[5], :, 0] = 1e38
    odd = torch.zeros(c.N, NH, dtype=torch.bool, device=DEV)
    heads[new - 1, 0, 0] = -1e38                         # all scores minus infinity
    odd[new - 1, 0] = True
    heads[new - 1, NH - 1, 0] = 1e38                     # infinity
    odd[new - 1, NH - 1] = True
    heads[new:2 * new, NH - 1, 0] = -1e38                # minus infinity at one key
    heads[3 * new - 1, 1, 2] = float("nan")
    odd[3 * new - 1, 1] = True
    masks = None
    if tree:
        masks = ops.tree_masks([O.random_tree(new, i) for i in range(3)])
        ops.paged_tree_attention(c.out, c.q, c.cache(ops), torch.cat([masks, masks[:3]]).to(DEV), NH)
    else:
        ops.paged_attention(c.out, c.q, c.cache(ops), NH)
    assert _lib.read_status() == 0
    got = c.out[:c.N].view(c.N, NH, HS)
    assert torch.equal(got.isnan().all(-1), odd) and torch.equal(got.isnan().any(-1), odd)
    # the oracle without the odd rows, and without the key that has no weight
    heads[odd] = 0
    heads[:, :, 0] = 0
    exact, size = O.attention(c, masks)
    gap = O.Case(c.keys, c.new, NH, NKV, HS, 16, seed=new, layers=1)
    gap.flat[1] = torch.cat([gap.flat[1][:5], gap.flat[1][6:]])          # (a cached key: all rows see it)
    gap.keys[1] -= 1
    gap.q.copy_(c.q)
    e, s = O.attention(gap, masks)
    rows, h = slice(new, 2 * new), slice((NH - 1) * HS, NH * HS)
    exact[rows, h], size[rows, h] = e[rows, h], s[rows, h]
    near = (got.double().cpu().view(c.N, -1) - exact).abs() <= 2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -12) * size
    assert bool((near.view(c.N, NH, HS).all(-1) | odd.cpu()).all())


@pytest.mark.parametrize("new,NH,NKV", [(1, 8, 2), (9, 8, 2), (64, 8, 2)])
def test_rows_without_a_key_beside_scores_of_minus_infinity(new, NH, NKV):
    """More new tokens than keys, masks that leave a row empty: 0, though scores that others see are minus infinity."""
    HS = 64
    c = O.Case((new, new, 900), (new, new, new), NH, NKV, HS, 16, device=DEV, pad=0)
    c.lengths[0] = new // 2
    heads, pages = c.q.view(c.N, NH, HS), c.kpages[0].view(-1, NKV, HS)
    for f in c.flat:
        pages[f.to(DEV), :, 0] = 1e38
    heads[:, :, 0] = -1e38
    ops.paged_attention(c.out, c.q, c.cache(ops), NH)
    none = new - new // 2
    assert bool((c.out[:none] == 0).all()) and bool(c.out[none:].isnan().all())
    masks = ops.tree_masks([O.random_tree(new, i) for i in range(3)])
    masks[new] = 0
    masks[:none] &= (1 << none) - 1                      # (of the first sequence, new tokens that have no slot)
    masks[2 * new:] = 0
    ops.paged_tree_attention(c.out, c.q, c.cache(ops), masks.to(DEV), NH)
    seen = [(m & (1 << 64) - 1) >> none > 0 for m in masks[:new].tolist()]
    assert c.out[:new].isnan().all(-1).tolist() == seen and bool((c.out[:new][~torch.tensor(seen, device=DEV)] == 0).all())
    assert bool((c.out[new] == 0).all()) and bool(c.out[new + 1:].isnan().all())
