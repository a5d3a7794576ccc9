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
