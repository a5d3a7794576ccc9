"""Attention over a key / value cache in pages, cut in each way that its kernels know: groups of 8 or 16 rows, or row tiles of 128; shares of a warp or of a block; few pieces, about as many as
SMs, and many; heads of whole chunks of channels and others."""
import pytest
import torch

from llmc_b200 import _lib, ops

import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(c, tree=None):
    """Half a step of bf16 for the result, and as much of sum |p v| for probabilities rounded to bf16; 32-bit sums are far below the last term."""
    exact, size = O.attention(c, tree)
    assert bool(((c.out[:c.N].cpu().double() - exact).abs() <= 2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -12) * size).all())
    assert bool((c.out[c.N:] == 7).all())


# sequences, new tokens of one at most, query and cached heads
CUTS = [(2, 1, 4, 4), (16, 1, 24, 12), (40, 1, 24, 24), (2, 12, 4, 4), (12, 12, 12, 12), (20, 3, 32, 8), (1, 3, 32, 8), (1, 12, 32, 8), (1, 13, 32, 8), (9, 4, 32, 8), (1, 48, 2, 2), (1, 49, 2, 2), (4, 30, 6, 2),
        (3, 5, 16, 1), (2, 64, 8, 4)]


@pytest.mark.parametrize("HS", [64, 128, 40, 104])
@pytest.mark.parametrize("B,new,NH,NKV", CUTS)
def test_trees(B, new, NH, NKV, HS):
    g = torch.Generator().manual_seed(B * 100 + new)
    counts = [new] + torch.randint(0, new + 1, (B - 1,), generator=g).tolist()
    keys = [n + int(k) for n, k in zip(counts, torch.randint(0, 700, (B,), generator=g))]
    keys[-1] = counts[-1]                                   # nothing in front of the new tokens
    c = O.Case(keys, counts, NH, NKV, HS, 16, seed=new, device=DEV)
    parents = [O.random_tree(n, i) for i, n in enumerate(counts)]
    tree = ops.tree_masks(parents)
    tree[0] = 0                                             # sees only what was cached before
    masks = torch.cat([tree, torch.zeros(3, dtype=torch.int64)]).to(DEV)
    ops.paged_tree_attention(c.out, c.q, c.cache(ops), masks, NH)
    _check(c, tree)
    assert _lib.read_status() == 0


@pytest.mark.parametrize("HS", [64, 128])
@pytest.mark.parametrize("B,new,NH,NKV", CUTS)
def test_parts_of_prompts(B, new, NH, NKV, HS):
    g = torch.Generator().manual_seed(B * 100 + new)
    counts = torch.randint(0, new + 1, (B - 1,), generator=g).tolist() + [new]
    keys = [n + int(k) for n, k in zip(counts, torch.randint(0, 900, (B,), generator=g))]
    c = O.Case(keys, counts, NH, NKV, HS, 32, seed=new, device=DEV, layout="heads")
    ops.paged_attention(c.out, c.q, c.cache(ops), NH)
    _check(c)
    assert _lib.read_status() == 0


@pytest.mark.parametrize("HS", [64, 128])
@pytest.mark.parametrize("new", [1, 6])
def test_results_do_not_depend_on_the_run(HS, new):
    c = O.Case([3000, 17, 0, 911], [new, new, 0, new], 8, 2, HS, 16, device=DEV)
    cache = c.cache(ops)
    ops.paged_attention(c.out, c.q, cache, 8)
    first = c.out.clone()
    for _ in range(20):
        c.out.fill_(7.0)
        ops.paged_attention(c.out, c.q, cache, 8)
        assert torch.equal(c.out, first)
