"""Attention of few rows over a cache in pages keeps 16 bits of a probability: a bound that 8 bits miss (test_paged_bits_cpu.py)."""
import pytest
import torch

from llmc_b200 import _lib, ops

import paged_bits
import paged_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("args", paged_bits.CASES)
def test_sixteen_bits_of_a_probability(args, tree):
    c = paged_bits.case(*args, device="cuda")
    masks = None
    if tree:
        masks = ops.tree_masks([O.random_tree(n, i) for i, n in enumerate(c.new)])
        ops.paged_tree_attention(c.out, c.q, c.cache(ops), masks.cuda(), c.NH)
    else:
        ops.paged_attention(c.out, c.q, c.cache(ops), c.NH)
    assert _lib.read_status() == 0
    exact, size = O.attention(c, masks)
    off = (c.out.cpu().double() - exact).abs() / paged_bits.bound(c, exact, size)
    assert float(off.max()) <= 1, float(off.max())
