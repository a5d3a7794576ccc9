"""Operators on a key / value cache in pages, on the host: numbers that are not finite, memory that is shared, what a refused call leaves behind."""
import math

import pytest
import torch

from llmc_b200 import ops

import paged_oracle as O

BF16 = torch.bfloat16


@pytest.mark.parametrize("tree", [False, True])
def test_numbers_that_are_not_finite_stay(tree):
    """A query that is not a number, scores that 32 bits do not hold, and visible scores that are all minus infinity give what a softmax gives: no number.  Only a row that sees no key is 0."""
    c = O.Case((20, 9, 4), (3, 2, 4), 2, 1, 16, 8, dtype=torch.float32, pad=0)
    c.q[1, 3] = math.nan                                 # head 0 of token 1
    c.q[3] = 1e30                                        # every key of the second sequence: scores past 32 bits
    c.kpages[0].view(-1, 1, 16)[c.flat[1]] = 1e30
    c.q[4] = -1e30
    c.lengths[2] = 2                                     # four new tokens, two slots: the first two have none
    masks = ops.tree_masks([[-1, 0, 1], [-1, 0], [-1, 0, 1, 2]])
    if tree:
        masks[5:7] = 0
        ops.paged_tree_attention(c.out, c.q, c.cache(ops), masks, 2)
    else:
        ops.paged_attention(c.out, c.q, c.cache(ops), 2)
    wrong = c.out.isnan().view(9, 2, 16).all(-1)
    assert wrong.tolist() == [[False, False], [True, False], [False, False], [True, True], [True, True]] + [[False, False]] * 4
    assert bool((c.out[5:7] == 0).all()) and bool((c.out[7:] != 0).all())
    assert not bool(c.out.isinf().any())
