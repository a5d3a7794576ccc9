"""Operators on a key / value cache in pages, on the host: numbers that are not finite, memory that is shared, what a refused call leaves behind."""
import math

import pytest
import torch

from llmc_b200 import _lib, ops
from llmc_b200.ops import kernels as KN

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


def test_angles_off_8_bytes_are_refused():
    """A cosine and its sine are read together.  On the host before a launch, by the operator and by the entry point alike; host tensors may lie anywhere."""
    c = O.Case((20, 9), (4, 2), 2, 1, 16, 8, pad=0)
    room = torch.zeros(30 * 8 * 2 + 1)
    f = room[1:].view(30, 8, 2)
    f.copy_(O.angles(30, 16))
    assert f.is_contiguous() and f.data_ptr() % 8 == 4
    cache = c.cache(KN)
    with pytest.raises(ValueError, match="8-byte"):
        KN.paged_rope_cache(c.out, cache, c.raw, f, 2)
    call = KN._pack_append(cache.address, c.out.data_ptr(), c.raw.data_ptr(), f.data_ptr(), 0, c.N, 32, 64, 2, 16, 30, 0, 0, 0)
    assert _lib.cuda().llmc_paged_rope_cache(call) == -1
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, f, 2)
    plain = torch.empty_like(c.out)
    ops.paged_rope_cache(plain, c.cache(ops), c.raw, O.angles(30, 16), 2)
    assert torch.equal(c.out, plain)
