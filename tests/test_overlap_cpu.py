"""Outputs that share memory with what is still read are refused, before anything is written; those that lie between the rows of an input are not."""
import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops


def test_clipping_refuses_tensors_that_overlap():
    a, b = torch.ones(64), torch.ones(64)
    for outs, grads in [(None, [a, a]), (None, [a, a[10:20]]), ([a[8:40], b[:32]], [a[:32], a[32:]]), ([b, b], [a, a.clone()]), ([b[:32], b[31:63]], [a[:32], a[32:]])]:
        with pytest.raises(ValueError, match="overlap"):
            ops.clip_plan(outs, grads)
    ops.clip_plan([a[:32], b[:32]], [a[:32], a[32:]])            # one in place, one not
    ops.clip_plan(None, [a[:0], a, a[5:5]])                      # empty ones overlap nothing
