"""Arguments that the head's operators cannot do without."""
import pytest
import torch

import linear_ce_oracle as O
from llmc_b200 import ops
from llmc_b200.ops import kernels as KN


@pytest.mark.parametrize("which", [ops, KN])
def test_losses_and_lse_are_needed(which):
    """Only the forward pass's lse may be left out.  (The launchers refuse before they ask for a GPU.)"""
    x, w, t = O.make(4, 16, 20)
    with pytest.raises(ValueError, match="losses"):
        which.linear_cross_entropy_forward(None, torch.zeros(4), x, w, t, 20)
    with pytest.raises(ValueError, match="lse"):
        which.linear_cross_entropy_backward(torch.zeros_like(x), None, x, w, t, None, 1.0, 20)
