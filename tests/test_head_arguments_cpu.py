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


def test_arguments_by_name():
    """The argument that decides where the operators run may be given by its name, as the others."""
    x, w, t = O.make(4, 16, 20, dtype=torch.float32)
    a, b, lse = torch.zeros(4), torch.zeros(4), torch.zeros(4)
    ops.linear_cross_entropy_forward(a, lse, x, w, t, 20)
    ops.linear_cross_entropy_forward(losses=b, lse=None, inp=x, weight=w, targets=t, V=20)
    assert torch.equal(a, b)
    dinp, dw, other = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(x)
    ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, 0.5, 20)
    ops.linear_cross_entropy_backward(dinp=other, dweight=None, inp=x, weight=w, targets=t, lse=lse, dloss=0.5, V=20)
    assert torch.equal(dinp, other)
    ops.gelu_forward(out=other, inp=x)
    assert torch.allclose(other, torch.nn.functional.gelu(x, approximate="tanh"), atol=1e-6)
