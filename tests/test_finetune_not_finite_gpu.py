"""A batch whose gradient is not finite leaves a head that is trained alone as it was, on the sm_100a kernels."""
import pytest
import torch

from test_finetune_not_finite_cpu import spoiled_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_gradient_that_is_not_finite(value):
    norm, before, after, later, loss = spoiled_step("cuda:0", torch.bfloat16, value)
    assert norm != norm or norm == float("inf")
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert all(torch.isfinite(a).all() and not torch.equal(a, b) for a, b in zip(later, after)) and loss == loss
