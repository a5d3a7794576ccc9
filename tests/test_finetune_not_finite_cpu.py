"""A batch whose gradient is not finite leaves a head that is trained alone as it was, on the host."""
import pytest
import torch

from llmc_b200 import finetune_head
from llmc_b200.models import llama3


def spoiled_step(device, dtype, value):
    """A step whose head gradient has one such element; parameters and state of the optimizer before, after, and after a step like any other."""
    cfg = llama3.config_from_descriptor("llama3:l=1,c=128,h=2,kv=1,t=32,v=200,m=16,f=1.0")
    m = llama3.Llama(cfg, device, dtype, head_pieces=True)
    m.init_random(42)
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randint(0, 200, (2, 32), generator=g, dtype=torch.int32) for _ in range(2))
    tuner = finetune_head.HeadTuner(m)
    state = lambda: [t.clone() for t in (m.params_flat, tuner.master, tuner.m, tuner.v)]
    tuner.step(x.to(device), y, 1e-2)
    before = state()
    clip = finetune_head.ops.clip_grad_norm

    def spoil(norm, plan, limit):
        tuner.head_grad[3, 5] = value
        clip(norm, plan, limit)

    try:
        finetune_head.ops.clip_grad_norm = spoil
        norm = float(tuner.step(x.to(device), y, 1e-2)[1])
    finally:
        finetune_head.ops.clip_grad_norm = clip
    after = state()
    loss = float(tuner.step(x.to(device), y, 1e-2)[0])
    return norm, before, after, state(), loss


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_gradient_that_is_not_finite(value):
    norm, before, after, later, loss = spoiled_step("cpu", torch.float32, value)
    assert norm != norm or norm == float("inf")
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert all(torch.isfinite(a).all() and not torch.equal(a, b) for a, b in zip(later, after)) and loss == loss
