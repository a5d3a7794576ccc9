"""Targets that are left out of a step that trains a head alone."""
import torch

from llmc_b200 import finetune_head
from llmc_b200.models import llama3


def test_targets_past_the_vocabulary_are_left_out_of_the_mean():
    """Like negative ones: the loss is the mean over the tokens that count."""
    cfg = llama3.config_from_descriptor("llama3:l=1,c=64,h=4,kv=2,t=32,v=200,m=16,f=1.0")
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randint(0, 200, (2, 16), generator=g, dtype=torch.int32) for _ in range(2))
    results = []
    for out in (-1, 200, 10 ** 6):
        m = llama3.Llama(cfg, "cpu", torch.float32, head_pieces=True)
        m.init_random(42)
        z = y.clone()
        z[:, :6] = out
        results.append([float(v) for v in finetune_head.HeadTuner(m).step(x, z, 1e-2)] + [m.params_flat.clone()])
    for r in results[1:]:
        assert r[:2] == results[0][:2] and torch.equal(r[2], results[0][2])
