"""Training without a logits buffer through the trainer, on the sm_100a kernels."""
import numpy as np
import pytest
import torch

from llmc_b200.train import TrainConfig, Trainer
from llmc_b200.utils.dataloader import write_datafile

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model,kind", [("llama3:l=2,c=128,h=2,kv=1,t=64,v=1003,m=64,f=1.0", "llama-3"), ("d6", "gpt-2")])
@pytest.mark.parametrize("recompute", [0, 2])
def test_trainer(tmp_path, model, kind, recompute):
    """Two micro-steps a step, validation and sampling between them.  The losses of a few steps stay with those of a model with logits, which rounds each of them to bf16 (2^-8 of a logit, a
    loss by twice that of the largest; logits of a model that has just been initialised are below 4)."""
    V = 1003
    rng = np.random.default_rng(0)
    write_datafile(str(tmp_path / "train.bin"), rng.integers(0, V, size=8000), kind)
    write_datafile(str(tmp_path / "val.bin"), rng.integers(0, V, size=2000), kind)
    results = []
    for pieces in (0, 1):
        torch.manual_seed(0)
        t = Trainer(TrainConfig(train_data_pattern=str(tmp_path / "train.bin"), val_data_pattern=str(tmp_path / "val.bin"), load_filename=model, output_log_dir=str(tmp_path / ("log%d" % pieces)),
                                B=4, T=64, total_batch_size=512, max_steps=6, learning_rate=1e-4, val_loss_every=2, val_max_steps=2, sample_every=3, genT=8, quiet=True, recompute=recompute,
                                tokenizer_path=str(tmp_path / "none.bin"), head_pieces=pieces))
        try:
            first = t.validate()
            t.run()
            assert t.model.head_pieces == bool(pieces) and ("logits" in t.model.acts) != bool(pieces)
            results.append((first, t.validate()))
        finally:
            t.close()
    for a, b in zip(*results):
        assert abs(a - b) <= 2 * 2.0 ** -8 * 4
    assert results[1][1] < results[1][0]
