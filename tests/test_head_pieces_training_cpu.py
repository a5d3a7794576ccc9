"""Training without a logits buffer through the trainer and on several ranks, on the host."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from llmc_b200.train import TrainConfig, Trainer
from llmc_b200.utils.dataloader import write_datafile

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("model,kind", [("llama3:l=2,c=32,h=4,kv=2,t=16,v=300,m=16,f=1.3", "llama-3"), ("d2", "gpt-2")])
def test_trainer(tmp_path, model, kind):
    """Steps of two micro-steps, validation and sampling give what they give with logits: the same losses but for fp32 sums in another order."""
    from llmc_b200.models import gpt2
    if kind == "gpt-2":
        from llmc_b200.utils import checkpoint
        m = gpt2.GPT(gpt2.GPTConfig(max_seq_len=16, vocab_size=300, padded_vocab_size=384, num_layers=2, num_heads=2, channels=32), "cpu", torch.float32)
        m.init_random(42)
        model = str(tmp_path / "start.bin")
        checkpoint.write_model(model, m)
    rng = np.random.default_rng(0)
    write_datafile(str(tmp_path / "train.bin"), rng.integers(0, 300, size=4000), kind)
    write_datafile(str(tmp_path / "val.bin"), rng.integers(0, 300, size=600), kind)
    results = []
    for pieces in (0, 1):
        t = Trainer(TrainConfig(train_data_pattern=str(tmp_path / "train.bin"), val_data_pattern=str(tmp_path / "val.bin"), load_filename=model, output_log_dir=str(tmp_path / ("log%d" % pieces)),
                                B=2, T=16, total_batch_size=64, max_steps=4, learning_rate=1e-3, val_loss_every=2, val_max_steps=2, sample_every=3, genT=8, device="cpu", dtype="fp32", quiet=True,
                                tokenizer_path=str(tmp_path / "none.bin"), head_pieces=pieces))
        try:
            t.run()
            assert t.model.head_pieces == bool(pieces) and ("logits" in t.model.acts) != bool(pieces)
            results.append((t.validate(), t.model.params_flat.clone()))
        finally:
            t.close()
    assert abs(results[0][0] - results[1][0]) < 1e-4
    # AdamW divides by sqrt(v): a gradient near 0 whose sum differs in its last bits may move by a fraction of the learning rate
    diff = (results[0][1] - results[1][1]).abs()
    assert (diff > 1e-4).float().mean().item() < 1e-3 and diff.max().item() < 5e-3


@pytest.mark.parametrize("family,zero,port", [("gpt2", 0, 29641), ("gpt2", 1, 29642), ("llama3", 1, 29643)])
def test_two_ranks_match_a_single_process_with_logits(tmp_path, family, zero, port):
    single, multi = str(tmp_path / "single.pt"), str(tmp_path / "multi.pt")
    env = dict(os.environ, OMP_NUM_THREADS="2")
    args = ["--device", "cpu", "--slots", "2", "--family", family]
    for cmd in ([sys.executable, os.path.join(HERE, "dist_worker.py"), "--out", single, "--zero", "0"] + args,
                [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1", "--master-port", str(port),
                 os.path.join(HERE, "head_pieces_dist_worker.py"), "--out", multi, "--zero", str(zero)] + args):
        r = subprocess.run(cmd, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
        assert r.returncode == 0, r.stdout[-2000:]
    a, b = torch.load(single), torch.load(multi)
    assert b["zero"] == zero and max(abs(x - y) for x, y in zip(a["losses"], b["losses"])) < 1e-4
    diff = (a["params"] - b["params"]).abs()
    assert (diff > 1e-4).float().mean().item() < 1e-3 and diff.max().item() < 5e-3
