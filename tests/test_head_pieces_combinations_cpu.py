"""What does not go together with a model that keeps no logits is refused before anything is computed or written."""
import importlib.util
import os

import pytest
import torch

from llmc_b200.models import gpt2


def _script(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(os.path.dirname(__file__), "..", name + ".py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_writing_tensors_needs_logits(tmp_path):
    script = _script("train_llama3")
    args = ["--model", "llama3:l=1,c=64,h=2,kv=1,t=32,v=200,m=16,f=1.0", "--output_dir", str(tmp_path / "out"), "--write_tensors", "1"]
    parse = lambda a: script.train_config(script.build_parser().parse_args(a))
    with pytest.raises(SystemExit, match="write_tensors"):
        parse(args + ["--head_pieces", "1"])
    assert parse(args).head_pieces == 0 and not (tmp_path / "out").exists()


def test_fp32_on_a_gpu():
    """GPT-2's full-precision mode runs on kernels of its own, the classifier among them; none of them forms the head in pieces."""
    cfg = gpt2.GPTConfig(max_seq_len=32, vocab_size=200, padded_vocab_size=256, num_layers=1, num_heads=2, channels=32)
    with pytest.raises(ValueError, match="head_pieces"):
        gpt2.GPT(cfg, "cuda:0", torch.float32, head_pieces=True)
    assert gpt2.GPT(cfg, "cpu", torch.float32, head_pieces=True).head_pieces
