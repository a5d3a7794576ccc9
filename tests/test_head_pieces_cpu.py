"""Models without a logits buffer, and training of a head alone, on the host."""
import pytest
import torch

from llmc_b200 import finetune_head
from llmc_b200.models import gpt2, llama3
from llmc_b200.ops import reference as RF
from llmc_b200.train import parse_args
from llmc_b200.utils import checkpoint
from llmc_b200.utils.dataloader import write_datafile


def _pair(family):
    if family == "gpt2":
        cfg = gpt2.GPTConfig(max_seq_len=32, vocab_size=200, padded_vocab_size=256, num_layers=2, num_heads=2, channels=32)
        make = lambda **k: gpt2.GPT(cfg, "cpu", torch.float32, **k)
    else:
        cfg = llama3.config_from_descriptor("llama3:l=2,c=64,h=4,kv=2,t=32,v=200,m=16,f=1.0")
        make = lambda **k: llama3.Llama(cfg, "cpu", torch.float32, **k)
    a, b = make(), make(head_pieces=True)
    a.init_random(3)
    b.params_flat.copy_(a.params_flat)
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randint(0, 200, (2, 16), generator=g, dtype=torch.int32) for _ in range(2))
    return a, b, x, y


@pytest.mark.parametrize("family", ["gpt2", "llama3"])
def test_model_without_logits(family, monkeypatch):
    """Same losses and gradients, fp32 sums in another order: a few eps of sums of 200 logits and 32 rows."""
    monkeypatch.setattr(RF, "HEAD_PIECE", 64)
    a, b, x, y = _pair(family)
    for micro in range(2):
        for m in (a, b):
            m.forward(x, y, grad_accum_steps=2, micro_step=micro)
            m.backward(micro_step=micro)
    assert "logits" not in b.acts and b.activation_bytes() < a.activation_bytes()
    assert torch.allclose(a.acts["losses"], b.acts["losses"], rtol=1e-5, atol=0)
    for n in a.grads:
        scale = float(a.grads[n].abs().max())
        assert torch.allclose(a.grads[n], b.grads[n], rtol=0, atol=2e-5 * scale), n
    b.forward(x)
    with pytest.raises(ValueError):
        b.logits()
    with pytest.raises(ValueError):
        b.backward()


def test_flag():
    assert parse_args(["-hl", "1"]).head_pieces == 1 and parse_args([]).head_pieces == 0


def test_finetune_head(tmp_path):
    cfg = llama3.config_from_descriptor("llama3:l=2,c=64,h=4,kv=2,t=64,v=200,m=16,f=1.0")
    m = llama3.Llama(cfg, "cpu", torch.float32, head_pieces=True)
    m.init_random(42)
    before = {n: p.clone() for n, p in m.params.items()}
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randint(0, 200, (2, 32), generator=g, dtype=torch.int32) for _ in range(2))
    y[:, :8] = -1
    tuner = finetune_head.HeadTuner(m, clip=0.05)
    first = [float(v) for v in tuner.step(x, y, 1e-2)]
    # the gradient that the optimizer saw has been clipped to the norm asked for
    assert first[1] > 0.05 and abs(float(tuner.grads.norm()) - 0.05) < 1e-6
    for _ in range(30):
        loss, _ = tuner.step(x, y, 1e-2)
    assert float(loss) < 0.5 * first[0]
    for n, p in m.params.items():
        assert torch.equal(p, before[n]) == (n not in ("lnfw", "lmhead")), n
    with pytest.raises(ValueError):
        finetune_head.HeadTuner(llama3.Llama(cfg, "cpu", torch.float32))
    with pytest.raises(ValueError):
        finetune_head.HeadTuner(gpt2.GPT(gpt2.GPTConfig(32, 200, 256, 1, 2, 32), "cpu", torch.float32, head_pieces=True))


def test_finetune_command(tmp_path, capsys):
    data, out = str(tmp_path / "tokens.bin"), str(tmp_path / "tuned.bin")
    write_datafile(data, torch.randint(0, 200, (2000,), generator=torch.Generator().manual_seed(2)).tolist(), "llama-3")
    finetune_head.main(["--model", "llama3:l=1,c=32,h=2,kv=1,t=32,v=200,m=16,f=1.0", "--data", data, "--steps", "3", "-b", "2", "-t", "16", "--prompt", "4",
                        "--device", "cpu", "--out", out])
    assert capsys.readouterr().out.count("loss") == 3
    cfg, _ = checkpoint.read_model_header(out)
    assert cfg.channels == 32
