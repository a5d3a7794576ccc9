"""Models without a logits buffer, and training of a head alone, on the sm_100a kernels."""
import pytest
import torch

from llmc_b200 import finetune_head
from llmc_b200.models import gpt2, llama3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _make(family, **k):
    if family == "gpt2":
        cfg = gpt2.GPTConfig(max_seq_len=128, vocab_size=1003, padded_vocab_size=1024, num_layers=2, num_heads=2, channels=128)
        return gpt2.GPT(cfg, DEV, torch.bfloat16, **k)
    return llama3.Llama(llama3.config_from_descriptor("llama3:l=2,c=128,h=2,kv=1,t=128,v=1003,m=64,f=1.0"), DEV, torch.bfloat16, **k)


@pytest.mark.parametrize("family", ["gpt2", "llama3"])
def test_model_without_logits(family):
    """Against the model with logits, which rounds them to bf16: a logit z is off by 2^-8 |z|, a loss by the largest of its row twice, each factor of a gradient by as much
    again; some twenty roundings of 2^-8 on the way through two layers leave the gradients apart by 0.05 of their norm at most."""
    a, b = _make(family), _make(family, head_pieces=True)
    a.init_random(3)
    b.params_flat.copy_(a.params_flat)
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randint(0, 1003, (3, 77), generator=g, dtype=torch.int32).to(DEV) for _ in range(2))
    a.forward(x, y, write_dlogits=False)
    largest = float(a.logits().float().abs().max())
    results = []
    for turn in range(4):                                     # the last two are replays of a captured pass
        for m in (a, b):
            m.forward(x, y)
            m.backward()
        results.append([b.acts["losses"].clone(), b.grads_flat.clone()])
    assert all(torch.equal(r[0], results[0][0]) and torch.equal(r[1], results[0][1]) for r in results)
    assert (a.acts["losses"] - b.acts["losses"]).abs().max() <= 2 * 2.0 ** -8 * largest + 1e-4
    for n in a.grads:
        p, q = a.grads[n].double(), b.grads[n].double()
        assert float((p - q).norm()) <= 0.05 * float(p.norm()), n
    assert b.activation_bytes() < a.activation_bytes()
    before = b.grads["wpe" if family == "gpt2" else "qkvw"].double().clone()
    b.forward(x, y)
    b.backward(micro_step=1)                                  # adds to what is there: two roundings of 2^-8 of the sum
    after = b.grads["wpe" if family == "gpt2" else "qkvw"].double()
    assert ((after - 2 * before).abs() <= 2.0 ** -7 * 2 * before.abs() + 1e-8).all()


def test_finetune_head():
    m = _make("llama3", head_pieces=True)
    m.init_random(42)
    before = {n: p.clone() for n, p in m.params.items()}
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randint(0, 1003, (2, 64), generator=g, dtype=torch.int32) for _ in range(2))
    y[:, :8] = -1
    x = x.to(DEV)
    tuner = finetune_head.HeadTuner(m, clip=0.05)
    first = [float(v) for v in tuner.step(x, y, 1e-2)]
    # 128 K elements rounded to bf16 after the factor: the sum of their squares is off by 2^-7 at most
    assert first[1] > 0.05 and abs(float(tuner.grads.double().norm()) - 0.05) <= 0.05 * 2.0 ** -7
    for _ in range(30):
        loss, _ = tuner.step(x, y, 1e-2)
    assert float(loss) < 0.5 * first[0]
    for n, p in m.params.items():
        assert torch.equal(p, before[n]) == (n not in ("lnfw", "lmhead")), n
