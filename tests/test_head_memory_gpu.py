"""Memory of training without a logits buffer, as the allocator counts it."""
import pytest
import torch

from llmc_b200.models import gpt2, llama3

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _peak(family, pieces, B, T, turns):
    """Largest number of bytes held at once, beyond what was held before, and the gradients."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    if family == "gpt2":
        m = gpt2.GPT(gpt2.GPTConfig(max_seq_len=T, vocab_size=50257, padded_vocab_size=50304, num_layers=1, num_heads=2, channels=128), DEV, torch.bfloat16, head_pieces=pieces)
    else:
        m = llama3.Llama(llama3.config_from_descriptor("llama3:l=1,c=128,h=2,kv=1,t=%d,v=50257,m=64,f=1.0" % T), DEV, torch.bfloat16, head_pieces=pieces)
    m.init_random(3)
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randint(0, 50257, (B, T), generator=g, dtype=torch.int32).to(DEV) for _ in range(2))
    torch.cuda.reset_peak_memory_stats()
    for _ in range(turns):
        m.forward(x, y)
        m.backward()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before, m.head_scratch_bytes(), m.activation_bytes()


@pytest.mark.parametrize("family", ["gpt2", "llama3"])
@pytest.mark.parametrize("B,T,turns", [(8, 1024, 2), (4, 1024, 5)])
def test_a_model_without_logits_holds_less(family, B, T, turns):
    """Half of the logits' bytes less at least, captured passes (4096 tokens) and launched ones."""
    logits = 2 * B * T * 50304
    with_logits, none, _ = _peak(family, False, B, T, turns)
    without, scratch, acts = _peak(family, True, B, T, turns)
    assert none == 0 and 0 < scratch < logits // 2
    assert without < with_logits - logits // 2
