"""The decoder on a cache in pages on a GPU: logits of prompts, parts of prompts, single tokens and trees against the fp32 model, no further off than those from the rectangular cache."""
import pytest
import torch

from llmc_b200.models import generate as G
from llmc_b200.models import llama3
from llmc_b200.models import paged as P

pytestmark = pytest.mark.gpu


def _models(desc):
    m = llama3.Llama(llama3.config_from_descriptor(desc), "cuda", torch.bfloat16, recompute=0)
    m.init_random(7)
    ref = llama3.Llama(llama3.config_from_descriptor(desc), "cpu", torch.float32, recompute=0)
    for n in m.params:
        if n in ("qkvw", "attprojw", "fc12w", "fcprojw", "lmhead"):
            m.params[n].mul_(4.0)
        ref.params[n].copy_(m.params[n].float().cpu())
    return m, ref


@pytest.mark.parametrize("desc,rows", [("llama3:l=2,c=256,h=4,kv=2,t=512,v=1000,m=64,f=1.0", 16), ("llama3:l=2,c=512,h=4,kv=1,t=512,v=1000,m=128,f=1.0", 64),
                                       ("llama3:l=1,c=288,h=3,kv=3,t=512,v=500,m=32,f=1.0", 8)])
def test_logits(desc, rows):
    m, ref = _models(desc)
    V = m.cfg.vocab_size
    g = torch.Generator().manual_seed(0)
    tok = torch.randint(0, V, (2, 320), generator=g, dtype=torch.int32)
    ref.forward(tok)
    full = ref.logits()[..., :V].clone()
    rect = G.CachedDecoder(m, 2, 512)
    off = [(rect.forward(tok[:, :300].contiguous().cuda(), 0).cpu() - full[:, 299]).norm() / full[:, 299].norm()]
    for t in range(300, 304):
        off.append((rect.forward(tok[:, t:t + 1].contiguous().cuda(), t).cpu() - full[:, t]).norm() / full[:, t].norm())
    # the same roundings in other places: errors of the same size
    allowed = 1.5 * float(max(off))
    near = lambda a, b: float((a.cpu() - b).norm() / b.norm()) <= allowed
    d = P.PagedDecoder(m, 2 * 320 // rows + 2, rows)
    a, b = d.open(), d.open()
    assert near(d.forward([a], [tok[0, :150].tolist()]), full[:1, 149])
    assert near(d.forward([b, a], [tok[1, :290].tolist(), tok[0, 150:299].tolist()]), torch.stack([full[1, 289], full[0, 298]]))
    assert near(d.forward([a, b], [tok[0, 299:300].tolist(), tok[1, 290:300].tolist()], every=True), torch.cat([full[0, 299:300], full[1, 290:300]]))
    for t in range(300, 303):
        assert near(d.forward([a, b], [tok[0, t:t + 1].tolist(), tok[1, t:t + 1].tolist()]), full[:, t])
    t = tok[:, 303:306].tolist()
    got = d.forward([a, b], [[t[0][0], 1, t[0][1], t[0][2], 4], [7, t[1][0], 3, t[1][1]]], [[-1, 0, 0, 2, -1], [-1, -1, 1, 1]], every=True)
    assert near(got[[0, 2, 3, 6, 8]], torch.cat([full[0, 303:306], full[1, 303:305]]))
    d.keep([a, b], [5, 4], [[0, 2, 3], [1, 3]])
    assert near(d.forward([a, b], [tok[0, 306:310].tolist(), tok[1, 305:320].tolist()]), torch.stack([full[0, 309], full[1, 319]]))


def test_generation_with_drafts():
    m, _ = _models("llama3:l=2,c=256,h=4,kv=2,t=256,v=64,m=64,f=1.0")
    prompts = [[5, 9, 5, 9, 5], [3], list(range(40, 59)), [8, 8]]
    got = P.generate_paged(m, prompts, 60, temperature=0.0, drafts=15)
    assert [len(t) for t in got] == [60] * 4 and all(0 <= t < 64 for text in got for t in text)
    # each token is the model's first choice, or within its rounding of it, when the whole text goes through the training forward pass
    for prompt, text in zip(prompts, got):
        tok = torch.tensor([prompt + text], dtype=torch.int32)[:, :-1]
        pad = torch.nn.functional.pad(tok, (0, -tok.shape[1] % 8))
        m.forward(pad.cuda())
        z = m.logits()[0, len(prompt) - 1:tok.shape[1], :64].float().cpu()
        chosen = z.gather(1, torch.tensor(text)[:, None])[:, 0]
        # bf16 activations of a few roundings each way: 2 % of the spread of the logits
        assert bool((z.max(1).values - chosen <= 0.02 * (z.max() - z.min())).all())
