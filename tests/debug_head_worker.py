"""Runs in a child process with LLMC_DEBUG_CHECKS=1 (see test_debug_head_gpu.py): the head's operators and clipping of the debug library keep a clean status word and give what 64 bits give.
Prints one JSON line."""
import json
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.dirname(HERE), HERE]

import linear_ce_oracle as O  # noqa: E402
from llmc_b200 import _lib, finetune_head, ops  # noqa: E402
from llmc_b200.models import llama3  # noqa: E402
from llmc_b200.ops import kernels as KN  # noqa: E402

DEV = "cuda:0"


def main():
    out = {"debug_lib": int(_lib.cuda().llmc_debug_checks_enabled()), "passes": 0, "status": []}
    if out["debug_lib"] != 1:
        print(json.dumps(out))
        return 1
    for N, C, V, piece, moved in [(7, 72, 63, None, 0), (40, 264, 20001, None, 0), (128, 520, 50257, None, 0), (200, 264, 20001, None, 0), (300, 264, 20001, None, 0), (700, 1032, 3001, 1024, 0), (700, 264, 3001, None, 1)]:
        KN.HEAD_KEPT_WORK = 0 if moved else 10 ** 11
        x, w, t = (a.to(DEV) for a in O.make(N, C, V, seed=N, left_out=0.1))
        losses, lse = torch.zeros(N, device=DEV), torch.zeros(N, device=DEV)
        ops.linear_cross_entropy_forward(losses, lse, x, w, t, V)
        want, _, e, _ = O.forward(x, w, t, V)
        O.within(losses, want, e)
        for accumulate in (False, True):
            old = torch.randn(V, C, generator=torch.Generator().manual_seed(1)).mul_(1e-3).to(torch.bfloat16).to(DEV)
            dinp, dw = torch.full_like(x, 7.0), old.clone()
            ops.linear_cross_entropy_backward(dinp, dw, x, w, t, lse, 0.3, V, accumulate=accumulate, piece=piece)
            want, want_w, e, e_w = O.gradient(x, w, t, V, lse, torch.full((N,), 0.3), old if accumulate else None, pieces=V // 256 + 1)
            O.within(dinp, want, e)
            O.within(dw, want_w, e_w)
        out["passes"] += 1
        out["status"].append(_lib.read_status())
    m = llama3.Llama(llama3.config_from_descriptor("llama3:l=1,c=128,h=2,kv=1,t=32,v=200,m=16,f=1.0"), DEV, torch.bfloat16, head_pieces=True)
    m.init_random(42)
    tuner, g = finetune_head.HeadTuner(m), torch.Generator().manual_seed(1)
    a, b = (torch.randint(0, 200, (2, 32), generator=g, dtype=torch.int32) for _ in range(2))
    out["losses"] = [float(tuner.step(a.to(DEV), b, 1e-2)[0]) for _ in range(10)]
    out["status"].append(_lib.read_status())
    print(json.dumps(out))
    return 0


if __name__ == "__main__":
    sys.exit(main())
