"""Trains the final norm and the LM head of a LLaMA-3 model whose other weights stay as they are.

    python -m llmc_b200.finetune_head --model llama3.bin --data 'data/answers_*.bin' --steps 200 -b 4 -t 1024 --prompt 64 --out tuned.bin

The end of a training step on the operators made for it: the loss at the head without its logits in memory (``ops.linear_cross_entropy_forward``), its
gradients with a weight for each token (``ops.linear_cross_entropy_backward``; the first ``--prompt`` targets of every row are left out), the
norm of the gradients and their clipping (``ops.clip_grad_norm``), then AdamW.
"""
import argparse
import sys

import torch

from . import ops


class HeadTuner:
    """Owns gradients and optimizer state of the two tensors; ``step`` trains them in place."""

    def __init__(self, model, clip=1.0, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0):
        if getattr(model, "family", "") != "llama3":
            raise ValueError("the head of this model is its embedding table; only untied heads are trained alone")
        if not model.head_pieces:
            raise ValueError("the model keeps logits that nobody reads: build it with head_pieces=True")
        cfg, self.model, self.clip = model.cfg, model, clip
        self.betas, self.eps = (beta1, beta2), eps
        C, Vp = cfg.channels, cfg.padded_vocab_size
        n = C + Vp * C
        o = model.offsets["lnfw"]                    # the head follows the norm's weights, at the end of the buffer
        self.params = model.params_flat[o:o + n]
        self.grads = torch.zeros_like(self.params)
        self.norm_grad, self.head_grad = self.grads[:C], self.grads[C:].view(Vp, C)
        self.plan = ops.clip_plan(None, [self.norm_grad, self.head_grad])
        self.norm = torch.zeros(1, dtype=torch.float32, device=model.device)
        self.m, self.v, self.master = (torch.zeros(n, dtype=torch.float32, device=model.device) for _ in range(3))
        self.master.copy_(self.params)
        self.views = [dict(p_base=0, p_stride=C, o_base=0, o_stride=C, n=C, L=1, wd=0.0),
                      dict(p_base=C, p_stride=Vp * C, o_base=C, o_stride=Vp * C, n=Vp * C, L=1, wd=weight_decay)]
        self.losses = self.lse = None
        self.t = 0

    def step(self, tokens, targets, lr):
        """One update on tokens and targets (B, T); targets outside the vocabulary are left out.  Returns loss and gradient norm as device tensors, without synchronising."""
        m, cfg, p = self.model, self.model.cfg, self.model.params
        m.forward(tokens)
        a, N = m.acts, tokens.numel()
        targets = targets.to(m.device, torch.int32).reshape(-1).contiguous()
        if self.losses is None or self.losses.numel() != N:
            self.losses, self.lse = (torch.zeros(N, dtype=torch.float32, device=m.device) for _ in range(2))
        counted = ((targets >= 0) & (targets < cfg.vocab_size)).float()
        weight = counted / counted.sum().clamp(min=1.0)
        ops.linear_cross_entropy_forward(self.losses, self.lse, a["lnf"], p["lmhead"], targets, cfg.vocab_size)
        ops.linear_cross_entropy_backward(a["scratch_btc"], self.head_grad, a["lnf"], p["lmhead"], targets, self.lse, weight, cfg.vocab_size, accumulate=False,
                                          piece=m.head_piece())
        ops.rmsnorm_backward(a["dresidual"], self.norm_grad, a["scratch_btc"], a["residual3"][cfg.num_layers - 1], p["lnfw"], a["lnf_rstd"],
                             accumulate_dinp=False, accumulate_dw=False)
        ops.clip_grad_norm(self.norm, self.plan, self.clip)
        self.t += 1
        for i, v in enumerate(self.views):
            v["seed"] = self.t * 2 + i               # of the stochastic rounding
        # a norm that is not finite leaves parameters and state as they are; the gradients have been clipped, so that is all it decides
        ops.adamw_update(self.params, self.master, self.grads, self.m, self.v, self.views, lr, *self.betas, self.eps, self.t, norm_sq=self.norm, grad_clip=float("inf"))
        return (self.losses * weight).sum(), self.norm[0]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model", required=True, help="model file, or a llama3: descriptor for random weights")
    ap.add_argument("--data", required=True, help="token shards")
    ap.add_argument("--out", default="", help="model file to write")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("-b", type=int, default=4)
    ap.add_argument("-t", type=int, default=256)
    ap.add_argument("--lr", type=float, default=1e-4)
    ap.add_argument("--clip", type=float, default=1.0)
    ap.add_argument("--prompt", type=int, default=0, help="targets at the start of every row that are left out")
    ap.add_argument("--device", default="")
    a = ap.parse_args(argv)

    from .models import llama3
    from .utils import checkpoint
    from .utils.dataloader import DataLoader
    dev = torch.device(a.device or ("cuda:0" if torch.cuda.is_available() else "cpu"))
    if a.model.endswith(".bin"):
        model = llama3.Llama(checkpoint.read_model_header(a.model)[0], dev, head_pieces=True)
        checkpoint.load_model(a.model, model)
    else:
        model = llama3.Llama(llama3.config_from_descriptor(a.model), dev, head_pieces=True)
        model.init_random(42)
    tuner = HeadTuner(model, a.clip)
    loader = DataLoader(a.data, a.b, a.t, 0, 1, 0)
    for step in range(a.steps):
        inputs, targets = loader.next_batch()
        targets = targets.clone()
        targets[:, :a.prompt] = -1
        loss, norm = tuner.step(inputs.to(dev), targets, a.lr)
        print("step %d loss %.4f norm %.4f" % (step + 1, float(loss), float(norm)), flush=True)
    if a.out:
        checkpoint.write_model(a.out, model)


if __name__ == "__main__":
    main(sys.argv[1:])
