"""Cases of the end of a training step: the loss of an LM head without its logits in memory (linear layer and softmax cross-entropy in one,
``linear_cross_entropy_forward``), the gradients of that loss (``linear_cross_entropy_backward``), and the global norm of many gradient
tensors with their clipping (``clip_grad_norm``).

``listed()`` gives the standing cases, ``draw(rng)`` one more of the same ranges.  ``run`` takes one pass: through the framework's public entry
points where ``own`` is set, else through elementary torch operations in 32 bits.  ``exact`` restates the pass in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # scoring the continuations of a multiple-choice question with GPT-2 124M: few tokens, the time is that of reading the weights
        {"name": "loss_24_gpt2_124M", "kind": "loss", "N": 24, "C": 768, "V": 50257, "Vp": 50304, "left_out": 0.0},
        # validation on the 4 x 64 tokens of the reference's numerics test
        {"name": "loss_256_gpt2_124M", "kind": "loss", "N": 256, "C": 768, "V": 50257, "Vp": 50304, "left_out": 0.0},
        # validation on one text of odd length, GPT-2 350M, some tokens (padding) left out
        {"name": "loss_1021_gpt2_350M", "kind": "loss", "N": 1021, "C": 1024, "V": 50257, "Vp": 50304, "left_out": 0.1},
        # validation at the full context of LLaMA-3 8B
        {"name": "loss_8192_llama_8B", "kind": "loss", "N": 8192, "C": 4096, "V": 128256, "Vp": 128256, "left_out": 0.0},
        # training on a short answer: LLaMA-sized vocabulary, 1.4 B model, a weight for each token, most of a prompt left out
        {"name": "gradient_77_llama_1.4B", "kind": "gradient", "N": 77, "C": 2048, "V": 128256, "Vp": 128256, "left_out": 0.5, "weighted": True},
        # micro-step on the 4 x 64 tokens of the reference's numerics test
        {"name": "gradient_256_gpt2_124M", "kind": "gradient", "N": 256, "C": 768, "V": 50257, "Vp": 50304, "left_out": 0.0, "weighted": False},
        # micro-step of 16 x 1024 tokens of GPT-2 124M
        {"name": "gradient_16384_gpt2_124M", "kind": "gradient", "N": 16384, "C": 768, "V": 50257, "Vp": 50304, "left_out": 0.0, "weighted": False},
        # packed texts of odd total length in LLaMA-3 8B, a weight for each token
        {"name": "gradient_3001_llama_8B", "kind": "gradient", "N": 3001, "C": 4096, "V": 128256, "Vp": 128256, "left_out": 0.1, "weighted": True},
        # adapters: many small tensors, latency
        {"name": "clip_adapters", "kind": "clip", "model": "adapters", "C": 768, "L": 12, "dtypes": "f32"},
        # every parameter tensor of every layer of GPT-2 124M, bf16
        {"name": "clip_gpt2_124M", "kind": "clip", "model": "gpt2", "C": 768, "L": 12, "dtypes": "bf16"},
        # the same of GPT-2 350M, matrices in bf16 and vectors in fp32
        {"name": "clip_gpt2_350M_mixed", "kind": "clip", "model": "gpt2", "C": 1024, "L": 24, "dtypes": "mixed"},
        # pieces of a sharded flat buffer: odd sizes, starts on any element, fp32
        {"name": "clip_pieces_f32", "kind": "clip", "model": "pieces", "count": 301, "total": 30_000_001, "dtypes": "f32"},
    ]


LARGEST_LOSS = 8192 * 4096 * 128256
LARGEST_GRADIENT = 3001 * 4096 * 128256


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "gradient", "gradient", "clip"])
    if kind == "clip":
        dtypes = rng.choice(["bf16", "f32", "mixed"])
        model = rng.choice(["adapters", "gpt2", "pieces", "pieces"])
        if model == "pieces":
            return {"kind": kind, "model": model, "count": _log(rng, 1, 1500), "total": _log(rng, 1000, 200_000_000), "dtypes": dtypes}
        if model == "adapters":
            return {"kind": kind, "model": model, "C": 8 * rng.randint(16, 512), "L": rng.randint(1, 48), "dtypes": dtypes}
        C, L = rng.choice([(384, 6), (768, 12), (768, rng.randint(1, 12)), (1024, rng.randint(1, 24))])
        return {"kind": kind, "model": model, "C": C, "L": L, "dtypes": dtypes}
    C = rng.choice([384, 768, 1024, 1280, 1600, 2048, 4096, 8 * rng.randint(16, 512)])
    V, Vp = rng.choice([(50257, 50304), (128256, 128256), (_log(rng, 500, 128256), None)])
    Vp = Vp or (V + 127) // 128 * 128
    largest = LARGEST_LOSS if kind == "loss" else LARGEST_GRADIENT
    N = _log(rng, 1, max(1, min(16384, largest // (C * V))))
    case = {"kind": kind, "N": N, "C": C, "V": V, "Vp": Vp, "left_out": rng.choice([0.0, 0.0, 0.1, 0.5, 1.0])}
    if kind == "gradient":
        case["weighted"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs

def _normal(g, *shape, std=1.0, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype).mul_(std)


def _head(case, seed):
    """Outputs of the final norm, head weights and targets.  The weights have the norm of a trained head's, so that logits spread over a few units,
    and a row leans towards the weights of its target, as in a model that predicts some tokens well and some badly."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    N, C, V, Vp = case["N"], case["C"], case["V"], case["Vp"]
    weight = _normal(g, Vp, C, std=2.0 / math.sqrt(C), dtype=BF16)
    targets = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    lean = 3.0 * torch.rand(N, 1, generator=g, device=DEV)
    inp = (_normal(g, N, C) + lean * weight[targets.long()].float()).to(BF16)
    out = torch.rand(N, generator=g, device=DEV) < case["left_out"]
    out[0] = False
    targets[out] = -1
    return inp, weight, targets, g


def _shapes(case):
    if case["model"] == "pieces":
        return None
    C, L = case["C"], case["L"]
    if case["model"] == "adapters":       # low-rank pairs beside the four products of a layer
        return [s for _ in range(L) for s in ((8, C), (3 * C, 8), (8, C), (C, 8), (8, C), (4 * C, 8), (8, 4 * C), (C, 8))]
    layer = [(C,), (C,), (3 * C, C), (3 * C,), (C, C), (C,), (C,), (C,), (4 * C, C), (4 * C,), (C, 4 * C), (C,)]
    return [(50304, C), (1024, C)] + layer * L + [(C,), (C,)]


def _pieces(case):
    """Sizes of the pieces: a fixed sequence of ragged shares of the total, one of them empty where there are more than ten."""
    count, total = case["count"], case["total"]
    share = [1.0 + (i * 2654435761 % 1000) / 50.0 for i in range(count)]
    cut, done, acc = [], 0, 0.0
    for i, s in enumerate(share):
        acc += s
        end = total if i == count - 1 else int(total * acc / sum(share))
        cut.append(max(0, end - done))
        done = max(done, end)
    if count > 10:
        cut[5] += cut[4]
        cut[4] = 0
    return cut


def _dtype(case, i, dims):
    if case["dtypes"] == "mixed":
        return (BF16 if dims > 1 else F32) if case["model"] != "pieces" else (BF16, F32)[i % 2]
    return BF16 if case["dtypes"] == "bf16" else F32


def _gradients(case, seed):
    """Gradient tensors whose magnitude differs from tensor to tensor; the clipped ones go to views of one flat buffer per type, as an optimizer
    keeps them.  Pieces are views of such a flat buffer themselves, on any element."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    shapes = _shapes(case) or [(n,) for n in _pieces(case)]
    types = [_dtype(case, i, len(s)) for i, s in enumerate(shapes)]
    size = {dt: sum(math.prod(s) for s, d in zip(shapes, types) if d == dt) for dt in (BF16, F32) if dt in types}
    flat = {dt: torch.zeros(n, dtype=dt, device=DEV) for dt, n in size.items()}
    whole = {dt: _normal(g, n, std=1e-3, dtype=dt) for dt, n in size.items()} if case["model"] == "pieces" else None
    at = dict.fromkeys(size, 0)
    grads, outs = [], []
    for i, (shape, dt) in enumerate(zip(shapes, types)):
        lo, hi = at[dt], at[dt] + math.prod(shape)
        at[dt] = hi
        grads.append(whole[dt][lo:hi] if whole else _normal(g, *shape, std=1e-3 * (1 + i % 7), dtype=dt))
        outs.append(flat[dt][lo:hi].view(shape))
    return grads, outs, list(flat.values())


def _joined(tensors, like):
    """The elements of a list of tensors type by type, in the order of ``like``."""
    return [torch.cat([t.reshape(-1) for t, l in zip(tensors, like) if l.dtype == dt]) for dt in (BF16, F32) if any(l.dtype == dt for l in like)]


def _weights_of_tokens(case, g):
    """The factor of each token's loss: 1 / N, or a number per token."""
    if case["weighted"]:
        return torch.rand(case["N"], generator=g, device=DEV).add_(0.1).div_(case["N"])
    return 1.0 / case["N"]


def _lse64(inp, weight, V):
    lse = torch.empty(inp.shape[0], dtype=F64, device=DEV)
    w = weight[:V].to(F64).t()
    for r in range(0, inp.shape[0], 1024):
        lse[r:r + 1024] = torch.logsumexp(inp[r:r + 1024].to(F64) @ w, 1)
    return lse


def _lse32(inp, weight, V):
    lse = torch.empty(inp.shape[0], dtype=F32, device=DEV)
    for r in range(0, inp.shape[0], 1024):
        lse[r:r + 1024] = torch.logsumexp((inp[r:r + 1024] @ weight[:V].t()).float(), 1)
    return lse


def prepare(case, seed):
    kind = case["kind"]
    if kind == "clip":
        grads, outs, flat = _gradients(case, seed)
        state = {"kind": kind, "grads": grads, "outs": outs, "flat": flat, "norm": torch.zeros(1, device=DEV), "max_norm": 1e-2}
        if own:
            _plan(state)
        return state
    inp, weight, targets, g = _head(case, seed)
    N = case["N"]
    state = {"kind": kind, "inp": inp, "weight": weight, "targets": targets, "V": case["V"]}
    if kind == "loss":
        state["losses"] = torch.zeros(N, device=DEV)
        state["lse"] = torch.zeros(N, device=DEV)
        return state
    # the statistics of the rows, as the forward pass left them
    state["lse"] = _lse32(inp, weight, case["V"])
    state["dloss"] = _weights_of_tokens(case, g)
    state["dinp"] = torch.zeros_like(inp)
    state["dweight"] = torch.zeros_like(weight)
    return state


# ---------------------------------------------------------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _plan(s):
    """Where the tensors lie, which a program with gradient buffers that stay finds out once."""
    from llmc_b200 import ops
    if "plan" not in s:
        s["plan"] = ops.clip_plan(s["outs"], s["grads"])
    return s["plan"]


def _run_own(s):
    from llmc_b200 import ops
    if s["kind"] == "clip":
        ops.clip_grad_norm(s["norm"], _plan(s), s["max_norm"])
        return [s["norm"]] + s["flat"]
    if s["kind"] == "loss":
        ops.linear_cross_entropy_forward(s["losses"], s["lse"], s["inp"], s["weight"], s["targets"], s["V"])
        return [s["losses"], s["lse"]]
    ops.linear_cross_entropy_backward(s["dinp"], s["dweight"], s["inp"], s["weight"], s["targets"], s["lse"], s["dloss"], s["V"], accumulate=False)
    return [s["dinp"], s["dweight"]]


def _run_plain(s):
    if s["kind"] == "clip":
        total = torch.zeros((), device=DEV)
        for g in s["grads"]:
            f = g.float()
            total = total + (f * f).sum()
        norm = torch.sqrt(total)
        scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm))
        return [norm.reshape(1)] + _joined([(g.float() * scale).to(g.dtype) for g in s["grads"]], s["grads"])
    V, targets = s["V"], s["targets"].long()
    x, w = s["inp"].float(), s["weight"][:V].float()
    z = x @ w.t()
    keep = (targets >= 0) & (targets < V)
    at = targets.clamp(0, V - 1)[:, None]
    if s["kind"] == "loss":
        m = z.max(1, keepdim=True).values
        lse = (m + torch.log(torch.exp(z - m).sum(1, keepdim=True)))[:, 0]
        return [torch.where(keep, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse)), lse]
    p = torch.exp(z.sub_(s["lse"][:, None]))
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=F32))
    p.mul_((keep * s["dloss"]).float()[:, None])
    dweight = torch.zeros_like(s["weight"])
    dweight[:V] = (p.t() @ x).to(dweight.dtype)
    return [(p @ w).to(s["inp"].dtype), dweight]


# ---------------------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    if case["kind"] == "clip":
        grads, _, _ = _gradients(case, seed)
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.to(F64))) ** 2 for g in grads if g.numel()))
        factor = min(1.0, 1e-2 / norm) if norm > 0 else 1.0
        return [torch.tensor([norm], dtype=F64, device=DEV)] + _joined([g.to(F64) * factor for g in grads], grads)
    inp, weight, targets, g = _head(case, seed)
    N, C, V = case["N"], case["C"], case["V"]
    kept = torch.nonzero((targets >= 0) & (targets < V))[:, 0]
    if case["kind"] == "loss":
        lse = _lse64(inp, weight, V)
        losses = torch.zeros(N, dtype=F64, device=DEV)
        losses[kept] = lse[kept] - torch.einsum("nc,nc->n", inp[kept].to(F64), weight[targets[kept].long()].to(F64))
        return [losses, lse]
    lse = _lse32(inp, weight, V).to(F64)
    factor = torch.zeros(N, dtype=F64, device=DEV)
    factor[kept] = _weights_of_tokens(case, g)[kept].to(F64) if case["weighted"] else 1.0 / N
    wide = weight[:V].to(F64)
    dinp = torch.zeros(N, C, dtype=F64, device=DEV)
    dweight = torch.zeros(weight.shape, dtype=F64, device=DEV)
    for r in range(0, N, 1024):
        x, f = inp[r:r + 1024].to(F64), factor[r:r + 1024, None]
        p = torch.exp(x @ wide.t() - lse[r:r + 1024, None]) * f
        dinp[r:r + 1024] = p @ wide
        dweight[:V].addmm_(p.t(), x)
    dinp[kept] -= factor[kept, None] * wide[targets[kept].long()]
    dweight.index_add_(0, targets[kept].long(), -factor[kept, None] * inp[kept].to(F64))
    return [dinp, dweight]


# ---------------------------------------------------------------------------------------------------------------- work

def work(case):
    if case["kind"] == "clip":
        shapes = _shapes(case) or [(n,) for n in _pieces(case)]
        held = sum(math.prod(s) * (2 if _dtype(case, i, len(s)) == BF16 else 4) for i, s in enumerate(shapes))
        return {"bytes": 2 * held + 4, "flops": 3 * sum(math.prod(s) for s in shapes)}
    N, C, V = case["N"], case["C"], case["V"]
    if case["kind"] == "loss":
        # inputs, weights and targets read, losses and row statistics written
        return {"bytes": 2 * (N + V) * C + 12 * N, "flops": 2 * N * V * C}
    # the logits formed again, two products with their gradients
    return {"bytes": 4 * (N + V) * C + (12 if case["weighted"] else 8) * N, "flops": 6 * N * V * C}
