"""Cases of serving on a paged key / value cache: rotated keys and values of new tokens written into pages (``paged_rope_cache``), attention of ragged new
tokens over the pages (``paged_attention``), the same for a tree of drafted tokens (``paged_tree_attention``), and the drafted tokens that a step accepts moved
together (``paged_keep``).

``listed()`` gives the standing cases, ``draw(rng)`` one more of the same ranges.  ``run`` takes one pass: through the framework's public entry
points where ``own`` is set, else through elementary torch operations in 32 bits.  ``exact`` restates the pass in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64

LLAMA_8B = {"NH": 32, "NKV": 8, "HS": 128}
LLAMA_1B = {"NH": 32, "NKV": 8, "HS": 64}
GPT2_124M = {"NH": 12, "NKV": 12, "HS": 64}


def listed():
    return [
        # one decoding step of eight conversations, one layer: latency
        {"name": "append_8_llama_8B", "kind": "append", **LLAMA_8B, "B": 8, "new": 1, "longest": 2000, "page": 16, "R": 128, "halves": False},
        # parts of prompts of odd lengths; two halves rotated against one another, in half of the head, every head with keys of its own
        {"name": "append_ragged_halves", "kind": "append", "NH": 16, "NKV": 16, "HS": 96, "B": 5, "new": 111, "longest": 700, "page": 32, "R": 48, "halves": True},
        # prompts of up to 2048 tokens entering the cache of a 1.4 B model
        {"name": "append_16_prompts_llama_1.4B", "kind": "append", **LLAMA_1B, "B": 16, "new": 2048, "longest": 2048, "page": 64, "R": 64, "halves": False},
        # a decoding step of one short conversation: latency
        {"name": "attention_1x161_llama_1.4B", "kind": "attention", **LLAMA_1B, "B": 1, "new": 1, "longest": 161, "page": 16},
        # a decoding step of 32 conversations of very different lengths
        {"name": "attention_32x8192_llama_8B", "kind": "attention", **LLAMA_8B, "B": 32, "new": 1, "longest": 8192, "page": 16},
        # a decoding step over the longest context of LLaMA 3.1
        {"name": "attention_1x131072_llama_8B", "kind": "attention", **LLAMA_8B, "B": 1, "new": 1, "longest": 131072, "page": 64},
        # a prompt of the training context
        {"name": "attention_prompt_8192_llama_8B", "kind": "attention", **LLAMA_8B, "B": 1, "new": 8192, "longest": 8192, "page": 16},
        # parts of prompts next to each other, GPT-2's heads, some of them behind a cached context
        {"name": "attention_ragged_gpt2_124M", "kind": "attention", **GPT2_124M, "B": 9, "new": 300, "longest": 1024, "page": 16},
        # a dozen drafted tokens of one conversation
        {"name": "tree_1x12_llama_8B", "kind": "tree", **LLAMA_8B, "B": 1, "new": 12, "longest": 1500, "page": 16},
        # trees of up to 64 drafted tokens of sixteen conversations
        {"name": "tree_16x64_llama_8B", "kind": "tree", **LLAMA_8B, "B": 16, "new": 64, "longest": 4096, "page": 16},
        # four drafted continuations of one conversation, part of one accepted, all layers
        {"name": "keep_1_llama_8B", "kind": "keep", **LLAMA_8B, "B": 1, "chains": 4, "chain": 5, "L": 32, "longest": 300, "page": 16},
        # eight drafted continuations of 64 conversations, all layers
        {"name": "keep_64_llama_1.4B", "kind": "keep", **LLAMA_1B, "B": 64, "chains": 8, "chain": 8, "L": 16, "longest": 500, "page": 16},
    ]


# what the largest listed cases hold: fp32 scores of the plain form, cached tokens times channels
SCORES = 32 * 8192 * 8192
CACHED = 32 * 8192 * 1024


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "tree", "keep"])
    NKV = rng.choice([1, 2, 4, 8, 8, 12, 16, 32])
    G = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 16]) if NKV <= 8 else 1
    HS = rng.choice([64, 128, 64, 128, 8 * rng.randint(2, 16)])
    case = {"kind": kind, "NH": G * NKV, "NKV": NKV, "HS": HS, "page": rng.choice([8, 16, 16, 32, 64, 128, 256]), "B": _log(rng, 1, 128)}
    if kind == "keep":
        case |= {"chains": rng.randint(1, 8), "chain": rng.randint(1, 8), "L": rng.randint(1, 32)}
        case["longest"] = _log(rng, 64, max(64, min(2000, CACHED // (8 * case["B"] * NKV * HS * case["L"]))))
        return case
    case["longest"] = _log(rng, 64 if kind == "tree" else 1, max(64, min(131072, CACHED // (case["B"] * NKV * HS))))
    if kind == "append":
        case["new"] = _log(rng, 1, min(case["longest"], max(1, 32768 // case["B"])))
        return case | {"R": rng.choice([HS, HS, 8 * max(1, HS // 16)]), "halves": rng.random() < 0.5}
    most = SCORES // (case["B"] * case["NH"] * case["longest"])
    case["new"] = _log(rng, 1, max(1, min(64 if kind == "tree" else case["longest"], most)))
    if kind == "attention" and rng.random() < 0.4:
        case["new"] = 1
    return case


# ---------------------------------------------------------------------------------------------------------------- inputs

def _lengths(case):
    """Keys and new tokens of every sequence, from the case alone: a fixed sequence of ragged shares; the first sequence has the longest of both."""
    B = case["B"]
    share = [1.0] + [(1 + i * 2654435761 % 1009) / 1009 for i in range(1, B)]
    if case["kind"] == "keep":
        new = [case["chains"] * case["chain"]] * B
        return [n + max(0, int(case["longest"] * s) - n) for n, s in zip(new, share)], new
    keys = [max(1, int(round(case["longest"] * s))) for s in share]
    new = [min(k, max(1, int(round(case["new"] * s)))) for k, s in zip(keys, share[:1] + share[:0:-1])]
    return keys, new


def _parents(count, g):
    """A tree of drafted tokens, parents before their children (-1: a child of the last accepted token)."""
    draws = torch.rand(count, generator=g).tolist()
    return [-1 if i == 0 or u < 0.1 else i - 1 if u < 0.6 else int(u * 7919 * i) % i for i, u in enumerate(draws)]


def _trees(new, seed):
    """One 64-bit mask per new token: bit j says that it sees drafted token j of its sequence (its ancestors and itself)."""
    g = torch.Generator().manual_seed(seed)
    masks = []
    for n in new:
        own_masks = []
        for i, parent in enumerate(_parents(n, g)):
            own_masks.append((own_masks[parent] if parent >= 0 else 0) | 1 << i)
        masks += own_masks
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _table(case, keys, g):
    """Which page holds which part of a sequence: pages in no order, one page behind them all that no sequence has; entries behind a sequence's last page are -1."""
    page = case["page"]
    count = [-(-k // page) for k in keys]
    pages = sum(count) + 1
    order = torch.randperm(pages - 1, generator=g).tolist()
    table = torch.full((len(keys), max(count)), -1, dtype=I32)
    at = 0
    for b, c in enumerate(count):
        table[b, :c] = torch.tensor(order[at:at + c], dtype=I32)
        at += c
    return table, pages


def _angles(length, R, dtype):
    inv = 500000.0 ** (-torch.arange(0, R, 2, dtype=F64, device=DEV) / R)
    a = torch.arange(length, dtype=F64, device=DEV)[:, None] * inv
    return torch.stack([torch.cos(a), torch.sin(a)], -1).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    keys, new = _lengths(case)
    NH, NKV, HS = case["NH"], case["NKV"], case["HS"]
    table, pages = _table(case, keys, torch.Generator().manual_seed(seed))
    N = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    normal = lambda *shape, std=1.0: torch.randn(*shape, generator=g, device=DEV, dtype=BF16).mul_(std)
    L = case.get("L", 1)
    s = {"kind": case["kind"], "NH": NH, "NKV": NKV, "HS": HS, "page": case["page"], "S": max(keys), "most": max(new),
         "kpages": normal(L, pages, case["page"], NKV, HS), "vpages": normal(L, pages, case["page"], NKV, HS),
         "table": table.to(DEV), "lengths": torch.tensor(keys, dtype=I32, device=DEV), "starts": torch.tensor(starts, dtype=I32, device=DEV)}
    if case["kind"] == "append":
        s |= {"raw": normal(N, (NH + 2 * NKV) * HS), "freqs": _angles(max(keys), case["R"], F32), "halves": case["halves"], "q": torch.zeros(N, NH * HS, dtype=BF16, device=DEV)}
    elif case["kind"] == "keep":
        # of each sequence, the first few tokens of one of its drafted chains
        c, n = case["chains"], case["chain"]
        which = torch.randint(0, c, (case["B"], 1), generator=g, device=DEV, dtype=I32)
        s |= {"kept": which * n + torch.arange(n, device=DEV, dtype=I32), "counts": torch.randint(0, n + 1, (case["B"],), generator=g, device=DEV, dtype=I32)}
    else:
        s |= {"q": normal(N, NH * HS, std=1.5), "out": torch.zeros(N, NH * HS, dtype=BF16, device=DEV)}
        if case["kind"] == "tree":
            s["tree"] = torch.tensor(_trees(new, seed), dtype=I64, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from llmc_b200 import ops
    cache = s.get("cache")
    if cache is None:
        # where the pages are, which a program finds out once for its cache
        cache = s["cache"] = ops.paged_cache(s["kpages"], s["vpages"], s["table"], s["lengths"], s["starts"])
    if s["kind"] == "append":
        ops.paged_rope_cache(s["q"], cache, s["raw"], s["freqs"], s["NH"], halves=s["halves"])
        return [s["q"], s["kpages"], s["vpages"]]
    if s["kind"] == "keep":
        ops.paged_keep(cache, s["kept"], s["counts"])
        return [s["kpages"], s["vpages"]]
    if s["kind"] == "tree":
        ops.paged_tree_attention(s["out"], s["q"], cache, s["tree"], s["NH"])
    else:
        ops.paged_attention(s["out"], s["q"], cache, s["NH"])
    return s["out"]


def _rotated(x, f, halves):
    """x (N, heads, HS) rotated by f (N, R / 2, 2): neighbours, or the two halves of the first R channels, are a pair."""
    R = 2 * f.shape[1]
    c, s = f[:, None, :, 0], f[:, None, :, 1]
    if halves:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., R:]], -1)
    a, b = x[..., 0:R:2], x[..., 1:R:2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), x[..., R:]], -1)


def _rows(s, N):
    """Sequence of every new token, its number there, and its position."""
    starts, n = s["starts"].long(), torch.arange(N, device=DEV)
    b = (n[:, None] >= starts[None, 1:]).sum(1)
    i = n - starts[b]
    return b, i, s["lengths"].long()[b] - (starts[b + 1] - starts[b]) + i


def _run_plain(s):
    page, NH, NKV, HS = s["page"], s["NH"], s["NKV"], s["HS"]
    table, lengths = s["table"].long(), s["lengths"].long()
    if s["kind"] == "keep":
        base = (lengths - (s["starts"][1:] - s["starts"][:-1]).long())[:, None]
        B, D = s["kept"].shape
        to = base + torch.arange(D, device=DEV)
        which = torch.arange(D, device=DEV)[None, :] < s["counts"].long()[:, None]
        seq = torch.arange(B, device=DEV)[:, None].expand(B, D)[which]
        src, dst = (base + s["kept"].long())[which], to[which]
        sp, dp = table[seq, src // page], table[seq, dst // page]
        k, v = s["kpages"][:, sp, src % page], s["vpages"][:, sp, src % page]
        s["kpages"][:, dp, dst % page] = k
        s["vpages"][:, dp, dst % page] = v
        return [s["kpages"], s["vpages"]]
    if s["kind"] == "append":
        N = s["raw"].shape[0]
        b, _, pos = _rows(s, N)
        x = s["raw"].view(N, NH + 2 * NKV, HS)
        r = _rotated(x[:, :NH + NKV].float(), s["freqs"][pos], s["halves"]).to(BF16)
        s["q"].copy_(r[:, :NH].reshape(N, NH * HS))
        p = table[b, pos // page]
        s["kpages"][0, p, pos % page] = r[:, NH:]
        s["vpages"][0, p, pos % page] = x[:, NH + NKV:]
        return [s["q"], s["kpages"], s["vpages"]]
    N, S, G = s["q"].shape[0], s["S"], NH // NKV
    b, i, pos = _rows(s, N)
    B, most = table.shape[0], s["most"]
    # every sequence's keys side by side, its queries in rows of a padded batch
    at = table.clamp(min=0)
    k = s["kpages"][0][at].view(B, -1, NKV, HS)[:, :S].float()
    v = s["vpages"][0][at].view(B, -1, NKV, HS)[:, :S].float()
    q = torch.zeros(B, most, NKV, G, HS, device=DEV)
    q[b, i] = s["q"].view(N, NKV, G, HS).float()
    key = torch.arange(S, device=DEV)
    seen = torch.zeros(B, most, S, dtype=torch.bool, device=DEV)
    if s["kind"] == "tree":
        context = (pos - i)[:, None]
        drafted = (key - context).clamp(0, 63)
        bit = (s["tree"][:, None] >> drafted) & 1
        seen[b, i] = (key < context) | ((key < lengths[b][:, None]) & (bit == 1))
    else:
        seen[b, i] = key <= pos[:, None]
    z = torch.einsum("bnghd,bsgd->bghns", q, k).mul_(1.0 / math.sqrt(HS))
    z.masked_fill_(~seen[:, None, None], -math.inf)
    z = z.sub_(z.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    y = torch.einsum("bghns,bsgd->bnghd", z, v) / z.sum(-1).clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
    s["out"].copy_(y[b, i].reshape(N, NH * HS))
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    keys, new = _lengths(case)
    page, NH, NKV, HS = case["page"], case["NH"], case["NKV"], case["HS"]
    slots = [torch.arange(k, device=DEV) for k in keys]
    flat = [s["table"][b].long()[t // page] * page + t % page for b, t in enumerate(slots)]      # where in the pages key t of sequence b lies
    if case["kind"] == "keep":
        pools = [s["kpages"].to(F64).view(case["L"], -1, NKV, HS), s["vpages"].to(F64).view(case["L"], -1, NKV, HS)]
        for b, c in enumerate(s["counts"].tolist()):
            base = keys[b] - new[b]
            for pool in pools:
                pool[:, flat[b][base:base + c]] = pool[:, flat[b][base + s["kept"][b, :c].long()]]
        return [p.view(s["kpages"].shape) for p in pools]
    if case["kind"] == "append":
        x = s["raw"].to(F64).view(-1, NH + 2 * NKV, HS)
        R = case["R"]
        f = s["freqs"].to(F64)
        first = torch.arange(R // 2, device=DEV) * (1 if case["halves"] else 2)
        second = first + (R // 2 if case["halves"] else 1)
        pool_k, pool_v = s["kpages"].to(F64).view(-1, NKV, HS), s["vpages"].to(F64).view(-1, NKV, HS)
        at = 0
        for b, n in enumerate(new):
            t = slots[b][keys[b] - n:]
            c, d = f[t][:, None, :, 0], f[t][:, None, :, 1]
            rows = x[at:at + n, :NH + NKV]
            one, two = rows[..., first], rows[..., second]
            rows[..., first], rows[..., second] = one * c - two * d, one * d + two * c
            pool_k[flat[b][t]], pool_v[flat[b][t]] = rows[:, NH:], x[at:at + n, NH + NKV:]
            at += n
        return [x[:, :NH].reshape(-1, NH * HS), pool_k.view(s["kpages"].shape), pool_v.view(s["vpages"].shape)]
    out = torch.zeros(sum(new), NH, HS, dtype=F64, device=DEV)
    pool_k, pool_v = s["kpages"][0].view(-1, NKV, HS), s["vpages"][0].view(-1, NKV, HS)
    at = 0
    for b, n in enumerate(new):
        q = s["q"][at:at + n].to(F64).view(n, NH, HS)
        context = keys[b] - n
        if case["kind"] == "tree":
            sees = torch.zeros(n, keys[b], dtype=torch.bool, device=DEV)
            sees[:, :context] = True
            bits = [[m >> j & 1 for j in range(n)] for m in s["tree"][at:at + n].tolist()]
            sees[:, context:] = torch.tensor(bits, dtype=torch.bool, device=DEV)
        else:
            sees = slots[b][None, :] <= slots[b][context:, None]
        for h in range(NH):
            k, v = pool_k[flat[b], h // (NH // NKV)].to(F64), pool_v[flat[b], h // (NH // NKV)].to(F64)
            z = torch.where(sees, q[:, h] @ k.t() / math.sqrt(HS), -math.inf)
            out[at:at + n, h] = torch.softmax(z, 1) @ v
        at += n
    return out.view(-1, NH * HS)


# ---------------------------------------------------------------------------------------------------------------- work

def work(case):
    keys, new = _lengths(case)
    NH, NKV, HS = case["NH"], case["NKV"], case["HS"]
    if case["kind"] == "keep":
        # half of a chain on average, moved
        moved = case["B"] * case["chain"] / 2 * case["L"] * NKV * HS
        return {"bytes": 8 * moved, "flops": 0}
    rows = sum(new) * (NH + 2 * NKV) * HS
    if case["kind"] == "append":
        return {"bytes": 4 * rows + 4 * sum(new) * case["R"], "flops": 3 * sum(new) * (NH + NKV) * case["R"]}
    pairs = sum(n * (k - n) + (n * n if case["kind"] == "tree" else n * (n + 1) // 2) for k, n in zip(keys, new))
    return {"bytes": 4 * sum(new) * NH * HS + 4 * sum(keys) * NKV * HS, "flops": 4 * pairs * NH * HS}
