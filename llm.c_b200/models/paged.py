"""Generation from a key / value cache in pages for the LLaMA family: sequences of any lengths side by side, each with as much of the cache as it needs, and several drafted tokens of a
sequence checked in one step.

``models.generate`` keeps a rectangle (rows of the batch x positions) and steps every row by the same position (train_llama3.py:156-190 and :476-556 of the reference).  Here a step takes any
number of new tokens of any of the open sequences: whole prompts, single tokens, or a tree of drafts, one behind the other without padding (``ops.paged_rope_cache``, ``ops.paged_attention``,
``ops.paged_tree_attention``); of a tree, the tokens that turn out to be right stay in the cache (``ops.paged_keep``).
"""
import numpy as np
import torch

from .. import ops
from ..ops import kernels
from .generate import CachedDecoder, _whole_tiles, sample_top_p


class Sequence:
    """An open sequence: how many keys it has in the cache, and in which pages."""

    def __init__(self):
        self.length, self.pages = 0, []


class PagedDecoder:
    """Runs tokens of many sequences through a ``models.llama3.Llama``, with ``pages`` pages of ``rows`` keys and values in every layer for all of them."""

    def __init__(self, model, pages, rows=16):
        cfg = model.cfg
        self.model, self.rows = model, rows
        self.kpages = torch.zeros(cfg.num_layers, pages, rows, cfg.num_kv_heads, cfg.head_size, dtype=model.dtype, device=model.device)
        self.vpages = torch.zeros_like(self.kpages)
        self.free = list(range(pages - 1, -1, -1))
        self._rows = self._last_rows = 0
        self._bufs = {}
        # products of at most this many rows run on exactly their rows, larger ones on rows padded to whole 128-row tiles
        self.skinny_rows = kernels.STREAM_MAX_ROWS if model.device.type == "cuda" and model.dtype == torch.bfloat16 else 0
        self.whole_tiles = model.device.type == "cuda"

    _buffers = CachedDecoder._buffers

    def open(self):
        return Sequence()

    def close(self, sequence):
        self.free += sequence.pages
        sequence.length, sequence.pages = 0, []

    def _reserve(self, sequences, new):
        """Pages for the new tokens of all sequences, or none at all."""
        needs = [max(0, -(-(s.length + n) // self.rows) - len(s.pages)) for s, n in zip(sequences, new)]
        if sum(needs) > len(self.free):
            raise RuntimeError("the cache has %d free pages of %d keys, %d are needed" % (len(self.free), self.rows, sum(needs)))
        for s, need in zip(sequences, needs):
            for _ in range(need):
                s.pages.append(self.free.pop())

    def _batch(self, sequences, new, parents, masks, tokens):
        """Handle of the cache for this batch, and the tokens, positions and masks on the device."""
        dev, B = self.model.device, len(sequences)
        width = max(len(s.pages) for s in sequences)
        table = np.zeros((B, width), dtype=np.int32)
        for b, s in enumerate(sequences):
            table[b, :len(s.pages)] = s.pages
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        positions = np.empty(sum(new) if parents is not None else 0, dtype=np.int32)
        if parents is not None:
            for s, tree, at in zip(sequences, parents, starts):
                for i, parent in enumerate(tree):
                    positions[at + i] = s.length if parent < 0 else positions[at + parent] + 1
        # one copy for all of them; what a kernel reads by 16 bytes is not among them
        parts = [table.ravel(), np.array([s.length + n for s, n in zip(sequences, new)], dtype=np.int32), starts, np.array(tokens, dtype=np.int32), positions]
        packed = torch.from_numpy(np.concatenate(parts)).to(dev)
        table, lengths, starts, tokens, positions = packed.split([len(p) for p in parts])
        cache = ops.paged_cache(self.kpages, self.vpages, table.view(B, width), lengths, starts)
        if parents is None:
            return cache, tokens, None, None
        return cache, tokens, positions, masks.to(dev)

    def forward(self, sequences, tokens, parents=None, every=False):
        """``tokens``: for each of the open ``sequences`` a list of new tokens, at least one.  With ``parents`` each list is a tree: the parent of each token, the number of a token in front of
        it in the list or -1 for what the cache holds (at most 64 tokens).  Keys and values of all tokens enter the cache.  Returns fp32 logits (rows, vocab_size): of the last token of each
        sequence, or of ``every`` token."""
        m = self.model
        cfg, p = m.cfg, m.params
        new = [len(t) for t in tokens]
        if not new or min(new) == 0 or len(sequences) != len(new) or len(set(map(id, sequences))) != len(new):
            raise ValueError("every sequence of a batch needs at least one new token, and is in it once")
        if parents is not None and [len(t) for t in parents] != new:
            raise ValueError("trees of %s tokens for %s tokens" % ([len(t) for t in parents], new))
        if max(s.length + n for s, n in zip(sequences, new)) > m.freqs.shape[0]:
            raise ValueError("positions up to %d exceed the model's context of %d" % (max(s.length + n for s, n in zip(sequences, new)), m.freqs.shape[0]))
        masks = None if parents is None else ops.tree_masks(parents)
        self._reserve(sequences, new)
        if m.param_sync is not None:
            m.param_sync.wait_all()
        cache, ids, positions, tree = self._batch(sequences, new, parents, masks, [t for l in tokens for t in l])
        N = sum(new)
        out_rows = None if every or N == len(new) else torch.tensor(np.cumsum(new) - 1, device=m.device)
        M = N if out_rows is None else len(new)
        a, _ = self._buffers(N, M)
        L, NH, eps, C = cfg.num_layers, cfg.num_heads, cfg.norm_eps, cfg.channels
        x, ln, rstd, q = a["x"], a["ln"], a["rstd"], a["q"]

        def mm(out, inp, weight, n):
            if self.whole_tiles and n > self.skinny_rows:
                n = _whole_tiles(n)                             # the rows beyond n are never read
            ops.matmul_forward(out[:n], inp[:n], weight, None)

        ops.encoder_forward(x[:N].view(1, N, C), ids.view(1, N), p["wte"], None)
        ops.rmsnorm_forward(ln[:N], rstd[:N], x[:N], p["ln1w"][0], eps)
        for l in range(L):
            mm(a["raw"], ln, p["qkvw"][l], N)
            ops.paged_rope_cache(q[:N], cache, a["raw"][:N], m.freqs, NH, layer=l, positions=positions)
            if tree is None:
                ops.paged_attention(a["atty"][:N], q[:N], cache, NH, layer=l)
            else:
                ops.paged_tree_attention(a["atty"][:N], q[:N], cache, tree, NH, layer=l)
            mm(a["proj"], a["atty"], p["attprojw"][l], N)
            ops.rmsnorm_fused_residual_forward(a["res"][:N], ln[:N], rstd[:N], x[:N], a["proj"][:N], p["ln2w"][l], eps)
            if N <= min(self.skinny_rows, 128) and cfg.hidden_dim % 64 == 0:
                ops.matmul_swiglu(a["h"][:N], ln[:N], p["fc12w"][l])
            elif self.skinny_rows and N > 128 and cfg.hidden_dim % 128 == 0:
                ops.matmul_swiglu_prompt(a["h"][:N], ln[:N], p["fc12w"][l])
            else:
                mm(a["fc12"], ln, p["fc12w"][l], N)
                ops.swiglu_forward(a["h"][:N], a["fc12"][:N])
            mm(a["proj"], a["h"], p["fcprojw"][l], N)
            w = p["ln1w"][l + 1] if l + 1 < L else p["lnfw"]
            ops.rmsnorm_fused_residual_forward(x[:N], ln[:N], rstd[:N], a["res"][:N], a["proj"][:N], w, eps)
        last = ln
        if out_rows is not None:
            last = a["last"]
            last[:M].copy_(ln[out_rows])
        mm(a["logits"], last, p["lmhead"], M)
        for s, n in zip(sequences, new):
            s.length += n
        return a["logits"][:M, :cfg.vocab_size].float()

    def keep(self, sequences, new, kept):
        """Of the last step's ``new`` tokens of each sequence only those stay that ``kept`` lists, in ascending order; they become the newest of the sequence."""
        dev, B = self.model.device, len(sequences)
        if not len(new) == len(kept) == B == len(set(map(id, sequences))) or B == 0:
            raise ValueError("%d new and %d kept tokens' lists for %d sequences, each of which is in it once" % (len(new), len(kept), B))
        if any(not 0 <= n <= s.length for s, n in zip(sequences, new)):
            raise ValueError("%s new tokens in sequences of %s" % (list(new), [s.length for s in sequences]))
        width = max(1, max(len(s.pages) for s in sequences))
        table = np.zeros((B, width), dtype=np.int32)
        for b, s in enumerate(sequences):
            table[b, :len(s.pages)] = s.pages
        most = max(1, max(len(k) for k in kept))
        lists = np.zeros((B, most), dtype=np.int32)
        for b, k in enumerate(kept):
            if list(k) != sorted(set(k)) or (k and not 0 <= k[0] <= k[-1] < new[b]):
                raise ValueError("kept tokens %s of %d" % (list(k), new[b]))
            lists[b, :len(k)] = k
        parts = [table.ravel(), np.array([s.length for s in sequences], dtype=np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32), lists.ravel(),
                 np.array([len(k) for k in kept], dtype=np.int32)]
        table, lengths, starts, lists, counts = torch.from_numpy(np.concatenate(parts)).to(dev).split([len(p) for p in parts])
        if any(list(k) != list(range(len(k))) for k in kept):
            ops.paged_keep(ops.paged_cache(self.kpages, self.vpages, table.view(B, width), lengths, starts), lists.view(B, most), counts)
        for s, n, k in zip(sequences, new, kept):
            s.length -= n - len(k)


def drafted_tree(tokens, most, branches=4):
    """Drafts of what may follow ``tokens``, looked up in themselves: the continuations of the latest earlier occurrences of their last two tokens (or of the last one), at most ``branches`` of
    them and ``most`` tokens in all, with common beginnings once.  Returns (tokens, parents): token 0 is the last of ``tokens``, the others are drafts."""
    tree, parents, children = [tokens[-1]], [-1], [{}]
    for n in (2, 1):
        if len(tokens) <= n or most <= 0:
            continue
        tail, found = tokens[-n:], 0
        for at in range(len(tokens) - n - 1, -1, -1):
            if tokens[at:at + n] != tail:
                continue
            node = 0
            # the first continuations get most of the room
            for t in tokens[at + n:at + n + max(1, most // 2 if found == 0 else most // branches)]:
                if t not in children[node]:
                    if len(tree) > most:
                        break
                    children[node][t] = len(tree)
                    tree.append(t)
                    parents.append(node)
                    children.append({})
                node = children[node][t]
            found += 1
            if found == branches or len(tree) > most:
                break
        if found:
            break
    return tree, parents


def generate_paged(model, prompt_tokens, max_gen_len, temperature=0.6, top_p=0.9, echo=False, stop_tokens=(), generator=None, drafts=0, rows=16, decoder=None):
    """``models.generate.generate`` on a cache in pages: the prompts enter in one step without padding, and a sequence that has ended gives its pages back.  With ``drafts`` (at most 63) each
    step also checks that many drafted tokens of every sequence (``drafted_tree``); a token that the model samples is always the model's own choice, so the drafts change how many steps it takes
    and not what may come out.  Returns the list of generated id lists (with the prompt in front if ``echo``), each cut at its first stop token."""
    cfg = model.cfg
    if not prompt_tokens or min(len(t) for t in prompt_tokens) == 0:
        raise ValueError("every prompt needs at least one token")
    if max(len(t) for t in prompt_tokens) > cfg.max_seq_len:
        raise ValueError("prompt of %d tokens exceeds the context of %d" % (max(len(t) for t in prompt_tokens), cfg.max_seq_len))
    if not 0 <= drafts <= 63:
        raise ValueError("%d drafted tokens; 0 to 63 can be checked in a step" % drafts)
    if decoder is None:
        longest = [min(cfg.max_seq_len, len(t) + max_gen_len) for t in prompt_tokens]
        decoder = PagedDecoder(model, sum(-(-min(cfg.max_seq_len, n + drafts) // rows) for n in longest), rows)
    stops = set(stop_tokens)
    texts = [list(t) for t in prompt_tokens]
    limits = [min(cfg.max_seq_len, len(t) + max_gen_len) for t in prompt_tokens]

    def pick(logits):
        if temperature > 0:
            return sample_top_p(torch.softmax(logits / temperature, dim=-1), top_p, generator).tolist()
        return torch.argmax(logits, dim=-1).tolist()

    running = [(i, decoder.open()) for i in range(len(texts)) if limits[i] > len(texts[i])]
    opened = [s for _, s in running]
    try:
        fresh = True
        while running:
            sequences = [s for _, s in running]
            if fresh or not drafts:
                chosen = pick(decoder.forward(sequences, [texts[i] if fresh else texts[i][-1:] for i, _ in running]).cpu())
                gained = [[t] for t in chosen]
            else:
                # room for the drafts in the text and in the context
                trees = [drafted_tree(texts[i], min(drafts, limits[i] - len(texts[i]) - 1)) for i, _ in running]
                chosen = pick(decoder.forward(sequences, [t for t, _ in trees], [p for _, p in trees], every=True).cpu())
                gained, kept, at = [], [], 0
                for tree, parents in trees:
                    path, got = [0], []
                    while True:
                        got.append(chosen[at + path[-1]])
                        following = [j for j in range(len(tree)) if parents[j] == path[-1] and tree[j] == got[-1]]
                        if not following:
                            break
                        path += following
                    gained.append(got)
                    kept.append(path)
                    at += len(tree)
                decoder.keep(sequences, [len(t) for t, _ in trees], kept)
            fresh = False
            still = []
            for (i, s), got in zip(running, gained):
                for t in got:
                    texts[i].append(t)
                    if t in stops or len(texts[i]) == limits[i]:
                        decoder.close(s)
                        break
                else:
                    still.append((i, s))
            running = still
    finally:
        for s in opened:
            decoder.close(s)
    out = []
    for prompt, text in zip(prompt_tokens, texts):
        body = text[(0 if echo else len(prompt)):]
        for at, t in enumerate(body):
            if t in stops:
                body = body[:at]
                break
        out.append(body)
    return out
