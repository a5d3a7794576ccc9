"""Plain 64-bit form of the operators on a key / value cache in pages, and caches to try them on."""
import math

import torch

F64 = torch.float64


class Case:
    """A batch of sequences: ``keys`` and ``new`` tokens of each, pages in no order.  What no sequence has is NaN: slots behind a sequence's length, pages of none, rows behind the last
    sequence, table entries behind a sequence's last page."""

    def __init__(self, keys, new, NH, NKV, HS, rows, seed=0, layers=1, device="cpu", dtype=torch.bfloat16, pad=3, width=0, std=1.0, layout="rows"):
        g = torch.Generator().manual_seed(seed)
        self.keys, self.new, self.NH, self.NKV, self.HS, self.rows = list(keys), list(new), NH, NKV, HS, rows
        B = len(self.keys)
        count = [-(-k // rows) for k in self.keys]
        pages = sum(count) + 2
        order = torch.randperm(pages, generator=g).tolist()
        table = torch.full((B, max(count + [1]) + width), 2 ** 30, dtype=torch.int32)
        self.flat = []                                   # of each sequence: where its slots lie among all rows of all pages
        at = 0
        for b, c in enumerate(count):
            table[b, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
            at += c
            slot = torch.arange(self.keys[b])
            self.flat.append(table[b].long()[slot // rows] * rows + slot % rows)
        self.N = sum(self.new)
        starts = [0]
        for n in self.new:
            starts.append(starts[-1] + n)
        pools = []
        for _ in range(2):
            pool = torch.full((layers, pages * rows, NKV, HS), math.nan)
            for f in self.flat:
                pool[:, f] = torch.randn(layers, len(f), NKV, HS, generator=g) * std
            pools.append(pool.view(layers, pages, rows, NKV, HS).to(dtype))
        if layout == "heads":                            # (layers, pages, heads, rows, channels) in memory
            pools = [p.permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4) for p in pools]
        elif layout == "both":                           # keys and values of a page next to each other
            both = torch.stack(pools, 2).to(device)
            pools = [both[:, :, 0], both[:, :, 1]]
        to = lambda t: t.to(device)
        self.kpages, self.vpages = (to(p) for p in pools)
        self.table, self.lengths, self.starts = to(table), to(torch.tensor(self.keys, dtype=torch.int32)), to(torch.tensor(starts, dtype=torch.int32))
        rowsof = lambda cols: to(torch.cat([torch.randn(self.N, cols, generator=g), torch.full((pad, cols), math.nan)]).to(dtype))
        self.q, self.raw = rowsof(NH * HS), rowsof((NH + 2 * NKV) * HS)
        self.out = torch.full((self.N + pad, NH * HS), 7.0, dtype=dtype, device=device)
        self.device = device

    def cache(self, ops):
        return ops.paged_cache(self.kpages, self.vpages, self.table, self.lengths, self.starts)

    def pool(self, pages, layer=0):
        return pages[layer].reshape(-1, self.NKV, self.HS).to("cpu", F64)


def attention(case, tree=None, layer=0):
    """Outputs of the rows that belong to a sequence, and sum |p v| of each (what roundings of probabilities scale with)."""
    K, V = case.pool(case.kpages, layer), case.pool(case.vpages, layer)
    q = case.q[:case.N].to("cpu", F64).view(case.N, case.NH, case.HS)
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    G, at = case.NH // case.NKV, 0
    for b, n in enumerate(case.new):
        context = case.keys[b] - n
        for i in range(n):
            if tree is None:
                seen = case.flat[b][:max(0, context + i + 1)]
            else:
                mask = int(tree[at + i])
                seen = case.flat[b][[s for s in range(case.keys[b]) if s < context or mask >> (s - context) & 1]]
            if len(seen):
                k, v = K[seen].repeat_interleave(G, 1), V[seen].repeat_interleave(G, 1)
                p = torch.softmax(torch.einsum("hd,khd->hk", q[at + i], k) / math.sqrt(case.HS), 1)
                out[at + i] = torch.einsum("hk,khd->hd", p, v)
                size[at + i] = torch.einsum("hk,khd->hd", p, v.abs())
        at += n
    return out.view(case.N, -1), size.view(case.N, -1)


def rotated(x, angles, halves):
    """x (N, heads, HS), angles (N, R / 2, 2), both in 64 bits."""
    R = 2 * angles.shape[1]
    y = x.clone()
    for i in range(R // 2):
        a, b = (i, i + R // 2) if halves else (2 * i, 2 * i + 1)
        c, s = angles[:, None, i, 0], angles[:, None, i, 1]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def angles(length, R, device="cpu"):
    a = torch.arange(length, dtype=F64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=F64) / R)
    return torch.stack([a.cos(), a.sin()], -1).float().to(device)


def random_tree(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(n)]
