"""Operators on a key / value cache in pages, on the host: against 64 bits, what is left alone, what is refused."""
import math

import pytest
import torch

from llmc_b200 import ops
from llmc_b200.ops import kernels as KN

import paged_oracle as O

SHAPES = [((1,), (1,), 2, 2, 16, 8), ((40, 0, 17, 8), (3, 0, 17, 0), 4, 2, 24, 8), ((3, 65), (3, 1), 6, 2, 64, 16)]


def _attention_bound(exact, size, dtype):
    # the result's rounding; products and sums of 32 bits over at most a hundred keys and channels each
    return torch.finfo(dtype).eps / 2 * exact.abs() + 2.0 ** -14 * size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keys,new,NH,NKV,HS,rows", SHAPES)
def test_attention(keys, new, NH, NKV, HS, rows, dtype):
    c = O.Case(keys, new, NH, NKV, HS, rows, dtype=dtype, layers=2)
    ops.paged_attention(c.out, c.q, c.cache(ops), NH, layer=1)
    exact, size = O.attention(c, layer=1)
    assert bool(((c.out[:c.N].double() - exact).abs() <= _attention_bound(exact, size, dtype)).all())
    assert bool((c.out[c.N:] == 7).all())


def test_tree_attention_and_an_empty_row():
    parents = [O.random_tree(9, 1), O.random_tree(64, 2)]
    c = O.Case((30, 64), (9, 64), 4, 2, 32, 16)
    tree = ops.tree_masks(parents)
    tree[9] = 0                                          # the second sequence has nothing but its new tokens
    ops.paged_tree_attention(c.out, c.q, c.cache(ops), torch.cat([tree, tree[:3]]), 4)
    exact, size = O.attention(c, tree)
    assert bool(((c.out[:c.N].double() - exact).abs() <= _attention_bound(exact, size, torch.bfloat16)).all())
    assert bool((c.out[9] == 0).all()) and bool((c.out[c.N:] == 7).all())


def test_tree_masks():
    assert ops.tree_masks([[-1, 0, 0, 2, -1], [], [-1]]).tolist() == [1, 3, 5, 13, 16, 1]
    assert ops.tree_masks([list(range(-1, 63))]).tolist()[-1] == -1
    for bad in ([[0]], [[-1, -2]], [[-1] * 65]):
        with pytest.raises(ValueError):
            ops.tree_masks(bad)


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("R", [16, 8])
def test_append(R, halves):
    c = O.Case((9, 0, 40, 16), (9, 0, 5, 1), 4, 2, 16, 8, layers=2)
    before = c.kpages.clone(), c.vpages.clone()
    f = O.angles(40, R)
    ops.paged_rope_cache(c.out[:, :c.NH * c.HS], c.cache(ops), c.raw, f, 4, layer=1, halves=halves)
    x = c.raw[:c.N].double().view(c.N, 8, 16)
    pos = torch.cat([torch.arange(k - n, k) for k, n in zip(c.keys, c.new)])
    y = O.rotated(x[:, :6], f[pos].double(), halves)
    # the result's rounding and three operations in 32 bits
    near = lambda a, b: bool(((a.double() - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -22 * x.abs().max()).all())
    assert near(c.out[:c.N].view(c.N, 4, 16), y[:, :4]) and bool((c.out[c.N:] == 7).all())
    at = torch.cat([f[k - n:] for f, k, n in zip(c.flat, c.keys, c.new)])
    k, v = c.kpages[1].reshape(-1, 2, 16), c.vpages[1].reshape(-1, 2, 16)
    assert near(k[at], y[:, 4:]) and torch.equal(v[at], c.raw[:c.N].view(c.N, 8, 16)[:, 6:])
    rest = torch.ones(k.shape[0], dtype=torch.bool)
    rest[at] = False
    for now, then in ((k, before[0]), (v, before[1])):
        assert torch.equal(now[rest].nan_to_num(9.0), then[1].reshape(-1, 2, 16)[rest].nan_to_num(9.0))
    assert torch.equal(c.kpages[0].nan_to_num(9.0), before[0][0].nan_to_num(9.0))


def test_append_with_positions_is_the_rotation_of_those_positions():
    c = O.Case((30,), (3,), 2, 1, 16, 8, pad=0)
    f = O.angles(64, 16)
    q = torch.empty(3, 32, dtype=torch.bfloat16)
    ops.paged_rope_cache(q, c.cache(ops), c.raw, f, 2, positions=torch.tensor([27, 28, 28], dtype=torch.int32))
    y = O.rotated(c.raw.double().view(3, 4, 16)[:, :2], f[[27, 28, 28]].double(), False)
    assert bool(((q.double().view(3, 2, 16) - y).abs() <= 2.0 ** -8 * y.abs() + 1e-6).all())


def test_keep():
    c = O.Case((9, 33, 20, 12), (4, 33, 7, 0), 2, 2, 16, 8, layers=3)
    kept = torch.zeros(4, 33, dtype=torch.int32)
    lists = [[1, 3], list(range(0, 33, 2)), [6, 6, 6], []]
    for b, l in enumerate(lists):
        kept[b, :len(l)] = torch.tensor(l, dtype=torch.int32)
    old = c.kpages.clone(), c.vpages.clone()
    ops.paged_keep(c.cache(ops), kept, torch.tensor([len(l) for l in lists], dtype=torch.int32))
    for then, now in zip(old, (c.kpages, c.vpages)):
        want = then.clone().view(3, -1, 2, 16)
        source = then.view(3, -1, 2, 16)
        for f, n, l in zip(c.flat, c.new, lists):
            base = len(f) - n
            for j, s in enumerate(l):
                want[:, f[base + j]] = source[:, f[base + s]]
        assert torch.equal(now.view(3, -1, 2, 16).nan_to_num(9.0), want.nan_to_num(9.0))


def test_host_refuses_entries_that_make_no_sense():
    def case(**k):
        c = O.Case((20, 9), (4, 2), 2, 2, 16, 8, pad=0)
        for name, (at, value) in k.items():
            getattr(c, name)[at] = value
        return c
    for wrong in ({"table": ((0, 1), -1)}, {"table": ((0, 0), 99)}, {"lengths": (0, 25)}, {"lengths": (0, -1)}, {"starts": (1, 7)}, {"starts": (0, -1)}):
        c = case(**wrong)
        with pytest.raises(ValueError):
            ops.paged_attention(c.out, c.q, c.cache(ops), 2)
        with pytest.raises(ValueError):
            ops.paged_rope_cache(c.out, c.cache(ops), c.raw, O.angles(64, 16), 2)
    c = case()
    for positions in ([0, 0, 0, 0, 0, 64], [-1, 0, 0, 0, 0, 0]):
        with pytest.raises(ValueError):
            ops.paged_rope_cache(c.out, c.cache(ops), c.raw, O.angles(64, 16), 2, positions=torch.tensor(positions, dtype=torch.int32))
    for kept, counts in (([[1, 0], [0, 1]], [2, 2]), ([[1, 4], [0, 1]], [2, 2]), ([[0, 1], [0, 1]], [3, 2]), ([[0, 1], [0, 1]], [2, -1])):
        with pytest.raises(ValueError):
            ops.paged_keep(c.cache(ops), torch.tensor(kept, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32))


@pytest.mark.parametrize("handle", [ops.paged_cache, KN.paged_cache])
def test_handle_refuses(handle):
    c = O.Case((20, 9), (4, 2), 2, 2, 16, 8)
    good = dict(kpages=c.kpages, vpages=c.vpages, table=c.table, lengths=c.lengths, starts=c.starts)
    handle(**good)
    handle(**dict(good, kpages=c.kpages[0], vpages=c.vpages[0]))
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    one = z(4, 2, 8, 2, 16)
    for wrong in (dict(kpages=c.kpages[:, :-1]), dict(vpages=c.vpages.float()), dict(kpages=z(4, 2, 16), vpages=z(4, 2, 16)), dict(table=c.table.long()), dict(table=c.table[:1]),
                  dict(lengths=c.lengths[:1]), dict(starts=c.starts[:-1]), dict(lengths=c.lengths.float()), dict(kpages=z(4, 12, 2, 16), vpages=z(4, 12, 2, 16)),
                  dict(kpages=z(4, 4, 2, 16), vpages=z(4, 4, 2, 16)), dict(kpages=z(4, 8, 2, 20), vpages=z(4, 8, 2, 20)), dict(kpages=z(4, 8, 2, 8), vpages=z(4, 8, 2, 8)),
                  dict(kpages=z(4, 8, 2, 136), vpages=z(4, 8, 2, 136)), dict(vpages=c.kpages), dict(table=c.table.t().contiguous().t()),
                  dict(kpages=z(1, 8, 2, 16).expand(4, 8, 2, 16), vpages=z(4, 8, 2, 16)), dict(kpages=one.view(8, 8, 2, 16)[:7], vpages=one.view(8, 8, 2, 16)[1:]),
                  dict(starts=c.starts.to("meta"))):
        with pytest.raises(ValueError):
            handle(**dict(good, **wrong))
    handle(**dict(good, kpages=one[:, 0], vpages=one[:, 1]))


def test_device_handle_refuses_what_the_kernels_cannot_read():
    c = O.Case((20, 9), (4, 2), 2, 2, 16, 8)
    odd = torch.zeros(4 * 8 * 2 * 16 + 4, dtype=torch.bfloat16)[4:].view(4, 8, 2, 16)
    wide = torch.zeros(4, 8, 2, 20, dtype=torch.bfloat16)[..., :16]
    turned = torch.zeros(4, 8, 16, 2, dtype=torch.bfloat16).transpose(2, 3)
    for pages in (odd, wide, turned):
        with pytest.raises(ValueError):
            KN.paged_cache(pages, torch.zeros(4, 8, 2, 16, dtype=torch.bfloat16), c.table, c.lengths, c.starts)
    with pytest.raises(ValueError):
        KN.paged_cache(c.kpages.float(), c.vpages.float(), c.table, c.lengths, c.starts)


@pytest.mark.parametrize("K", [ops, KN])
def test_calls_refuse(K):
    c = O.Case((20, 9), (4, 2), 4, 2, 16, 8)
    cache, f, n = c.cache(K), O.angles(64, 16), c.q.shape[0]
    tree = torch.zeros(n, dtype=torch.int64)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    for wrong in (dict(NH=3), dict(NH=0), dict(layer=1), dict(layer=-1), dict(out=c.q), dict(out=c.out[:-1]), dict(q=c.q[:, :-8]), dict(q=c.q.float()), dict(out=c.out.float())):
        with pytest.raises(ValueError):
            K.paged_attention(**dict(dict(out=c.out, q=c.q, cache=cache, NH=4, layer=0), **wrong))
        with pytest.raises(ValueError):
            K.paged_tree_attention(**dict(dict(out=c.out, q=c.q, cache=cache, tree=tree, NH=4, layer=0), **wrong))
    for wrong in (tree[:-1], tree.int()):
        with pytest.raises(ValueError):
            K.paged_tree_attention(c.out, c.q, cache, wrong, 4)
    good = dict(q=c.out, cache=cache, raw=c.raw, freqs=f, NH=4)
    for wrong in (dict(freqs=f.double()), dict(freqs=f[:, :, 0]), dict(freqs=O.angles(64, 18)), dict(freqs=f.transpose(0, 1)), dict(positions=tree), dict(positions=tree.int()[:-1]),
                  dict(raw=c.raw[:, :-16]), dict(raw=c.raw.float()), dict(q=c.out[:-1]), dict(q=c.raw[:, :64]), dict(layer=2), dict(NH=5)):
        with pytest.raises(ValueError):
            K.paged_rope_cache(**dict(good, **wrong))
    counts = torch.zeros(2, dtype=torch.int32)
    for kept, cnt in ((z(2, 4, dtype=torch.int64), counts), (z(3, 4, dtype=torch.int32), counts), (z(2, 257, dtype=torch.int32), counts), (z(2, 0, dtype=torch.int32), counts),
                      (z(2, 4, dtype=torch.int32), counts[:1]), (z(2, 4, dtype=torch.int32), counts.long()), (z(4, 2, dtype=torch.int32).t(), counts)):
        with pytest.raises(ValueError):
            K.paged_keep(cache, kept, cnt)


def test_device_calls_refuse_rows_off_16_bytes():
    c = O.Case((20, 9), (4, 2), 4, 2, 16, 8)
    cache = c.cache(KN)
    for wrong in (torch.zeros(c.q.shape[0], 68, dtype=torch.bfloat16)[:, :64], torch.zeros(c.q.shape[0], 72, dtype=torch.bfloat16)[:, 4:68], torch.zeros(64, c.q.shape[0], dtype=torch.bfloat16).t()):
        with pytest.raises(ValueError):
            KN.paged_attention(c.out, wrong, cache, 4)
        with pytest.raises(ValueError):
            KN.paged_attention(wrong, c.q, cache, 4)


def test_nothing_to_do():
    c = O.Case((), (), 2, 1, 16, 8, pad=2)
    ops.paged_attention(c.out, c.q, c.cache(ops), 2)
    KN.paged_attention(c.out, c.q, c.cache(KN), 2)
    KN.paged_keep(c.cache(KN), torch.zeros(0, 4, dtype=torch.int32), torch.zeros(0, dtype=torch.int32))
    assert bool((c.out == 7).all())
    assert math.isnan(float(c.q[0, 0]))


@pytest.mark.parametrize("handle", [ops.paged_cache, KN.paged_cache])
def test_handle_refuses_room_for_more_keys_than_counts_hold(handle):
    pages = torch.zeros(2, 1, 1 << 10, 1, 16, dtype=torch.bfloat16)
    lengths, starts = torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    handle(pages[0], pages[1], torch.zeros(1, 1 << 20, dtype=torch.int32), lengths, starts)
    with pytest.raises(ValueError):
        handle(pages[0], pages[1], torch.zeros(1, (1 << 20) + 1, dtype=torch.int32), lengths, starts)
