"""Operators on a key / value cache in pages, on the host: numbers that are not finite, memory that is shared, what a refused call leaves behind."""
import ctypes
import math
import struct

import pytest
import torch

from llmc_b200 import _lib, ops
from llmc_b200.ops import kernels as KN

import paged_oracle as O

BF16 = torch.bfloat16


@pytest.mark.parametrize("tree", [False, True])
def test_numbers_that_are_not_finite_stay(tree):
    """A query that is not a number, scores that 32 bits do not hold, and visible scores that are all minus infinity give what a softmax gives: no number.  Only a row that sees no key is 0."""
    c = O.Case((20, 9, 4), (3, 2, 4), 2, 1, 16, 8, dtype=torch.float32, pad=0)
    c.q[1, 3] = math.nan                                 # head 0 of token 1
    c.q[3] = 1e30                                        # every key of the second sequence: scores past 32 bits
    c.kpages[0].view(-1, 1, 16)[c.flat[1]] = 1e30
    c.q[4] = -1e30
    c.lengths[2] = 2                                     # four new tokens, two slots: the first two have none
    masks = ops.tree_masks([[-1, 0, 1], [-1, 0], [-1, 0, 1, 2]])
    if tree:
        masks[5:7] = 0
        ops.paged_tree_attention(c.out, c.q, c.cache(ops), masks, 2)
    else:
        ops.paged_attention(c.out, c.q, c.cache(ops), 2)
    wrong = c.out.isnan().view(9, 2, 16).all(-1)
    assert wrong.tolist() == [[False, False], [True, False], [False, False], [True, True], [True, True]] + [[False, False]] * 4
    assert bool((c.out[5:7] == 0).all()) and bool((c.out[7:] != 0).all())
    assert not bool(c.out.isinf().any())


def test_angles_off_8_bytes_are_refused():
    """A cosine and its sine are read together.  On the host before a launch, by the operator and by the entry point alike; host tensors may lie anywhere."""
    c = O.Case((20, 9), (4, 2), 2, 1, 16, 8, pad=0)
    room = torch.zeros(30 * 8 * 2 + 1)
    f = room[1:].view(30, 8, 2)
    f.copy_(O.angles(30, 16))
    assert f.is_contiguous() and f.data_ptr() % 8 == 4
    cache = c.cache(KN)
    with pytest.raises(ValueError, match="8-byte"):
        KN.paged_rope_cache(c.out, cache, c.raw, f, 2)
    call = KN._pack_append(cache.address, c.out.data_ptr(), c.raw.data_ptr(), f.data_ptr(), 0, c.N, 32, 64, 2, 16, 30, 0, 0, 0)
    assert _lib.cuda().llmc_paged_rope_cache(call) == -1
    ops.paged_rope_cache(c.out, c.cache(ops), c.raw, f, 2)
    plain = torch.empty_like(c.out)
    ops.paged_rope_cache(plain, c.cache(ops), c.raw, O.angles(30, 16), 2)
    assert torch.equal(c.out, plain)


def _bytes(t):
    """Offsets of all elements of a view."""
    at = torch.zeros((), dtype=torch.int64) + t.storage_offset()
    for s, n in zip(t.stride(), t.shape):
        at = at[..., None] + torch.arange(n) * s
    return set(at.flatten().tolist())


@pytest.mark.parametrize("handle", [ops.paged_cache, KN.paged_cache])
def test_keys_and_values_that_share_memory_are_refused(handle):
    lengths, starts, table = torch.ones(2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    flat = torch.zeros(20000, dtype=BF16)
    at = lambda offset, *strides: flat.as_strided((3, 8, 2, 16), strides + (1,), offset)
    rows, heads = (512, 32, 16), (512, 16, 128)          # a page's rows beside each other with room for twice as many; a head's
    pairs = [(at(0, *rows), at(o, *rows)) for o in (0, 8, 16, 32, 128, 248, 256, 264, 496, 504, 512, 1024, 1528, 1536)]
    pairs += [(at(512, *rows), at(o, *rows)) for o in (0, 256, 264, 248)]
    pairs += [(at(0, 512, 64, 32), at(o, 512, 64, 32)) for o in (8, 16, 24, 48, 1000, 1040)]
    pairs += [(at(0, *rows), at(o, *heads)) for o in (0, 8, 1272, 1280, 1536)] + [(at(o, 256, 32, 16), at(p, *rows)) for o, p in ((64, 0), (0, 256), (2000, 0), (0, 760), (0, 768))]
    seen = set()
    for k, v in pairs:
        shared = bool(_bytes(k) & _bytes(v))
        if not shared and k.stride() != v.stride() and max(min(_bytes(k)), min(_bytes(v))) < min(max(_bytes(k)), max(_bytes(v))):
            continue                                     # in one another's gaps
        seen.add(shared)
        if shared:
            with pytest.raises(ValueError, match="share memory"):
                handle(k, v, table, lengths, starts)
        else:
            handle(k, v, table, lengths, starts)
    assert seen == {True, False}


def test_whether_a_pool_lies_in_a_range():
    g = torch.Generator().manual_seed(0)
    draw = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))
    flat = torch.zeros(4000, dtype=torch.uint8)
    for _ in range(300):
        strides, shape, end = [], [], 1
        for _ in range(3):
            strides.append(end + draw(0, 4)), shape.append(draw(1, 5))
            end = strides[-1] * (shape[-1] - 1) + end
        pool = flat.as_strided(shape, strides, 100)
        has = _bytes(pool)
        for _ in range(20):
            lo = draw(90, 110 + end)
            hi = lo + draw(0, 12)
            assert KN._pool_meets(KN._pool(pool), flat.data_ptr() + lo, flat.data_ptr() + hi) == any(b in has for b in range(lo, hi))
        for apart in range(-end - 3, end + 4):
            assert KN._pools_meet(apart, *KN._pool(pool)[2:]) == any(b + apart in has for b in has)


@pytest.mark.parametrize("K", [ops, KN])
def test_matrices_inside_the_pages_are_refused(K):
    """What a call writes, and what an append reads beside its writes.  A matrix in a gap between pages is taken: the call gets as far as it does with one that lies elsewhere."""
    N, NH, HS = 6, 2, 16
    lengths, starts, table = torch.tensor([20, 9], dtype=torch.int32), torch.tensor([0, 4, 6], dtype=torch.int32), torch.arange(6, dtype=torch.int32).view(2, 3)
    flat = torch.zeros(2, 40000, dtype=BF16)
    pool = lambda i: flat[i].as_strided((2, 6, 8, 1, HS), (8192, 1024, 16, 16, 1))             # 128 elements of each 1024
    cache = K.paged_cache(pool(0), pool(1), table, lengths, starts)
    rows = lambda i, at, cols, ld: flat[i].as_strided((N, cols), (ld, 1), 40000 * i + at)
    q, raw, f = torch.zeros(N, NH * HS, dtype=BF16), torch.zeros(N, (NH + 2) * HS, dtype=BF16), O.angles(64, HS)
    fine = [rows(0, 128, 32, 32), rows(1, 1024 + 512, 32, 32), rows(1, 128, 32, 1024), rows(0, 6144, 32, 256), rows(1, 8192 + 6144, 32, 48)]
    shared = [rows(0, 0, 32, 32), rows(1, 64, 32, 32), rows(0, 1024 - 32, 32, 40), rows(1, 1024 - 32 * 5, 32, 32), rows(0, 128, 32, 1024 + 8 * 28), rows(1, 8192 + 5 * 1024 + 96, 32, 1024)]

    def attempt(call):
        try:
            call()
        except ValueError as e:
            return "share memory" in str(e)
        except Exception as e:                           # the device's form stops at the missing device
            assert K is KN, e
        return False

    for places, wrong in ((fine, False), (shared, True)):
        for m in places:
            assert attempt(lambda: K.paged_attention(m, q, cache, NH)) == wrong
            assert attempt(lambda: K.paged_tree_attention(m, q, cache, torch.zeros(N, dtype=torch.int64), NH)) == wrong
            assert attempt(lambda: K.paged_rope_cache(m, cache, raw, f, NH)) == wrong
            wide = m.as_strided((N, 64), (max(64, m.stride(0)), 1))
            if wrong or m.stride(0) >= 64:
                assert attempt(lambda: K.paged_rope_cache(q, cache, wide, f, NH)) == wrong
            # attention reads both
            assert not attempt(lambda: K.paged_attention(q, m, cache, NH))


def test_rows_that_32_bit_counts_do_not_hold_are_refused():
    """By the entry point, before it looks at anything else."""
    c = O.Case((9,), (1,), 2, 1, 16, 8, pad=0)
    cache, lib = c.cache(KN), _lib.cuda()
    for N in (0, -1, (1 << 30) + 1, 1 << 31, 1 << 40):
        assert lib.llmc_paged_attention(KN._pack_attention(cache.address, 0, 0, 0, 0, N, 32, 32, 2, 0, 0)) == -1


def test_two_graphs_of_attention_share_no_scratch(monkeypatch):
    """Seen from the host: what a captured call asks for, in the graphs of two owners that keep their buffers.  (What a graph's pool hands out stays the graph's; here the test keeps it.)"""
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True, raising=False)
    monkeypatch.setattr(KN, "_stream_of", lambda op, device: 0)
    calls = []

    class Lib:
        llmc_paged_attention_workspace = llmc_paged_attention_launches = staticmethod(lambda cache, N, NH: 1000)
        llmc_paged_attention = staticmethod(lambda call: calls.append(struct.unpack("11q", call)[4]) or 0)

    monkeypatch.setattr(_lib, "cuda", lambda: Lib)
    empty, kept = torch.empty, []
    monkeypatch.setattr(torch, "empty", lambda *a, **k: kept.append(empty(*a, **k)) or kept[-1])
    c = O.Case((20, 9), (4, 2), 2, 1, 16, 8, pad=0)
    for _ in range(2):
        with KN.scratch_taken():
            KN.paged_attention(c.out, c.q, c.cache(KN), 2)
    assert len(calls) == 2 and calls[0] != calls[1]


def _decoder(pages, rows=8):
    from llmc_b200.models import paged
    from test_paged_generate_cpu import small_model
    return paged.PagedDecoder(small_model(), pages, rows)


def test_a_refused_step_takes_no_pages():
    d = _decoder(3)
    a, b = d.open(), d.open()
    with pytest.raises(RuntimeError):
        d.forward([a, b], [[1] * 9, [2] * 9])            # two pages each
    assert not a.pages and not b.pages and len(d.free) == 3
    for parents in ([[-1, 1]], [[-1, -2]], [[-1, 7]]):
        with pytest.raises(ValueError):
            d.forward([a], [[1, 2]], parents)
        assert not a.pages and a.length == 0
    d.forward([b], [[2] * 9])
    d.forward([a], [[1] * 8])
    assert (len(a.pages), len(b.pages), len(d.free)) == (1, 2, 0)
    d.forward([b], [[2] * 7])                            # what the pages have room for
    with pytest.raises(RuntimeError):
        d.forward([b, a], [[2], [1]])
    assert (a.length, b.length, len(a.pages), len(b.pages)) == (8, 16, 1, 2)


def test_keep_refuses_lists_that_do_not_fit_the_sequences():
    d = _decoder(8)
    a, b = d.open(), d.open()
    d.forward([a, b], [[1, 2, 3], [4, 5]])
    for sequences, new, kept in (([a, b], [3, 2], [[0, 1]]), ([a, b], [3], [[0], [0]]), ([a], [3, 2], [[0]]), ([a, a], [3, 3], [[0], [0]]), ([], [], []), ([a], [4], [[0]]), ([b], [-1], [[]]),
                                 ([a, b], [3, 3], [[0], [0]])):
        with pytest.raises(ValueError):
            d.keep(sequences, new, kept)
        assert (a.length, b.length) == (3, 2)
    d.keep([a, b], [3, 2], [[0, 1], []])
    assert (a.length, b.length) == (2, 0)


def test_the_command_line_is_refused_before_a_model_is_made():
    import train_llama3
    parse = lambda *a: train_llama3.build_parser().parse_args(["--model", "llama3:l=1,c=64,h=4,kv=1,t=48,v=13,m=16,f=1.3", *a])
    for wrong in (["--drafts", "4"], ["--page_rows", "12"], ["--page_rows", "4"], ["--page_rows", "-8"], ["--page_rows", "8", "--drafts", "64"], ["--page_rows", "8", "--use_kv", "0"]):
        with pytest.raises(SystemExit):
            train_llama3.train_config(parse(*wrong))
    train_llama3.train_config(parse("--page_rows", "8", "--drafts", "63"))
    train_llama3.train_config(parse())


def test_the_host_launches_nothing_and_a_handle_fits_its_entry_points():
    before = KN.launch_count()
    c = O.Case((20, 9), (4, 2), 4, 2, 16, 8)
    cache = c.cache(ops)
    ops.paged_rope_cache(c.out, cache, c.raw, O.angles(64, 16), 4)
    ops.paged_attention(c.out, c.q, cache, 4)
    ops.paged_tree_attention(c.out, c.q, cache, torch.zeros(c.q.shape[0], dtype=torch.int64), 4)
    ops.paged_keep(cache, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    d = _decoder(4)
    d.forward([d.open()], [[1, 2, 3]])
    assert KN.launch_count() == before
    assert ctypes.sizeof(_lib.PagedCache) == _lib.cuda().llmc_paged_cache_size()
    handle = c.cache(KN).call
    assert (handle.layers, handle.pages, handle.page_shift, handle.heads, handle.hs, handle.sequences, handle.table_width) == (1, c.kpages.shape[1], 3, 2, 16, 2, c.table.shape[1])
    assert handle.k == c.kpages.data_ptr() and handle.starts == c.starts.data_ptr() and (handle.k_page, handle.k_row, handle.k_head) == c.kpages.stride()[1:4]
