// A key / value cache in pages: slot s of sequence b is row s % page of page table[b][s / page], and a row holds NKV heads of HS channels.  What is new in a call are
// rows starts[b] .. starts[b + 1] - 1 of a batch without padding; the last of them lies in slot lengths[b] - 1.  Table, lengths and starts are read from device memory when a
// kernel runs, so that a captured graph follows them, and a kernel checks what it reads there: a wrong entry is recorded in the status word, and nothing outside the tensors is touched.
#pragma once
#include "common.cuh"

// What a caller's handle holds (the fields of _lib.PagedCache); strides in elements
struct PagedCache {
    bf16 *k, *v;
    const int *table, *lengths, *starts;
    long long k_layer, k_page, k_row, k_head, v_layer, v_page, v_row, v_head;
    long long table_row;                // entries from one sequence's row of the table to the next's
    int layers, pages, page_shift, heads, hs, sequences, table_width, align;
};

struct PagedSpan { int first, count, keys; };       // rows of a sequence and its keys; count and keys are 0 where its entries make no sense

// N: rows of the batch.  A sequence is left out whose start lies in front of the one before it, since its rows may be another's.
DEVINL PagedSpan paged_span(const PagedCache& c, int b, int N, unsigned int* status, unsigned int where) {
    const int before = c.starts[b > 0 ? b - 1 : 0], s0 = c.starts[b], s1 = c.starts[b + 1], len = c.lengths[b];
    if (before < 0 || s0 < before || s1 < s0 || s1 > N || len < 0 || (long long)len > ((long long)c.table_width << c.page_shift)) {
        record_error(status, ST_BAD_ARG, where);
        return {0, 0, 0};
    }
    return {s0, s1 - s0, len};
}

// The page of a slot below the sequence's length, -1 (and the status word) where the table names no page
DEVINL int paged_page(const PagedCache& c, int b, int slot, unsigned int* status, unsigned int where) {
    const int p = c.table[b * c.table_row + (slot >> c.page_shift)];
    if ((unsigned)p >= (unsigned)c.pages) { record_error(status, ST_BAD_ARG, where); return -1; }
    return p;
}

// The sequence that row n belongs to (the first one that claims it), found by a warp; as many as there are: none, it lies behind the last one
DEVINL int paged_sequence(const PagedCache& c, int n) {
    int b = c.sequences;
    for (int i = threadIdx.x & 31; i < c.sequences; i += 32)
        if (c.starts[i] <= n && n < c.starts[i + 1]) b = min(b, i);
    return __reduce_min_sync(0xffffffffu, b);
}
