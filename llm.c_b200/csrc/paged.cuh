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
    int layers, pages, page_shift, heads, hs, sequences, table_width;
};

// Arguments of the entry points, a 64-bit word each: a caller packs them in one go (a call through ctypes with ten arguments takes the host 2.3 us, with one 0.5)
struct PagedAppendCall {
    const PagedCache* cache;
    bf16* q;
    const bf16* raw;
    const float2* freqs;               // (freqs_len, R / 2) cos, sin
    const int* positions;              // null, or one per row
    long long N, ldq, ldr, NH, R, freqs_len, halves, layer;
    cudaStream_t stream;
};
struct PagedAttentionCall {
    const PagedCache* cache;
    bf16* out;
    const bf16* q;
    const long long* tree;             // null, or one per row
    float* ws;
    long long N, ldo, ldq, NH, layer;
    cudaStream_t stream;
};
struct PagedKeepCall {
    const PagedCache* cache;
    const int *kept, *counts;
    long long D, kept_row;
    cudaStream_t stream;
};

// n / d for n below 2^31, by a product (Granlund and Montgomery's round-up method)
struct FastDiv {
    unsigned mul, shift;
    FastDiv() = default;
    explicit FastDiv(unsigned d) {
        for (shift = 0; (1ull << shift) < d; ) shift++;
        mul = (unsigned)((((1ull << shift) - d) << 32) / d + 1);
    }
    DEVINL unsigned operator()(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct PagedSpan { int first, count, keys; };       // rows of a sequence and its keys; count and keys are 0 where its entries make no sense

// N: rows of the batch.  A sequence is left out whose start lies in front of the one before it, since its rows may be another's.
DEVINL PagedSpan paged_span(const PagedCache& c, int before, int s0, int s1, int len, int N, unsigned int* status, unsigned int where) {
    if (before < 0 || s0 < before || s1 < s0 || s1 > N || len < 0 || (long long)len > ((long long)c.table_width << c.page_shift)) {
        record_error(status, ST_BAD_ARG, where);
        return {0, 0, 0};
    }
    return {s0, s1 - s0, len};
}
DEVINL PagedSpan paged_span(const PagedCache& c, int b, int N, unsigned int* status, unsigned int where) {
    return paged_span(c, c.starts[b > 0 ? b - 1 : 0], c.starts[b], c.starts[b + 1], c.lengths[b], N, status, where);
}

// The page of a slot below the sequence's length, -1 (and the status word) where the table names no page
DEVINL int paged_page(const PagedCache& c, int b, int slot, unsigned int* status, unsigned int where) {
    const int p = c.table[b * c.table_row + (slot >> c.page_shift)];
    if ((unsigned)p >= (unsigned)c.pages) { record_error(status, ST_BAD_ARG, where); return -1; }
    return p;
}


// A row's maximum is -inf where it has seen no key, and its result is then 0.  Where all scores that it sees are -inf its sum is 0 too, but the result is no number, as of any softmax: such a maximum
// becomes the lowest finite number when a piece ends, which weighs nothing beside another one, and 0 / 0 is left.
// limit: keys in front of it are visible; bits: new tokens that are, of `count` in a sequence of `keys`
DEVINL float paged_maximum(float m, int limit, unsigned long long bits, int count, int keys) {
    if (m != -INFINITY || keys == 0) return m;
    const unsigned long long there = count < 64 ? bits & ((1ull << count) - 1) : bits;
    return limit > 0 || (there >> min(63, max(0, count - keys))) != 0 ? -3.402823466e38f : m;      // (with bits there are at most 64 new tokens)
}
DEVINL float paged_inverse(float m, float l) { return m == -INFINITY ? 0.f : 1.0f / l; }

// How the attention kernels cut their work.  A piece is what one block does without a pause: the keys of one cached head for a group of query rows.  A piece is counted in units
// of `unit` keys (one at least, which writes the zeros of rows without keys), and the units of all pieces, one behind the other, are dealt to the blocks in equal and contiguous shares, so that
// sequences of any lengths load all SMs alike.  A piece that a share ends in leaves partial results, which a second kernel joins in the order of the keys.
struct PagedShares {
    int blocks;                // shares that have units, one to a block or to a warp
    int size, longer;          // the first `longer` shares have size + 1 units, the others size
    // total units among at most `most` blocks
    DEVINL PagedShares(int total, int most) {
        blocks = min(most, total);
        size = blocks ? total / blocks : 0;
        longer = total - size * blocks;
    }
    DEVINL int first(int share) const { return size * share + min(share, longer); }
    // the share that unit u lies in
    DEVINL int share_of(int u) const { return u < longer * (size + 1) ? u / (size + 1) : min(blocks - 1, longer + (u - longer * (size + 1)) / size); }
};

// Where a unit lies: the sequence, and the units of it in front
struct PagedPlace { int b, offset; PagedSpan s; };
// Sums of units stay below this: a call whose work cannot be more is all that the host lets through.  More of them come of starts that claim rows many times.
constexpr unsigned PAGED_UNITS = 1u << 30;
// units_of(span): units of a sequence; wanted(total): the unit that is looked for, below 0: none.  A warp calls this; the sum of all units (0, and the status word, where it is too large).
// Sequences are dealt to the lanes.  Entries are read once more where the unit is looked for and where the shares are walked: of a caller that changes them meanwhile the result is anything, but each
// span is checked by itself, and no walk goes past the last sequence.
template <class F, class W>
DEVINL int paged_find(const PagedCache& c, int N, unsigned int* status, unsigned int where, F units_of, W wanted, PagedPlace& place) {
    const int lane = threadIdx.x & 31;
    const int per = (c.sequences + 31) / 32, b0 = min(c.sequences, lane * per), b1 = min(c.sequences, b0 + per);
    PagedSpan s = {0, 0, 0};
    unsigned sum = 0;
    for (int b = b0; b < b1; b += 4) {
        // four sequences' entries on their way at a time
        int before[4], s0[4], s1[4], len[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = min(b + i, b1 - 1);
            before[i] = c.starts[at > 0 ? at - 1 : 0]; s0[i] = c.starts[at]; s1[i] = c.starts[at + 1]; len[i] = c.lengths[at];
        }
        #pragma unroll
        for (int i = 0; i < 4; i++)
            if (b + i < b1) {
                s = paged_span(c, before[i], s0[i], s1[i], len[i], N, status, where);
                sum = min(sum + units_of(s), PAGED_UNITS);
            }
    }
    unsigned upto = sum;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto = min(upto + v, PAGED_UNITS); }
    int total = (int)__shfl_sync(0xffffffffu, upto, 31);
    if (total == PAGED_UNITS) {
        record_error(status, ST_BAD_ARG, where);
        total = 0;
    }
    const int u = wanted(total);
    int at = (int)(upto - sum), b = b0;
    const bool mine = u >= at && u < (int)upto;
    if (mine && per > 1)
        for (;; b++) {
            s = b < b1 ? paged_span(c, b, N, status, where) : PagedSpan{0, 0, 0};      // (b1: only where the entries are no longer those that were added up)
            const int n = units_of(s);
            if (u < at + n || b >= b1) break;
            at += n;
        }
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    const int from = who ? __ffs(who) - 1 : 0;
    place.b = __shfl_sync(0xffffffffu, b, from);
    place.offset = __shfl_sync(0xffffffffu, u - at, from);
    place.s.first = __shfl_sync(0xffffffffu, s.first, from);
    place.s.count = __shfl_sync(0xffffffffu, s.count, from);
    place.s.keys = __shfl_sync(0xffffffffu, s.keys, from);
    return total;
}

// What the first share that begins inside a piece leaves for the kernel that joins the parts, in front of the partials in the workspace: 8 words for each share
struct PagedJoin {
    int parts;                 // of shares k - 1, k, ...; 0: nothing to join
    int first, count, g, row;  // rows of the sequence in the batch, the cached head, the first query row of the piece
    int pad[3];
};

// Shared memory of a kernel, asked for once on each device
template <typename K>
inline int paged_shared_memory(K kernel, int bytes, bool (&done)[64]) {
    int dev = 0;
    CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 64 && done[dev]) return 0;
    CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 64) done[dev] = true;
    return 0;
}
