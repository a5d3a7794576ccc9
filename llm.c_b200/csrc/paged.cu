// Writing into a key / value cache in pages (paged.cuh):
//
//   paged_rope_cache   raw (N, (NH + 2 NKV) HS), the new tokens of all sequences behind one another -> q (N, NH, HS) rotated queries; rotated keys and values to the tokens' slots.
//                      The first R channels of a head are rotated, in pairs of neighbours (2 i, 2 i + 1) or of two halves (i, i + R / 2), by the angle of the token's slot or of a position given.
//   paged_keep         of the newest tokens of every sequence, those that `kept` lists move to the front, in all layers (what remains of a tree of drafted tokens).
//
// Both move every byte once and compute next to nothing.
#include "paged.cuh"
#include "pdl.cuh"

namespace {

// One rotary pair.  The fused product of each sum is written out, as in decode.cu: the same bits
DEVINL float2 rotate(float re, float im, float c, float s) { return make_float2(fmaf(re, c, -__fmul_rn(im, s)), fmaf(re, s, __fmul_rn(im, c))); }

constexpr int PR_THREADS = 256;        // at most
constexpr int PR_TOKENS = 256;         // whose places a block looks up at once

struct AppendArgs {
    bf16* q;
    const bf16* raw;
    const float2* freqs;
    const int* positions;
    long long ldq, ldr;
    int N, NH, R, freqs_len, layer;
    int head_chunks, chunks;           // 16-byte chunks of a head, of a token
    int lanes;                         // tokens side by side in a block
    unsigned int* status;
};

// A thread has one chunk of 8 channels of a head and goes from token to token, so that where it reads and writes in a token, and whether it rotates, is worked out once; a block has a slice of a
// token's chunks (blockIdx.y), or several tokens side by side where they are small.  The places of all tokens of the block are looked up at once, a token a thread, while its first loads are on
// their way; then a thread has one token at hand and the next one on its way.
// FORM: the pairs of a rotation are 0 neighbours, 1 two halves whose chunks go together, 2 either, with a number of channels that is not made of whole chunks.
// 11769 tokens of 48 heads of 64 channels: 29 us, as two halves 37.5 (a second load for the other half's chunk, and fewer threads on an SM); FORM 2, whatever it rotates, 68 to 69: eight loads of a
// partner and eight of an angle for each chunk.  With two or four tokens at hand, and fewer threads on an SM, 32 and 37; with chunks dealt to the threads one by one, whose addresses took
// most of the instructions, 37; a block to a token, which looked its place up before it loaded, 70.
// Blocks of 256 threads on an SM: 40 registers do for neighbours; the other forms would spill
__host__ __device__ constexpr int append_blocks(int form) { return form == 0 ? 6 : 4; }
template <int FORM>
__global__ void __launch_bounds__(PR_THREADS, append_blocks(FORM))
paged_rope_cache_kernel(const PagedCache c, const AppendArgs a, int halves) {
    struct Place { long long k, v; int pos; };                 // pos < 0: the token has no place
    __shared__ Place places[PR_TOKENS];
    const int lane = a.lanes > 1 ? threadIdx.x / a.chunks : 0, col = blockIdx.y * blockDim.x + threadIdx.x - lane * a.chunks;
    const bool works = lane < a.lanes && col < a.chunks;
    const int h = col / a.head_chunks, ch = (col - h * a.head_chunks) * 8;
    const bool is_q = h < a.NH, is_k = !is_q && h < a.NH + c.heads, rotates = (is_q || is_k) && ch < a.R;
    const bf16* src = a.raw + h * c.hs + ch;
    bf16* dst = is_q ? a.q + h * c.hs + ch : is_k ? c.k + (h - a.NH) * c.k_head + ch : c.v + (h - a.NH - c.heads) * c.v_head + ch;
    // FORM 1: the other half's chunk
    const bool second = FORM == 1 && ch >= (a.R >> 1);
    const int across = second ? -(a.R >> 1) : a.R >> 1, pair0 = FORM == 1 ? (second ? ch - (a.R >> 1) : ch) : ch >> 1;
    pdl_wait();
    pdl_trigger();
    // the block's tokens, PR_TOKENS at a time
    const int own0 = (int)((long long)a.N * blockIdx.x / gridDim.x), own1 = (int)((long long)a.N * (blockIdx.x + 1) / gridDim.x);
    // (a load that is left out leaves its register as it was: with zeros in its place the loop takes 34 us instead of 29)
    bf16x8 x, next;
    if (works && own0 + lane < own1) x = ld128cs(src + (own0 + lane) * a.ldr);
    for (int batch = own0; batch < own1; batch += PR_TOKENS) {
        const int batch_end = min(own1, batch + PR_TOKENS);
        for (int t = threadIdx.x; t < batch_end - batch; t += blockDim.x) {
            const int n = batch + t;
            int lo = 0, hi = c.sequences;                      // the last sequence that begins at or before n lies in [lo, hi)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (c.starts[mid] <= n) lo = mid; else hi = mid;
            }
            Place p = {0, 0, -1};
            if (n < c.starts[lo + 1] && n >= c.starts[lo]) {   // otherwise the row lies behind the last sequence
                const PagedSpan s = paged_span(c, lo, a.N, a.status, 0x40);
                const int slot = s.keys - s.count + (n - s.first);
                if (s.count > s.keys) record_error(a.status, ST_BAD_ARG, 0x41);
                else if ((unsigned)(n - s.first) < (unsigned)s.count) {
                    const int pos = a.positions ? a.positions[n] : slot, page = paged_page(c, lo, slot, a.status, 0x42), row = slot & ((1 << c.page_shift) - 1);
                    if (pos < 0 || pos >= a.freqs_len) record_error(a.status, ST_BAD_ARG, 0x43);
                    else if (page >= 0) p = {a.layer * c.k_layer + page * c.k_page + row * c.k_row, a.layer * c.v_layer + page * c.v_page + row * c.v_row, pos};
                }
            }
            places[t] = p;
        }
        __syncthreads();
        for (int n0 = batch; n0 < batch_end; n0 += a.lanes, x = next) {
            const int n = n0 + lane;
            if (works && n + a.lanes < own1) next = ld128cs(src + (n + a.lanes) * a.ldr);      // (the first of the next batch at the end of this one: lanes divides PR_TOKENS)
            if (!works || n >= batch_end) continue;
            bf16x8 y = x;
            const Place* p = &places[n - batch];
            const int pos = p->pos;
            if (pos < 0) continue;
            const bf16x8 was = y;
            uint32_t* yw = reinterpret_cast<uint32_t*>(&y);
            if (rotates) {
                const float2* f = a.freqs + (size_t)pos * (a.R >> 1) + pair0;
                if (FORM == 0) {
                    const float4 f0 = *reinterpret_cast<const float4*>(f), f1 = *reinterpret_cast<const float4*>(f + 2);
                    const float cs[4] = {f0.x, f0.z, f1.x, f1.z}, sn[4] = {f0.y, f0.w, f1.y, f1.w};
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 v = unpack_bf16x2(yw[j]), r = rotate(v.x, v.y, cs[j], sn[j]);
                        yw[j] = pack_bf16x2(r.x, r.y);
                    }
                } else if (FORM == 1) {
                    const bf16x8 other = ld128(src + n * a.ldr + across);
                    const uint32_t* ow = reinterpret_cast<const uint32_t*>(&other);
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float4 fj = *reinterpret_cast<const float4*>(f + 2 * j);
                        const float2 m = unpack_bf16x2(yw[j]), o = unpack_bf16x2(ow[j]);
                        const float2 r0 = second ? rotate(o.x, m.x, fj.x, fj.y) : rotate(m.x, o.x, fj.x, fj.y);
                        const float2 r1 = second ? rotate(o.y, m.y, fj.z, fj.w) : rotate(m.y, o.y, fj.z, fj.w);
                        yw[j] = second ? pack_bf16x2(r0.y, r1.y) : pack_bf16x2(r0.x, r1.x);
                    }
                } else {
                    const bf16* row = src + n * a.ldr - ch;
                    f -= pair0;
                    #pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int at = ch + j;
                        if (at >= a.R) continue;
                        const bool late = halves ? at >= (a.R >> 1) : at & 1;
                        const int pair = halves ? (late ? at - (a.R >> 1) : at) : at >> 1;
                        const float2 fj = f[pair];
                        const float mine = __bfloat162float(was[j]), its = __bfloat162float(row[halves ? (late ? pair : pair + (a.R >> 1)) : at ^ 1]);
                        const float2 r = late ? rotate(its, mine, fj.x, fj.y) : rotate(mine, its, fj.x, fj.y);
                        y[j] = __float2bfloat16_rn(late ? r.y : r.x);
                    }
                }
            }
            st128(dst + (is_q ? n * a.ldq : is_k ? p->k : p->v), y);
        }
        __syncthreads();                                       // the next batch's places take these ones'
    }
}

constexpr int PK_THREADS = 128;
constexpr int PK_MOST = 256;           // tokens that a sequence may keep
constexpr int PK_EACH = 8;             // chunks that a thread carries at a time

// A block: keys or values of one layer of one sequence.  Its threads carry a number of tokens, 16 bytes of a row each: all are read before any is written, and since a token only ever moves to
// the front (kept[j] >= j), no write meets what the block reads later.
__global__ void __launch_bounds__(PK_THREADS)
paged_keep_kernel(const PagedCache c, const int* __restrict__ kept, const int* __restrict__ counts, int D, long long kept_row, FastDiv by_token, FastDiv by_head, unsigned int* status) {
    __shared__ long long from[PK_MOST], to[PK_MOST];
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.x, layer = blockIdx.y;
    const bool values = blockIdx.z;
    const int count = counts[b], mine = threadIdx.x < D ? kept[b * kept_row + threadIdx.x] : 0;
    const PagedSpan s = paged_span(c, b, 0x7fffffff, status, 0x44);
    if (count == 0) return;
    if (count < 0 || count > D || count > s.count || s.count > s.keys) { if (threadIdx.x == 0) record_error(status, ST_BAD_ARG, 0x45); return; }
    const long long page_stride = values ? c.v_page : c.k_page, row_stride = values ? c.v_row : c.k_row, head_stride = values ? c.v_head : c.k_head;
    const int base = s.keys - s.count, in_page = (1 << c.page_shift) - 1;
    bool fine = true;
    for (int j = threadIdx.x; j < count; j += PK_THREADS) {
        const int src = j == (int)threadIdx.x ? mine : kept[b * kept_row + j];
        if (src < j || src >= s.count) { record_error(status, ST_BAD_ARG, 0x46); fine = false; continue; }
        const int ps = paged_page(c, b, base + src, status, 0x47), pd = paged_page(c, b, base + j, status, 0x47);
        fine = fine && ps >= 0 && pd >= 0;
        from[j] = ps * page_stride + ((base + src) & in_page) * row_stride;
        to[j] = pd * page_stride + ((base + j) & in_page) * row_stride;
    }
    if (!__syncthreads_and(fine)) return;
    bf16* pool = values ? c.v + layer * c.v_layer : c.k + layer * c.k_layer;
    const unsigned chunks = c.heads * (c.hs >> 3), total = count * chunks;
    for (unsigned i0 = 0; i0 < total; i0 += PK_THREADS * PK_EACH) {
        bf16x8 x[PK_EACH];
        long long dst[PK_EACH];
        #pragma unroll
        for (int e = 0; e < PK_EACH; e++) {
            const unsigned i = i0 + e * PK_THREADS + threadIdx.x;
            dst[e] = -1;
            if (i < total) {
                const unsigned j = by_token(i), r = i - j * chunks, h = by_head(r);
                const long long at = h * head_stride + (r - h * (c.hs >> 3)) * 8;
                if (from[j] != to[j]) {
                    x[e] = ld128(pool + from[j] + at);
                    dst[e] = to[j] + at;
                }
            }
        }
        __syncthreads();
        #pragma unroll
        for (int e = 0; e < PK_EACH; e++) if (dst[e] >= 0) st128(pool + dst[e], x[e]);
    }
}

template <int FORM>
cudaError_t append_launch(const PagedCache& c, const AppendArgs& a, int halves, dim3 block, int slices, int sms, cudaStream_t stream) {
    // the blocks that are resident at once share the tokens
    const int most = sms * (append_blocks(FORM) * PR_THREADS / (int)block.x) / slices, turns = CEIL_DIV(a.N, a.lanes);
    return launch_pdl(paged_rope_cache_kernel<FORM>, dim3(turns < most ? turns : most > 0 ? most : 1, slices), block, 0, stream, 0, c, a, halves);
}

}  // namespace

extern "C" int llmc_paged_cache_size() { return (int)sizeof(PagedCache); }

extern "C" int llmc_paged_rope_cache(const PagedAppendCall* call) {
    const PagedCache* c = call->cache;
    if (call->N <= 0 || call->N > 1 << 30 || call->NH <= 0 || call->NH > 0xffffff) return -1;
    const int N = (int)call->N, NH = (int)call->NH, R = (int)call->R, halves = (int)call->halves, layer = (int)call->layer;
    const long long ldq = call->ldq, ldr = call->ldr;
    if (R <= 0 || R % 2 || R > c->hs || layer < 0 || layer >= c->layers || ldq % 8 || ldr % 8 || call->freqs_len > 0x7fffffff || (reinterpret_cast<uintptr_t>(call->freqs) & 7)) return -1;
    cudaStream_t stream = call->stream;
    const int hp = c->hs / 8, chunks = (NH + 2 * c->heads) * hp, most = PR_THREADS / chunks;
    // a power of two, so that a batch is whole turns
    const int lanes = most >= 32 ? 32 : most >= 16 ? 16 : most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
    const int slices = CEIL_DIV(chunks, PR_THREADS);
    if (slices > 65535) return -7;
    const dim3 block(lanes > 1 ? PR_THREADS : CEIL_DIV(CEIL_DIV(chunks, slices), 32) * 32);
    const AppendArgs a = {call->q, call->raw, call->freqs, call->positions, ldq, ldr, N, NH, R, (int)call->freqs_len, layer, hp, chunks, lanes, llmc_status_ptr()};
    const int form = R % 8 || (halves && R % 16) || (reinterpret_cast<uintptr_t>(call->freqs) & 15) ? 2 : halves ? 1 : 0;
    int sms = llmc_device_sm_count(); if (sms <= 0) sms = 148;
    CUDA_CHECK(form == 0 ? append_launch<0>(*c, a, halves, block, slices, sms, stream) : form == 1 ? append_launch<1>(*c, a, halves, block, slices, sms, stream)
                                                                                                : append_launch<2>(*c, a, halves, block, slices, sms, stream));
    return 0;
}

extern "C" int llmc_paged_keep(const PagedKeepCall* call) {
    const PagedCache* c = call->cache;
    const int D = (int)call->D;
    const long long kept_row = call->kept_row;
    const int *kept = call->kept, *counts = call->counts;
    cudaStream_t stream = call->stream;
    if (call->D <= 0 || call->D > PK_MOST || c->layers > 65535) return -1;
    CUDA_CHECK(launch_pdl(paged_keep_kernel, dim3(c->sequences, c->layers, 2), dim3(PK_THREADS), 0, stream, 0, *c, kept, counts, D, kept_row, FastDiv(c->heads * (c->hs / 8)), FastDiv(c->hs / 8), llmc_status_ptr()));
    return 0;
}
