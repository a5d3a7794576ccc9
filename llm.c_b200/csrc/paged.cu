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

// n / d for n below 2^31, by a product (Granlund and Montgomery's round-up method)
struct FastDiv {
    unsigned mul, shift;
    explicit FastDiv(unsigned d) {
        for (shift = 0; (1ull << shift) < d; ) shift++;
        mul = (unsigned)((((1ull << shift) - d) << 32) / d + 1);
    }
    DEVINL unsigned operator()(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

constexpr int PR_THREADS = 256;

struct AppendArgs {
    bf16* q;
    const bf16* raw;
    const float2* freqs;
    const int* positions;
    long long ldq, ldr;
    int N, NH, R, freqs_len, layer;
    FastDiv by_token, by_head;     // 16-byte chunks of a token, of a head
    int chunks, head_chunks;
    unsigned int* status;
};

// A thread takes PER chunks of 8 channels, PR_THREADS apart; they are on their way while the first threads of the block find out, a token each, where the block's tokens belong.
// FORM: the pairs of a rotation are 0 neighbours, 1 two halves whose chunks go together, 2 either, with a number of channels that is not made of whole chunks.
// 11769 tokens of 48 heads of 64 channels: TODO us.  A block to a token, which looked its place up before it loaded, took 70.
template <int PER, int FORM>
__global__ void __launch_bounds__(PR_THREADS, 4)
paged_rope_cache_kernel(const PagedCache c, const AppendArgs a, int halves) {
    struct Place { long long k, v; int pos; };                 // pos < 0: the token has no place
    __shared__ Place places[PR_THREADS];
    pdl_wait();
    pdl_trigger();
    const unsigned total = (unsigned)a.N * a.chunks, base = blockIdx.x * (PR_THREADS * PER), i0 = base + threadIdx.x;
    const int n0 = a.by_token(base), tokens = (int)a.by_token(min(base + PR_THREADS * PER, total) - 1) - n0 + 1;
    bf16x8 x[PER];
    int token[PER], head[PER], ch[PER];
    #pragma unroll
    for (int e = 0; e < PER; e++) {
        const unsigned i = i0 + e * PR_THREADS;
        token[e] = a.by_token(i);
        const unsigned r = i - token[e] * a.chunks;
        head[e] = a.by_head(r);
        ch[e] = (r - head[e] * a.head_chunks) * 8;
        if (i < total) x[e] = ld128cs(a.raw + token[e] * a.ldr + head[e] * c.hs + ch[e]);
    }
    // (at most PR_THREADS tokens at a time: a token has 6 chunks at least, of which a block has PR_THREADS * PER)
    for (int t0 = 0; t0 < tokens; t0 += PR_THREADS) {
        const int n = n0 + t0 + (int)threadIdx.x;
        if ((int)threadIdx.x < tokens - t0) {
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
                else if (s.count > 0) {
                    const int pos = a.positions ? a.positions[n] : slot, page = paged_page(c, lo, slot, a.status, 0x42), row = slot & ((1 << c.page_shift) - 1);
                    if (pos < 0 || pos >= a.freqs_len) record_error(a.status, ST_BAD_ARG, 0x43);
                    else if (page >= 0) p = {a.layer * c.k_layer + page * c.k_page + row * c.k_row, a.layer * c.v_layer + page * c.v_page + row * c.v_row, pos};
                }
            }
            places[threadIdx.x] = p;
        }
        __syncthreads();
        #pragma unroll
        for (int e = 0; e < PER; e++) {
            const int at = token[e] - n0 - t0, h = head[e];
            if (i0 + e * PR_THREADS >= total || at < 0 || at >= PR_THREADS) continue;
            const Place p = places[at];
            if (p.pos < 0) continue;
            bf16x8 y = x[e];
            if (h < a.NH + c.heads && ch[e] < a.R) {
                const float2* f = a.freqs + (size_t)p.pos * (a.R >> 1);
                const bf16* src = a.raw + token[e] * a.ldr + h * c.hs;
                if (FORM == 0) {
                    const float4 f0 = *reinterpret_cast<const float4*>(f + ch[e] / 2), f1 = *reinterpret_cast<const float4*>(f + ch[e] / 2 + 2);
                    const float cs[4] = {f0.x, f0.z, f1.x, f1.z}, sn[4] = {f0.y, f0.w, f1.y, f1.w};
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 r = rotate(__bfloat162float(x[e][2 * j]), __bfloat162float(x[e][2 * j + 1]), cs[j], sn[j]);
                        y[2 * j] = __float2bfloat16_rn(r.x);
                        y[2 * j + 1] = __float2bfloat16_rn(r.y);
                    }
                } else if (FORM == 1) {
                    const bool second = ch[e] >= (a.R >> 1);
                    const int first = second ? ch[e] - (a.R >> 1) : ch[e];
                    const bf16x8 other = ld128(src + (second ? first : first + (a.R >> 1)));
                    #pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float2 fj = f[first + j];
                        const float mine = __bfloat162float(x[e][j]), its = __bfloat162float(other[j]);
                        const float2 r = second ? rotate(its, mine, fj.x, fj.y) : rotate(mine, its, fj.x, fj.y);
                        y[j] = __float2bfloat16_rn(second ? r.y : r.x);
                    }
                } else {
                    #pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int at_ch = ch[e] + j;
                        if (at_ch >= a.R) continue;
                        const bool second = halves ? at_ch >= (a.R >> 1) : at_ch & 1;
                        const int pair = halves ? (second ? at_ch - (a.R >> 1) : at_ch) : at_ch >> 1;
                        const float2 fj = f[pair];
                        const float mine = __bfloat162float(x[e][j]), its = __bfloat162float(src[halves ? (second ? pair : pair + (a.R >> 1)) : at_ch ^ 1]);
                        const float2 r = second ? rotate(its, mine, fj.x, fj.y) : rotate(mine, its, fj.x, fj.y);
                        y[j] = __float2bfloat16_rn(second ? r.y : r.x);
                    }
                }
            }
            bf16* dst = h < a.NH ? a.q + token[e] * a.ldq + h * c.hs : h < a.NH + c.heads ? c.k + p.k + (h - a.NH) * c.k_head : c.v + p.v + (h - a.NH - c.heads) * c.v_head;
            st128(dst + ch[e], y);
        }
        if (t0 + PR_THREADS < tokens) __syncthreads();         // the next tokens' places take these ones'
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

template <int PER>
cudaError_t append_launch(const PagedCache& c, const AppendArgs& a, int form, int halves, cudaStream_t stream) {
    const dim3 grid((unsigned)CEIL_DIV((long long)a.N * a.chunks, PR_THREADS * PER));
    if (form == 0) return launch_pdl(paged_rope_cache_kernel<PER, 0>, grid, dim3(PR_THREADS), 0, stream, 0, c, a, halves);
    if (form == 1) return launch_pdl(paged_rope_cache_kernel<PER, 1>, grid, dim3(PR_THREADS), 0, stream, 0, c, a, halves);
    return launch_pdl(paged_rope_cache_kernel<PER, 2>, grid, dim3(PR_THREADS), 0, stream, 0, c, a, halves);
}

}  // namespace

extern "C" int llmc_paged_cache_size() { return (int)sizeof(PagedCache); }

// R: channels of a head that are rotated, a multiple of 2; positions: null, or one per row
extern "C" int llmc_paged_rope_cache(bf16* q, const PagedCache* c, const bf16* raw, const float* freqs, const int* positions, int N, long long ldq, long long ldr, int NH, int R, int freqs_len,
                                     int halves, int layer, cudaStream_t stream) {
    if (N <= 0 || NH <= 0 || R <= 0 || R % 2 || R > c->hs || layer < 0 || layer >= c->layers || ldq % 8 || ldr % 8) return -1;
    const int hp = c->hs / 8, chunks = (NH + 2 * c->heads) * hp;
    if ((long long)N * chunks > 0x7fffffff - PR_THREADS * 4) return -7;
    const AppendArgs a = {q, raw, reinterpret_cast<const float2*>(freqs), positions, ldq, ldr, N, NH, R, freqs_len, layer, FastDiv(chunks), FastDiv(hp), chunks, hp, llmc_status_ptr()};
    const int form = R % 8 || (halves && R % 16) || (reinterpret_cast<uintptr_t>(freqs) & 15) ? 2 : halves ? 1 : 0;
    // few tokens: a chunk a thread, so that they are spread over more SMs
    int sms = llmc_device_sm_count(); if (sms <= 0) sms = 148;
    CUDA_CHECK((long long)N * chunks < 4LL * PR_THREADS * 4 * sms ? append_launch<1>(*c, a, form, halves, stream) : append_launch<4>(*c, a, form, halves, stream));
    return 0;
}

extern "C" int llmc_paged_keep(const PagedCache* c, const int* kept, const int* counts, int D, long long kept_row, cudaStream_t stream) {
    if (D <= 0 || D > PK_MOST || c->layers > 65535) return -1;
    CUDA_CHECK(launch_pdl(paged_keep_kernel, dim3(c->sequences, c->layers, 2), dim3(PK_THREADS), 0, stream, 0, *c, kept, counts, D, kept_row, FastDiv(c->heads * (c->hs / 8)), FastDiv(c->hs / 8), llmc_status_ptr()));
    return 0;
}
