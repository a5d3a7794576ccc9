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

constexpr int PR_THREADS = 256;

// A block takes one token at a time: which sequence it belongs to and where its slot lies are found by every warp once, while the loads of its channels are on their way.
// A thread takes 8 channels of a head.
__global__ void __launch_bounds__(PR_THREADS)
paged_rope_cache_kernel(bf16* __restrict__ q, const PagedCache c, const bf16* __restrict__ raw, const float2* __restrict__ freqs, const int* __restrict__ positions, int N,
                        long long ldq, long long ldr, int NH, int R, int freqs_len, int halves, int layer, unsigned int* status) {
    pdl_wait();
    pdl_trigger();
    const int n = blockIdx.x;
    const int hs = c.hs, hp = hs >> 3, items = (NH + 2 * c.heads) * hp;
    const int b = paged_sequence(c, n);
    if (b >= c.sequences) return;
    const PagedSpan s = paged_span(c, b, N, status, 0x40);
    const int slot = s.keys - s.count + (n - s.first);
    if (s.count == 0) return;
    if (s.count > s.keys) { if (threadIdx.x == 0) record_error(status, ST_BAD_ARG, 0x41); return; }
    const int pos = positions ? positions[n] : slot;
    const int page = paged_page(c, b, slot, status, 0x42);
    if (page < 0) return;
    if (pos < 0 || pos >= freqs_len) { if (threadIdx.x == 0) record_error(status, ST_BAD_ARG, 0x43); return; }
    const float2* f = freqs + (size_t)pos * (R >> 1);
    const int row = slot & ((1 << c.page_shift) - 1);
    bf16* kdst = c.k + layer * c.k_layer + page * c.k_page + row * c.k_row;
    bf16* vdst = c.v + layer * c.v_layer + page * c.v_page + row * c.v_row;
    for (int i = threadIdx.x; i < items; i += PR_THREADS) {
        const int h = i / hp, ch = (i - h * hp) * 8;
        const bf16* src = raw + n * ldr + h * hs;
        bf16x8 a = ld128cs(src + ch);
        if (h < NH + c.heads && ch < R) {
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const int x = ch + e;
                if (x < R) {
                    const bool second = halves ? x >= (R >> 1) : x & 1;
                    const int pair = halves ? (second ? x - (R >> 1) : x) : x >> 1;
                    const float2 cs = f[pair];
                    const float mine = __bfloat162float(src[x]), other = __bfloat162float(src[halves ? (second ? pair : pair + (R >> 1)) : x ^ 1]);
                    a[e] = __float2bfloat16_rn(second ? fmaf(other, cs.y, __fmul_rn(mine, cs.x)) : fmaf(mine, cs.x, -__fmul_rn(other, cs.y)));
                }
            }
        }
        bf16* dst = h < NH ? q + n * ldq + h * hs : h < NH + c.heads ? kdst + (h - NH) * c.k_head : vdst + (h - NH - c.heads) * c.v_head;
        st128(dst + ch, a);
    }
}

constexpr int PK_THREADS = 256;
constexpr int PK_MOST = 256;           // tokens that a sequence may keep
constexpr int PK_BATCH = 8;

// A block: keys or values of one layer of one sequence.  A thread carries 16 bytes of a row from token to token: it reads up to 8 tokens before it writes any, and since a token only ever
// moves to the front (kept[j] >= j), no write meets what a later batch reads.
__global__ void __launch_bounds__(PK_THREADS)
paged_keep_kernel(const PagedCache c, const int* __restrict__ kept, const int* __restrict__ counts, int D, long long kept_row, unsigned int* status) {
    pdl_wait();
    pdl_trigger();
    __shared__ long long from[PK_MOST], to[PK_MOST];
    const int b = blockIdx.x, layer = blockIdx.y;
    const bool values = blockIdx.z;
    const PagedSpan s = paged_span(c, b, 0x7fffffff, status, 0x44);
    const int count = counts[b];
    if (count == 0) return;
    if (count < 0 || count > D || count > s.count || s.count > s.keys) { if (threadIdx.x == 0) record_error(status, ST_BAD_ARG, 0x45); return; }
    const long long page_stride = values ? c.v_page : c.k_page, row_stride = values ? c.v_row : c.k_row, head_stride = values ? c.v_head : c.k_head;
    const int base = s.keys - s.count, in_page = (1 << c.page_shift) - 1;
    bool fine = true;
    if (threadIdx.x < count) {
        const int j = threadIdx.x, src = kept[b * kept_row + j];
        if (src < j || src >= s.count) { record_error(status, ST_BAD_ARG, 0x46); fine = false; }
        else {
            const int ps = paged_page(c, b, base + src, status, 0x47), pd = paged_page(c, b, base + j, status, 0x47);
            fine = ps >= 0 && pd >= 0;
            from[j] = ps * page_stride + ((base + src) & in_page) * row_stride;
            to[j] = pd * page_stride + ((base + j) & in_page) * row_stride;
        }
    }
    if (!__syncthreads_and(fine)) return;
    bf16* pool = values ? c.v + layer * c.v_layer : c.k + layer * c.k_layer;
    const int hp = c.hs >> 3;
    for (int i = threadIdx.x; i < c.heads * hp; i += PK_THREADS) {
        const int h = i / hp;
        bf16* p = pool + h * head_stride + (i - h * hp) * 8;
        for (int j0 = 0; j0 < count; j0 += PK_BATCH) {
            bf16x8 x[PK_BATCH];
            #pragma unroll
            for (int j = 0; j < PK_BATCH; j++) if (j0 + j < count) x[j] = ld128(p + from[j0 + j]);
            #pragma unroll
            for (int j = 0; j < PK_BATCH; j++) if (j0 + j < count && from[j0 + j] != to[j0 + j]) st128(p + to[j0 + j], x[j]);
        }
    }
}

}  // namespace

extern "C" int llmc_paged_cache_size() { return (int)sizeof(PagedCache); }

// R: channels of a head that are rotated, a multiple of 2; positions: null, or one per row
extern "C" int llmc_paged_rope_cache(bf16* q, const PagedCache* c, const bf16* raw, const float* freqs, const int* positions, int N, long long ldq, long long ldr, int NH, int R, int freqs_len,
                                     int halves, int layer, cudaStream_t stream) {
    if (N <= 0 || NH <= 0 || R <= 0 || R % 2 || R > c->hs || layer < 0 || layer >= c->layers || ldq % 8 || ldr % 8) return -1;
    CUDA_CHECK(launch_pdl(paged_rope_cache_kernel, dim3(N), dim3(PR_THREADS), 0, stream, 0, q, *c, raw, reinterpret_cast<const float2*>(freqs), positions, N, ldq, ldr, NH, R, freqs_len, halves,
                          layer, llmc_status_ptr()));
    return 0;
}

extern "C" int llmc_paged_keep(const PagedCache* c, const int* kept, const int* counts, int D, long long kept_row, cudaStream_t stream) {
    if (D <= 0 || D > PK_MOST || c->layers > 65535) return -1;
    CUDA_CHECK(launch_pdl(paged_keep_kernel, dim3(c->sequences, c->layers, 2), dim3(PK_THREADS), 0, stream, 0, *c, kept, counts, D, kept_row, llmc_status_ptr()));
    return 0;
}
