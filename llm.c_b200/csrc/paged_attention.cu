// Attention of ragged new tokens over a key / value cache in pages (paged.cuh):
//
//   out[n, h] = sum over the keys s that row n sees of softmax_s(q[n, h] . K[s, g] / sqrt(HS)) V[s, g],  g = h / (NH / NKV); 0 where it sees none.
//   Token i of a sequence of `len` keys with `count` new ones sees slots 0 .. len - count + i; with `tree` it sees slots below len - count, and slot len - count + j
//   where bit j of tree[n] is set (at most 64 new tokens of a sequence).
#include "paged.cuh"
#include "pdl.cuh"

namespace {

constexpr int PA_THREADS = 128;
constexpr int PA_CHUNK = 512;       // keys whose scores sit in shared memory at a time
constexpr int PA_MAX_HS = 128;

// One block per head and row.  Scores: a thread per key; weighted sum of the values: a thread per channel.
__global__ void __launch_bounds__(PA_THREADS)
paged_attention_kernel(bf16* __restrict__ out, const bf16* __restrict__ q, const PagedCache c, const long long* __restrict__ tree, int N, long long ldo, long long ldq, int NH, int layer,
                       float scale, unsigned int* status) {
    pdl_wait();
    pdl_trigger();
    __shared__ float qs[PA_MAX_HS];
    __shared__ float sc[PA_CHUNK];
    __shared__ float red[32];
    const int tid = threadIdx.x, h = blockIdx.x, n = blockIdx.y, g = h / (NH / c.heads), hs = c.hs;
    const int b = paged_sequence(c, n);
    if (b >= c.sequences) return;
    const PagedSpan s = paged_span(c, b, N, status, 0x48);
    if (s.count == 0) return;
    if (tree && s.count > 64) { if (tid == 0) record_error(status, ST_BAD_ARG, 0x49); return; }
    const int context = s.keys - s.count, last = tree ? s.keys : min(s.keys, max(0, context + (n - s.first) + 1));
    const unsigned long long bits = tree ? (unsigned long long)tree[n] : 0;
    if (tid < hs) qs[tid] = __bfloat162float(q[n * ldq + h * hs + tid]) * scale;
    __syncthreads();
    const bf16 *kb = c.k + layer * c.k_layer + g * c.k_head, *vb = c.v + layer * c.v_layer + g * c.v_head;
    const int in_page = (1 << c.page_shift) - 1;
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int base = 0; base < last; base += PA_CHUNK) {
        const int cnt = min(PA_CHUNK, last - base);
        float lmax = -INFINITY;
        for (int j = tid; j < cnt; j += PA_THREADS) {
            const int slot = base + j;
            float x = -INFINITY;
            if (!tree || slot < context || (bits >> (slot - context) & 1)) {
                const int page = paged_page(c, b, slot, status, 0x4A);
                x = 0.f;
                if (page >= 0) {
                    const bf16* k = kb + page * c.k_page + (slot & in_page) * c.k_row;
                    for (int d = 0; d < hs; d += 8) {
                        const bf16x8 kk = ld128(k + d);
                        #pragma unroll
                        for (int e = 0; e < 8; e++) x = fmaf(qs[d + e], __bfloat162float(kk[e]), x);
                    }
                }
            }
            sc[j] = x;
            lmax = fmaxf(lmax, x);
        }
        const float mn = fmaxf(m, block_max(lmax, red)), ref = mn == -INFINITY ? 0.f : mn;
        float lsum = 0.f;
        for (int j = tid; j < cnt; j += PA_THREADS) { sc[j] = __expf(sc[j] - ref); lsum += sc[j]; }
        const float corr = __expf(m - ref);
        l = l * corr + block_sum(lsum, red);
        acc *= corr;
        m = mn;
        if (tid < hs)
            for (int j = 0; j < cnt; j++) {
                const int slot = base + j, page = c.table[b * c.table_row + (slot >> c.page_shift)];
                if (sc[j] > 0.f && (unsigned)page < (unsigned)c.pages) acc = fmaf(sc[j], __bfloat162float(vb[page * c.v_page + (slot & in_page) * c.v_row + tid]), acc);
            }
        __syncthreads();
    }
    if (tid < hs) out[n * ldo + h * hs + tid] = __float2bfloat16_rn(l > 0.f ? acc / l : 0.f);
}

}  // namespace

extern "C" int llmc_paged_attention(bf16* out, const PagedCache* c, const bf16* q, const long long* tree, int N, long long ldo, long long ldq, int NH, int layer, cudaStream_t stream) {
    if (N <= 0 || N > 65535 || NH <= 0 || NH % c->heads || layer < 0 || layer >= c->layers || c->hs > PA_MAX_HS || ldq % 8 || ldo % 8) return -1;
    CUDA_CHECK(launch_pdl(paged_attention_kernel, dim3(NH, N), dim3(PA_THREADS), 0, stream, 0, out, q, *c, tree, N, ldo, ldq, NH, layer, 1.0f / sqrtf((float)c->hs), llmc_status_ptr()));
    return 0;
}
