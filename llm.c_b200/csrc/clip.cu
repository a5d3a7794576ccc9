// Global norm of many gradient tensors and clipping by it.
//
//   norm = sqrt(sum of g^2 over all elements of all tensors);   s = max_norm / norm if norm > max_norm, else 1;   out = s g
//
// The tensors are described by one list of chunks of 16 KB that the host lays out once (ops/kernels.py, ClipPlan): a block takes a chunk, whatever tensor it is
// of, so hundreds of small tensors cost no more than one large one.  Chunks end at 16-byte boundaries of the gradients; what lies in front of the
// first and behind the last boundary of a tensor is moved by element.
//
// Two launches, bound by memory: the first reads everything once, the second reads it again and writes the result.  The second goes through the chunks
// backwards, so that what the first has read last comes from L2 (126 MB).
//
// Squares and the sums of a thread's chunk are fp32, everything across chunks is 64-bit, in an order that the launch geometry fixes: the same norm on every run.
#include "common.cuh"
#include "pdl.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int PACKS = 4;                         // 128-bit loads of a thread in flight
constexpr int CHUNK_BYTES = THREADS * PACKS * 16;
constexpr int BLOCKS_PER_SM = 8;

// n elements at src (and dst); only the first chunk of a tensor starts off a 16-byte boundary.  type: 0 bf16, 1 fp32
struct alignas(8) Chunk { const void* src; void* dst; int n, type; };

template <typename T> DEVINL float to_f(T v);
template <> DEVINL float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <> DEVINL float to_f<float>(float v) { return v; }
template <typename T> DEVINL T from_f(float v);
template <> DEVINL bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> DEVINL float from_f<float>(float v) { return v; }

// The packs of a chunk: this thread's PACKS of them, element by element where a pack reaches over an end of the chunk (absent elements are 0)
template <typename T>
DEVINL void load_packs(Pack128<T> (&g)[PACKS], const Chunk& c, int lead) {
    constexpr int E = 16 / sizeof(T);
    const T* base = static_cast<const T*>(c.src) - lead;
    const int end = lead + c.n;
    #pragma unroll
    for (int u = 0; u < PACKS; u++) {
        const int e0 = (u * THREADS + (int)threadIdx.x) * E;
        if (e0 >= lead && e0 + E <= end) {
            g[u] = ld128(base + e0);
        } else {
            #pragma unroll
            for (int e = 0; e < E; e++) g[u][e] = e0 + e >= lead && e0 + e < end ? base[e0 + e] : (T)0.f;
        }
    }
}

template <typename T>
DEVINL float chunk_sumsq(const Chunk& c) {
    const int lead = (int)((reinterpret_cast<uintptr_t>(c.src) & 15) / sizeof(T));
    Pack128<T> g[PACKS];
    load_packs(g, c, lead);
    float a[PACKS];
    #pragma unroll
    for (int u = 0; u < PACKS; u++) {
        a[u] = 0.f;
        #pragma unroll
        for (int e = 0; e < Pack128<T>::size; e++) { const float f = to_f(g[u][e]); a[u] = fmaf(f, f, a[u]); }
    }
    return (a[0] + a[1]) + (a[2] + a[3]);
}

template <typename T>
DEVINL void scale_chunk(const Chunk& c, float s) {
    constexpr int E = 16 / sizeof(T);
    const int lead = (int)((reinterpret_cast<uintptr_t>(c.src) & 15) / sizeof(T));
    Pack128<T> g[PACKS];
    load_packs(g, c, lead);
    T* base = static_cast<T*>(c.dst) - lead;
    const int end = lead + c.n;
    const bool whole = ((reinterpret_cast<uintptr_t>(c.dst) ^ reinterpret_cast<uintptr_t>(c.src)) & 15) == 0;      // the packs of dst are aligned too
    #pragma unroll
    for (int u = 0; u < PACKS; u++) {
        const int e0 = (u * THREADS + (int)threadIdx.x) * E;
        #pragma unroll
        for (int e = 0; e < E; e++) g[u][e] = from_f<T>(to_f(g[u][e]) * s);
        if (whole && e0 >= lead && e0 + E <= end) {
            st128(base + e0, g[u]);
        } else {
            #pragma unroll
            for (int e = 0; e < E; e++) if (e0 + e >= lead && e0 + e < end) base[e0 + e] = g[u][e];
        }
    }
}

DEVINL double warp_sum(double v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
DEVINL double block_sum(double v, double* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_sum(v);
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < THREADS / 32 ? red[lane] : 0.0;
    return warp_sum(v);
}

// result[0] = norm, result[1] = factor
__global__ void __launch_bounds__(THREADS)
clip_norm_kernel(float* __restrict__ norm, float* __restrict__ factor, double* __restrict__ partials, unsigned int* __restrict__ ticket,
                 const Chunk* __restrict__ chunks, int count, float max_norm) {
    __shared__ double red[32];
    __shared__ bool last;
    pdl_wait();
    pdl_trigger();
    double acc = 0.0;
    for (int i = blockIdx.x; i < count; i += gridDim.x) {
        const Chunk c = chunks[i];
        acc += (double)(c.type ? chunk_sumsq<float>(c) : chunk_sumsq<bf16>(c));
    }
    acc = block_sum(acc, red);
    if (threadIdx.x == 0) {
        partials[blockIdx.x] = acc;
        __threadfence();
        last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    // the block that arrives last adds the sums of all blocks, in block order whichever it is
    __threadfence();
    acc = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += THREADS) acc += __ldcg(partials + i);
    acc = block_sum(acc, red);
    if (threadIdx.x == 0) {
        const float n = (float)sqrt(acc);
        norm[0] = n;
        factor[0] = n > max_norm ? max_norm / n : 1.0f;
        *ticket = 0;
    }
}

__global__ void __launch_bounds__(THREADS)
clip_scale_kernel(const float* __restrict__ factor, const Chunk* __restrict__ chunks, int count) {
    pdl_wait();
    pdl_trigger();
    const float s = factor[0];
    for (int i = count - 1 - (int)blockIdx.x; i >= 0; i -= gridDim.x) {
        const Chunk c = chunks[i];
        if (s == 1.0f && c.src == c.dst) continue;
        if (c.type) scale_chunk<float>(c, s); else scale_chunk<bf16>(c, s);
    }
}

int blocks_for(int count) {
    int sms = llmc_device_sm_count(); if (sms <= 0) sms = 148;
    return count < sms * BLOCKS_PER_SM ? (count < 1 ? 1 : count) : sms * BLOCKS_PER_SM;
}

}  // namespace

extern "C" int llmc_clip_chunk_bytes() { return CHUNK_BYTES; }
// 64-bit words of scratch: partial sums, the factor, the ticket (0 before the first call)
extern "C" int llmc_clip_scratch(int count) { return blocks_for(count) + 2; }

// norm[0] = the global norm of the chunks' elements; with `scale` the clipped elements go to the chunks' destinations
extern "C" int llmc_clip(float* norm, double* scratch, const void* chunks, int count, float max_norm, int scale, cudaStream_t stream) {
    if (count < 0 || !(max_norm > 0.f)) return -1;
    const int blocks = blocks_for(count);
    float* factor = reinterpret_cast<float*>(scratch + blocks);
    unsigned int* ticket = reinterpret_cast<unsigned int*>(scratch + blocks + 1);
    const Chunk* c = static_cast<const Chunk*>(chunks);
    CUDA_CHECK(launch_pdl(clip_norm_kernel, dim3(blocks), dim3(THREADS), 0, stream, 0, norm, factor, scratch, ticket, c, count, max_norm));
    if (scale && count > 0) CUDA_CHECK(launch_pdl(clip_scale_kernel, dim3(blocks), dim3(THREADS), 0, stream, 0, factor, c, count));
    return 0;
}
