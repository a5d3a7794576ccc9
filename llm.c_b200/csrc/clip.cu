// Global norm of many gradient tensors and clipping by it.
//
//   norm = sqrt(sum of g^2 over all elements of all tensors);   s = max_norm / norm if norm > max_norm, else 1;   out = s g
//
// The tensors are described by one list of chunks of at most 16 KB that the host lays out once (ops/kernels.py, ClipPlan): a block takes a chunk, whatever tensor
// it is of, so hundreds of small tensors cost no more than one large one.  Chunks end at 16-byte boundaries of the gradients; the elements in
// front of a tensor's first boundary and behind its last are read one by one.
//
// One cooperative launch, bound by memory: every block reads its chunks and sums their squares, waits for the others' sums, and writes its chunks' results.  Chunks that a block has kept in shared memory (its last two: 19 MB on 148 SMs) are written from there,
// some that it read before them come from L2, the rest is read twice.
// us: 324 chunks of 96 tensors 8.2, 249 MB of 148 tensors 117 (three passes over them at the copy rate: 114), 710 MB 330 (326), 120 MB in 301 ragged pieces 57 (55).  The last three in place 112, 331 and 46, and below
// the limit, where nothing is written, 46, 124 and 23; of elements of 1e-25, whose squares are summed in 64 bits, 124, 353 and 54.  Outputs that lie on another element of a 16-byte unit than their gradients are written one by one: 347 us instead of 113 for the 249 MB, 65 instead of 53 for the pieces.  Four blocks
// of 64 KB in flight per SM: five 118 / 342 / 58, three 129 / 359 / 64.  With three kept chunks per block L1 is too small for the loads in flight: 139 / 400 / 69.
//
// Squares and the sums of a thread's part of a chunk are fp32 (64-bit where that overflows or loses them), everything across chunks is 64-bit, in an order that the launch geometry fixes: the same norm on every run.
#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int PACKS = 4;                         // 128-bit loads of a thread in flight
constexpr int CHUNK_BYTES = THREADS * PACKS * 16;
constexpr int BLOCKS_PER_SM = 4;
constexpr int KEPT = 2;                          // chunks that a block keeps in shared memory between reading and writing
constexpr int SMEM = KEPT * (CHUNK_BYTES + THREADS * 4);

// n elements at src (and dst).  type: 0 bf16, 1 fp32.  aligned: src and dst lie on the same byte of a 16-byte unit
struct alignas(16) Chunk { const void* src; void* dst; int n, type, aligned, pad; };
static_assert(sizeof(Chunk) == 32, "ClipPlan lays out 32 bytes");

DEVINL Chunk load_chunk(const Chunk* p) {
    Chunk c;
    reinterpret_cast<int4*>(&c)[0] = __ldg(reinterpret_cast<const int4*>(p));
    reinterpret_cast<int4*>(&c)[1] = __ldg(reinterpret_cast<const int4*>(p) + 1);
    return c;
}

template <typename T> DEVINL float to_f(T v);
template <> DEVINL float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <> DEVINL float to_f<float>(float v) { return v; }
template <typename T> DEVINL T from_f(float v);
template <> DEVINL bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> DEVINL float from_f<float>(float v) { return v; }

// What a thread holds of a chunk: packs (absent ones are 0) and, at the ends, up to one element
struct Part { int4 g[PACKS]; float edge; };
struct Ends { int head, packs, tail; };          // elements before the first pack, packs, elements behind the last
template <typename T> DEVINL Ends ends_of(const Chunk& c) {
    constexpr int E = 16 / (int)sizeof(T);
    Ends e;
    e.head = min(c.n, (int)((0 - reinterpret_cast<uintptr_t>(c.src)) & 15) / (int)sizeof(T));
    e.packs = (c.n - e.head) / E;
    e.tail = c.n - e.head - e.packs * E;
    return e;
}
// the element at an end of the chunk that this thread takes: threads 0 .. 7 those in front, 8 .. 15 those behind (-1: none)
template <typename T> DEVINL int edge_of(const Chunk& c, const Ends& e) {
    const int t = threadIdx.x;
    return t < e.head ? t : t >= 8 && t - 8 < e.tail ? c.n - e.tail + t - 8 : -1;
}

template <typename T, bool STREAM>
DEVINL void load_part(Part& p, const Chunk& c) {
    const Ends e = ends_of<T>(c);
    const int4* body = reinterpret_cast<const int4*>(static_cast<const T*>(c.src) + e.head);
    #pragma unroll
    for (int u = 0; u < PACKS; u++) {
        const int i = u * THREADS + (int)threadIdx.x;
        p.g[u] = make_int4(0, 0, 0, 0);
        if (i < e.packs) p.g[u] = STREAM ? __ldcs(body + i) : body[i];
    }
    const int k = edge_of<T>(c, e);
    p.edge = k >= 0 ? to_f(static_cast<const T*>(c.src)[k]) : 0.f;
}

// In fp32 where its range holds the squares; else (an element past 1.8e19, or none above 1e-12 or so; an inf or a NaN too) the same in 64 bits.  Nothing but zeros, as behind a chunk's end, is 0.
template <typename T>
DEVINL double sumsq(const Part& p) {
    float a[PACKS];
    #pragma unroll
    for (int u = 0; u < PACKS; u++) {
        const Pack128<T> g = *reinterpret_cast<const Pack128<T>*>(&p.g[u]);
        a[u] = u ? 0.f : p.edge * p.edge;
        #pragma unroll
        for (int e = 0; e < Pack128<T>::size; e++) { const float f = to_f(g[e]); a[u] = fmaf(f, f, a[u]); }
    }
    const float s = (a[0] + a[1]) + (a[2] + a[3]);
    if (s >= 1e-24f && s < INFINITY) return (double)s;
    int bits = __float_as_int(p.edge);
    #pragma unroll
    for (int u = 0; u < PACKS; u++) bits |= p.g[u].x | p.g[u].y | p.g[u].z | p.g[u].w;
    if (bits == 0) return 0.0;
    double d = (double)p.edge * p.edge;
    #pragma unroll
    for (int u = 0; u < PACKS; u++) {
        const Pack128<T> g = *reinterpret_cast<const Pack128<T>*>(&p.g[u]);
        #pragma unroll
        for (int e = 0; e < Pack128<T>::size; e++) { const double f = to_f(g[e]); d = fma(f, f, d); }
    }
    return d;
}

// The results are read by nothing here: they leave L2 first
template <typename T>
DEVINL void store_part(const Part& p, const Chunk& c, float s) {
    constexpr int E = 16 / (int)sizeof(T);
    const Ends e = ends_of<T>(c);
    T* dst = static_cast<T*>(c.dst);
    #pragma unroll
    for (int u = 0; u < PACKS; u++) {
        const int i = u * THREADS + (int)threadIdx.x;
        Pack128<T> g = *reinterpret_cast<const Pack128<T>*>(&p.g[u]);
        #pragma unroll
        for (int k = 0; k < E; k++) g[k] = from_f<T>(to_f(g[k]) * s);
        if (i < e.packs) {
            T* to = dst + e.head + i * E;
            if (c.aligned) {
                st128cs(to, g);
            } else {
                #pragma unroll
                for (int k = 0; k < E; k++) to[k] = g[k];
            }
        }
    }
    const int k = edge_of<T>(c, e);
    if (k >= 0) dst[k] = from_f<T>(p.edge * s);
}

DEVINL double warp_sum(double v) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
DEVINL double block_sum(double v, double* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < THREADS / 32 ? red[lane] : 0.0;
    return warp_sum(v);
}

// `keep`: chunks in front of those that are kept in shared memory that may stay in L2; everything else passes through it as a stream.  arrivals: blocks that have come
// to the barrier in all calls so far (each call adds the size of its grid, which is the plan's)
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM)
clip_kernel(float* __restrict__ norm, double* __restrict__ partials, unsigned long long* __restrict__ arrivals, const Chunk* __restrict__ chunks, int count, int keep,
            float max_norm, unsigned int* status) {
    extern __shared__ int4 smem[];
    __shared__ double red[32];
    __shared__ bool gave_up;
    int4* kept = smem + threadIdx.x;                                              // this thread's packs of the kept chunks: nobody else touches them
    float* kept_edge = reinterpret_cast<float*>(smem + KEPT * PACKS * THREADS) + threadIdx.x;
    const int G = gridDim.x, mine = (int)blockIdx.x < count ? (count - 1 - (int)blockIdx.x) / G + 1 : 0;       // this block's chunks: blockIdx.x + k G

    double acc = 0.0;
    Chunk next;
    if (mine > 0) next = load_chunk(chunks + blockIdx.x);
    for (int k = 0; k < mine; k++) {
        const Chunk c = next;
        const int i = blockIdx.x + k * G, slot = mine - 1 - k;
        if (slot > 0) next = load_chunk(chunks + i + G);
        const bool stream = slot < KEPT || i < count - KEPT * G - keep;
        Part p;
        if (c.type) { if (stream) load_part<float, true>(p, c); else load_part<float, false>(p, c); }
        else { if (stream) load_part<bf16, true>(p, c); else load_part<bf16, false>(p, c); }
        acc += c.type ? sumsq<float>(p) : sumsq<bf16>(p);
        if (slot < KEPT) {
            #pragma unroll
            for (int u = 0; u < PACKS; u++) kept[(slot * PACKS + u) * THREADS] = p.g[u];
            kept_edge[slot * THREADS] = p.edge;
        }
    }

    // when all blocks have arrived, each adds up all sums, in the same order: one trip to L2 less than a block that does it for the others (1.5 us)
    acc = block_sum(acc, red);
    if (threadIdx.x == 0) {
        partials[blockIdx.x] = acc;
        __threadfence();
        const unsigned long long before = atomicAdd(arrivals, 1ull), all = (before / G + 1) * G;
        const long long t0 = clock64();
        unsigned long long now;
        gave_up = false;
        while (true) {
            asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(now) : "l"(arrivals) : "memory");
            if (now >= all) break;
            if (clock64() - t0 > WAIT_LIMIT_CYCLES) { record_error(status, ST_FLAG_TIMEOUT, 0xC11); gave_up = true; break; }
        }
    }
    __syncthreads();
    if (gave_up) return;
    acc = 0.0;
    for (int i = threadIdx.x; i < G; i += THREADS) acc += __ldcg(partials + i);
    const float n = (float)sqrt(block_sum(acc, red)), s = n > max_norm ? max_norm / n : 1.0f;
    if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = n;

    for (int slot = 0; slot < mine; slot++) {
        const Chunk c = next;                                                     // the last one that was read comes first
        if (slot + 1 < mine) next = load_chunk(chunks + blockIdx.x + (mine - 2 - slot) * G);
        if (s == 1.0f && c.src == c.dst) continue;
        Part p;
        if (slot < KEPT) {
            #pragma unroll
            for (int u = 0; u < PACKS; u++) p.g[u] = kept[(slot * PACKS + u) * THREADS];
            p.edge = kept_edge[slot * THREADS];
        } else if (c.type) load_part<float, true>(p, c);
        else load_part<bf16, true>(p, c);
        if (c.type) store_part<float>(p, c, s); else store_part<bf16>(p, c, s);
    }
}

// Blocks that are resident at once, on every SM; 0: the launch is not possible
int resident() {
    static int per_sm = -1;
    if (per_sm < 0) {
        int n = 0;
        if (cudaFuncSetAttribute(clip_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, clip_kernel, THREADS, SMEM) != cudaSuccess) { (void)cudaGetLastError(); n = 0; }
        per_sm = n < BLOCKS_PER_SM ? n : BLOCKS_PER_SM;
    }
    return per_sm * llmc_device_sm_count();
}

}  // namespace

extern "C" int llmc_clip_chunk_bytes() { return CHUNK_BYTES; }
// 64-bit words of scratch (0 before the first call): the blocks' sums and the count of their arrivals.  It serves calls with one number of chunks.
extern "C" int llmc_clip_scratch() { return BLOCKS_PER_SM * llmc_device_sm_count() + 1; }

// norm[0] = the global norm of the chunks' elements; the clipped elements go to the chunks' destinations.  keep_bytes: what may be expected to stay in L2
extern "C" int llmc_clip(float* norm, double* scratch, const void* chunks, int count, int keep_bytes, float max_norm, cudaStream_t stream) {
    const int most = resident();
    if (count < 0 || !(max_norm > 0.f) || most <= 0) return -1;           // chunks holds at least one entry, also where count is 0
    unsigned long long* arrivals = reinterpret_cast<unsigned long long*>(scratch + BLOCKS_PER_SM * llmc_device_sm_count());
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(count < 1 ? 1 : count < most ? count : most); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM; cfg.stream = stream;
    cfg.attrs = attr; cfg.numAttrs = 1;
    CUDA_CHECK(cudaLaunchKernelEx(&cfg, clip_kernel, norm, scratch, arrivals, static_cast<const Chunk*>(chunks), count, keep_bytes / CHUNK_BYTES, max_norm, llmc_status_ptr()));
    return 0;
}
