// The tiles of csrc/linear_ce.cu for at most 128 rows, where the time is that of reading the weights once: the roles of the operands are swapped, up to 256 rows
// of the weights on the M side of the tensor core (two accumulators of 128), the rows of x on its N side, padded to a multiple of 16 only.
//
// The vocabulary is cut into equal tiles, as many for each CTA, one CTA on every SM with all of its shared memory in flight: at 50257 x 768 two
// tiles of 176 weight rows for 143 CTAs, where tiles of 256 columns would keep CTA pairs busy for three rounds with a third of the last one idle.
//
// A thread of the epilogue owns a row of the weights and has its products with all rows of x, so the softmax statistics of a row of x go across the lanes: each of five
// steps halves the number of values that a lane still carries, 31 exchanges for 32 rows instead of 160.  Whether a warp holds the target of one of 32 rows of x is one vote;
// comparing each of its products with the target took 27.2 instead of 23.2 us with 128 rows at 50257 x 768 (64 rows: 20.6 and 19.4, 24 rows: 18.8 and 18.4).
#include "common.cuh"
#include "linear_ce_ops.h"
#include "pdl.cuh"

namespace {

constexpr int BK = 64, UMMA_K = 16;
constexpr int MAX_ROWS = 128;                 // rows of x
constexpr int MAX_TILE = 256;                 // weight rows of a tile
constexpr int EPI_WARPS = 8;
constexpr int NUM_THREADS = 64 + EPI_WARPS * 32;
constexpr int MAX_STAGES = 12;
constexpr int SMEM_MAX = 226 * 1024;
constexpr float LOG2E = 1.4426950408889634f;

enum Mode : int { LSE = 0, GRAD = 1 };

// shared memory behind the stages
struct Tables {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2];
    float lse2[MAX_ROWS], dl[MAX_ROWS];
    int target[MAX_ROWS];                     // -1: left out
    uint32_t kept[MAX_ROWS / 32];             // a bit for each row
    float ref[EPI_WARPS][32];                 // references of the 32 rows that a warp is at
    float2 stat[EPI_WARPS][MAX_ROWS];
    uint32_t tmem_slot;
    int abort;
};

struct Args {
    int N, V, num_kb, kb_part;                // k-blocks that are summed in tensor memory, as in linear_ce.cu
    int tile, tiles, nb, stages, w_bytes;     // weight rows of a tile, rows of x padded to 16, bytes of a stage's weights
    const int* targets;
    float2* part; int part_rows; float* z_target;                 // LSE
    const float* lse; const float* dloss_rows;                    // GRAD; null: all 1
    bf16* out; int ldg;
    LinearCeRows rows; LinearCeOld old;
    unsigned int* status;
};

// op over the 32 lanes of each of 32 values: lane j gets that of value j
template <typename F>
DEVINL float across(float (&v)[32], F op) {
    const int lane = threadIdx.x & 31;
    #pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        const bool up = lane & s;
        #pragma unroll
        for (int i = 0; i < s; i++) {
            const float send = up ? v[i] : v[i + s], keep = up ? v[i + s] : v[i];
            v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, s));
        }
    }
    return v[0];
}

// CHUNKS: groups of 32 rows of x
template <int MODE, int CHUNKS>
__global__ void __launch_bounds__(NUM_THREADS, 1)
linear_ce_few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const Args g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stage_bytes = g.w_bytes + g.nb * (BK * 2);
    Tables& t = *reinterpret_cast<Tables*>(smem + g.stages * stage_bytes);
    volatile int* abort_flag = &t.abort;
    const int warp = warp_index(), lane = threadIdx.x & 31;
    constexpr int nbp = CHUNKS * 32;                                      // accumulator columns
    constexpr uint32_t tmem_cols = nbp <= 32 ? 128 : nbp <= 64 ? 256 : 512;
    const bool two = g.tile > 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < g.stages; s++) { mbar_init(&t.full[s], 1); mbar_init(&t.empty[s], 1); }
        for (int b = 0; b < 2; b++) { mbar_init(&t.acc_full[b], 1); mbar_init(&t.acc_empty[b], EPI_WARPS); }
        t.abort = 0;
        mbar_fence_init();
        tma_prefetch_desc(&tmX); tma_prefetch_desc(&tmW);
    }
    if (warp == 1) { tmem_alloc(&t.tmem_slot, tmem_cols); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = t.tmem_slot;
    // the first weights come to L2 (a hint: whatever the kernel before writes is read after it has completed)
    if (threadIdx.x == 0 && blockIdx.x * g.tile < g.V)
        for (int kb = 0; kb < min(g.stages, g.num_kb); kb++) tma_prefetch_2d(&tmW, kb * BK, blockIdx.x * g.tile);
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            int st = 0; uint32_t phase = 0;
            bool ok = true;
            for (int i = blockIdx.x; i < g.tiles && ok; i += gridDim.x) {
                for (int kb = 0; kb < g.num_kb; kb++) {
                    if (!(ok = mbar_wait_relaxed(&t.empty[st], phase ^ 1, abort_flag, g.status, 0xD00 + st))) break;
                    uint8_t* w = smem + st * stage_bytes;
                    mbar_expect_tx(&t.full[st], (g.tile + g.nb) * (BK * 2));
                    tma_load_2d(w, &tmW, &t.full[st], kb * BK, i * g.tile);                  // box {64 k, tile rows}
                    tma_load_2d(w + g.w_bytes, &tmX, &t.full[st], kb * BK, 0);               // box {64 k, nb rows}
                    if (++st == g.stages) { st = 0; phase ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        const bool leader = elect_one();
        const uint32_t idesc = umma_idesc_bf16(128, 0, 0, 0) | ((uint32_t)(g.nb >> 3) << 17);
        int st = 0; uint32_t phase = 0;
        int it = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < g.tiles && ok; i += gridDim.x) {
            for (int kb0 = 0; kb0 < g.num_kb && ok; kb0 += g.kb_part, it++) {
                const int buf = it & 1;
                ok = __all_sync(0xffffffffu, mbar_wait_relaxed(&t.acc_empty[buf], ((uint32_t)(it >> 1) & 1) ^ 1, abort_flag, g.status, 0xD40 + buf)) != 0;
                if (!ok) break;
                tc_fence_after();
                const uint32_t acc = tmem_base + buf * 2 * nbp;
                const int kb1 = min(g.num_kb, kb0 + g.kb_part);
                for (int kb = kb0; kb < kb1; kb++) {
                    ok = __all_sync(0xffffffffu, mbar_wait_relaxed(&t.full[st], phase, abort_flag, g.status, 0xD20 + st)) != 0;
                    if (!ok) break;
                    tc_fence_after();
                    // rows of the second accumulator past the tile are whatever the stage holds: nobody reads their products
                    const uint64_t dw = umma_desc_sw128(smem_u32(smem + st * stage_bytes), 16, 1024), dx = umma_desc_sw128(smem_u32(smem + st * stage_bytes + g.w_bytes), 16, 1024);
                    if (leader) {
                        #pragma unroll
                        for (int k = 0; k < BK / UMMA_K; k++) {
                            const uint32_t add = (kb > kb0 || k > 0) ? 1u : 0u;
                            umma_ss(acc, dw + k * (UMMA_K * 2 >> 4), dx + k * (UMMA_K * 2 >> 4), idesc, add);
                            if (two) umma_ss(acc + nbp, dw + (128 * 128 >> 4) + k * (UMMA_K * 2 >> 4), dx + k * (UMMA_K * 2 >> 4), idesc, add);
                        }
                        umma_commit(&t.empty[st]);
                    }
                    __syncwarp();
                    if (++st == g.stages) { st = 0; phase ^= 1; }
                }
                if (ok && leader) umma_commit(&t.acc_full[buf]);
                __syncwarp();
            }
        }
    } else {
        const int ew = warp - 2, half = ew >> 2, q = warp & 3;
        const int e = threadIdx.x - 64;
        if (e < MAX_ROWS) {
            const int tg = e < g.N ? g.targets[e] : -1;
            const bool kept = tg >= 0 && tg < g.V;
            t.target[e] = kept ? tg : -1;
            const uint32_t bits = __ballot_sync(0xffffffffu, kept);
            if (lane == 0) t.kept[e >> 5] = bits;
            if (MODE == GRAD) {
                t.lse2[e] = kept ? g.lse[e] * LOG2E : 0.f;
                t.dl[e] = kept ? (g.dloss_rows != nullptr ? g.dloss_rows[e] : 1.f) : 0.f;
            }
        }
        if (MODE == GRAD) {
            linear_ce_copy_rows(g.rows, blockIdx.x * EPI_WARPS + ew, gridDim.x * EPI_WARPS);
            linear_ce_save_rows(g.old, blockIdx.x * EPI_WARPS + ew, gridDim.x * EPI_WARPS);
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        float run_r[CHUNKS], run_s[CHUNKS];
        #pragma unroll
        for (int c = 0; c < CHUNKS; c++) { run_r[c] = -INFINITY; run_s[c] = 0.f; }
        const int in_tile = half * 128 + q * 32 + lane;
        const bool has_rows = half * 128 + q * 32 < g.tile;               // of this warp
        int it = 0;
        for (int i = blockIdx.x; i < g.tiles; i += gridDim.x) {
            const int v_row = i * g.tile + in_tile;                       // this thread's row of the weights
            const bool valid = in_tile < g.tile && v_row < g.V;
            bool ok = true;
            auto acquire = [&] {
                ok = mbar_wait_relaxed(&t.acc_full[it & 1], (uint32_t)(it >> 1) & 1, abort_flag, g.status, 0xD60 + (it & 1)) && ok;
                tc_fence_after();
                return tmem_base + ((uint32_t)(q * 32) << 16) + ((it & 1) * 2 + half) * nbp;
            };
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t.acc_empty[it & 1]);
                it++;
            };
            // which of 32 rows of x have their target among this warp's rows of the weights
            const int warp_row = v_row - lane, warp_end = i * g.tile + min(g.tile, half * 128 + q * 32 + 32);
            auto targets_here = [&](int c) {
                const int tg = t.target[c * 32 + lane];
                return __ballot_sync(0xffffffffu, tg >= warp_row && tg < warp_end);
            };
            if (MODE == LSE) {
                float z[CHUNKS][32];
                uint32_t acc = acquire();
                if (has_rows) {
                    #pragma unroll
                    for (int c = 0; c < CHUNKS; c++) tmem_ld32(acc + c * 32, reinterpret_cast<uint32_t*>(z[c]));
                    tmem_ld_wait();
                }
                release();
                #pragma unroll 1
                for (int kb = g.kb_part; kb < g.num_kb; kb += g.kb_part) {
                    acc = acquire();
                    if (has_rows) {
                        #pragma unroll
                        for (int c = 0; c < 2 * CHUNKS; c++) {
                            uint32_t u[16];
                            tmem_ld16(acc + c * 16, u);
                            tmem_ld_wait();
                            #pragma unroll
                            for (int j = 0; j < 16; j++) z[c / 2][(c & 1) * 16 + j] += __uint_as_float(u[j]);
                        }
                    }
                    release();
                }
                if (has_rows) {
                    #pragma unroll
                    for (int c = 0; c < CHUNKS; c++) {
                        float* f = z[c];
                        const uint32_t hits = targets_here(c);
                        if (hits) {
                            #pragma unroll
                            for (int j = 0; j < 32; j++)
                                if ((hits >> j & 1) && t.target[c * 32 + j] == v_row && ok) g.z_target[c * 32 + j] = f[j];
                        }
                        float y[32];
                        #pragma unroll
                        for (int j = 0; j < 32; j++) { f[j] = valid ? f[j] : -INFINITY; y[j] = f[j]; }
                        const float mx = across(y, [](float a, float b) { return fmaxf(a, b); });
                        const float r = fminf(fmaxf(mx * LOG2E, -3e38f), 3e38f);      // finite, as in linear_ce.cu
                        t.ref[ew][lane] = r;
                        __syncwarp();
                        const float4* ref = reinterpret_cast<const float4*>(t.ref[ew]);
                        #pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 w = ref[j / 4];
                            f[j] = ex2_fast(fmaf(f[j], LOG2E, -w.x)); f[j + 1] = ex2_fast(fmaf(f[j + 1], LOG2E, -w.y));
                            f[j + 2] = ex2_fast(fmaf(f[j + 2], LOG2E, -w.z)); f[j + 3] = ex2_fast(fmaf(f[j + 3], LOG2E, -w.w));
                        }
                        __syncwarp();
                        const float s = across(z[c], [](float a, float b) { return a + b; });
                        const float hi = fmaxf(run_r[c], r);
                        run_s[c] = run_s[c] * ex2_fast(run_r[c] - hi) + s * ex2_fast(r - hi);
                        run_r[c] = hi;
                    }
                }
            } else {
                const uint32_t acc = acquire();
                if (has_rows) {
                    #pragma unroll
                    for (int c = 0; c < CHUNKS; c++) {
                        uint32_t u[32];
                        tmem_ld32(acc + c * 32, u);
                        tmem_ld_wait();
                        float* f = reinterpret_cast<float*>(u);
                        const float4 *l4 = reinterpret_cast<const float4*>(t.lse2 + c * 32), *d4 = reinterpret_cast<const float4*>(t.dl + c * 32);
                        #pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 l = l4[j / 4];
                            f[j] = ex2_fast(fmaf(f[j], LOG2E, -l.x)); f[j + 1] = ex2_fast(fmaf(f[j + 1], LOG2E, -l.y));
                            f[j + 2] = ex2_fast(fmaf(f[j + 2], LOG2E, -l.z)); f[j + 3] = ex2_fast(fmaf(f[j + 3], LOG2E, -l.w));
                        }
                        const uint32_t hits = targets_here(c);
                        if (hits) {
                            #pragma unroll
                            for (int j = 0; j < 32; j++)
                                if ((hits >> j & 1) && t.target[c * 32 + j] == v_row) f[j] -= 1.f;
                        }
                        #pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 d = d4[j / 4];
                            f[j] *= d.x; f[j + 1] *= d.y; f[j + 2] *= d.z; f[j + 3] *= d.w;
                        }
                        // rows that are left out and columns past the vocabulary are 0, whatever their logits are
                        const uint32_t kept = t.kept[c];
                        if (kept != 0xffffffffu || !__all_sync(0xffffffffu, valid)) {
                            #pragma unroll
                            for (int j = 0; j < 32; j++) f[j] = valid && (kept >> j & 1) ? f[j] : 0.f;
                        }
                        // two lanes share two rows of x: each stores a pair of columns of one (both gradients with 128 rows at 50257 x 768: 63.6 us, one column of a lane 65.9)
                        const int odd = lane & 1;
                        bf16* out = g.out + (size_t)(c * 32 + odd) * g.ldg + (v_row - odd);
                        const bool stored = ok && (in_tile | 1) < g.tile && (v_row | 1) < g.ldg;       // tiles and rows of g have even lengths
                        #pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float got = __shfl_xor_sync(0xffffffffu, odd ? f[j] : f[j + 1], 1);
                            if (stored && c * 32 + j + odd < g.N)
                                *reinterpret_cast<uint32_t*>(out + (size_t)j * g.ldg) = odd ? pack_bf16x2(got, f[j + 1]) : pack_bf16x2(f[j], got);
                        }
                    }
                }
                release();
            }
            if (__any_sync(0xffffffffu, *abort_flag)) break;
        }
        if (MODE == LSE) {
            #pragma unroll
            for (int c = 0; c < CHUNKS; c++) t.stat[ew][c * 32 + lane] = make_float2(run_r[c], run_s[c]);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (e < g.N) {
                float r = -INFINITY, s = 0.f;
                #pragma unroll
                for (int w = 0; w < EPI_WARPS; w++) r = fmaxf(r, t.stat[w][e].x);
                #pragma unroll
                for (int w = 0; w < EPI_WARPS; w++) s += t.stat[w][e].y * ex2_fast(t.stat[w][e].x - r);
                g.part[(size_t)blockIdx.x * g.part_rows + e] = make_float2(r, s);
            }
        }
    }
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000ll) { __nanosleep(1000); }
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem_base, tmem_cols);
}

int sms() { const int n = llmc_device_sm_count(); return n > 0 ? n : 148; }

// Weight rows of a tile: equal tiles, as many for each SM, of at most 256 rows
int tile_rows(int cols) {
    const int rounds = CEIL_DIV(cols, sms() * MAX_TILE);
    return CEIL_DIV(CEIL_DIV(cols, sms() * rounds), 8) * 8;
}

int make(Args& g, CUtensorMap& tmX, CUtensorMap& tmW, const bf16* x, const bf16* w, const int* targets, int N, int C, int V, int cols, int ldx, int ldw) {
    if (N <= 0 || N > MAX_ROWS || C <= 0 || V <= 0 || (C % 8) || (ldx % 8) || (ldw % 8) || ldx < C || ldw < C) return -1;
    g = Args{};
    g.N = N; g.V = V; g.targets = targets; g.num_kb = CEIL_DIV(C, BK);
    g.tile = tile_rows(cols); g.tiles = CEIL_DIV(cols, g.tile);
    g.kb_part = g.num_kb;
    g.nb = CEIL_DIV(N, 16) * 16;
    g.w_bytes = (g.tile > 128 ? 256 : 128) * (BK * 2);
    g.stages = (SMEM_MAX - 1024 - (int)sizeof(Tables)) / (g.w_bytes + g.nb * (BK * 2));
    if (g.stages > MAX_STAGES) g.stages = MAX_STAGES;
    g.status = llmc_status_ptr();
    uint64_t dx[2] = {(uint64_t)C, (uint64_t)N}, sx[2] = {2, (uint64_t)ldx * 2};
    uint64_t dw[2] = {(uint64_t)C, (uint64_t)V}, sw[2] = {2, (uint64_t)ldw * 2};
    uint32_t bx[2] = {BK, (uint32_t)g.nb}, bw[2] = {BK, (uint32_t)g.tile};
    const int rc = llmc_get_tensormap(&tmX, x, 2, 2, dx, sx, bx, 3);
    return rc ? rc : llmc_get_tensormap(&tmW, w, 2, 2, dw, sw, bw, 3);
}

template <int MODE, int CHUNKS>
int launch(const Args& g, const CUtensorMap& tmX, const CUtensorMap& tmW, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        CUDA_CHECK(cudaFuncSetAttribute(linear_ce_few_kernel<MODE, CHUNKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX));
        configured = true;
    }
    CUDA_CHECK(launch_pdl(linear_ce_few_kernel<MODE, CHUNKS>, dim3(g.tiles < sms() ? g.tiles : sms()), dim3(NUM_THREADS), SMEM_MAX, stream, 0, tmX, tmW, g));
    return 0;
}

template <int MODE>
int launch(const Args& g, const CUtensorMap& tmX, const CUtensorMap& tmW, cudaStream_t stream) {
    return g.nb <= 32 ? launch<MODE, 1>(g, tmX, tmW, stream) : g.nb <= 64 ? launch<MODE, 2>(g, tmX, tmW, stream) : launch<MODE, 4>(g, tmX, tmW, stream);
}

}  // namespace

// CTAs, each of which leaves a pair (reference, sum) for each row
int llmc_linear_ce_few_slots(int V) {
    const int tiles = CEIL_DIV(V, tile_rows(V));
    return tiles < sms() ? tiles : sms();
}

int llmc_linear_ce_few_stats(void* part, int part_rows, float* z_target, const bf16* x, const bf16* w, const int* targets, int N, int C, int V, int ldx, int ldw,
                             cudaStream_t stream) {
    Args g;
    CUtensorMap tmX, tmW;
    const int rc = make(g, tmX, tmW, x, w, targets, N, C, V, V, ldx, ldw);
    if (rc) return rc;
    g.kb_part = LINEAR_CE_FEW_PART;
    g.part = static_cast<float2*>(part); g.part_rows = part_rows; g.z_target = z_target;
    return launch<LSE>(g, tmX, tmW, stream);
}

int llmc_linear_ce_few_dlogits(bf16* out, bf16* copy, int* copied, const bf16* dw, bf16* old, const bf16* x, const bf16* w, const int* targets, const float* lse, const float* dloss_rows, int N, int C, int V,
                               int ldx, int ldw, int ldg, int lddw, cudaStream_t stream) {
    Args g;
    CUtensorMap tmX, tmW;
    const int rc = make(g, tmX, tmW, x, w, targets, N, C, V, ldg, ldx, ldw);
    if (rc) return rc;
    g.lse = lse; g.dloss_rows = dloss_rows; g.out = out; g.ldg = ldg; g.rows = {x, copy, copied, N, C, V, ldx, targets}; g.old = {dw, old, N, C, V, lddw, targets, nullptr};
    return launch<GRAD>(g, tmX, tmW, stream);
}
