// Softmax cross-entropy of a linear layer without its logits in memory (the LM head and the loss in one operator).
//
//   z[n,v] = sum_c x[n,c] w[v,c],  v < V;   lse[n] = log sum_v exp z[n,v];   loss[n] = lse[n] - z[n,t[n]]
//   g[n,v] = (exp(z[n,v] - lse[n]) - [v = t[n]]) dloss[n];   dx = g w,  dw = g^T x
//
// Forward: the tiles of x w^T are formed in tensor memory and never leave it.  A thread of the epilogue owns a row of the tile and turns 64 of its
// columns into a reference (their maximum) and the sum of the exponentials below it; the thread whose columns hold the target stores its logit.  A second
// launch joins the pairs of a row.  All of it in fp32 from the accumulators: no logit is ever rounded.
// Backward: the same tiles again, piece of the vocabulary by piece, now with the row's lse known: the epilogue leaves g of the piece in bf16 (the one
// rounding on the way to both gradients, of the same size as that of the gradients themselves), and two products take it from there.  What the rounding takes from a row's
// largest entry, the target's, is put back at the end (finish_kernel).
//
// Exponentials are taken to the base 2: with r = max z log2(e), s = sum 2^(z log2(e) - r), lse = (r + log2 s) ln 2.  The rounding of r cancels, since
// the same r stands on both sides.
//
// The tensor cores cut the running sum off towards zero at each addition, so that a logit of many channels comes out too small, by about C 2^-31 of its size.  The loss
// is what is read to six digits: its logits are summed in parts of 512 channels, which are added in registers.  Error of lse against 64 bits at C = 4096: 1.5e-6
// in one part, 3.5e-7 in four, 1.8e-7 in eight, 1e-7 in sixteen, which took 0, 0 to 1 and 5 to 9 % longer; of the mean loss 2.0e-6, 4.5e-7, 2.3e-7 and 1.2e-7 (plain fp32 products 6e-7),
// of a single loss of 0.3 at C = 1280 6e-6 in parts of 1024 and 2e-6 in parts of 512 channels (plain 1e-6).
//
// The kernel is the 256 x 256 tile pipeline of the two-SM products (gemm2.cu): a cluster of two CTAs, each staging its halves of both operands, the
// accumulators double buffered in tensor memory.  The 2048 cycles of exponentials of a tile hide behind the products of the next from C = 256 on.
#include "common.cuh"
#include "decoder_ops.h"
#include "linear_ce_ops.h"
#include "pdl.cuh"
#include "two_sm.cuh"

namespace {

constexpr int BM = 128;               // rows per CTA (256 per pair)
constexpr int BN = 256;               // vocabulary columns per pair; each CTA stages the weights of 128 of them
constexpr int BK = 64, UMMA_K = 16;
constexpr int A_STAGE_BYTES = BM * BK * 2;            // 16 KB
constexpr int B_STAGE_BYTES = (BN / 2) * BK * 2;      // 16 KB
constexpr int STAGE_BYTES = A_STAGE_BYTES + B_STAGE_BYTES;
constexpr int GROUPS = 4;             // epilogue groups of four warps, each owning 64 columns of the tile
constexpr int GROUP_COLS = BN / GROUPS;
constexpr int WARP_BUF_BYTES = 32 * GROUP_COLS * 2;   // 4 KB: the staged piece of g of a warp
constexpr int NUM_THREADS = 576;      // TMA warp + MMA warp + 16 epilogue warps
constexpr int TMEM_COLS = 512;
constexpr int RASTER_GROUP = 8;       // row tiles that share the weights of a column tile while these are in L2
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

enum Mode : int { LSE = 0, GRAD = 1 };
__host__ __device__ constexpr int stages_for(int mode) { return mode == LSE ? 6 : 5; }
__host__ __device__ constexpr int smem_for(int mode) { return stages_for(mode) * STAGE_BYTES + (mode == GRAD ? 4 * GROUPS * WARP_BUF_BYTES : 0) + 1024 + 512; }

struct Args {
    int N, V, num_m_tiles, num_n_tiles, num_kb;
    int kb_part;                      // k-blocks that are summed in tensor memory; the sums of more of them are added in registers
    int col0, cols;                   // the piece: columns col0 .. col0 + cols of the vocabulary
    const int* targets;
    // LSE: pairs (reference, sum) of a row, [slot][part_rows]; logits of the targets
    float2* part; int part_rows;
    float* z_target;
    // GRAD
    const float* lse; const float* dloss_rows;      // null: all 1
    float* at_target;                 // the stored entry of each row at its target, where g does not stay (several pieces); else null
    int ldg;                          // columns of the stored piece: those past `cols` are 0
    const int* rows;                  // not null: how many of the N rows there are
    LinearCeRows copy; LinearCeOld old;
    unsigned int* status;
};

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
linear_ce_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmG, const Args g) {
    constexpr int STAGES = stages_for(MODE);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* epi_smem = smem + STAGES * STAGE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(epi_smem + (MODE == GRAD ? 4 * GROUPS * WARP_BUF_BYTES : 0));
    uint64_t* full = bars;                    // [STAGES]  used in the leader CTA: bytes of both CTAs' loads
    uint64_t* empty = bars + STAGES;          // [STAGES]  one per CTA, raised by the leader's commit
    uint64_t* acc_full = bars + 2 * STAGES;   // [2]       one per CTA, raised by the leader's commit
    uint64_t* acc_empty = acc_full + 2;       // [2]       used in the leader CTA: all epilogue warps of the pair arrive
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();              // 0 = leader
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; b++) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * 4 * GROUPS); }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 0 && lane == 0) { tma_prefetch_desc(&tmX); tma_prefetch_desc(&tmW); if (MODE == GRAD) tma_prefetch_desc(&tmG); }
    cluster_sync_all();                                   // both CTAs' barriers exist before anyone signals them
    if (warp == 1) { tmem_alloc_2sm(tmem_slot, TMEM_COLS); tmem_relinquish_2sm(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // the first weights come to L2 (a hint: whatever the kernel before writes is read after it has completed)
    if (threadIdx.x == 0) {
        const int gh = min(RASTER_GROUP, g.num_m_tiles);
        for (int kb = 0; kb < min(STAGES, g.num_kb); kb++) tma_prefetch_2d(&tmW, kb * BK, pair / gh * BN + (int)rank * (BN / 2));
    }
    pdl_wait();

    const int num_m_tiles = MODE == GRAD && g.rows != nullptr ? (*g.rows + 255) / 256 : g.num_m_tiles;
    const int total = num_m_tiles * g.num_n_tiles;
    auto decode = [&](int t, int& mt, int& nt) {
        const int per_group = RASTER_GROUP * g.num_n_tiles;
        const int grp = t / per_group, within = t - grp * per_group;
        const int gh = min(RASTER_GROUP, num_m_tiles - grp * RASTER_GROUP);
        nt = within / gh;
        mt = grp * RASTER_GROUP + within - nt * gh;
    };

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs; each loads its own halves) ----------------
        const bool leader = elect_one();
        int stage = 0; uint32_t phase = 0;
        bool go = true;
        for (int w = pair; w < total && go; w += npairs) {
            int mt, nt; decode(w, mt, nt);
            const int m0 = mt * 256 + (int)rank * BM, n0 = nt * BN + (int)rank * (BN / 2);
            for (int kb = 0; kb < g.num_kb; kb++) {
                go = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, abort_flag, g.status, 0x900 + stage)) != 0;
                if (!go) break;
                uint8_t* sa = smem + stage * STAGE_BYTES;
                const uint32_t lead_full = map_to_cta(smem_u32(&full[stage]), 0);
                if (leader) {
                    if (rank == 0) mbar_expect_tx(&full[stage], 2 * STAGE_BYTES);     // bytes of both CTAs
                    tma_load_2d_2sm(sa, &tmX, lead_full, kb * BK, m0);                // box {64 k, 128 rows}
                    tma_load_2d_2sm(sa + A_STAGE_BYTES, &tmW, lead_full, kb * BK, n0);
                }
                __syncwarp();
                if (++stage == STAGES) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader CTA only) ----------------
        if (rank == 0) {
            const bool leader = elect_one();
            constexpr uint32_t idesc = umma_idesc_bf16(256, BN, 0, 0);
            const uint64_t da0 = umma_desc_sw128(smem_u32(smem), 16, 1024), db0 = umma_desc_sw128(smem_u32(smem) + A_STAGE_BYTES, 16, 1024);
            int stage = 0; uint32_t phase = 0;
            int it = 0;
            bool go = true;
            for (int w = pair; w < total && go; w += npairs) {
                for (int kb0 = 0; kb0 < g.num_kb && go; kb0 += g.kb_part, it++) {
                    const int buf = it & 1;
                    go = __all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((uint32_t)(it >> 1) & 1) ^ 1, abort_flag, g.status, 0xA00 + buf)) != 0;
                    if (!go) break;
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + buf * BN;
                    const int kb1 = min(g.num_kb, kb0 + g.kb_part);
                    for (int kb = kb0; kb < kb1; kb++) {
                        go = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort_flag, g.status, 0xB00 + stage)) != 0;
                        if (!go) break;
                        tc_fence_after();
                        const uint64_t da = da0 + (uint64_t)(stage * (STAGE_BYTES >> 4)), db = db0 + (uint64_t)(stage * (STAGE_BYTES >> 4));
                        if (leader) {
                            #pragma unroll
                            for (int k = 0; k < BK / UMMA_K; k++)
                                umma_ss_2sm(d_tmem, da + k * (UMMA_K * 2 >> 4), db + k * (UMMA_K * 2 >> 4), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
                            umma_commit_2sm(&empty[stage]);      // frees this stage in both CTAs
                        }
                        __syncwarp();
                        if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    }
                    if (go && leader) umma_commit_2sm(&acc_full[buf]);
                    __syncwarp();
                }
            }
        }
    } else {
        // ---------------- epilogue (warps 2..17 of each CTA, on that CTA's 128 rows): every warp on its own ----------------
        const int ew = warp - 2, grp = ew >> 2, q = warp & 3;
        uint8_t* wbuf = epi_smem + ew * WARP_BUF_BYTES;
        const uint32_t lead_acc_empty0 = map_to_cta(smem_u32(&acc_empty[0]), 0);
        const uint32_t lead_acc_empty1 = map_to_cta(smem_u32(&acc_empty[1]), 0);
        // one row tile: a pair's tiles all have the same rows, and their statistics join in registers
        const bool one_tile = g.num_m_tiles == 1;
        float run_r = -INFINITY, run_s = 0.f;
        if (MODE == GRAD) {
            linear_ce_copy_rows(g.copy, blockIdx.x * 4 * GROUPS + ew, gridDim.x * 4 * GROUPS);
            linear_ce_save_rows(g.old, blockIdx.x * 4 * GROUPS + ew, gridDim.x * 4 * GROUPS);
        }
        int it = 0;
        for (int w = pair; w < total; w += npairs) {
            int mt, nt; decode(w, mt, nt);
            const int m = mt * 256 + (int)rank * BM + q * 32 + lane;
            const bool row = m < g.N;
            const int c0 = nt * BN + grp * GROUP_COLS;                    // within the piece
            const int left = g.cols - c0;                                 // columns of the vocabulary from here on
            const int target = row ? g.targets[m] : -1;
            const bool kept = target >= 0 && target < g.V;
            const int tj = kept ? target - g.col0 - c0 : -1;              // the target's place among this thread's columns
            float lse2 = 0.f, dl = 0.f;
            if (MODE == GRAD && row) {
                lse2 = g.lse[m] * LOG2E;
                dl = g.dloss_rows != nullptr ? g.dloss_rows[m] : 1.f;
            }
            // the accumulator that is next: waits for it and gives its place in tensor memory
            auto acquire = [&](bool& ok) {
                ok = mbar_wait(&acc_full[it & 1], (uint32_t)(it >> 1) & 1, abort_flag, g.status, 0xC00 + (it & 1)) && ok;
                tc_fence_after();
                return tmem_base + ((uint32_t)(q * 32) << 16) + (it & 1) * BN + grp * GROUP_COLS;
            };
            auto release = [&] {                                          // the leader's MMA thread may refill it
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(it & 1 ? lead_acc_empty1 : lead_acc_empty0);
                it++;
            };
            bool ok = true;
            uint32_t t_row = acquire(ok);
            const bool mine = tj >= 0 && tj < GROUP_COLS;
            if (MODE == LSE) {
                uint32_t v[GROUP_COLS];
                tmem_ld32(t_row, v);
                tmem_ld32(t_row + 32, v + 32);
                tmem_ld_wait();
                release();
                float* f = reinterpret_cast<float*>(v);
                #pragma unroll 1
                for (int kb = g.kb_part; kb < g.num_kb; kb += g.kb_part) {
                    t_row = acquire(ok);
                    #pragma unroll
                    for (int h = 0; h < GROUP_COLS; h += 16) {
                        uint32_t u[16];
                        tmem_ld16(t_row + h, u);
                        tmem_ld_wait();
                        #pragma unroll
                        for (int j = 0; j < 16; j++) f[h + j] += __uint_as_float(u[j]);
                    }
                    release();
                }
                if (left < GROUP_COLS) {
                    #pragma unroll
                    for (int j = 0; j < GROUP_COLS; j++) if (j >= left) f[j] = -INFINITY;
                }
                if (__any_sync(0xffffffffu, mine)) {
                    float z = 0.f;
                    #pragma unroll
                    for (int j = 0; j < GROUP_COLS; j++) if (j == tj) z = f[j];
                    if (mine && ok) g.z_target[m] = z;
                }
                float mx = f[0];
                #pragma unroll
                for (int j = 1; j + 1 < GROUP_COLS; j += 2) mx = max3(mx, f[j], f[j + 1]);
                mx = fmaxf(mx, f[GROUP_COLS - 1]);
                // kept finite: all logits -inf, or one of them +inf, would make NaN of inf - inf (their sums are 0 and inf)
                const float r = fminf(fmaxf(mx * LOG2E, -3e38f), 3e38f);
                float s0 = 0.f, s1 = 0.f;
                #pragma unroll
                for (int j = 0; j < GROUP_COLS; j += 2) {
                    s0 += ex2_fast(fmaf(f[j], LOG2E, -r));
                    s1 += ex2_fast(fmaf(f[j + 1], LOG2E, -r));
                }
                const float s = s0 + s1;
                if (one_tile) {
                    const float hi = fmaxf(run_r, r);
                    run_s = run_s * ex2_fast(run_r - hi) + s * ex2_fast(r - hi);
                    run_r = hi;
                } else if (row && ok) {
                    g.part[(size_t)(nt * GROUPS + grp) * g.part_rows + m] = make_float2(r, s);
                }
            } else {
                // rows that are left out and columns past the vocabulary are 0, whatever their logits are
                const int valid = kept ? left : 0;
                const bool any_kept = __any_sync(0xffffffffu, kept), any_mine = __any_sync(0xffffffffu, mine);
                uint8_t* srow = wbuf + lane * 128;
                const int swz = lane & 7;
                #pragma unroll
                for (int h = 0; h < GROUP_COLS; h += 32) {
                    uint32_t v[32];
                    tmem_ld32(t_row + h, v);
                    tmem_ld_wait();
                    if (h) release();
                    float* f = reinterpret_cast<float*>(v);
                    uint32_t pk[16];
                    if (any_kept) {
                        #pragma unroll
                        for (int j = 0; j < 32; j++) f[j] = ex2_fast(fmaf(f[j], LOG2E, -lse2));
                        if (any_mine) {
                            float e = 0.f;
                            #pragma unroll
                            for (int j = 0; j < 32; j++) if (h + j == tj) { f[j] -= 1.f; e = f[j]; }
                            if (g.at_target != nullptr && kept && tj >= h && tj < h + 32 && ok) g.at_target[m] = __bfloat162float(__float2bfloat16_rn(e * dl));
                        }
                    }
                    #pragma unroll
                    for (int j = 0; j < 32; j += 2)
                        pk[j / 2] = pack_bf16x2(h + j < valid ? f[j] * dl : 0.f, h + j + 1 < valid ? f[j + 1] * dl : 0.f);
                    if (h == 0) {
                        if (lane == 0) tma_store_wait_read<0>();          // the previous tile's store has had a whole tile's time
                        __syncwarp();
                    }
                    #pragma unroll
                    for (int j = 0; j < 4; j++)
                        *reinterpret_cast<uint4*>(srow + ((h / 8 + j) ^ swz) * 16) = make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0 && ok && c0 < g.ldg && m < g.N) { tma_store_2d(&tmG, wbuf, c0, m); tma_store_commit(); }
            }
            if (__any_sync(0xffffffffu, *abort_flag)) break;
        }
        if (MODE == LSE && one_tile) {
            const int m = (int)rank * BM + q * 32 + lane;
            if (m < g.N) g.part[(size_t)(pair * GROUPS + grp) * g.part_rows + m] = make_float2(run_r, run_s);
        }
        if (MODE == GRAD && lane == 0) tma_store_wait<0>();
    }

    pdl_trigger();
    // teardown: the pair meets (nobody may still signal a barrier of a CTA that has left), then TMEM is freed
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        long long t0 = clock64();
        while (clock64() - t0 < 2000000ll) { __nanosleep(1000); }
    }
    cluster_sync_all();
    tc_fence_after();
    if (warp == 1) tmem_dealloc_2sm(tmem_base, TMEM_COLS);
}

// Joins the pairs of a row: lse = (R + log2 sum s 2^(r - R)) ln 2 with R the largest reference.  The loss of a target whose softmax is near 1 is far below its logit: it is formed
// from R - z log2(e), in which the rounding of R (half an ulp of the logit) stands as it does in the sum, not from the rounded lse.  (Logits past 1e30 might overflow in it.)  A block takes 32 rows, a lane each; its warps take the slots in turn.
constexpr int JOIN_WARPS = 32;
__global__ void __launch_bounds__(JOIN_WARPS * 32)
linear_ce_join_kernel(float* __restrict__ losses, float* __restrict__ lse, const float2* __restrict__ part, const float* __restrict__ z_target,
                      const int* __restrict__ targets, int N, int V, int slots, int part_rows, int accumulate) {
    __shared__ float2 red[JOIN_WARPS][33];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m = blockIdx.x * 32 + lane;
    float r = -INFINITY, s = 0.f;
    if (m < N) {
        #pragma unroll 8
        for (int i = warp; i < slots; i += JOIN_WARPS) {
            const float2 p = __ldcg(part + (size_t)i * part_rows + m);
            const float hi = fmaxf(r, p.x);
            s = s * ex2_fast(r - hi) + p.y * ex2_fast(p.x - hi);
            r = hi;
        }
    }
    red[warp][lane] = make_float2(r, s);
    __syncthreads();
    if (warp != 0 || m >= N) return;
    for (int i = 1; i < JOIN_WARPS; i++) r = fmaxf(r, red[i][lane].x);
    s = 0.f;
    for (int i = 0; i < JOIN_WARPS; i++) s += red[i][lane].y * ex2_fast(red[i][lane].x - r);
    const float l2 = log2f(s), l = (r + l2) * LN2;
    if (lse != nullptr) lse[m] = l;
    const int t = targets[m];
    float loss = 0.f;
    if (t >= 0 && t < V) {
        const float z = z_target[m];
        loss = fabsf(z) < 1e30f ? (fmaf(-z, LOG2E, r) + l2) * LN2 : l - z;
    }
    losses[m] = accumulate ? losses[m] + loss : loss;
}

// Rows that count, moved together.  Where many are left out (the prompts of a fine-tuning set) the products of the backward pass are formed for the others alone: every block
// finds the places of all rows, in order, keeps those of its own and copies them; up to the next tile's end rows of zeros without a target follow.  How many there are stays on the
// device.  Whole backward passes without / with it, us: half of the rows left out 2048 x 768 x 50257 379 / 290, 4096 x 768 750 / 518, 16384 x 768 2995 / 1779, 2048 x 2048 x 128256
// 2250 / 1666; a tenth 16384 x 768 3155 / 3008, 3001 x 4096 x 128256 6961 / 6745; none 1024 x 768 210 / 218, 2048 x 768 414 / 427, 4096 x 768 826 / 838, 16384 x 768 3212 / 3190.
constexpr int KEPT_THREADS = 1024, KEPT_MOST = 4096;          // rows of a block
struct Kept {
    int *count, *place;                      // how many; place of each row of x that counts
    int* targets; float *lse, *dloss; bf16* x;      // theirs
};
__global__ void __launch_bounds__(KEPT_THREADS)
kept_rows_kernel(const Kept k, const bf16* __restrict__ x, const int* __restrict__ targets, const float* __restrict__ lse, const float* __restrict__ dloss, int N, int C, int V, int ldx, int each) {
    __shared__ int row_of[KEPT_MOST], per_warp[32];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lo = blockIdx.x * each;
    constexpr int EACH = 8;
    int count = 0;
    for (int base = 0; base < N; base += KEPT_THREADS * EACH) {
        const int from = base + threadIdx.x * EACH;
        uint32_t mine = 0;
        #pragma unroll
        for (int j = 0; j < EACH; j++) {
            const int t = from + j < N ? targets[from + j] : -1;
            mine |= (t >= 0 && t < V ? 1u : 0u) << j;
        }
        int before = __popc(mine);                            // inclusive sums over the lanes, then over the warps
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += v; }
        if (lane == 31) per_warp[warp] = before;
        __syncthreads();
        int w = per_warp[lane];
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += v; }
        const int all = __shfl_sync(0xffffffffu, w, 31), warps_before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
        int at = count + before - __popc(mine) + (warp > 0 ? warps_before : 0);
        #pragma unroll
        for (int j = 0; j < EACH; j++)
            if (mine >> j & 1) {
                if (at >= lo && at < lo + each) { row_of[at - lo] = from + j; k.place[from + j] = at; }
                at++;
            }
        count += all;
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *k.count = count;
    const int most = min(N, (count + 255) / 256 * 256);
    for (int i = lo + warp; i < min(lo + each, most); i += 32) {
        const int n = i < count ? row_of[i - lo] : -1;
        if (lane == 0) {
            k.targets[i] = n >= 0 ? targets[n] : -1;
            k.lse[i] = n >= 0 ? lse[n] : 0.f;
            if (dloss != nullptr) k.dloss[i] = n >= 0 ? dloss[n] : 0.f;
        }
        #pragma unroll 4
        for (int c = lane * 8; c < C; c += 256)
            *reinterpret_cast<uint4*>(k.x + (size_t)i * C + c) = n >= 0 ? *reinterpret_cast<const uint4*>(x + (size_t)n * ldx + c) : make_uint4(0u, 0u, 0u, 0u);
    }
}

// The end of a backward pass.  In each row of g the target's entry is the largest (the others are positive and add up to it), and bf16 takes up to 2^-9 of it: an error along one
// vector, the target's weights in the input gradient, the row of x in the weight gradient, where those of the other entries are independent and cancel.  It is also the one that
// loses digits, in softmax - 1.  So that entry is formed again in fp32, from one dot product whose sums are shorter than those of the tensor core, and the gradients get the difference.  Relative errors (2-norm, 1 row, 50257 x 768): input 0.0039 -> 0.0017, weights 0.0036 -> 0.0017;
// passes of 24, 64, 77 and 128 rows take 0.8, 2, 6 (2048 x 128256) and 0 us longer, of 54, 57, 310 and 65.
//
// Input gradients: the threads of a row add up the fp32 slots and the difference times the target's weights and round once.  Four elements of a thread, eight slots in flight.
// Weight gradients: where at most FEW_KEPT rows of x count and the vocabulary is in one piece, the rows of their targets are formed again, from fp32 entries, and added to what they held before
// (linear_ce_save_rows) where the pass adds.  (With many rows the errors of their entries are independent too.  In several pieces a row's entries at the other rows' targets are gone by then.)  A block takes 256 channels of the target of one row that counts; the first row with a target does it for all.
// The dot products and the lists of rows read what no kernel of this pass writes, before the wait: they run under the end of the products.
constexpr int FEW_KEPT = LINEAR_CE_KEPT;
struct Finish {
    bf16* dx; const float* slots; int lddx, count, team_log, blocks_x;
    bf16* dw; const bf16* old; int lddw, slices;      // dw: null where the rows are left as they are; old: not null: what is added to, LinearCeOld
    const bf16* g; int ldg; const float* at_target;      // g of the whole vocabulary, or (not null) its entries at the targets
    const bf16 *x, *w; int ldx, ldw;
    const int* targets; const float *lse, *dloss_rows; float alpha;
    const int* place;                        // not null: rows of g and of the slots are those of x that count; which one a row of x is
    int N, C, V;
};

// g of row n at its target t, by a warp
__device__ __forceinline__ float target_entry(const Finish& f, int n, int t, int lane) {
    const bf16 *x = f.x + (size_t)n * f.ldx, *w = f.w + (size_t)t * f.ldw;
    float z = 0.f;
    #pragma unroll 4
    for (int c = lane * 8; c < f.C; c += 256) {
        const bf16x8 a = ld128(x + c), b = ld128(w + c);
        #pragma unroll
        for (int k = 0; k < 8; k++) z = fmaf(__bfloat162float(a[k]), __bfloat162float(b[k]), z);
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    const float e = expm1f(z - f.lse[n]);                     // softmax - 1 without cancellation
    return f.dloss_rows != nullptr ? e * f.dloss_rows[n] : e;
}

// a + e * w: an infinite weight has decided the sum already, and times a difference of the other sign (or of 0) it would make it a NaN
__device__ __forceinline__ float put_back(float a, float e, float w) { return isfinite(w) ? fmaf(e, w, a) : a; }

__global__ void __launch_bounds__(256)
finish_kernel(const Finish f) {
    const int lane = threadIdx.x & 31;
    if ((int)blockIdx.x < f.blocks_x) {
        const int team = 1 << f.team_log, n = blockIdx.x * (256 >> f.team_log) + (threadIdx.x >> f.team_log);        // one or more warps
        const int t = n < f.N ? f.targets[n] : -1;
        const bool kept = t >= 0 && t < f.V;
        float lost = 0.f;
        if (kept) lost = target_entry(f, n, t, lane);         // in each warp: no exchange between them
        pdl_wait();
        pdl_trigger();
        if (n >= f.N) return;
        const int at = f.place != nullptr && kept ? f.place[n] : n, count = kept ? f.count : 0;
        if (kept) lost -= f.at_target != nullptr ? f.at_target[at] : __bfloat162float(f.g[(size_t)at * f.ldg + t]);
        const size_t step = (size_t)f.N * f.C;
        for (int c = (threadIdx.x & (team - 1)) * 4; c < f.C; c += team * 4) {
            const float* src = f.slots + (size_t)at * f.C + c;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            #pragma unroll 8
            for (int k = 0; k < count; k++) {
                const float4 v = __ldcs(reinterpret_cast<const float4*>(src + k * step));
                a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
            }
            if (kept) {
                const uint2 u = *reinterpret_cast<const uint2*>(f.w + (size_t)t * f.ldw + c);
                const float2 lo = unpack_bf16x2(u.x), hi = unpack_bf16x2(u.y);
                a.x = put_back(a.x, lost, lo.x); a.y = put_back(a.y, lost, lo.y); a.z = put_back(a.z, lost, hi.x); a.w = put_back(a.w, lost, hi.y);
            }
            *reinterpret_cast<uint2*>(f.dx + (size_t)n * f.lddx + c) = make_uint2(pack_bf16x2(a.x * f.alpha, a.y * f.alpha), pack_bf16x2(a.z * f.alpha, a.w * f.alpha));
        }
        return;
    }
    // ---- rows of dw.  The rows of x that count, in order
    __shared__ int row_of[FEW_KEPT], target_of[FEW_KEPT], per_warp[8];
    __shared__ float entry[FEW_KEPT];
    constexpr int EACH = 8;                                   // targets of a thread at a time
    const int warp = threadIdx.x >> 5;
    const int mine = ((int)blockIdx.x - f.blocks_x) / f.slices, slice = ((int)blockIdx.x - f.blocks_x) % f.slices;
    int kept = 0;
    for (int base = 0; base < f.N && kept <= FEW_KEPT; base += 256 * EACH) {
        const int from = base + threadIdx.x * EACH;
        int t[EACH], n = 0;
        #pragma unroll
        for (int k = 0; k < EACH; k++) {
            t[k] = from + k < f.N ? f.targets[from + k] : -1;
            if (t[k] >= f.V) t[k] = -1;
            n += t[k] >= 0;
        }
        int before = n;                                       // inclusive sum over the lanes
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += v; }
        if (lane == 31) per_warp[warp] = before;
        before -= n;
        __syncthreads();
        int all = 0;
        #pragma unroll
        for (int k = 0; k < 8; k++) { if (k < warp) before += per_warp[k]; all += per_warp[k]; }
        int at = kept + before;
        kept += all;
        if (kept <= FEW_KEPT) {
            #pragma unroll
            for (int k = 0; k < EACH; k++)
                if (t[k] >= 0) { row_of[at] = from + k; target_of[at] = t[k]; at++; }
        }
        __syncthreads();
    }
    const bool none = kept > FEW_KEPT || mine >= kept;        // the same in the whole block
    const bool skip = __syncthreads_or(none || ((int)threadIdx.x < mine && target_of[threadIdx.x] == target_of[mine]));
    const int t = skip ? -1 : target_of[mine];
    if (!skip)
        for (int j = warp; j < kept; j += 8)
            if (target_of[j] == t) {
                const float e = target_entry(f, row_of[j], t, lane);
                if (lane == 0) entry[j] = e;
            }
    pdl_wait();
    pdl_trigger();
    if (skip) return;
    if ((int)threadIdx.x < kept && target_of[threadIdx.x] != t) {
        const int at = f.place != nullptr ? f.place[row_of[threadIdx.x]] : row_of[threadIdx.x];
        entry[threadIdx.x] = __bfloat162float(f.g[(size_t)at * f.ldg + t]);
    }
    __syncthreads();
    const int col = slice * 256 + threadIdx.x;
    if (col >= f.C) return;
    float a = 0.f;
    #pragma unroll 16
    for (int j = 0; j < kept; j++) a = fmaf(entry[j], __bfloat162float(f.x[(size_t)row_of[j] * f.ldx + col]), a);
    const float old = f.old != nullptr ? __bfloat162float(f.old[(size_t)mine * f.C + col]) : 0.f;
    f.dw[(size_t)t * f.lddw + col] = __float2bfloat16_rn(fmaf(a, f.alpha, old));
}

int sm_pairs() { int sms = llmc_device_sm_count(); return (sms > 0 ? sms : 148) / 2; }

int make_args(Args& g, CUtensorMap& tmX, CUtensorMap& tmW, const bf16* x, const bf16* w, const int* targets, int N, int C, int V, int col0, int cols, int ldx, int ldw) {
    if (N <= 0 || C <= 0 || V <= 0 || cols <= 0 || col0 < 0 || cols > V - col0 || (C % 8) || (ldx % 8) || (ldw % 8) || ldx < C || ldw < C) return -1;
    g = Args{};
    g.N = N; g.V = V; g.col0 = col0; g.cols = cols; g.targets = targets;
    g.num_m_tiles = CEIL_DIV(N, 256); g.num_n_tiles = CEIL_DIV(cols, BN); g.num_kb = CEIL_DIV(C, BK);
    if ((long long)g.num_m_tiles * g.num_n_tiles > 0x3fffffffll) return -1;
    g.kb_part = g.num_kb;
    g.status = llmc_status_ptr();
    uint64_t dx[2] = {(uint64_t)C, (uint64_t)N}, sx[2] = {2, (uint64_t)ldx * 2};
    uint64_t dw[2] = {(uint64_t)C, (uint64_t)cols}, sw[2] = {2, (uint64_t)ldw * 2};
    uint32_t box[2] = {BK, 128};
    int rc = llmc_get_tensormap(&tmX, x, 2, 2, dx, sx, box, 3);
    return rc ? rc : llmc_get_tensormap(&tmW, w + (size_t)col0 * ldw, 2, 2, dw, sw, box, 3);
}

template <int MODE>
int launch(const Args& g, const CUtensorMap& tmX, const CUtensorMap& tmW, const CUtensorMap& tmG, int pairs, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        CUDA_CHECK(cudaFuncSetAttribute(linear_ce_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_for(MODE)));
        configured = true;
    }
    CUDA_CHECK(launch_pdl(linear_ce_kernel<MODE>, dim3(2 * pairs), dim3(NUM_THREADS), smem_for(MODE), stream, 0, tmX, tmW, tmG, g));
    return 0;
}

int pairs_for(int tiles) { const int p = sm_pairs(); return p < tiles ? p : tiles; }
int slots_for(int N, int V) {
    if (N <= LINEAR_CE_FEW) return llmc_linear_ce_few_slots(V);
    const int tiles = CEIL_DIV(V, BN);
    return GROUPS * (N <= 256 ? pairs_for(tiles) : tiles);
}

}  // namespace

// fp32 words of scratch that llmc_linear_ce_fwd needs
extern "C" long long llmc_linear_ce_fwd_scratch(int N, int V) {
    const long long rows = (N + 31ll) / 32 * 32;
    return 2 * rows * slots_for(N, V) + rows;
}

// losses (N) (+)= the cross-entropy of x (N, C) . w (V, C)^T at the targets, lse (N; null: not wanted) the logarithm of the sum of the exponentials of a row.
// A target outside 0 .. V-1 leaves its row out: loss 0.
extern "C" int llmc_linear_ce_fwd(float* losses, float* lse, float* scratch, const bf16* x, const bf16* w, const int* targets, int N, int C, int V, int ldx, int ldw,
                                  int accumulate, cudaStream_t stream) {
    if (N <= 0 || V <= 0) return -1;
    const int slots = slots_for(N, V), part_rows = CEIL_DIV(N, 32) * 32;
    float2* part = reinterpret_cast<float2*>(scratch);
    float* z_target = scratch + 2ll * part_rows * slots;
    int rc;
    if (N <= LINEAR_CE_FEW) {
        rc = llmc_linear_ce_few_stats(part, part_rows, z_target, x, w, targets, N, C, V, ldx, ldw, stream);
    } else {
        Args g;
        CUtensorMap tmX, tmW;
        if ((rc = make_args(g, tmX, tmW, x, w, targets, N, C, V, 0, V, ldx, ldw))) return rc;
        g.kb_part = LINEAR_CE_PART;
        g.part_rows = part_rows; g.part = part; g.z_target = z_target;
        rc = launch<LSE>(g, tmX, tmW, tmX, pairs_for(g.num_m_tiles * g.num_n_tiles), stream);
    }
    if (rc) return rc;
    CUDA_CHECK(launch_pdl(linear_ce_join_kernel, dim3(CEIL_DIV(N, 32)), dim3(JOIN_WARPS * 32), 0, stream, 0, losses, lse, part, z_target, targets, N, V, slots,
                          part_rows, accumulate));
    return 0;
}

namespace {

// dlogits (N, ldg) = (softmax - onehot) * dloss_rows (null: 1) of the columns col0 .. col0 + cols of the vocabulary, then zeros; ldg: a multiple of 64 within the last 256-column tile
int dlogits(bf16* out, bf16* copy, int* copied, const bf16* dw, bf16* old, float* at_target, const int* rows, const bf16* x, const bf16* w, const int* targets, const float* lse, const float* dloss_rows,
            int N, int C, int V, int col0, int cols, int ldx, int ldw, int ldg, int lddw, cudaStream_t stream) {
    Args g;
    CUtensorMap tmX, tmW, tmG;
    int rc = make_args(g, tmX, tmW, x, w, targets, N, C, V, col0, cols, ldx, ldw);
    if (rc) return rc;
    g.lse = lse; g.dloss_rows = dloss_rows; g.ldg = ldg; g.at_target = at_target; g.rows = rows; g.copy = {x, copy, copied, N, C, V, ldx, targets}; g.old = {dw, old, N, C, V, lddw, targets, rows};
    uint64_t dg[2] = {(uint64_t)ldg, (uint64_t)N}, sg[2] = {2, (uint64_t)ldg * 2};
    uint32_t box[2] = {GROUP_COLS, 32};
    if ((rc = llmc_get_tensormap(&tmG, out, 2, 2, dg, sg, box, 3))) return rc;
    return launch<GRAD>(g, tmX, tmW, tmG, pairs_for(g.num_m_tiles * g.num_n_tiles), stream);
}

int finish(Finish f, cudaStream_t stream) {
    // threads of a row: since each warp forms the dot product, as few as still fill half of the GPU (16384 x 768: 28 us with 32, 40 with 128) and have no
    // more than 8 times 4 channels each (3001 x 4096: 29 us with 128, 38 with 64)
    f.team_log = 8;
    while (f.team_log > 5 && ((long long)f.N << (f.team_log - 1)) >= 2ll * sm_pairs() * 768 && f.C <= 32 << (f.team_log - 1)) f.team_log--;
    f.blocks_x = f.dx ? CEIL_DIV(f.N, 256 >> f.team_log) : 0;
    f.slices = CEIL_DIV(f.C, 256);
    const int blocks_w = f.dw ? (f.N < FEW_KEPT ? f.N : FEW_KEPT) * f.slices : 0;
    CUDA_CHECK(launch_pdl(finish_kernel, dim3(f.blocks_x + blocks_w), dim3(256), 0, stream, 0, f));
    return 0;
}

// How a backward pass is cut: columns of the vocabulary at a time, row length of the stored piece, slots of the input gradient, K slices
// of the weight gradient; whether both gradients go to one launch; and where its parts lie in the scratch, in bytes.
struct Plan { int cols, ldg, slots, splits; bool both, kept; long long at_target, at_kept, at_kept_x, at_copied, at_old, at_slots, at_ws, at_cnt, bytes; };
constexpr int MAX_SLOTS = 32;

Plan make_plan(int N, int C, int V, int piece, int want_dx, int want_dw, int kept) {
    Plan p = {};
    const int sms = 2 * sm_pairs();
    p.cols = piece < V ? piece : V;
    p.ldg = CEIL_DIV(p.cols, 128) * 128;
    if (want_dx && want_dw && p.cols == V) p.slots = llmc_gemm2_both_slots(N, C, V, sms);
    p.both = p.slots > 0;
    if (want_dx && !p.both) p.slots = llmc_gemm2_sum32_slots(N, C, p.cols, sms, MAX_SLOTS);
    auto align = [](long long b) { return (b + 255) / 256 * 256; };
    p.at_target = align((long long)N * p.ldg * 2);
    p.kept = kept && N > 256;                                 // fewer rows are a tile
    p.at_kept = align(p.at_target + (p.cols < V ? 4ll * N : 0));
    p.at_kept_x = align(p.at_kept + (p.kept ? 256 + 16ll * N : 0));
    p.at_copied = align(p.at_kept_x + (p.kept || want_dw ? 2ll * N * C : 0));      // those that count, or those of LinearCeRows
    p.at_old = align(p.at_copied + (p.kept || !want_dw ? 0 : 4ll * CEIL_DIV(N, 64)));
    p.at_slots = align(p.at_old + (want_dw && p.cols == V ? 2ll * LINEAR_CE_KEPT * C : 0));
    p.at_ws = align(p.at_slots + 4ll * p.slots * N * C);
    long long ws = 0; int cnt = 0;
    if (want_dw && !p.both) {
        p.splits = llmc_gemm2_pick_splits(p.ldg, C, N, sms);
        llmc_gemm2_workspace(p.ldg, C, p.splits, &ws, &cnt);
    }
    p.at_cnt = align(p.at_ws + 4 * ws);
    p.bytes = align(p.at_cnt + 4ll * cnt);
    return p;
}

}  // namespace

// Bytes of scratch of llmc_linear_ce_bwd
extern "C" long long llmc_linear_ce_bwd_scratch(int N, int C, int V, int piece, int want_dx, int want_dw, int kept) { return make_plan(N, C, V, piece, want_dx, want_dw, kept).bytes; }

// dx (N, C) = g w, dw (rows, C) = or += g^T x with g = (softmax - onehot) * dloss (one number, or dloss_rows); either may be null.  `piece` columns of the
// vocabulary at a time, a multiple of 256 or at least V.  Rows of dw from V on: zeros, or left alone when it is added to.  kept: the products are formed for the rows that count alone
// (more than 256 rows).  launches: number of kernels issued.
extern "C" int llmc_linear_ce_bwd(bf16* dx, bf16* dw, void* scratch, const bf16* x, const bf16* w, const int* targets, const float* lse, float dloss, const float* dloss_rows,
                                  int N, int C, int V, int ldx, int ldw, int lddx, int lddw, int dw_rows, int accumulate, int piece, int kept, int* launches, cudaStream_t stream) {
    if (N <= 0 || C <= 0 || V <= 0 || piece <= 0 || (piece < V && piece % 256) || (C % 8) || (dx && ((lddx % 8) || lddx < C)) || (dw && ((lddw % 8) || lddw < C || dw_rows < V))) return -1;
    const Plan p = make_plan(N, C, V, piece, dx != nullptr, dw != nullptr, kept);
    char* s = static_cast<char*>(scratch);
    bf16* g = reinterpret_cast<bf16*>(s);
    float *slots = reinterpret_cast<float*>(s + p.at_slots), *at_target = p.cols < V ? reinterpret_cast<float*>(s + p.at_target) : nullptr;
    // One dloss for all rows multiplies the gradients: as a part of g it would give the entries of all targets of a small softmax, -dloss, the same rounding error
    // (2-norm of the weight gradients' error, of many rows: 0.0022 to 0.0027 so, 0.0019 to 0.0021 like this)
    const float alpha = dloss_rows != nullptr ? 1.f : dloss;
    int rc, n = 0;
#define GO(call) do { if ((rc = (call))) return rc; n++; } while (0)
    bf16* const rows_x = reinterpret_cast<bf16*>(s + p.at_kept_x);       // those that count, or a copy of blocks of 64 rows
    int* const copied = p.kept ? nullptr : reinterpret_cast<int*>(s + p.at_copied);       // which
    const bf16* const x_dw = p.kept ? rows_x : x;
    const int ldx_dw = p.kept ? C : ldx;
    // rows of dw are formed again only from g of the whole vocabulary; where they are added to, from what they were
    bf16 *const again = p.cols < V ? nullptr : dw, *const old = again && accumulate ? reinterpret_cast<bf16*>(s + p.at_old) : nullptr;
    Kept k = {};
    if (p.kept) {
        char* at = s + p.at_kept;
        auto take = [&](long long bytes) { char* a = at; at += bytes; return a; };
        k.count = reinterpret_cast<int*>(take(256));
        k.place = reinterpret_cast<int*>(take(4ll * N)); k.targets = reinterpret_cast<int*>(take(4ll * N));
        k.lse = reinterpret_cast<float*>(take(4ll * N)); k.dloss = reinterpret_cast<float*>(take(4ll * N));
        k.x = rows_x;
        int each = CEIL_DIV(N, 2 * sm_pairs());
        if (each < 32) each = 32;
        if (each > KEPT_MOST) each = KEPT_MOST;
        CUDA_CHECK(launch_pdl(kept_rows_kernel, dim3(CEIL_DIV(N, each)), dim3(KEPT_THREADS), 0, stream, 0, k, x, targets, lse, dloss_rows, N, C, V, ldx, each));
        n++;
    }
    for (int c0 = 0; c0 < V; c0 += p.cols) {
        const int cols = V - c0 < p.cols ? V - c0 : p.cols;
        const bf16* wp = w + (size_t)c0 * ldw;
        const int ldg = cols == p.cols ? p.ldg : CEIL_DIV(cols, 128) * 128;
        bf16* const copy = dw && c0 == 0 ? rows_x : nullptr;
        if (N <= LINEAR_CE_FEW && cols == V) GO(llmc_linear_ce_few_dlogits(g, copy, copied, dw, old, x, w, targets, lse, dloss_rows, N, C, V, ldx, ldw, ldg, lddw, stream));
        else if (p.kept) GO(dlogits(g, nullptr, nullptr, dw, old, at_target, k.count, k.x, w, k.targets, k.lse, dloss_rows ? k.dloss : nullptr, N, C, V, c0, cols, C, ldw, ldg, lddw, stream));
        else GO(dlogits(g, copy, copied, dw, old, at_target, nullptr, x, w, targets, lse, dloss_rows, N, C, V, c0, cols, ldx, ldw, ldg, lddw, stream));
        // the zeros behind the last column give the first rows behind the vocabulary
        const int more = dw && c0 + cols == V && !accumulate ? (dw_rows - V < ldg - cols ? dw_rows - V : ldg - cols) : 0;
        if (p.both) {
            GO(llmc_gemm2_both(slots, p.slots, dw, g, x_dw, rows_x, copied, w, N, C, V, V + more, ldg, ldx_dw, ldw, lddw, accumulate, alpha, k.count, stream));
        } else {
            if (dx) GO(llmc_gemm2_sum32(g, wp, slots, N, C, cols, ldg, ldw, p.slots, c0 > 0, k.count, stream));
            if (dw) GO(llmc_gemm2_wgrad(g, x_dw, rows_x, copied, dw + (size_t)c0 * lddw, cols + more, C, N, ldg, ldx_dw, lddw, accumulate, alpha, p.splits,
                                        reinterpret_cast<float*>(s + p.at_ws), reinterpret_cast<unsigned int*>(s + p.at_cnt), k.count, stream));
            if (dw && p.splits > 1) n++;
        }
        if (dw && c0 + cols == V && !accumulate && dw_rows - V > more)
            CUDA_CHECK(cudaMemset2DAsync(dw + (size_t)(V + more) * lddw, (size_t)lddw * 2, 0, (size_t)C * 2, dw_rows - V - more, stream));
    }
    if (dx || again) GO(finish({dx, slots, lddx, p.slots, 0, 0, again, old, lddw, 0, g, p.ldg, at_target, x, w, ldx, ldw, targets, lse, dloss_rows, alpha, k.place, N, C, V}, stream));
#undef GO
    if (launches) *launches = n;
    return 0;
}
