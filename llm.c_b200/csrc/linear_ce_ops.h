// What csrc/linear_ce.cu calls from csrc/gemm2.cu and csrc/linear_ce_few.cu.  The definitions include this header too, so that an argument list that changes on one
// side alone does not compile.
#pragma once
#include "common.cuh"

extern "C" {
int llmc_gemm2_sum32_slots(int M, int N, int K, int sm_count, int most);
int llmc_gemm2_sum32(const bf16* A, const bf16* B, float* slots, int M, int N, int K, int lda, int ldb, int S, int accumulate, const int* rows, cudaStream_t stream);
int llmc_gemm2_both_slots(int M, int N, int K, int sm_count);
int llmc_gemm2_both(float* slots, int S, bf16* dw, const bf16* G, const bf16* x, const bf16* w, int M, int N, int K, int dw_rows, int ldg, int ldx, int ldw, int lddw,
                    int accumulate, float alpha, const int* rows, cudaStream_t stream);
int llmc_gemm2_wgrad(const bf16* A, const bf16* B, bf16* D, int M, int N, int K, int lda, int ldb, int ldd, int accumulate, float alpha, int splits, float* workspace,
                     unsigned int* counters, const int* rows, cudaStream_t stream);
int llmc_gemm2_pick_splits(int M, int N, int K, int sm_count);
void llmc_gemm2_workspace(int M, int N, int splits, long long* ws_floats, int* num_counters);
}

// the tiles of at most 128 rows
constexpr int LINEAR_CE_FEW = 128;
// k-blocks of 64 channels whose products a logit of the loss sums in tensor memory.  At most 128 rows: half as many cost nothing at 24 x 768 x 50257 and 2 % at 128 x 2048 x 50257
constexpr int LINEAR_CE_PART = 8, LINEAR_CE_FEW_PART = 4;
// Rows of x as the weight gradient reads them: those that are left out may hold anything, an inf or a NaN, which would not vanish under their 0 in g.  The epilogue warps of the kernels that
// form g leave a copy with zeros in their place while the first products run (to null: not wanted); the `warp`-th of `warps` takes its strips of 256 channels.
struct LinearCeRows { const bf16* x; bf16* to; int N, C, V, ldx; const int* targets; };
#ifdef __CUDACC__
DEVINL void linear_ce_copy_rows(const LinearCeRows& r, int warp, int warps) {
    if (r.to == nullptr) return;
    const int lane = threadIdx.x & 31, strips = CEIL_DIV(r.C, 256);
    for (long long i = warp; i < (long long)r.N * strips; i += warps) {
        const int n = (int)(i / strips), c = (int)(i - (long long)n * strips) * 256 + lane * 8;
        const int t = r.targets[n];
        if (c < r.C)
            *reinterpret_cast<uint4*>(r.to + (size_t)n * r.C + c) = t >= 0 && t < r.V ? *reinterpret_cast<const uint4*>(r.x + (size_t)n * r.ldx + c) : make_uint4(0u, 0u, 0u, 0u);
    }
}
#endif
// Rows of dw that few rows of x (at most LINEAR_CE_KEPT) have their targets in, as they are before the weight gradient is added to them: the same warps leave the row of the target of the i-th row of x
// that counts in row i of `to` (null: not wanted).  The end of the pass, which forms those rows again, adds to what they were.  Two passes over the targets, the first of which ends where too many count.
constexpr int LINEAR_CE_KEPT = 64;
struct LinearCeOld { const bf16* dw; bf16* to; int N, C, V, lddw; const int *targets, *rows; };       // rows: not null: how many of the N rows there are
#ifdef __CUDACC__
DEVINL void linear_ce_save_rows(const LinearCeOld& o, int warp, int warps) {
    if (o.to == nullptr) return;
    constexpr int EACH = 8;                                   // targets of a lane in flight
    const int N = o.rows != nullptr ? *o.rows : o.N, lane = threadIdx.x & 31, strips = CEIL_DIV(o.C, 256);
    int kept = 0;
    for (int base = 0; base < N && kept <= LINEAR_CE_KEPT; base += 32 * EACH) {
        #pragma unroll
        for (int j = 0; j < EACH; j++) {
            const int n = base + j * 32 + lane, t = n < N ? o.targets[n] : -1;
            kept += __popc(__ballot_sync(0xffffffffu, t >= 0 && t < o.V));
        }
    }
    if (kept > LINEAR_CE_KEPT || warp >= kept * strips) return;
    int at = 0;
    for (int base = 0; base < N && at < kept; base += 32) {
        const int n = base + lane, t = n < N ? o.targets[n] : -1;
        for (uint32_t left = __ballot_sync(0xffffffffu, t >= 0 && t < o.V); left != 0; left &= left - 1, at++) {
            const bf16* row = o.dw + (size_t)__shfl_sync(0xffffffffu, t, __ffs(left) - 1) * o.lddw;
            // strips at strips + k, k = 0 .. strips - 1, of which this warp's are those that leave `warp` when divided by `warps`
            for (int k = ((warp - at * strips) % warps + warps) % warps; k < strips; k += warps) {
                const int c = k * 256 + lane * 8;
                if (c < o.C) *reinterpret_cast<uint4*>(o.to + (size_t)at * o.C + c) = *reinterpret_cast<const uint4*>(row + c);
            }
        }
    }
}
#endif
int llmc_linear_ce_few_slots(int V);
int llmc_linear_ce_few_stats(void* part, int part_rows, float* z_target, const bf16* x, const bf16* w, const int* targets, int N, int C, int V, int ldx, int ldw,
                             cudaStream_t stream);
int llmc_linear_ce_few_dlogits(bf16* out, bf16* copy, const bf16* dw, bf16* old, const bf16* x, const bf16* w, const int* targets, const float* lse, const float* dloss_rows, int N, int C, int V,
                               int ldx, int ldw, int ldg, int lddw, cudaStream_t stream);
