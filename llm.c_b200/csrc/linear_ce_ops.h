// What csrc/linear_ce.cu calls from csrc/gemm2.cu and csrc/linear_ce_few.cu.  The definitions include this header too, so that an argument list that changes on one
// side alone does not compile.
#pragma once
#include "common.cuh"

extern "C" {
int llmc_gemm2_sum32_slots(int M, int N, int K, int sm_count, int most);
int llmc_gemm2_sum32(const bf16* A, const bf16* B, float* slots, int M, int N, int K, int lda, int ldb, int S, int accumulate, const int* rows, cudaStream_t stream);
int llmc_gemm2_both_slots(int M, int N, int K, int sm_count);
int llmc_gemm2_both(float* slots, int S, bf16* dw, const bf16* G, const bf16* x, const bf16* x2, const int* other_x, const bf16* w, int M, int N, int K, int dw_rows, int ldg, int ldx, int ldw, int lddw,
                    int accumulate, float alpha, const int* rows, cudaStream_t stream);
int llmc_gemm2_wgrad(const bf16* A, const bf16* B, const bf16* B2, const int* other_b, bf16* D, int M, int N, int K, int lda, int ldb, int ldd, int accumulate, float alpha, int splits, float* workspace,
                     unsigned int* counters, const int* rows, cudaStream_t stream);
int llmc_gemm2_pick_splits(int M, int N, int K, int sm_count);
void llmc_gemm2_workspace(int M, int N, int splits, long long* ws_floats, int* num_counters);
}

// the tiles of at most 128 rows
constexpr int LINEAR_CE_FEW = 128;
// k-blocks of 64 channels whose products a logit of the loss sums in tensor memory.  At most 128 rows: half as many cost nothing at 24 x 768 x 50257 and 2 % at 128 x 2048 x 50257
constexpr int LINEAR_CE_PART = 8, LINEAR_CE_FEW_PART = 4;
// Rows of x as the weight gradient reads them: those that are left out may hold anything, an inf or a NaN, which would not vanish under their 0 in g.  The epilogue warps of the kernels that
// form g leave a copy with zeros in their place while the first products run, of the blocks of 64 rows (a k-block of the weight gradient) that have such a row, and a word for each block that says so.  `to`
// null: not wanted.  The `warp`-th of `warps` takes pieces of a block, or of 8 of its rows where there are few, and 256 channels.  us, without a copy (a tenth of the rows left out) / with one, none left
// out / with one, a tenth: 16384 x 4096 x 500 336 / 324 / 332, 8192 x 1024 x 1000 83 / 88 / 94, 16384 x 2048 x 700 203 / 205 / 206, 16384 x 1024 x 3000 287 / 293 / 299, 1024 x 768 x 50257 185 / 213 (210 without) / 185.
// Every row copied, one strip in flight for a warp, made the first 410.
struct LinearCeRows { const bf16* x; bf16* to; int* copied; int N, C, V, ldx; const int* targets; };
#ifdef __CUDACC__
DEVINL void linear_ce_copy_rows(const LinearCeRows& r, int warp, int warps) {
    if (r.to == nullptr) return;
    const int lane = threadIdx.x & 31, strips = CEIL_DIV(r.C, 256);
    const int rows = (long long)CEIL_DIV(r.N, 64) * strips >= warps ? 64 : 8;          // of a piece
    const unsigned int pieces = (unsigned int)CEIL_DIV(r.N, rows) * strips;             // products of more than 1e11 rows x channels do not come here
    for (unsigned int i = warp; i < pieces; i += warps) {
        const int piece = (int)(i / (unsigned int)strips), strip = (int)i - piece * strips, n0 = piece * rows, block = n0 >> 6, c = strip * 256 + lane * 8;
        bool out[2];
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            const int n = block * 64 + h * 32 + lane, t = n < r.N ? r.targets[n] : 0;
            out[h] = t < 0 || t >= r.V;
        }
        const uint32_t lo = __ballot_sync(0xffffffffu, out[0]), hi = __ballot_sync(0xffffffffu, out[1]);
        if (strip == 0 && (n0 & 63) == 0 && lane == 0) r.copied[block] = (lo | hi) != 0;
        if ((lo | hi) == 0 || c >= r.C) continue;
        #pragma unroll 1
        for (int n = n0; n < n0 + rows; n += 8) {
            const uint32_t left = ((n & 32) ? hi : lo) >> (n & 31);                    // of these 8 rows
            uint4 v[8];
            #pragma unroll
            for (int j = 0; j < 8; j++)
                v[j] = n + j < r.N && !(left >> j & 1) ? *reinterpret_cast<const uint4*>(r.x + (size_t)(n + j) * r.ldx + c) : make_uint4(0u, 0u, 0u, 0u);
            #pragma unroll
            for (int j = 0; j < 8; j++) if (n + j < r.N) *reinterpret_cast<uint4*>(r.to + (size_t)(n + j) * r.C + c) = v[j];
        }
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
int llmc_linear_ce_few_dlogits(bf16* out, bf16* copy, int* copied, const bf16* dw, bf16* old, const bf16* x, const bf16* w, const int* targets, const float* lse, const float* dloss_rows, int N, int C, int V,
                               int ldx, int ldw, int ldg, int lddw, cudaStream_t stream);
