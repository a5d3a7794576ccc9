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
int llmc_linear_ce_few_slots(int V);
int llmc_linear_ce_few_stats(void* part, int part_rows, float* z_target, const bf16* x, const bf16* w, const int* targets, int N, int C, int V, int ldx, int ldw,
                             cudaStream_t stream);
int llmc_linear_ce_few_dlogits(bf16* out, const bf16* x, const bf16* w, const int* targets, const float* lse, const float* dloss_rows, int N, int C, int V,
                               int ldx, int ldw, int ldg, cudaStream_t stream);
