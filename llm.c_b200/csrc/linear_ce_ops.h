// Entry points of csrc/gemm2.cu that csrc/linear_ce.cu calls.  Their definitions include this header too, so that an argument list that changes on one side alone does
// not compile.
#pragma once
#include "common.cuh"

extern "C" {
int llmc_gemm2_sum32_slots(int M, int N, int K, int sm_count, int most);
int llmc_gemm2_sum32(const bf16* A, const bf16* B, float* slots, int M, int N, int K, int lda, int ldb, int S, int accumulate, cudaStream_t stream);
int llmc_gemm2_pick_splits(int M, int N, int K, int sm_count);
void llmc_gemm2_workspace(int M, int N, int splits, long long* ws_floats, int* num_counters);
}
