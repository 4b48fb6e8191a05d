// Host API of the experts' bf16 product with its gradients (csrc/grouped_linear.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace kiwi::gemm {

/// Rows of x [rows, k], y and dy [rows, n] belong to groups of counts[g]
/// consecutive rows; w is [num_groups * n, k].  n and k are multiples of 64;
/// rows start on 16-byte boundaries (bases and row strides of multiples of 16 bytes).
struct GroupedLinearArgs {
    const __nv_bfloat16* x;   // forward, wgrad
    int64_t ldx;
    const __nv_bfloat16* w;   // forward, dgrad
    int64_t ldw;
    const __nv_bfloat16* dy;  // dgrad, wgrad
    int64_t lddy;
    void* out;                // y [rows, n], dx [rows, k] (bf16) or dw [num_groups * n, k] (bf16 or fp32)
    int64_t ldo;
    bool out_fp32;            // wgrad only
    bool accumulate;          // wgrad only: out += instead of out =
    const int32_t* counts;
    int32_t num_groups;
    int32_t n;
    int32_t k;
    int64_t rows;
    bool zero_tail;           // forward, dgrad: rows past the last group's become zero (else are left as they were)
};

void grouped_linear_forward(const GroupedLinearArgs& args, cudaStream_t stream);
void grouped_linear_dgrad(const GroupedLinearArgs& args, cudaStream_t stream);
void grouped_linear_wgrad(const GroupedLinearArgs& args, cudaStream_t stream);

}  // namespace kiwi::gemm
