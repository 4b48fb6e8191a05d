// Host API of the block-scaled FP8 products (csrc/fp8_gemm.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace kiwi::gemm {

/// C[r, :] = sum over blocks kb of 128 columns of a_scale[r, kb] * b_scale[n / 128, kb] *
/// (A[r, kb] . B[g][n, kb]^T) for the rows r of every group g.  A [rows, k] and
/// B [num_groups * n, k] are e4m3 bytes; k is a multiple of 16 (a short last
/// block is fine), and with more than one group n is a multiple of 128.
struct Fp8GemmArgs {
    const uint8_t* a;
    int64_t lda;              // A row stride in bytes, a multiple of 16
    const uint8_t* b;
    int64_t ldb;
    const float* a_scale;     // [rows, ceil(k / 128)]
    int64_t a_scale_stride;   // elements between rows
    const float* b_scale;     // contiguous [num_groups * ceil(n / 128), ceil(k / 128)]
    const int32_t* counts;    // [num_groups] rows of each group (device), or null: one group of all rows
    int32_t num_groups;
    int32_t n;
    int32_t k;
    int64_t rows;             // rows of A and of the output
    __nv_bfloat16* c;         // [rows, n] ([rows, n / 2] with swiglu), or null with codes
    int64_t ldc;              // elements
    uint8_t* codes;           // swiglu only: [rows, n / 2] contiguous e4m3 codes, 16-byte aligned, instead of c ...
    float* scales;            // ... with [rows, n / 256] scales amax / 448 (1 for an all-zero block, 2^-128 at the least)
    const float* row_scale;   // optional [rows]: factor of an output row (bf16 output)
    bool swiglu;              // B holds blocks of 128 gate and 128 up rows; n a multiple of 256
    // Two products in a row on a stream, the second on the first's output: the
    // first sets feeds_next, the second follows, and its CTAs then start up while
    // the last of the first's are still running.  Nothing but the first's output
    // may be written by it and read by the second, and the first is launched
    // without `follows`, so that all earlier work is done.
    bool feeds_next;
    bool follows;
    bool zero_tail;           // rows past the last group's are set to zero (else left as they were)
    uint32_t* error;          // device word that errors are reported in (bits are set, never cleared), or null:
                              // gemm_error_word()
};

void fp8_gemm(const Fp8GemmArgs& args, cudaStream_t stream);

/// 128 x 128 block quantisation of bf16 w [rows, cols] (row stride ld elements)
/// to e4m3 codes [rows, cols] (16-byte aligned) and scales [ceil(rows / 128), ceil(cols / 128)] =
/// amax / 448 (1 for an all-zero block, 2^-128 where 448 / amax would overflow).
void quant_fp8_blocks(const __nv_bfloat16* w, int64_t ld, int64_t rows, int64_t cols, uint8_t* codes, float* scales,
                      cudaStream_t stream);

/// The current device's error word of fp8_gemm (where a call brings none of its
/// own) and grouped_linear: one for all callers, bits in group_table.cuh, sticky
/// until cleared.
uint32_t* gemm_error_word();

/// *out = the error word's bits, which are cleared in the same step: a bit that a
/// kernel on another stream sets meanwhile is either in *out or still in the word.
void take_error(uint32_t* word, uint32_t* out, cudaStream_t stream);

}  // namespace kiwi::gemm
