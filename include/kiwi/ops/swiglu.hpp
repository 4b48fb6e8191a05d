// Host API of SwiGLU and its gradient (csrc/swiglu_gpu.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace kiwi::ops {

/// h[r, j] = row_scale[r] * silu(gate) * up for y [rows, 2 * ffn] whose columns
/// come in blocks of 128 gate and 128 up columns (ffn is a multiple of 128);
/// h [rows, ffn] contiguous.  Row strides (ldy, lddh) are multiples of 8, all
/// bases on 16-byte boundaries.  row_scale may be null (1).
void swiglu_forward(const __nv_bfloat16* y, int64_t ldy, const float* row_scale, __nv_bfloat16* h, int64_t rows,
                    int ffn, cudaStream_t s);

/// Gradients of swiglu_forward: dy [rows, 2 * ffn] contiguous and, when
/// drow_scale is not null, drow_scale [rows].
void swiglu_backward(const __nv_bfloat16* dh, int64_t lddh, const __nv_bfloat16* y, int64_t ldy,
                     const float* row_scale, __nv_bfloat16* dy, float* drow_scale, int64_t rows, int ffn,
                     cudaStream_t s);

}  // namespace kiwi::ops
