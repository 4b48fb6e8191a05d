// SwiGLU between the experts' two products, with routing weights, and its gradients.
//
//   h = s * a * u                      a = g * sig(g)
//   du = dh * s * a
//   dg = dh * s * u * sig(g) * (1 + g * (1 - sig(g)))
//   ds = sum over the row of dh * a * u
//
// g and u are the gate and up columns of a row of y, in blocks of 128 each (the
// layout of the grouped products).  All arithmetic is fp32; each result is
// rounded once to bf16, ds is summed and kept in fp32 in an order that depends
// on nothing but the row's length.
//
// Bound by memory: forward reads 4 F bytes a row and writes 2 F, backward reads
// 6 F and writes 4 F.  One warp takes a row, 256 hidden columns a step, eight
// columns (one 16-byte access of each operand) a lane.  Measured on one B200 at
// 32768 x 2048: forward 73 us (5.6 TB/s), backward 111 us (6.1 TB/s) of a copy's
// 6.5.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kiwi/common.hpp"
#include "kiwi/ep/quant.cuh"
#include "kiwi/ops/swiglu.hpp"
#include "kiwi/ptx.cuh"

namespace kiwi::ops {

namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerBlock = kThreads / 32;

/// 1 / (1 + exp(-x)) from the approximate exponential and reciprocal: good to a
/// few steps of 2^-23 and |x| of them, far below a bf16 rounding; exact zeros
/// only where exp(-x) overflows.  (With expf and IEEE divisions the forward pass
/// was bound by their instructions: 83 us at 32768 x 2048.)
__device__ __forceinline__ float sigmoid(float x) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-x)));
    return r;
}

/// Column of y that holds the gate of hidden column j (its up column is 128 further).
__device__ __forceinline__ int gate_col(int j) { return (j >> 7) * 256 + (j & 127); }

__global__ void __launch_bounds__(kThreads) swiglu_forward_kernel(const __nv_bfloat16* __restrict__ y, int64_t ldy,
                                                                  const float* __restrict__ row_scale,
                                                                  __nv_bfloat16* __restrict__ h, int64_t rows,
                                                                  int ffn) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock + (threadIdx.x >> 5);
    if (r >= rows) return;
    const float s = row_scale ? __ldg(row_scale + r) : 1.0f;
    const __nv_bfloat16* yr = y + r * ldy;
    __nv_bfloat16* hr = h + r * ffn;
#pragma unroll 4
    for (int j = (threadIdx.x & 31) * 8; j < ffn; j += 256) {
        const int c = gate_col(j);
        float g[8], u[8], o[8];
        ep::bf16x8_to_f32(ptx::ld_nc_v4(yr + c), g);
        ep::bf16x8_to_f32(ptx::ld_nc_v4(yr + c + 128), u);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = g[i] * sigmoid(g[i]) * u[i] * s;
        *reinterpret_cast<uint4*>(hr + j) = ep::f32x8_to_bf16(o);
    }
}

__global__ void __launch_bounds__(kThreads)
    swiglu_backward_kernel(const __nv_bfloat16* __restrict__ dh, int64_t lddh, const __nv_bfloat16* __restrict__ y,
                           int64_t ldy, const float* __restrict__ row_scale, __nv_bfloat16* __restrict__ dy,
                           float* __restrict__ drow_scale, int64_t rows, int ffn) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock + (threadIdx.x >> 5);
    if (r >= rows) return;
    const float s = row_scale ? __ldg(row_scale + r) : 1.0f;
    const __nv_bfloat16* yr = y + r * ldy;
    const __nv_bfloat16* dhr = dh + r * lddh;
    __nv_bfloat16* dyr = dy + r * 2 * ffn;
    float sum = 0.f;
#pragma unroll 2
    for (int j = (threadIdx.x & 31) * 8; j < ffn; j += 256) {
        const int c = gate_col(j);
        float g[8], u[8], d[8], dg[8], du[8];
        ep::bf16x8_to_f32(ptx::ld_nc_v4(yr + c), g);
        ep::bf16x8_to_f32(ptx::ld_nc_v4(yr + c + 128), u);
        ep::bf16x8_to_f32(ptx::ld_nc_v4(dhr + j), d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sig = sigmoid(g[i]);
            const float a = g[i] * sig;
            const float ds = d[i] * s;
            sum += d[i] * a * u[i];
            du[i] = ds * a;
            dg[i] = ds * u[i] * sig * (1.0f + g[i] * (1.0f - sig));
        }
        *reinterpret_cast<uint4*>(dyr + c) = ep::f32x8_to_bf16(dg);
        *reinterpret_cast<uint4*>(dyr + c + 128) = ep::f32x8_to_bf16(du);
    }
    if (drow_scale) {
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if ((threadIdx.x & 31) == 0) drow_scale[r] = sum;
    }
}

unsigned blocks_for(int64_t rows) {
    const int64_t b = (rows + kRowsPerBlock - 1) / kRowsPerBlock;
    if (b > INT32_MAX) throw kiwi::error("swiglu: too many rows");
    return static_cast<unsigned>(b);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

void check(const __nv_bfloat16* y, int64_t ldy, const __nv_bfloat16* out, int ffn) {
    if (!y || !out) throw kiwi::error("swiglu: missing input or output");
    if (ffn < 128 || ffn % 128 || ffn > (INT32_MAX - 256) / 2) {
        throw kiwi::error("swiglu: the hidden columns must be a positive multiple of 128, in all fewer than 2^30");
    }
    if (ldy < 2 * static_cast<int64_t>(ffn)) throw kiwi::error("swiglu: row stride below the rows' length");
    if (!aligned16(y) || !aligned16(out) || ldy % 8) throw kiwi::error("swiglu: rows must start on 16-byte boundaries");
}

}  // namespace

void swiglu_forward(const __nv_bfloat16* y, int64_t ldy, const float* row_scale, __nv_bfloat16* h, int64_t rows,
                    int ffn, cudaStream_t s) {
    if (rows <= 0) return;
    check(y, ldy, h, ffn);
    swiglu_forward_kernel<<<blocks_for(rows), kThreads, 0, s>>>(y, ldy, row_scale, h, rows, ffn);
    KIWI_CUDA_CHECK(cudaGetLastError());
}

void swiglu_backward(const __nv_bfloat16* dh, int64_t lddh, const __nv_bfloat16* y, int64_t ldy,
                     const float* row_scale, __nv_bfloat16* dy, float* drow_scale, int64_t rows, int ffn,
                     cudaStream_t s) {
    if (rows <= 0) return;
    check(y, ldy, dy, ffn);
    if (!dh) throw kiwi::error("swiglu: missing dh");
    if (lddh < ffn) throw kiwi::error("swiglu: dh's row stride below its rows' length");
    if (!aligned16(dh) || lddh % 8) throw kiwi::error("swiglu: dh's rows must start on 16-byte boundaries");
    swiglu_backward_kernel<<<blocks_for(rows), kThreads, 0, s>>>(dh, lddh, y, ldy, row_scale, dy, drow_scale, rows,
                                                                 ffn);
    KIWI_CUDA_CHECK(cudaGetLastError());
}

}  // namespace kiwi::ops
