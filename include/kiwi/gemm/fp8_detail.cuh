// Shared by the two FP8 kernels: parameters, packed fp32 arithmetic, SwiGLU.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kiwi/common.hpp"
#include "kiwi/gemm/fp8_gemm.hpp"

namespace kiwi::gemm::fp8 {

inline constexpr int kBN = 256;  // columns (rows of B) of a tile: two scale blocks, one of gate and one of up with SwiGLU
inline constexpr int kBK = 128;  // bytes = e4m3 elements of K a stage: one scale block

enum Epi : int { kEpiStore = 0, kEpiSwiGLU = 1, kEpiSwiGLUQuant = 2 };

struct Params {
    Fp8GemmArgs a;
    int k_blocks;
    int nb;  // scale blocks of B per group along n
    uint32_t* error;
};

/// The kernel for few rows a group (csrc/fp8_few_rows.cu), for `split` CTAs a tile along K.
void launch_few_rows(const Params& p, int row_chunk, int split, cudaStream_t stream);

#if defined(__CUDACC__)

/// A launch in clusters of `cluster` CTAs that may start before the kernel ahead of it has ended (`follows`).
template <typename... Formal, typename... Actual>
void launch_kernel(void (*kernel)(Formal...), unsigned grid, int threads, int smem, int cluster, bool follows,
                   cudaStream_t stream, const Actual&... args) {
    cudaLaunchAttribute attr[2] = {};
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n++].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    }
    if (follows) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    KIWI_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, Formal(args)...));
}

__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}

__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}

/// acc += v * s on two fp32 lanes (one instruction).
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t v, uint64_t s) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(s));
}

/// A scale of A.  Not through the read-only path: in a product that follows
/// another one, the first may still be writing these while this kernel runs, up
/// to grid_wait_before(), and what that path reads has to stay as it is for the
/// whole kernel.
__device__ __forceinline__ float ld_a_scale(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}

/// x / (1 + exp(-x)) with the approximate division (2 steps of 2^-23; 0 where
/// exp(-x) exceeds 2^126): 64 of them are straight-line code in an epilogue, and
/// with IEEE divisions the SM spent 11 us a tile fetching it.
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

/// Sets one row of the output to zero (scale 1 where it is quantised): thread `t` of `threads`.
template <int EPI>
__device__ __forceinline__ void zero_row(const Fp8GemmArgs& a, int64_t r, int cols, int t, int threads) {
    if constexpr (EPI == kEpiSwiGLUQuant) {
        for (int c = t * 16; c < cols; c += threads * 16) {
            *reinterpret_cast<uint4*>(a.codes + r * cols + c) = make_uint4(0, 0, 0, 0);
        }
        for (int c = t; c < cols / 128; c += threads) a.scales[r * (cols / 128) + c] = 1.0f;
    } else {
        for (int c = t; c < cols; c += threads) a.c[r * a.ldc + c] = __float2bfloat16_rn(0.f);
    }
}

#endif  // __CUDACC__

}  // namespace kiwi::gemm::fp8
