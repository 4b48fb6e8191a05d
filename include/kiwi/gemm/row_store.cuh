// Coalesced stores of an epilogue whose threads each hold a piece of one row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kiwi/common.hpp"

namespace kiwi::gemm {

#if defined(__CUDACC__)

inline constexpr int kRowStoreBytes = 2048;  // shared memory of one warp

/// Where 16-byte piece `piece` of row `row` is in a warp's staging memory: pieces
/// are XOR-swizzled by row so that neither side of the exchange has a bank conflict.
__device__ __forceinline__ uint8_t* staged(uint8_t* stg, int row, int piece) {
    return stg + row * 64 + ((piece ^ ((row >> 1) & 3)) * 16);
}

/// Stores rows [0, rows) of the staged 32 x 64 bytes to dst + row * ld_bytes, the
/// first `bytes` (at least 1) of each.  Four lanes store a row's 64 bytes, so a
/// store instruction fills whole sectors of eight rows instead of half sectors
/// of 32.  `vec`: dst and ld_bytes are multiples of 16; else the columns go out
/// as 2-byte elements, 32 lanes along a row.
__device__ __forceinline__ void flush_rows64(uint8_t* stg, uint8_t* dst, int64_t ld_bytes, int rows, int bytes,
                                             bool vec) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    if (vec && bytes >= 64) {
        const int piece = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2);
            const uint4 x = *reinterpret_cast<const uint4*>(staged(stg, row, piece));
            if (row < rows) *reinterpret_cast<uint4*>(dst + row * ld_bytes + piece * 16) = x;
        }
    } else {
#pragma unroll 8
        for (int row = 0; row < rows; ++row) {
            const uint16_t x = *reinterpret_cast<const uint16_t*>(staged(stg, row, lane >> 3) + (lane & 7) * 2);
            if (lane * 2 < bytes) *reinterpret_cast<uint16_t*>(dst + row * ld_bytes + lane * 2) = x;
        }
    }
    __syncwarp();
}

/// Lane l of the warp holds 64 bytes of row l of a tile: through `stg` (2 KB of
/// shared memory of this warp) to memory.
__device__ __forceinline__ void store_rows64(uint8_t* stg, const uint4 (&w)[4], uint8_t* dst, int64_t ld_bytes,
                                             int rows, int bytes, bool vec) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(staged(stg, lane, j)) = w[j];
    flush_rows64(stg, dst, ld_bytes, rows, bytes, vec);
}

/// Lane l holds column l of 32 rows: v[j] is row j's, stored as bf16.
__device__ __forceinline__ void store_columns32(uint8_t* stg, const float (&v)[32], __nv_bfloat16* dst, int64_t ld,
                                                int rows) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        *reinterpret_cast<__nv_bfloat16*>(staged(stg, j, lane >> 3) + (lane & 7) * 2) = __float2bfloat16_rn(v[j]);
    }
    flush_rows64(stg, reinterpret_cast<uint8_t*>(dst), ld * 2, rows, 64, true);
}

/// The same for 16 fp32 values a lane that are added to dst's rows, of bf16 or
/// fp32 elements: one addition in fp32 and one rounding each.
template <typename T>
__device__ __forceinline__ void add_rows16(uint8_t* stg, const uint4 (&w)[4], T* dst, int64_t ld, int rows) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(staged(stg, lane, j)) = w[j];
    __syncwarp();
    const int piece = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (lane >> 2);
        if (row >= rows) continue;
        const float4 x = *reinterpret_cast<const float4*>(staged(stg, row, piece));
        T* at = dst + row * ld + piece * 4;
        if constexpr (sizeof(T) == 4) {
            float4 o = *reinterpret_cast<const float4*>(at);
            o.x += x.x;
            o.y += x.y;
            o.z += x.z;
            o.w += x.w;
            *reinterpret_cast<float4*>(at) = o;
        } else {
            __nv_bfloat162 o[2];
            *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(at);
            const float2 lo = __bfloat1622float2(o[0]), hi = __bfloat1622float2(o[1]);
            o[0] = __floats2bfloat162_rn(lo.x + x.x, lo.y + x.y);
            o[1] = __floats2bfloat162_rn(hi.x + x.z, hi.y + x.w);
            *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(o);
        }
    }
    __syncwarp();
}

#endif  // __CUDACC__

}  // namespace kiwi::gemm
