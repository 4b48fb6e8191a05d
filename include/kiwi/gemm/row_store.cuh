// Coalesced stores of an epilogue whose threads each hold a piece of one row.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kiwi/common.hpp"

namespace kiwi::gemm {

#if defined(__CUDACC__)

inline constexpr int kRowStoreBytes = 2048;  // shared memory of one warp

/// Lane l of the warp holds 64 bytes of row l of a tile; rows [0, rows) of them
/// go to dst + row * ld_bytes, the first `bytes` (at least 1) of each.  They pass
/// through `stg` (2 KB of shared memory of this warp, 16-byte pieces
/// XOR-swizzled so that neither side has a bank conflict): four lanes then store
/// a row's 64 bytes, so a store instruction fills whole sectors of eight rows
/// instead of half sectors of 32.  `vec`: dst and ld_bytes are multiples of 16;
/// else the columns go out as 2-byte elements, 32 lanes along a row.
__device__ __forceinline__ void store_rows64(uint8_t* stg, const uint4 (&w)[4], uint8_t* dst, int64_t ld_bytes,
                                             int rows, int bytes, bool vec) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stg + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16)) = w[j];
    __syncwarp();
    if (vec && bytes >= 64) {
        const int piece = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2);
            const uint4 x = *reinterpret_cast<const uint4*>(stg + row * 64 + ((piece ^ ((row >> 1) & 3)) * 16));
            if (row < rows) *reinterpret_cast<uint4*>(dst + row * ld_bytes + piece * 16) = x;
        }
    } else {
#pragma unroll 4
        for (int row = 0; row < rows; ++row) {
            const uint16_t x = *reinterpret_cast<const uint16_t*>(
                stg + row * 64 + (((lane >> 3) ^ ((row >> 1) & 3)) * 16) + (lane & 7) * 2);
            if (lane * 2 < bytes) *reinterpret_cast<uint16_t*>(dst + row * ld_bytes + lane * 2) = x;
        }
    }
    __syncwarp();
}

#endif  // __CUDACC__

}  // namespace kiwi::gemm
