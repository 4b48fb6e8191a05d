// Coalesced stores of an epilogue whose threads each hold a piece of one row.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kiwi/common.hpp"

namespace kiwi::gemm {

#if defined(__CUDACC__)

inline constexpr int kRowStoreBytes = 2048;  // shared memory of one warp

/// Lane l of the warp holds 64 bytes of row l.  They pass through `stg` (2 KB of
/// shared memory of this warp, 16-byte pieces XOR-swizzled so that neither side
/// has a bank conflict) and come back as emit(row, piece, 16 bytes), four lanes
/// to a row: a warp's store then fills eight rows' 64-byte segments, whole
/// sectors, instead of half sectors of 32 rows.
template <typename Emit>
__device__ __forceinline__ void emit_rows64(uint8_t* stg, const uint4 (&w)[4], Emit&& emit) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stg + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16)) = w[j];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (lane >> 2), piece = lane & 3;
        emit(row, piece, *reinterpret_cast<const uint4*>(stg + row * 64 + ((piece ^ ((row >> 1) & 3)) * 16)));
    }
    __syncwarp();
}

#endif  // __CUDACC__

}  // namespace kiwi::gemm
