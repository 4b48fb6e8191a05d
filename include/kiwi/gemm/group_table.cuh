// The tile schedule of a grouped product, built by every CTA in its own shared
// memory from the groups' row counts on the device: no schedule launch before
// the product, no host synchronisation, no workspace that two launches could
// share.  All warps of the CTA scan the counts, 32 groups at a time.  A launch
// whose groups are all empty takes 3.0 us with one group, 3.1 to 3.4 with 32 to
// 256 and 4.9 (bf16 product: 5.8) with 1024, in graphs on one B200: the table is
// 2 to 3 us of it at 1024 groups and nothing to speak of below 256.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kiwi/common.hpp"

namespace kiwi::gemm {

inline constexpr int kMaxGroups = 1024;

// Error bits of the products' device error word (see gemm_error_word()).
inline constexpr uint32_t kGemmTimeout = 1u;   // a bounded wait ran out: the output is incomplete
inline constexpr uint32_t kGemmCounts = 2u;    // a negative count, or counts whose sum exceeds the rows

#if defined(__CUDACC__)

/// off[g] .. off[g + 1] are group g's rows; tiles[g] its first tile.
struct GroupTable {
    int32_t off[kMaxGroups + 1];
    int32_t tiles[kMaxGroups + 1];
    int32_t chunk_tiles[kMaxGroups / 32];  // scratch of the scan: sums of 32 groups
    int64_t chunk_rows[kMaxGroups / 32];
};

template <typename T>
__device__ __forceinline__ T warp_inclusive_scan(T v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, v, d);
        if ((threadIdx.x & 31) >= d) v += y;
    }
    return v;
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

/// Whole CTA; ends with a __syncthreads().  Counts are clamped to what `rows`
/// can hold, so every offset is a valid row whatever the counts are (a bad
/// count sets kGemmCounts in *error).  counts == nullptr: one group of all rows.
/// `bm` rows and `n_tiles` column tiles make a tile.
__device__ __forceinline__ void build_group_table(GroupTable& t, const int32_t* counts, int groups, int64_t rows,
                                                  int bm, int n_tiles, uint32_t* error) {
    if (counts == nullptr) {
        if (threadIdx.x == 0) {
            t.off[0] = 0;
            t.off[1] = static_cast<int32_t>(rows);
            t.tiles[0] = 0;
            t.tiles[1] = static_cast<int32_t>((rows + bm - 1) / bm) * n_tiles;
        }
        __syncthreads();
        return;
    }
    bool bad = false;
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        int32_t c = __ldg(&counts[g]);
        if (c < 0) {
            bad = true;
            c = 0;
        }
        t.off[g + 1] = c;
    }
    __syncthreads();
    // A warp takes 32 groups at a time: first their rows, then, with the rows
    // before them known, their offsets and tiles, then the tiles before them.
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int ch = warp; ch * 32 < groups; ch += warps) {
        const int g = ch * 32 + lane;
        const int64_t sum = warp_sum(static_cast<int64_t>(g < groups ? t.off[g + 1] : 0));
        if (lane == 0) t.chunk_rows[ch] = sum;
    }
    __syncthreads();
    for (int ch = warp; ch * 32 < groups; ch += warps) {
        const int g = ch * 32 + lane;
        const int32_t c = g < groups ? t.off[g + 1] : 0;
        const int64_t before = warp_sum(lane < ch ? t.chunk_rows[lane] : int64_t{0});
        const int64_t upto = before + warp_inclusive_scan(static_cast<int64_t>(c));
        const int64_t first = upto - c < rows ? upto - c : rows;
        const int64_t last = upto < rows ? upto : rows;
        if (upto > rows) bad = true;
        const int32_t tl = warp_inclusive_scan(static_cast<int32_t>((last - first + bm - 1) / bm) * n_tiles);
        if (g < groups) {
            t.off[g + 1] = static_cast<int32_t>(last);
            t.tiles[g + 1] = tl;
        }
        if (lane == 31) t.chunk_tiles[ch] = tl;
    }
    __syncthreads();
    for (int ch = warp; ch * 32 < groups; ch += warps) {
        const int g = ch * 32 + lane;
        const int32_t before = warp_sum(lane < ch ? t.chunk_tiles[lane] : 0);
        if (g < groups) t.tiles[g + 1] += before;
    }
    if (threadIdx.x == 0) {
        t.off[0] = 0;
        t.tiles[0] = 0;
    }
    if (bad && error && blockIdx.x == 0) atomicOr(error, kGemmCounts);
    __syncthreads();
}

/// Group, row block and column block of a tile.  The column block is outermost
/// within a group: the row blocks that share one weight tile are neighbours in
/// the schedule, run at the same time and read it from L2.
__device__ __forceinline__ void find_tile(const GroupTable& t, int groups, int n_tiles, int tile, int& g, int& mt,
                                          int& nt) {
    int lo = 0, hi = groups - 1;
    while (lo < hi) {  // first g with tiles[g + 1] > tile
        const int mid = (lo + hi) >> 1;
        if (t.tiles[mid + 1] > tile) hi = mid;
        else lo = mid + 1;
    }
    g = lo;
    const int local = tile - t.tiles[g];
    const int m_tiles = (t.tiles[g + 1] - t.tiles[g]) / n_tiles;
    nt = local / m_tiles;
    mt = local - nt * m_tiles;
}

#endif  // __CUDACC__

}  // namespace kiwi::gemm
