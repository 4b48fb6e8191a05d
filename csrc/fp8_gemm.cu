// Block-scaled FP8 products on sm_100a tensor cores (tcgen05 + TMEM + TMA).
//
//   C[r, n] = sum over kb of sa[r, kb] * sb[n / 128, kb] * (A[r, kb] . B[g][n, kb])
//
// with e4m3 operands in blocks kb of 128 columns, one fp32 scale per 1 x 128
// block of A (the FP8 dispatch's wire format) and per 128 x 128 block of B,
// dense or grouped by expert with row counts on the device.
//
// The scales are any fp32 number, so they cannot ride along in the tensor core
// (its block scales are powers of two).  The four K = 32 MMAs of one
// 128-column block therefore go to a TMEM accumulator of their own; eight warps
// drain it into registers with one fused multiply-add per element,
// acc += (sa * sb) * partial, while the tensor core fills the other of the two
// accumulators that TMEM holds.
//
// What bounds it: a block's 128 x 256 x 128 multiply-adds are 512 tensor cycles
// and its drain 256 FP32-pipe cycles, but an accumulator's round trip (MMAs ~720
// cycles from issue to completion, drain, hand-over) makes a block ~820 cycles
// on an idle GPU; in long runs the power cap holds the clock at 1.4 to 1.6 GHz.
// Measured on one B200: 4096 x 4096 x 7168 in 117 us (2.05 PFLOP/s, 1.23 of the
// measured bf16 rate); gate and up product with SwiGLU and quantisation of
// 32768 rows over 32 experts (4096 x 7168) in 982 us (1.96 PFLOP/s), the down
// product (7168 x 2048) in 570 us (1.69).  Four accumulators of 128 columns,
// with twice the hand-overs, took 15 to 25 % longer; pairs of SMs sharing a tile
// took as long at the largest sizes and longer at others.
//
// Kernel shape (one CTA per SM, persistent over 128 x 256 tiles):
//   warps 0..7   drain and epilogue: TMEM lane quadrant = warp % 4 (32 rows),
//                columns [64 h, 64 h + 64) and [128 + 64 h, 128 + 64 h + 64) for
//                h = warp / 4, so that with SwiGLU a thread owns matching gate
//                and up columns; 128 fp32 sums in registers
//   warp 8       TMA producer: 128 x 128-byte A tile + 256 x 128-byte B tile
//   warp 9       TMEM owner and MMA issuer
//   warps 10..11 scales: sa * sb of every row, a block ahead, to shared memory
// Every wait is bounded; one that runs out sets the error word, and the CTA
// drains its loads, frees its TMEM and leaves.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "kiwi/ep/quant.cuh"
#include "kiwi/gemm/fp8_detail.cuh"
#include "kiwi/gemm/fp8_gemm.hpp"
#include "kiwi/gemm/group_table.cuh"
#include "kiwi/gemm/grouped_gemm.hpp"
#include "kiwi/gemm/row_store.cuh"
#include "kiwi/gemm/tensor_map.hpp"
#include "kiwi/sm100.cuh"

namespace kiwi::gemm {

namespace {

using namespace fp8;

constexpr int kBM = 128;
constexpr int kThreads = 384;  // two drain warpgroups; one with the producer, the MMA issuer and the scale warps
constexpr int kDrainThreads = 256;
constexpr int kScaleWarps = 2;
// 128 sums and a 32-column TMEM load do not fit the 168 registers that 384
// threads share evenly; the third warpgroup gives some of its own away.  How many
// the drain gets is what was fastest without spills; its loop is unrolled, which
// frees it of moves between the blocks' registers: 4096 x 4096 x 7168 in 117 us
// against 127, 32768 rows over 32 experts 982 + 570 against 1019 + 598.
template <int EPI>
struct Tuning {
    static constexpr int kDrainRegs = EPI == kEpiStore ? 192 : 208;
    static constexpr int kIssueRegs = EPI == kEpiStore ? 120 : 88;
    static constexpr int kUnroll = 4;
    static_assert(2 * kDrainRegs + kIssueRegs <= 3 * 168, "more registers than the CTA is launched with");
};

struct Smem {
    static constexpr int kStages = 4;
    static constexpr int kABytes = kBM * kBK;
    static constexpr int kBBytes = kBN * kBK;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kTableOffset = kStages * kStageBytes;
    static constexpr int kAmaxOffset = kTableOffset + static_cast<int>(round_up(sizeof(GroupTable), 16));
    static constexpr int kScaleOffset = kAmaxOffset + 2 * 2 * kBM * 4;
    static constexpr int kStgOffset = kScaleOffset + 2 * kBM * 8;
    static constexpr int kBarOffset = kStgOffset + kDrainThreads / 32 * kRowStoreBytes;
    static constexpr int kBytes = kBarOffset + 256 + 1024;  // barriers, TMEM slot, alignment slack
};
static_assert(Smem::kBytes <= 227 * 1024, "exceeds the shared-memory limit");

/// The warp's rows' 64 columns at `col` as bf16: row r0 + lane from v, of which
/// rows before `rows` and columns before `cols` are in the matrix.
__device__ __forceinline__ void store_rows(__nv_bfloat16* c, int64_t ldc, int64_t r0, int rows, int col, int cols,
                                           const float (&v)[64], uint8_t* stg, bool vec) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 32 columns = 64 bytes a row
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = v[32 * h + 8 * j + i];
            w[j] = ep::f32x8_to_bf16(f);
        }
        const int at = col + 32 * h;
        if (rows > 0 && at < cols) {
            store_rows64(stg, w, reinterpret_cast<uint8_t*>(c + r0 * ldc + at), ldc * 2, rows, (cols - at) * 2, vec);
        }
    }
}

template <int EPI>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ Params p) {
    using S = Smem;
    constexpr int kStages = S::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    GroupTable& table = *reinterpret_cast<GroupTable*>(smem + S::kTableOffset);
    float* s_amax = reinterpret_cast<float*>(smem + S::kAmaxOffset);  // [tile parity][column half][thread]
    float2* s_scale = reinterpret_cast<float2*>(smem + S::kScaleOffset);  // [block parity][row]: for each column part
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBarOffset);
    // done: a block's MMAs have run and its scales are in shared memory.  Its
    // operands may be overwritten, its partial sums drained.
    uint64_t* done = full + kStages;
    uint64_t* drained = done + kStages;  // [block parity] an accumulator and its scales have been read
    uint64_t* amax_bar = drained + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(amax_bar + 1);
    __shared__ int s_abort;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform: the roles' addresses stay in uniform registers
    const int lane = threadIdx.x & 31;
    const int groups = p.a.num_groups;
    const int n_tiles = (p.a.n + kBN - 1) / kBN;
    const int k_blocks = p.k_blocks;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < kStages; ++s) {
            sm100::mbar_init(&full[s], 1);
            sm100::mbar_init(&done[s], 1 + kScaleWarps);
        }
        for (int i = 0; i < 2; ++i) {
            sm100::mbar_init(&drained[i], kDrainThreads / 32);
        }
        sm100::mbar_init(amax_bar, kDrainThreads);
        sm100::fence_mbar_init();
    }
    if (warp == 8 && lane == 0) {
        sm100::tma_prefetch_desc(&tmap_a);
        sm100::tma_prefetch_desc(&tmap_b);
    }
    if (warp == 9) {
        sm100::tmem_alloc(tmem_slot, 2 * kBN);
    }
    build_group_table(table, p.a.counts, groups, p.a.rows, kBM, n_tiles, p.error);
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    if (p.a.feeds_next) sm100::grid_launch_dependents();
    if (p.a.follows) sm100::grid_wait_before();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = table.tiles[groups];

    // A tile with at most 64 rows of its group left runs M = 64 MMAs: half the
    // tensor work, the same sums.  Its row 16 q + i is in TMEM lane 32 q + i.
    auto half_tile = [&](int g, int mt) { return table.off[g + 1] - table.off[g] - mt * kBM <= 64; };

    auto aborted = [&]() { return *reinterpret_cast<volatile int*>(&s_abort) != 0; };
    auto fail = [&]() {
        *reinterpret_cast<volatile int*>(&s_abort) = 1;
        atomicOr(p.error, kGemmTimeout);
    };

    if (warp >= 8) {
        sm100::reg_dec<Tuning<EPI>::kIssueRegs>();
        if (warp == 8 && lane == 0) {
            uint32_t issued = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < total_tiles && !aborted(); tile += gridDim.x) {
                int g, mt, nt;
                find_tile(table, groups, n_tiles, tile, g, mt, nt);
                const int row0 = table.off[g] + mt * kBM;
                const int brow0 = g * p.a.n + nt * kBN;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    const uint32_t stage = issued % kStages;
                    if (!sm100::mbar_wait(&done[stage], ((issued / kStages) & 1) ^ 1)) {
                        fail();
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + stage * S::kStageBytes;
                    sm100::mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
                    sm100::tma_load_2d(sa, &tmap_a, &full[stage], kb * kBK, row0);
                    sm100::tma_load_2d(sa + S::kABytes, &tmap_b, &full[stage], kb * kBK, brow0);
                    ++issued;
                }
            }
            // No load may still be in flight when this CTA's shared memory goes away:
            // each has landed once the MMAs that read its stage are done.
            for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                if (!sm100::mbar_wait(&done[i % kStages], (i / kStages) & 1)) fail();
            }
        } else if (warp == 9) {
            // The whole warp walks the blocks and one elected lane issues, so that
            // descriptors and addresses are warp-uniform.
            const uint64_t desc0 = sm100::sw128_kmajor_desc(smem);
            const bool issuer = sm100::elect_one();
            uint32_t it = 0;
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < total_tiles && !aborted(); tile += gridDim.x) {
                int g, mt, nt;
                find_tile(table, groups, n_tiles, tile, g, mt, nt);
                const uint32_t idesc =
                    half_tile(g, mt) ? sm100::idesc_e4m3_f32(64, kBN) : sm100::idesc_e4m3_f32(kBM, kBN);
                for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                    const uint32_t buf = it & 1;
                    ok = sm100::mbar_wait(&full[stage], phase) && sm100::mbar_wait(&drained[buf], ((it >> 1) & 1) ^ 1);
                    if (!ok) {
                        if (issuer) fail();
                        break;
                    }
                    sm100::tc_fence_after();
                    const uint64_t ad = desc0 + stage * (S::kStageBytes >> 4);
                    const uint64_t bd = ad + (S::kABytes >> 4);
                    const uint32_t d = tmem_base + buf * kBN;
                    if (issuer) {
#pragma unroll
                        for (int kk = 0; kk < kBK / 32; ++kk) {  // 32 bytes of K = 2 descriptor units a step
                            sm100::mma_f8(d, ad + 2 * kk, bd + 2 * kk, idesc, kk != 0 ? 1u : 0u);
                        }
                        sm100::mma_commit(&done[stage]);
                    }
                    __syncwarp();
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Nor may an MMA still write the TMEM that is freed below.
            if (it > 0 && !sm100::mbar_wait(&done[(it - 1) % kStages], ((it - 1) / kStages) & 1) && issuer) fail();
        } else if (warp >= 10) {
            // Scale warps: each lane multiplies two rows' scales with those of the
            // tile's two column parts, a block ahead of the drain.
            uint32_t it = 0;
            uint32_t stage = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < total_tiles && !aborted(); tile += gridDim.x) {
                int g, mt, nt;
                find_tile(table, groups, n_tiles, tile, g, mt, nt);
                const int r = (warp - 10) * 64 + lane;
                const int64_t row = static_cast<int64_t>(table.off[g]) + mt * kBM + r;
                const int64_t last = table.off[g + 1] - 1;  // rows past the group's are not stored: any scale will do
                const float* sa0 = p.a.a_scale + (row < last ? row : last) * p.a.a_scale_stride;
                const float* sa1 = p.a.a_scale + (row + 32 < last ? row + 32 : last) * p.a.a_scale_stride;
                const float* sb0 = p.a.b_scale + (static_cast<int64_t>(g) * p.nb + 2 * nt) * k_blocks;
                const float* sb1 = 2 * nt + 1 < p.nb ? sb0 + k_blocks : sb0;
                float a0 = ld_a_scale(sa0), a1 = ld_a_scale(sa1), b0 = __ldg(sb0), b1 = __ldg(sb1);
                for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                    const float2 v0 = make_float2(a0 * b0, a0 * b1), v1 = make_float2(a1 * b0, a1 * b1);
                    if (kb + 1 < k_blocks) {
                        a0 = ld_a_scale(sa0 + kb + 1);
                        a1 = ld_a_scale(sa1 + kb + 1);
                        b0 = __ldg(sb0 + kb + 1);
                        b1 = __ldg(sb1 + kb + 1);
                    }
                    const uint32_t buf = it & 1;
                    if (!sm100::mbar_wait(&drained[buf], ((it >> 1) & 1) ^ 1)) {
                        if (lane == 0) fail();
                        ok = false;
                        break;
                    }
                    s_scale[buf * kBM + r] = v0;
                    s_scale[buf * kBM + r + 32] = v1;
                    __syncwarp();
                    if (lane == 0) sm100::mbar_arrive(&done[stage]);
                    if (++stage == kStages) stage = 0;
                }
            }
        }
    } else {
        sm100::reg_inc<Tuning<EPI>::kDrainRegs>();
        const int q = warp & 3;
        const int half = warp >> 2;
        uint8_t* stg = smem + S::kStgOffset + warp * kRowStoreBytes;
        const bool vec = p.a.ldc % 8 == 0 && reinterpret_cast<uintptr_t>(p.a.c) % 16 == 0;
        uint32_t it = 0;
        uint32_t stage = 0, phase = 0;
        uint32_t n_done = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < total_tiles && !aborted(); tile += gridDim.x, ++n_done) {
            int g, mt, nt;
            find_tile(table, groups, n_tiles, tile, g, mt, nt);
            // The warp's rows: r0 + lane, r_end of them in the group.
            const int span = half_tile(g, mt) ? 16 : 32;
            const int row_in_tile = q * span + lane;
            const int64_t r0 = static_cast<int64_t>(table.off[g]) + mt * kBM + q * span;
            const int64_t row = r0 + lane;
            const int r_end = static_cast<int>(table.off[g + 1] - r0 < span ? table.off[g + 1] - r0 : span);
            const bool valid = lane < r_end;
            uint64_t acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
#pragma unroll Tuning<EPI>::kUnroll
            for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                const uint32_t buf = it & 1;
                if (!sm100::mbar_wait(&done[stage], phase)) {
                    fail();
                    ok = false;
                    break;
                }
                sm100::tc_fence_after();
                const uint32_t taddr =
                    tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * kBN + static_cast<uint32_t>(half * 64);
                const float2 sc = s_scale[buf * kBM + row_in_tile];
                const uint64_t ss0 = pack2(sc.x, sc.x), ss1 = pack2(sc.y, sc.y);
                // Four loads of 32 columns; each but the first runs under the
                // multiply-adds of the one before.
                uint32_t v[2][32];
                sm100::tmem_issue_32cols(taddr, v[0]);
                sm100::tmem_wait_32cols(v[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c < 3) {
                        sm100::tmem_issue_32cols(taddr + ((c + 1) >> 1) * 128 + ((c + 1) & 1) * 32, v[(c + 1) & 1]);
                    } else {  // all of the accumulator is in registers: the next MMAs may have it
                        sm100::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) sm100::mbar_arrive(&drained[buf]);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        fma2(acc[c * 16 + i], pack2(v[c & 1][2 * i], v[c & 1][2 * i + 1]), c < 2 ? ss0 : ss1);
                    }
                    if (c < 3) sm100::tmem_wait_32cols(v[(c + 1) & 1]);
                }
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) break;
            if constexpr (EPI == kEpiStore) {
                const float scale = valid && p.a.row_scale ? __ldg(p.a.row_scale + row) : 1.0f;
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    float v[64];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 f = unpack2(acc[part * 32 + i]);
                        v[2 * i] = f.x * scale;
                        v[2 * i + 1] = f.y * scale;
                    }
                    const int col = nt * kBN + part * 128 + half * 64;
                    store_rows(p.a.c, p.a.ldc, r0, r_end, col, p.a.n, v, stg, vec);
                }
            } else {
                float h[64];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float2 gt = unpack2(acc[i]);
                    const float2 up = unpack2(acc[32 + i]);
                    h[2 * i] = silu(gt.x) * up.x;
                    h[2 * i + 1] = silu(gt.y) * up.y;
                }
                const int col = nt * (kBN / 2) + half * 64;
                if constexpr (EPI == kEpiSwiGLU) {
                    const float scale = valid && p.a.row_scale ? __ldg(p.a.row_scale + row) : 1.0f;
#pragma unroll
                    for (int i = 0; i < 64; ++i) h[i] *= scale;
                    store_rows(p.a.c, p.a.ldc, r0, r_end, col, p.a.n / 2, h, stg, vec);
                } else {
                    // The tile's 128 hidden columns are one scale block; its other 64
                    // columns are in the thread of the same row in the other four warps.
                    float amax = 0.f;
#pragma unroll
                    for (int i = 0; i < 64; ++i) amax = fmaxf(amax, fabsf(h[i]));
                    float* slot = s_amax + (n_done & 1) * 2 * kBM;
                    const int place = q * 32 + lane;  // this thread's own, whatever the tile's height
                    slot[half * kBM + place] = amax;
                    sm100::mbar_arrive(amax_bar);
                    if (!sm100::mbar_wait(amax_bar, n_done & 1)) {
                        fail();
                        break;
                    }
                    amax = fmaxf(amax, slot[(half ^ 1) * kBM + place]);
                    float scale, inv;
                    ep::fp8_block_scale(amax, scale, inv);
                    uint4 w[4];
                    uint32_t* wi = reinterpret_cast<uint32_t*>(w);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(h[4 * i] * inv, h[4 * i + 1] * inv),
                                                                     __NV_SATFINITE, __NV_E4M3);
                        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(h[4 * i + 2] * inv, h[4 * i + 3] * inv),
                                                                     __NV_SATFINITE, __NV_E4M3);
                        wi[i] = lo | (hi << 16);
                    }
                    if (r_end > 0) store_rows64(stg, w, p.a.codes + r0 * (p.a.n / 2) + col, p.a.n / 2, r_end, 64, true);
                    if (valid && half == 0) p.a.scales[row * (p.a.n / kBN) + nt] = scale;
                }
            }
        }
        if (p.a.zero_tail) {
            const int cols = EPI == kEpiStore ? p.a.n : p.a.n / 2;
            for (int64_t r = table.off[groups] + static_cast<int64_t>(blockIdx.x); r < p.a.rows; r += gridDim.x) {
                zero_row<EPI>(p.a, r, cols, threadIdx.x, kDrainThreads);
            }
        }
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    if (warp == 9) {
        sm100::tmem_dealloc(tmem_base, 2 * kBN);
    }
}

// ---------------------------------------------------------------------------
// 128 x 128 block quantisation of weights: one CTA per block, which stays in
// registers between its maximum and its conversion (32 bf16 values a thread:
// 4 rows of 8 columns), so w is read once.  Bound by memory; a one-time cost
// when weights are loaded (3.4 TB/s: 131072 x 7168 in 0.83 ms).
// ---------------------------------------------------------------------------
constexpr int kQuantThreads = 512;

__global__ void __launch_bounds__(kQuantThreads) quant_fp8_blocks_kernel(const __nv_bfloat16* __restrict__ w, int64_t ld,
                                                               int64_t rows, int64_t cols, int64_t col_blocks,
                                                               bool vec, uint8_t* __restrict__ codes,
                                                               float* __restrict__ scales) {
    __shared__ float s_max[kQuantThreads / 32];
    const int64_t rb = blockIdx.x / col_blocks, cb = blockIdx.x % col_blocks;
    const int64_t c = cb * 128 + (threadIdx.x & 15) * 8;
    const int64_t r0 = rb * 128 + (threadIdx.x >> 4);
    const bool whole = vec && c + 8 <= cols;
    uint4 in[4];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + 32 * i;
        in[i] = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            if (whole) {
                in[i] = *reinterpret_cast<const uint4*>(w + r * ld + c);
            } else {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = c + j < cols ? __bfloat162float(w[r * ld + c + j]) : 0.f;
                in[i] = ep::f32x8_to_bf16(f);
            }
        }
        float f[8];
        ep::bf16x8_to_f32(in[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]));
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQuantThreads / 32; ++i) amax = fmaxf(amax, s_max[i]);
    float scale, inv;
    ep::fp8_block_scale(amax, scale, inv);
    if (threadIdx.x == 0) scales[blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + 32 * i;
        if (r >= rows) continue;
        float f[8];
        ep::bf16x8_to_f32(in[i], f);
        uint16_t q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            q[j] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * j] * inv, f[2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        }
        uint8_t* dst = codes + r * cols + c;
        if (c + 8 <= cols && cols % 8 == 0) {
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(q[0] | (static_cast<uint32_t>(q[1]) << 16), q[2] | (static_cast<uint32_t>(q[3]) << 16));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (c + j < cols) dst[j] = static_cast<uint8_t>(q[j >> 1] >> (8 * (j & 1)));
            }
        }
    }
}

__device__ uint32_t g_error;

__global__ void take_error_kernel(uint32_t* word, uint32_t* out) { *out = atomicExch(word, 0u); }

template <int EPI>
void launch(const Params& p, cudaStream_t stream) {
    static std::atomic<uint64_t> attr{0};
    raise_smem_limit(reinterpret_cast<const void*>(fp8_gemm_kernel<EPI>), Smem::kBytes, attr);
    const Fp8GemmArgs& a = p.a;
    const CUtensorMap ta = make_tmap_2d(a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.rows, a.k, a.lda, kBM, kBK);
    const CUtensorMap tb = make_tmap_2d(a.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1,
                                        static_cast<uint64_t>(a.num_groups) * a.n, a.k, a.ldb, kBN, kBK);
    // At most this many tiles, however the rows fall into groups.
    const int64_t most = ((a.rows + kBM - 1) / kBM + (a.counts ? a.num_groups : 0)) * ((a.n + kBN - 1) / kBN);
    const int sms = num_sms();
    launch_kernel(fp8_gemm_kernel<EPI>, static_cast<unsigned>(most < sms ? most : sms), kThreads, Smem::kBytes, 1,
                  a.follows, stream, ta, tb, p);
}

struct Choice {
    int row_chunk;  // 0: this file's kernel, else the few-rows kernel with 16, 32 or 48 rows a tile
    int split;      // and its CTAs a tile
};

/// The kernel for a call, by a model of its time in microseconds that was fitted
/// to a sweep of 1 to 2000 rows (dense N x K 512 x 1024 to 7168 x 2048 and 4096 x
/// 7168; 16 and 32 experts).  A CTA needs 0.37 us a block of K here, and 0.285,
/// 0.315 or 0.33 us with 16, 32 or 48 rows a tile, plus 2.5 or 1.6 us a tile for
/// its start and epilogue.  Where a tile's K is split, the exchange of its sums
/// costs another 1.7 us, and several times that on a cluster's second tile, so a
/// split is only for tiles that the GPU runs all at once; clusters of 4 leave
/// some SMs of a GPC unused, and how rows fall into experts is not known here
/// (every expert is taken to end with half a tile), hence the margins.  (Splits
/// of 8 lost to splits of 4.)  No kernel is faster than the weights can be read,
/// at 6.4 TB/s; of kernels that this bounds, few rows are taken (they read with
/// more in flight) unless their own work is clearly more, and of their tiles the
/// smaller unless the larger mean clearly less.  The counts stay on the device, so
/// this goes by the rows of the buffer, taken to be full and evenly divided: with
/// 32 experts (7168 / 2048) the FFN takes 74 us for 8 rows in a buffer of 2048 and 53
/// in one of 8, for 1024 rows 266 and 238 (the zeroing of the rest of the result
/// included).  Measured, this file's kernel against few
/// rows: 1 row, 4096 x 7168: 25.7 / 10.1 us; 64 rows: 26.1 / 13.4; 200: 27.9 /
/// 24.4; 400: 28.6 / 26.4 (48 a tile) or 43.7 (32); 1000: 30.4 / 69; 32 experts of
/// 32 rows, 4096 x 7168: 162 / 149; of 64 rows: 169 / 199.
Choice choose(const Fp8GemmArgs& a, int k_blocks) {
    const double sms = num_sms(), n_tiles = (a.n + kBN - 1) / kBN;
    const double used = a.counts ? static_cast<double>(a.rows < a.num_groups ? a.rows : a.num_groups) : 1.0;
    const double hbm = used * a.n * a.k / 6.4e6;
    auto tiles = [&](double bm) {
        if (!a.counts) return std::ceil(a.rows / bm) * n_tiles;
        return std::max(used, a.rows / bm + used / 2) * n_tiles;
    };
    Choice best{0, 1};
    double work = std::ceil(tiles(kBM) / sms) * (0.37 * k_blocks + 2.5), time = std::max(work, hbm);
    for (int rows : {16, 32, 48}) {
        const double t = tiles(rows), block = rows == 16 ? 0.285 : rows == 32 ? 0.315 : 0.33;
        for (int split : {1, 2, 4}) {
            if (split > 1 && (t * split > (a.counts ? 0.6 : 0.87) * sms || split > k_blocks)) break;
            const double w = split > 1 ? std::ceil(k_blocks / static_cast<double>(split)) * block + 3.3
                                       : std::ceil(t / sms) * (block * k_blocks + 1.6);
            const double us = std::max(w, hbm);
            if (us < time || (us == time && w < (best.row_chunk == 0 ? 1.3 : 0.8) * work)) {
                best = {rows, split};
                work = w;
                time = us;
            }
        }
    }
    return best;
}

}  // namespace

uint32_t* gemm_error_word() {
    static std::mutex mu;
    static uint32_t* ptr[64] = {};
    int dev = 0;
    KIWI_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) throw kiwi::error("gemm_error_word: device index beyond 64");
    std::lock_guard<std::mutex> lock(mu);
    if (!ptr[dev]) {
        void* q = nullptr;
        KIWI_CUDA_CHECK(cudaGetSymbolAddress(&q, g_error));
        ptr[dev] = static_cast<uint32_t*>(q);
    }
    return ptr[dev];
}

void take_error(uint32_t* word, uint32_t* out, cudaStream_t stream) {
    if (!word || !out) throw kiwi::error("take_error: missing words");
    take_error_kernel<<<1, 1, 0, stream>>>(word, out);
    KIWI_CUDA_CHECK(cudaGetLastError());
}

void fp8_gemm(const Fp8GemmArgs& args, cudaStream_t stream) {
    if (args.num_groups < 1 || args.num_groups > kMaxGroups) throw kiwi::error("fp8_gemm: 1..1024 groups");
    if (!args.counts && args.num_groups != 1) throw kiwi::error("fp8_gemm: several groups need counts");
    if (args.n < 1 || args.k < 16 || args.k % 16 != 0) throw kiwi::error("fp8_gemm: K must be a positive multiple of 16");
    if (args.k > INT32_MAX - 256) throw kiwi::error("fp8_gemm: K must be below 2^31 - 256");
    if (args.num_groups > 1 && args.n % 128 != 0) throw kiwi::error("fp8_gemm: grouped N must be a multiple of 128");
    if (args.swiglu && args.n % kBN != 0) throw kiwi::error("fp8_gemm: SwiGLU needs N to be a multiple of 256");
    if (args.codes && !args.swiglu) throw kiwi::error("fp8_gemm: FP8 output needs swiglu");
    if (args.codes && (!args.scales || reinterpret_cast<uintptr_t>(args.codes) % 16 != 0)) {
        throw kiwi::error("fp8_gemm: FP8 output needs codes on a 16-byte boundary and scales");
    }
    if (args.rows < 0 || args.rows > INT32_MAX - kBM ||
        static_cast<int64_t>(args.num_groups) * args.n > INT32_MAX - kBN) {
        throw kiwi::error("fp8_gemm: more than 2^31 rows");
    }
    if (args.rows == 0) return;
    if (!args.a || !args.b || !args.a_scale || !args.b_scale || (!args.c && !args.codes)) {
        throw kiwi::error("fp8_gemm: missing operands or output");
    }
    Params p{};
    p.a = args;
    p.k_blocks = (args.k + kBK - 1) / kBK;
    p.nb = (args.n + 127) / 128;
    p.error = args.error ? args.error : gemm_error_word();
    const Choice c = choose(args, p.k_blocks);
    if (c.row_chunk) launch_few_rows(p, c.row_chunk, c.split, stream);
    else if (!args.swiglu) launch<kEpiStore>(p, stream);
    else if (!args.codes) launch<kEpiSwiGLU>(p, stream);
    else launch<kEpiSwiGLUQuant>(p, stream);
}

void quant_fp8_blocks(const __nv_bfloat16* w, int64_t ld, int64_t rows, int64_t cols, uint8_t* codes, float* scales,
                      cudaStream_t stream) {
    if (rows <= 0 || cols <= 0) return;
    if (!w || !codes || !scales || reinterpret_cast<uintptr_t>(codes) % 16 != 0) {
        throw kiwi::error("quant_fp8_blocks: missing tensors, or codes off a 16-byte boundary");
    }
    const int64_t cb = (cols + 127) / 128, blocks = (rows + 127) / 128 * cb;
    if (blocks > INT32_MAX) throw kiwi::error("quant_fp8_blocks: matrix too large");
    quant_fp8_blocks_kernel<<<static_cast<unsigned>(blocks), kQuantThreads, 0, stream>>>(
        w, ld, rows, cols, cb, ld % 8 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0, codes, scales);
    KIWI_CUDA_CHECK(cudaGetLastError());
}

}  // namespace kiwi::gemm
