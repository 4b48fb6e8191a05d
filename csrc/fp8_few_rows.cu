// Block-scaled FP8 products of few rows a group: single tokens, decode batches.
//
// The same sums as csrc/fp8_gemm.cu with the operands' places swapped: 256 rows
// of the weights are the tensor core's M operand (two of 128: with SwiGLU one
// of gate and one of up), and up to ROWS (16, 32 or 48) rows of the group its N operand.  What
// counts here is reading the weights once at the memory's rate: a stage holds
// 32 KB of weights and only ROWS * 128 bytes of rows, an accumulator 2 * ROWS
// TMEM columns, so that five of them are in flight and the drain (one FMA per
// weight row and token) hides.
//
// Where the tiles do not fill the GPU, a cluster of SPLIT CTAs shares a tile
// along K.  Each leaves its fp32 sums in its own shared memory, then
// CTA r adds up, in rank order, the sums of the tokens
// t % SPLIT == r from all of them and finishes those rows.  No workspace, no
// atomics: the result does not depend on the order of execution.
//
// A group with more than ROWS rows is cut into chunks of ROWS, which read the
// same weights, mostly from L2.  (With 64 rows only three
// stages fit; that was faster at no size.)
//
// Bound by weight streaming, and for the smallest calls by launch and set-up.
// Measured on one B200 (graph, warm): 1 row, 7168 x 2048 in 6.9 us; 33 rows,
// 4096 x 7168 in 13 us; 32 rows for each of 32 experts, 4096 x 7168 (940 MB of
// weights) in 142 to 147 us = 6.4 to 6.6 TB/s (2 % more without the evict-first
// policy on the weights, 5 % with 128-byte instead of 256-byte L2 promotion).
//
//   warps 0..7   drain: TMEM lane quadrant = warp % 4, weight block = warp / 4;
//                then a token's 256 columns a warp
//   warp 8       TMA producer      warp 9  TMEM owner and MMA issuer
//   warp 10      scales: sa * sb of every token and weight block, a block ahead
// Every wait is bounded; one that runs out sets the error word, and the CTA
// drains its loads, frees its TMEM and leaves.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>

#include "kiwi/ep/quant.cuh"
#include "kiwi/gemm/fp8_detail.cuh"
#include "kiwi/gemm/group_table.cuh"
#include "kiwi/gemm/grouped_gemm.hpp"
#include "kiwi/gemm/tensor_map.hpp"
#include "kiwi/sm100.cuh"

namespace kiwi::gemm::fp8 {

namespace {

constexpr int kThreads = 352;
constexpr int kDrainThreads = 256;

template <int ROWS>
struct Smem {
    // Stages, and TMEM accumulators: the most that fit (with 32 rows, 4 read weights 4 % slower than 5).
    static constexpr int kRing = ROWS <= 32 ? 5 : 4;
    static constexpr int kTmemCols = kRing * 2 * ROWS <= 256 ? 256 : 512;
    static constexpr int kWBytes = kBN * kBK;
    static constexpr int kStageBytes = kWBytes + ROWS * kBK;
    static constexpr int kSumOffset = kRing * kStageBytes;
    static constexpr int kTableOffset = kSumOffset + ROWS * kBN * 4;
    static constexpr int kScaleOffset = kTableOffset + static_cast<int>(round_up(sizeof(GroupTable), 16));
    static constexpr int kBarOffset = kScaleOffset + kRing * 2 * ROWS * 4;
    static constexpr int kBytes = kBarOffset + 256 + 1024;  // barriers, TMEM slot, alignment slack
};
static_assert(Smem<32>::kBytes <= 227 * 1024 && Smem<48>::kBytes <= 227 * 1024, "exceeds the shared-memory limit");

/// f += CTA `rank`'s four sums at the place of `p`.
__device__ __forceinline__ void add4(const float* p, int rank, int split, float* f) {
    const float4 v = split > 1 ? sm100::ld_cluster_f32x4(p, rank) : *reinterpret_cast<const float4*>(p);
    f[0] += v.x;
    f[1] += v.y;
    f[2] += v.z;
    f[3] += v.w;
}

__device__ __forceinline__ void add8(const float* p, int rank, int split, float* f) {
    add4(p, rank, split, f);
    add4(p + 4, rank, split, f + 4);
}

template <int EPI, int ROWS>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_few_rows_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                        const __grid_constant__ Params p, const int split) {
    using S = Smem<ROWS>;
    constexpr int kRing = S::kRing;
    constexpr int kCols = 2 * ROWS;  // TMEM columns of an accumulator
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* s_sum = reinterpret_cast<float*>(smem + S::kSumOffset);  // [token][256]
    GroupTable& table = *reinterpret_cast<GroupTable*>(smem + S::kTableOffset);
    float* s_scale = reinterpret_cast<float*>(smem + S::kScaleOffset);  // [ring][weight block][token]
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBarOffset);
    uint64_t* done = full + kRing;        // a block's MMAs have run and its scales are in shared memory
    uint64_t* drained = done + kRing;
    uint64_t* written = drained + kRing;  // this CTA's sums of a tile are in shared memory
    uint64_t* ready = written + 1;        // every CTA's are
    uint64_t* read = ready + 1;           // every CTA has read what it needs of this one's
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(read + 1);
    __shared__ int s_abort;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int groups = p.a.num_groups;
    const int n_tiles = (p.a.n + kBN - 1) / kBN;
    const int rank = split > 1 ? static_cast<int>(sm100::cluster_ctarank()) : 0;
    const int first_tile = blockIdx.x / split;
    const int tile_step = gridDim.x / split;
    const int kb0 = p.k_blocks * rank / split;  // this CTA's share of K: at least one block
    const int kb1 = p.k_blocks * (rank + 1) / split;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < kRing; ++s) {
            sm100::mbar_init(&full[s], 1);
            sm100::mbar_init(&done[s], 2);
            sm100::mbar_init(&drained[s], kDrainThreads / 32);
        }
        sm100::mbar_init(written, kDrainThreads);
        sm100::mbar_init(ready, split);
        sm100::mbar_init(read, split * (kDrainThreads / 32));
        sm100::fence_mbar_init();
    }
    if (warp == 8 && lane == 0) {
        sm100::tma_prefetch_desc(&tmap_a);
        sm100::tma_prefetch_desc(&tmap_b);
    }
    if (warp == 9) sm100::tmem_alloc(tmem_slot, S::kTmemCols);
    build_group_table(table, p.a.counts, groups, p.a.rows, ROWS, n_tiles, p.error);
    sm100::tc_fence_before();
    __syncthreads();
    if (split > 1) sm100::cluster_sync();  // every CTA's barriers exist before any arrival from another
    sm100::tc_fence_after();
    if (p.a.feeds_next) sm100::grid_launch_dependents();
    if (p.a.follows) sm100::grid_wait_before();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = table.tiles[groups];

    auto next = [](uint32_t& slot, uint32_t& phase) {
        if (++slot == kRing) {
            slot = 0;
            phase ^= 1;
        }
    };
    auto aborted = [&]() { return *reinterpret_cast<volatile int*>(&s_abort) != 0; };
    auto fail = [&]() {
        *reinterpret_cast<volatile int*>(&s_abort) = 1;
        atomicOr(p.error, kGemmTimeout);
    };

    if (warp == 8) {
        if (lane == 0) {
            const uint64_t policy = sm100::l2_evict_first();
            uint32_t issued = 0, stage = 0, phase = 0;
            bool ok = true;
            for (int tile = first_tile; ok && tile < total_tiles && !aborted(); tile += tile_step) {
                int g, mt, nt;
                find_tile(table, groups, n_tiles, tile, g, mt, nt);
                const int row0 = table.off[g] + mt * ROWS;
                const int brow0 = g * p.a.n + nt * kBN;
                for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                    if (!sm100::mbar_wait(&done[stage], phase ^ 1)) {
                        fail();
                        ok = false;
                        break;
                    }
                    uint8_t* sw = smem + stage * S::kStageBytes;
                    sm100::mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
                    sm100::tma_load_2d_hint(sw, &tmap_b, &full[stage], kb * kBK, brow0, policy);
                    sm100::tma_load_2d(sw + S::kWBytes, &tmap_a, &full[stage], kb * kBK, row0);
                    next(stage, phase);
                }
            }
            // No load may still be in flight when this CTA's shared memory goes away.
            for (uint32_t i = issued > kRing ? issued - kRing : 0; i < issued; ++i) {
                if (!sm100::mbar_wait(&full[i % kRing], (i / kRing) & 1)) fail();
            }
        }
    } else if (warp == 9) {
        const uint32_t idesc = sm100::idesc_e4m3_f32(128, ROWS);
        const uint64_t desc0 = sm100::sw128_kmajor_desc(smem);
        const bool issuer = sm100::elect_one();
        uint32_t it = 0, slot = 0, phase = 0;
        bool ok = true;
        for (int tile = first_tile; ok && tile < total_tiles && !aborted(); tile += tile_step) {
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                ok = sm100::mbar_wait(&drained[slot], phase ^ 1) && sm100::mbar_wait(&full[slot], phase);
                if (!ok) {
                    if (issuer) fail();
                    break;
                }
                sm100::tc_fence_after();
                const uint64_t wd = desc0 + slot * (S::kStageBytes >> 4);
                const uint64_t rd = wd + (S::kWBytes >> 4);
                if (issuer) {
#pragma unroll
                    for (int mb = 0; mb < 2; ++mb) {
#pragma unroll
                        for (int kk = 0; kk < kBK / 32; ++kk) {  // 32 bytes of K = 2 descriptor units a step
                            sm100::mma_f8(tmem_base + slot * kCols + mb * ROWS, wd + mb * (128 * kBK >> 4) + 2 * kk,
                                          rd + 2 * kk, idesc, kk != 0 ? 1u : 0u);
                        }
                    }
                    sm100::mma_commit(&done[slot]);
                }
                __syncwarp();
                next(slot, phase);
            }
        }
        // Nor may an MMA still write the TMEM that is freed below.
        if (it > 0 && !sm100::mbar_wait(&done[(it - 1) % kRing], ((it - 1) / kRing) & 1) && issuer) fail();
    } else if (warp == 10) {
        uint32_t slot = 0, phase = 0;
        bool ok = true;
        for (int tile = first_tile; ok && tile < total_tiles && !aborted(); tile += tile_step) {
            int g, mt, nt;
            find_tile(table, groups, n_tiles, tile, g, mt, nt);
            // A lane a token, and with 48 the first 16 lanes another.
            const int64_t row = static_cast<int64_t>(table.off[g]) + mt * ROWS + lane;
            const int64_t last = table.off[g + 1] - 1;  // rows past the group's are not stored: any scale will do
            const float* sa0 = p.a.a_scale + (row < last ? row : last) * p.a.a_scale_stride;
            const float* sa1 = p.a.a_scale + (row + 32 < last ? row + 32 : last) * p.a.a_scale_stride;
            const float* sb0 = p.a.b_scale + (static_cast<int64_t>(g) * p.nb + 2 * nt) * p.k_blocks;
            const float* sb1 = 2 * nt + 1 < p.nb ? sb0 + p.k_blocks : sb0;
            float a0 = ld_a_scale(sa0 + kb0), a1 = ROWS > 32 ? ld_a_scale(sa1 + kb0) : 0.f;
            float b0 = __ldg(sb0 + kb0), b1 = __ldg(sb1 + kb0);
            for (int kb = kb0; kb < kb1; ++kb) {
                const float v00 = a0 * b0, v01 = a0 * b1, v10 = a1 * b0, v11 = a1 * b1;
                if (kb + 1 < kb1) {
                    a0 = ld_a_scale(sa0 + kb + 1);
                    if (ROWS > 32) a1 = ld_a_scale(sa1 + kb + 1);
                    b0 = __ldg(sb0 + kb + 1);
                    b1 = __ldg(sb1 + kb + 1);
                }
                if (!sm100::mbar_wait(&drained[slot], phase ^ 1)) {
                    if (lane == 0) fail();
                    ok = false;
                    break;
                }
                float* to = s_scale + slot * 2 * ROWS + lane;
                if (lane < ROWS) {
                    to[0] = v00;
                    to[ROWS] = v01;
                }
                if (ROWS > 32 && lane + 32 < ROWS) {
                    to[32] = v10;
                    to[ROWS + 32] = v11;
                }
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&done[slot]);
                next(slot, phase);
            }
        }
    } else if (warp < 8) {
        const int q = warp & 3;
        const int mb = warp >> 2;  // weight block: with SwiGLU gate or up
        uint32_t slot = 0, phase = 0;
        uint32_t n_sum = 0;  // tiles whose sums were shared
        bool ok = true;
        for (int tile = first_tile; ok && tile < total_tiles && !aborted(); tile += tile_step, ++n_sum) {
            int g, mt, nt;
            find_tile(table, groups, n_tiles, tile, g, mt, nt);
            const int64_t row0 = static_cast<int64_t>(table.off[g]) + mt * ROWS;
            const int left = table.off[g + 1] - static_cast<int>(row0);
            const int here = left < ROWS ? left : ROWS;  // tokens of this tile
            // Lane t holds token t's factor (and token t + 32's), loaded now and used after the last block.
            const bool scaled = EPI != kEpiSwiGLUQuant && p.a.row_scale;
            const float factor0 = scaled && lane < here ? __ldg(p.a.row_scale + row0 + lane) : 1.0f;
            const float factor1 = ROWS > 32 && scaled && lane + 32 < here ? __ldg(p.a.row_scale + row0 + lane + 32) : 1.0f;
            uint64_t acc[ROWS / 2];
#pragma unroll
            for (int i = 0; i < ROWS / 2; ++i) acc[i] = 0;
#pragma unroll 1
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!sm100::mbar_wait(&done[slot], phase)) {
                    fail();
                    ok = false;
                    break;
                }
                sm100::tc_fence_after();
                const uint32_t taddr =
                    tmem_base + (static_cast<uint32_t>(q * 32) << 16) + slot * kCols + static_cast<uint32_t>(mb * ROWS);
                uint32_t v[ROWS];
                if constexpr (ROWS >= 32) sm100::tmem_issue_32cols(taddr, reinterpret_cast<uint32_t(&)[32]>(v));
                if constexpr (ROWS % 32 != 0) {
                    sm100::tmem_issue_16cols(taddr + ROWS / 32 * 32, reinterpret_cast<uint32_t(&)[16]>(v[ROWS / 32 * 32]));
                    sm100::tmem_wait_16cols(reinterpret_cast<uint32_t(&)[16]>(v[ROWS / 32 * 32]));
                }
                if constexpr (ROWS >= 32) sm100::tmem_wait_32cols(reinterpret_cast<uint32_t(&)[32]>(v));
                const float* sc = s_scale + (slot * 2 + mb) * ROWS;
#pragma unroll
                for (int i = 0; i < ROWS / 4; ++i) {
                    const float4 f = *reinterpret_cast<const float4*>(sc + 4 * i);
                    fma2(acc[2 * i], pack2(v[4 * i], v[4 * i + 1]), pack2(f.x, f.y));
                    fma2(acc[2 * i + 1], pack2(v[4 * i + 2], v[4 * i + 3]), pack2(f.z, f.w));
                }
                sm100::tc_fence_before();
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&drained[slot]);
                next(slot, phase);
            }
            if (!ok) break;
            // Every CTA has read the sums of the tile before this one.
            if (n_sum > 0 && !sm100::mbar_wait_cluster(read, (n_sum - 1) & 1)) {
                fail();
                break;
            }
            float* sums = s_sum + mb * 128 + q * 32 + lane;
#pragma unroll
            for (int i = 0; i < ROWS / 2; ++i) {
                const float2 f = unpack2(acc[i]);
                sums[(2 * i) * kBN] = f.x;
                sums[(2 * i + 1) * kBN] = f.y;
            }
            sm100::mbar_arrive(written);
            if (!sm100::mbar_wait(written, n_sum & 1)) {
                fail();
                break;
            }
            if (split > 1) {
                if (threadIdx.x < static_cast<unsigned>(split)) {
                    sm100::mbar_arrive_cluster(sm100::mapa(ready, threadIdx.x));
                }
                if (!sm100::mbar_wait_cluster(ready, n_sum & 1)) {
                    fail();
                    break;
                }
            }
            for (int t = warp * split + rank; t < here; t += 8 * split) {
                const int64_t row = row0 + t;
                const float scale = __shfl_sync(0xffffffffu, ROWS <= 32 || t < 32 ? factor0 : factor1, t & 31);
                if constexpr (EPI == kEpiStore) {
                    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // columns 8 * lane ..
                    for (int r = 0; r < split; ++r) add8(s_sum + t * kBN + 8 * lane, r, split, f);
                    const int col = nt * kBN + 8 * lane;
                    __nv_bfloat16* dst = p.a.c + row * p.a.ldc + col;
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] *= scale;
                    if (p.a.ldc % 8 == 0 && reinterpret_cast<uintptr_t>(p.a.c) % 16 == 0 && col + 8 <= p.a.n) {
                        *reinterpret_cast<uint4*>(dst) = ep::f32x8_to_bf16(f);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (col + i < p.a.n) dst[i] = __float2bfloat16_rn(f[i]);
                        }
                    }
                } else {
                    float gt[4] = {0.f, 0.f, 0.f, 0.f}, up[4] = {0.f, 0.f, 0.f, 0.f};
                    for (int r = 0; r < split; ++r) {
                        add4(s_sum + t * kBN + 4 * lane, r, split, gt);
                        add4(s_sum + t * kBN + 128 + 4 * lane, r, split, up);
                    }
                    float h[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[i] = silu(gt[i]) * up[i];
                    const int col = nt * (kBN / 2) + 4 * lane;
                    if constexpr (EPI == kEpiSwiGLU) {
                        __nv_bfloat16* dst = p.a.c + row * p.a.ldc + col;
#pragma unroll
                        for (int i = 0; i < 4; ++i) dst[i] = __float2bfloat16_rn(h[i] * scale);
                    } else {
                        float amax = fmaxf(fmaxf(fabsf(h[0]), fabsf(h[1])), fmaxf(fabsf(h[2]), fabsf(h[3])));
#pragma unroll
                        for (int d = 16; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
                        float s, inv;
                        ep::fp8_block_scale(amax, s, inv);
                        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(h[0] * inv, h[1] * inv),
                                                                     __NV_SATFINITE, __NV_E4M3);
                        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(h[2] * inv, h[3] * inv),
                                                                     __NV_SATFINITE, __NV_E4M3);
                        *reinterpret_cast<uint32_t*>(p.a.codes + row * (p.a.n / 2) + col) = lo | (hi << 16);
                        if (lane == 0) p.a.scales[row * (p.a.n / kBN) + nt] = s;
                    }
                }
            }
            __syncwarp();  // this warp has read its tokens' sums
            if (split > 1) {
                if (lane < split) sm100::mbar_arrive_cluster(sm100::mapa(read, lane));
            } else if (lane == 0) {
                sm100::mbar_arrive(read);
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
    if (split > 1) sm100::cluster_sync();  // no CTA leaves while another may read its sums
    sm100::tc_fence_after();
    if (warp == 9) sm100::tmem_dealloc(tmem_base, S::kTmemCols);
}

template <int EPI, int ROWS>
void launch(const Params& p, const CUtensorMap& tb, int split, cudaStream_t stream) {
    static std::atomic<uint64_t> attr{0};
    constexpr int smem = Smem<ROWS>::kBytes;
    raise_smem_limit(reinterpret_cast<const void*>(fp8_few_rows_kernel<EPI, ROWS>), smem, attr);
    const CUtensorMap ta =
        make_tmap_2d(p.a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.a.rows, p.a.k, p.a.lda, ROWS, kBK);
    const int64_t n_tiles = (p.a.n + kBN - 1) / kBN;
    // At most this many tiles, however the rows fall into groups.
    const int64_t most = p.a.counts
                             ? ((p.a.rows + ROWS - 1) / ROWS + (p.a.num_groups < p.a.rows ? p.a.num_groups : p.a.rows)) * n_tiles
                             : (p.a.rows + ROWS - 1) / ROWS * n_tiles;
    const int64_t workers = num_sms() / split;
    launch_kernel(fp8_few_rows_kernel<EPI, ROWS>, static_cast<unsigned>(most < workers ? most : workers) * split, kThreads,
                  smem, split, p.a.follows, stream, ta, tb, p, split);
}

template <int EPI>
void launch_rows(const Params& p, const CUtensorMap& tb, int rows, int split, cudaStream_t stream) {
    if (rows <= 16) launch<EPI, 16>(p, tb, split, stream);
    else if (rows <= 32) launch<EPI, 32>(p, tb, split, stream);
    else launch<EPI, 48>(p, tb, split, stream);
}

}  // namespace

void launch_few_rows(const Params& p, int row_chunk, int split, cudaStream_t stream) {
    if ((split != 1 && split != 2 && split != 4) || split > p.k_blocks) {
        throw kiwi::error("fp8_few_rows: split must be 1, 2 or 4, and at most the blocks of K");
    }
    const CUtensorMap tb =
        make_tmap_2d(p.a.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, static_cast<uint64_t>(p.a.num_groups) * p.a.n, p.a.k,
                     p.a.ldb, kBN, kBK);
    if (!p.a.swiglu) launch_rows<kEpiStore>(p, tb, row_chunk, split, stream);
    else if (!p.a.codes) launch_rows<kEpiSwiGLU>(p, tb, row_chunk, split, stream);
    else launch_rows<kEpiSwiGLUQuant>(p, tb, row_chunk, split, stream);
}

}  // namespace kiwi::gemm::fp8
