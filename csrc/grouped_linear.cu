// The experts' bf16 product with its gradients on sm_100a tensor cores.
//
//   forward  y[r, :]  = w[g] x[r, :]                  for the rows r of group g
//   dgrad    dx[r, :] = w[g]^T dy[r, :]
//   wgrad    dw[g]    = sum over r of dy[r, :] x[r, :]^T
//
// All three are the same kernel: a pair of SMs computes 256 x 256 tiles with
// 2-SM MMAs, each loading half of both operands.  They differ in which operand
// runs along the contraction in memory:
//
//            M operand               N operand              contraction
//   forward  w   n x k (K)           x   rows x k (K)       k
//   dgrad    w   n x k (MN)          dy  rows x n (K)       n
//   wgrad    dy  rows x n (MN)       x   rows x k (MN)      the group's rows
//
// (K): the contraction is the contiguous dimension; (MN): it is the row.  The
// tensor core takes either from 128-byte-swizzled shared memory, so no operand
// is ever transposed in memory: an MN operand's tile is loaded as boxes of 64
// contraction rows x 64 columns, and its descriptor says so.
//
// forward and dgrad take the group's rows as the N operand because N comes in
// steps of 32: a tile then costs what its rows cost, where M is 128 or 256.  Their
// accumulators have a result column a lane and a row a TMEM column; the epilogue
// turns them in shared memory.
//
// wgrad's contraction ends where the group does, which is anywhere: the last
// 64-row block then also holds rows of the next group, or whatever lies behind
// the last one.  Those rows are zeroed in both operands' tiles before the MMAs
// (zero times a stale infinity would not be zero): each CTA loads such a block
// onto a barrier of its own, clears the rows and arrives at the leader's.  A
// group without rows gets zeros.
//
// Bound where groups are long by the tensor cores and, in long runs, in part by
// the power cap: 1.35 to 1.53 PFLOP/s on even groups of 512 to 2048 rows in bursts
// (0.81 to 0.92 of the measured rate), 1.2 in a long run at 1.15 GHz, where a
// plain library product holds 1.39; wgrad, where groups are short, by writing dw:
// 3.4 to 3.6 TB/s of the 3.95 that a fill reaches.  Measured on one B200, n x k =
// 4096 x 7168, 16384 rows over 32 groups: even groups forward 702 us, dgrad 711,
// wgrad 857; uneven ones (Zipf 0.3) 842, 792, 990, and in a long run of all three
// 2984 together.  128 x 256 tiles on one SM each took 818, 828, 1043 and 3037;
// on 8 uneven groups (2560 x 4096, 6111 rows) 402 where the pairs take 377.
// Accumulators are handed back before the last of a tile is stored, by an
// arrival without a cluster-scope release, which would wait for the stores
// (wgrad at 128 rows a group: 209 -> 131 us).  wgrad's tiles go down the rows of
// dw first; along its columns first they took 5 to 10 % longer.
//
// Kernel shape (clusters of two, persistent): warps 0..7 epilogue (TMEM lane
// quadrant = warp % 4, column half = warp / 4), warp 8 TMA producer, warp 9
// TMEM owner and, in the leader, MMA issuer; 6 stages of 32 KB a CTA; two
// accumulators of 256 columns, so the epilogue of one tile runs under the MMAs
// of the next.  Every wait is bounded; one that runs out sets the error word, and
// the CTA drains its loads, frees its TMEM and leaves.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "kiwi/ep/quant.cuh"
#include "kiwi/gemm/fp8_gemm.hpp"
#include "kiwi/gemm/group_table.cuh"
#include "kiwi/gemm/grouped_gemm.hpp"
#include "kiwi/gemm/grouped_linear.hpp"
#include "kiwi/gemm/row_store.cuh"
#include "kiwi/gemm/tensor_map.hpp"
#include "kiwi/sm100.cuh"

namespace kiwi::gemm {

namespace {

enum Mode : int { kForward = 0, kDgrad = 1, kWgrad = 2 };

constexpr int kBM = 256;  // of the M operand across the pair, 128 a CTA
constexpr int kBN = 256;  // of the N operand, half of it in each CTA
constexpr int kBK = 64;
constexpr int kStages = 6;
constexpr int kThreads = 320;
constexpr int kEpiThreads = 256;
constexpr int kBox = 64 * 64 * 2;  // one 64 x 64 box of an MN operand

struct Smem {
    static constexpr int kOperandBytes = 128 * kBK * 2;  // a CTA's part of either operand
    static constexpr int kStageBytes = 2 * kOperandBytes;
    static constexpr int kTableOffset = kStages * kStageBytes;
    static constexpr int kStgOffset = kTableOffset + static_cast<int>(round_up(sizeof(GroupTable), 16));
    static constexpr int kBarOffset = kStgOffset + kEpiThreads / 32 * kRowStoreBytes;
    static constexpr int kBytes = kBarOffset + 256 + 1024;  // barriers, TMEM slot, alignment slack
};
static_assert(Smem::kBytes <= 227 * 1024, "exceeds the shared-memory limit");

struct Params {
    GroupedLinearArgs a;
    int m_size;    // of one group's M operand: n (forward, wgrad) or k (dgrad)
    int k_blocks;  // forward, dgrad: 64-wide blocks of the contraction
    uint32_t* error;
};

template <int MODE, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_linear_kernel(const __grid_constant__ CUtensorMap tmap_m, const __grid_constant__ CUtensorMap tmap_n,
                          const __grid_constant__ Params p) {
    constexpr bool kMMn = MODE != kForward;  // M operand stored contraction-row by contraction-row
    constexpr bool kNMn = MODE == kWgrad;    // N operand
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    GroupTable& table = *reinterpret_cast<GroupTable*>(smem + Smem::kTableOffset);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Smem::kBarOffset);  // the leader's: both CTAs' loads
    uint64_t* empty = full + kStages;
    uint64_t* tail = empty + kStages;      // wgrad: this CTA's loads of a group's last, partial block
    uint64_t* tmem_full = tail + kStages;
    uint64_t* tmem_empty = tmem_full + 2;  // the leader's: both CTAs' epilogue warps
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
    __shared__ int s_abort;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform: the roles' addresses stay in uniform registers
    const int lane = threadIdx.x & 31;
    const int crank = static_cast<int>(sm100::cluster_ctarank());
    const bool leader = crank == 0;
    const int groups = p.a.num_groups;
    const int m_tiles = (p.m_size + kBM - 1) / kBM;
    const int n_tiles = (p.a.k + kBN - 1) / kBN;  // wgrad

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < kStages; ++s) {
            sm100::mbar_init(&full[s], MODE == kWgrad ? 2 : 1);
            sm100::mbar_init(&empty[s], 1);
            sm100::mbar_init(&tail[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            sm100::mbar_init(&tmem_full[i], 1);
            sm100::mbar_init(&tmem_empty[i], 2 * kEpiThreads / 32);
        }
        sm100::fence_mbar_init();
    }
    if (warp == 8 && lane == 0) {
        sm100::tma_prefetch_desc(&tmap_m);
        sm100::tma_prefetch_desc(&tmap_n);
    }
    if (warp == 9) sm100::tmem_alloc_pair(tmem_slot, 2 * kBN);
    build_group_table(table, p.a.counts, groups, p.a.rows, kBN, m_tiles, p.error);
    sm100::tc_fence_before();
    __syncthreads();
    sm100::cluster_sync();  // both CTAs' barriers exist before any arrival from the other
    sm100::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // forward, dgrad: a group's tiles are blocks of 256 of its rows (nt, innermost:
    // neighbours share a weight tile) times blocks of 256 result columns (mt).
    // wgrad: every group has the same tiles, of a contraction as long as the group.
    const int total_tiles = MODE == kWgrad ? groups * m_tiles * n_tiles : table.tiles[groups];
    const int first_tile = blockIdx.x / 2, tile_step = gridDim.x / 2;
    auto locate = [&](int tile, int& g, int& mt, int& nt) {
        if constexpr (MODE == kWgrad) {
            g = tile / (m_tiles * n_tiles);
            const int local = tile - g * (m_tiles * n_tiles);
            nt = local / m_tiles;
            mt = local - nt * m_tiles;
        } else {
            find_tile(table, groups, m_tiles, tile, g, nt, mt);
        }
    };
    auto blocks_of = [&](int g) {
        return MODE == kWgrad ? (table.off[g + 1] - table.off[g] + kBK - 1) / kBK : p.k_blocks;
    };
    // forward, dgrad: a group's rows are cut into equal blocks of at most 256, in
    // steps of 32 (the N of the MMA), rather than into 256s and a rest: a tile
    // costs what its rows cost, and pairs that stride through tiles of like cost
    // end at like times (forward of 32 uneven groups: 5 % faster).
    auto block_rows = [&](int g) {
        const int c = table.off[g + 1] - table.off[g];
        const int blocks = (c + kBN - 1) / kBN;
        return ((c + blocks - 1) / blocks + 31) / 32 * 32;
    };
    // First row of the N operand's tile within the group, and its extent.
    auto start_of = [&](int g, int nt) { return MODE == kWgrad ? nt * kBN : nt * block_rows(g); };
    auto extent_of = [&](int g, int nt) {
        if constexpr (MODE == kWgrad) return kBN;
        const int size = block_rows(g), left = table.off[g + 1] - table.off[g] - nt * size;
        return left < size ? (left + 31) / 32 * 32 : size;
    };
    // Rows of block kb that are the group's (wgrad; 64 or more: all of them).
    auto rows_of = [&](int g, int kb) { return table.off[g + 1] - table.off[g] - kb * kBK; };

    auto next = [](uint32_t& stage, uint32_t& phase) {
        if (++stage == kStages) {
            stage = 0;
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
            uint32_t issued = 0, stage = 0, phase = 0;
            bool ok = true;
            for (int tile = first_tile; ok && tile < total_tiles && !aborted(); tile += tile_step) {
                int g, mt, nt;
                locate(tile, g, mt, nt);
                const int k_blocks = blocks_of(g);
                const int m0 = mt * kBM + crank * 128;
                const int n0 = MODE == kWgrad ? nt * kBN + crank * 128
                                              : table.off[g] + start_of(g, nt) + crank * (extent_of(g, nt) / 2);
                for (int kb = 0; kb < k_blocks; ++kb, ++issued) {
                    if (!sm100::mbar_wait(&empty[stage], phase ^ 1)) {
                        fail();
                        ok = false;
                        break;
                    }
                    uint8_t* sm = smem + stage * Smem::kStageBytes;
                    uint8_t* sn = sm + Smem::kOperandBytes;
                    const int krow = (MODE == kWgrad ? table.off[g] : g * p.a.n) + kb * kBK;
                    if (MODE == kWgrad && rows_of(g, kb) < kBK) {
                        // This CTA's warp 9 zeroes the rows behind the group's, then tells the leader.
                        sm100::mbar_arrive_expect_tx(&tail[stage], Smem::kStageBytes);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            sm100::tma_load_2d(sm + j * kBox, &tmap_m, &tail[stage], m0 + j * 64, krow);
                            sm100::tma_load_2d(sn + j * kBox, &tmap_n, &tail[stage], n0 + j * 64, krow);
                        }
                    } else {
                        if (leader) {
                            sm100::mbar_arrive_expect_tx(&full[stage], 2 * Smem::kStageBytes);
                            if (MODE == kWgrad) sm100::mbar_arrive(&full[stage]);
                        }
                        const uint32_t bar = sm100::mapa(&full[stage], 0);
                        if constexpr (kMMn) {
                            sm100::tma_load_2d_pair(sm, &tmap_m, bar, m0, krow);
                            sm100::tma_load_2d_pair(sm + kBox, &tmap_m, bar, m0 + 64, krow);
                        } else {
                            sm100::tma_load_2d_pair(sm, &tmap_m, bar, kb * kBK, g * p.a.n + m0);
                        }
                        if constexpr (kNMn) {
                            sm100::tma_load_2d_pair(sn, &tmap_n, bar, n0, krow);
                            sm100::tma_load_2d_pair(sn + kBox, &tmap_n, bar, n0 + 64, krow);
                        } else {
                            sm100::tma_load_2d_pair(sn, &tmap_n, bar, kb * kBK, n0);
                        }
                    }
                    next(stage, phase);
                }
            }
            // No load may still be in flight, and no MMA still at work, when this
            // CTA's shared memory and TMEM go away: a stage is empty once its MMAs
            // are done.
            for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                if (!sm100::mbar_wait(&empty[i % kStages], (i / kStages) & 1)) fail();
            }
        }
    } else if (warp == 9) {
        // The whole warp walks the blocks and one elected lane of the leader issues,
        // so that descriptors and addresses are warp-uniform.
        constexpr uint32_t majors = (kMMn ? sm100::kIdescAMn : 0u) | (kNMn ? sm100::kIdescBMn : 0u);
        const uint64_t m_desc0 = kMMn ? sm100::sw128_mnmajor_desc(smem) : sm100::sw128_kmajor_desc(smem);
        const uint64_t n_desc0 = (kNMn ? sm100::sw128_mnmajor_desc(smem) : sm100::sw128_kmajor_desc(smem)) +
                                 (Smem::kOperandBytes >> 4);
        const bool issuer = sm100::elect_one();
        uint32_t stage = 0, phase = 0, tail_phases = 0;
        uint32_t n_acc = 0;  // accumulators started
        bool ok = true;
        for (int tile = first_tile; ok && tile < total_tiles && !aborted(); tile += tile_step) {
            int g, mt, nt;
            locate(tile, g, mt, nt);
            const int k_blocks = blocks_of(g);
            if (k_blocks == 0) continue;
            const uint32_t acc = n_acc & 1;
            const uint32_t idesc = sm100::idesc_bf16_f32(kBM, extent_of(g, nt)) | majors;
            if (leader) ok = sm100::mbar_wait(&tmem_empty[acc], ((n_acc >> 1) & 1) ^ 1);
            const uint32_t d = tmem_base + acc * kBN;
            for (int kb = 0; ok && kb < k_blocks; ++kb) {
                if constexpr (MODE == kWgrad) {
                    const int left = rows_of(g, kb);
                    if (left < kBK) {
                        // A box row is 128 contiguous bytes (the swizzle permutes within it).
                        ok = sm100::mbar_wait(&tail[stage], (tail_phases >> stage) & 1);
                        if (!ok) break;
                        tail_phases ^= 1u << stage;
                        uint8_t* sm = smem + stage * Smem::kStageBytes;
                        for (int b = 0; b < 4; ++b) {
                            for (int o = left * 128 + lane * 16; o < kBox; o += 512) {
                                *reinterpret_cast<uint4*>(sm + b * kBox + o) = make_uint4(0, 0, 0, 0);
                            }
                        }
                        sm100::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) sm100::mbar_arrive_cluster(sm100::mapa(&full[stage], 0));
                    }
                }
                if (leader) {
                    ok = sm100::mbar_wait_cluster(&full[stage], phase);
                    if (!ok) break;
                    sm100::tc_fence_after();
                    const uint64_t md = m_desc0 + stage * (Smem::kStageBytes >> 4);
                    const uint64_t nd = n_desc0 + stage * (Smem::kStageBytes >> 4);
                    if (issuer) {
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; ++kk) {
                            // 16 of K: 32 bytes along a swizzled row, or 16 rows of 128 bytes.
                            sm100::mma_bf16_pair(d, md + (kMMn ? 128 : 2) * kk, nd + (kNMn ? 128 : 2) * kk, idesc,
                                                 (kb | kk) != 0 ? 1u : 0u);
                        }
                        sm100::mma_commit_both(&empty[stage]);
                        if (kb == k_blocks - 1) sm100::mma_commit_both(&tmem_full[acc]);
                    }
                    __syncwarp();
                }
                next(stage, phase);
            }
            if (!ok && issuer) fail();
            ++n_acc;
        }
    } else {
        const int q = warp & 3;
        const int half = warp >> 2;
        T* const out = static_cast<T*>(p.a.out);
        uint8_t* stg = smem + Smem::kStgOffset + warp * kRowStoreBytes;
        uint32_t n_acc = 0;
        for (int tile = first_tile; tile < total_tiles && !aborted(); tile += tile_step) {
            int g, mt, nt;
            locate(tile, g, mt, nt);
            const bool have = blocks_of(g) != 0;
            const uint32_t acc = n_acc & 1;
            if (have && !sm100::mbar_wait(&tmem_full[acc], (n_acc >> 1) & 1)) {
                fail();
                break;
            }
            sm100::tc_fence_after();
            const uint32_t taddr =
                tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * kBN + static_cast<uint32_t>(half * 128);
            const int m = mt * kBM + crank * 128 + q * 32;  // of this warp's lane 0
            // Called once the warp has read its part of the accumulator, before the
            // last of it is stored: the next tile's MMAs do not wait for stores.
            auto release = [&]() {
                sm100::tc_fence_before();
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive_remote(sm100::mapa(&tmem_empty[acc], 0));
            };
            if constexpr (MODE != kWgrad) {
                // Lanes are result columns, accumulator columns are rows of the group.
                const int at = start_of(g, nt) + half * 128;
                const int64_t r0 = static_cast<int64_t>(table.off[g]) + at;
                const int end = min(table.off[g + 1] - table.off[g], start_of(g, nt) + block_rows(g));
                const int rows = end - at < 128 ? end - at : 128;
                if (rows <= 0) release();
#pragma unroll 1
                for (int c = 0; c < rows; c += 32) {
                    float v[32];
                    sm100::tmem_ld_32cols(taddr + c, v);
                    if (c + 32 >= rows) release();
                    if (m < p.m_size) {
                        store_columns32(stg, v, out + (r0 + c) * p.a.ldo + m, p.a.ldo, rows - c < 32 ? rows - c : 32);
                    }
                }
            } else {
                const int n0 = nt * kBN + half * 128;
                const int cols = p.a.k - n0 < 128 ? p.a.k - n0 : 128;
                if (have && cols <= 0) release();
                // A group without rows has a zero gradient, or adds nothing.
                const bool store = m < p.m_size && (have || !p.a.accumulate);
#pragma unroll 1
                for (int c = 0; c < cols; c += 32) {
                    float v[32];
                    if (have) {
                        sm100::tmem_ld_32cols(taddr + c, v);
                        if (c + 32 >= cols) release();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0.f;
                    }
                    if (!store) continue;
                    T* dst = out + (static_cast<int64_t>(g) * p.m_size + m) * p.a.ldo + n0 + c;
                    if (sizeof(T) == 2 && !p.a.accumulate) {
                        uint4 w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float f[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) f[i] = v[8 * j + i];
                            w[j] = ep::f32x8_to_bf16(f);
                        }
                        store_rows64(stg, w, reinterpret_cast<uint8_t*>(dst), p.a.ldo * 2, 32, 64, true);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint4 w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float* f = v + 16 * h + 4 * j;
                                w[j] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                                  __float_as_uint(f[3]));
                            }
                            if (p.a.accumulate) add_rows16(stg, w, dst + 16 * h, p.a.ldo, 32);
                            else store_rows64(stg, w, reinterpret_cast<uint8_t*>(dst + 16 * h), p.a.ldo * sizeof(T), 32, 64, true);
                        }
                    }
                }
            }
            if (have) ++n_acc;
        }
        if (MODE != kWgrad && p.a.zero_tail) {
            for (int64_t r = table.off[groups] + static_cast<int64_t>(blockIdx.x); r < p.a.rows; r += gridDim.x) {
                for (int c = threadIdx.x * 8; c < p.m_size; c += kEpiThreads * 8) {
                    *reinterpret_cast<uint4*>(out + r * p.a.ldo + c) = make_uint4(0, 0, 0, 0);
                }
            }
        }
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::cluster_sync();  // neither CTA leaves while the other may touch its barriers
    sm100::tc_fence_after();
    if (warp == 9) sm100::tmem_dealloc_pair(tmem_base, 2 * kBN);
}

CUtensorMap bf16_map(const __nv_bfloat16* ptr, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    return make_tmap_2d(ptr, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, cols, ld * 2, box_rows, kBK);
}

void check(const GroupedLinearArgs& a, int out_bytes) {
    if (a.num_groups < 1 || a.num_groups > kMaxGroups) throw kiwi::error("grouped_linear: 1..1024 groups");
    if (a.n < 64 || a.n % 64 || a.k < 64 || a.k % 64) throw kiwi::error("grouped_linear: N and K must be multiples of 64");
    if (a.k > INT32_MAX - 256) throw kiwi::error("grouped_linear: K must be below 2^31 - 256");
    if (!a.counts || (!a.out && a.rows > 0)) throw kiwi::error("grouped_linear: counts and out are required");
    if (a.rows < 0 || a.rows > INT32_MAX - 256 || static_cast<int64_t>(a.num_groups) * a.n > INT32_MAX - 256) {
        throw kiwi::error("grouped_linear: more than 2^31 rows");
    }
    if (a.ldo * out_bytes % 16 || reinterpret_cast<uintptr_t>(a.out) % 16) {
        throw kiwi::error("grouped_linear: the result's rows must start on 16-byte boundaries");
    }
}

template <int MODE, typename T>
void launch(const CUtensorMap& tm, const CUtensorMap& tn, const Params& p, int64_t most_tiles, cudaStream_t stream) {
    static std::atomic<uint64_t> attr{0};
    raise_smem_limit(reinterpret_cast<const void*>(grouped_linear_kernel<MODE, T>), Smem::kBytes, attr);
    const int64_t pairs = num_sms() / 2;
    if (pairs < 1) throw kiwi::error("grouped_linear: needs at least two SMs");
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim = {2, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * static_cast<unsigned>(most_tiles < pairs ? most_tiles : pairs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem::kBytes;
    cfg.stream = stream;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    KIWI_CUDA_CHECK(cudaLaunchKernelEx(&cfg, grouped_linear_kernel<MODE, T>, tm, tn, p));
}

int64_t most_row_blocks(const GroupedLinearArgs& a) {
    return (a.rows + kBN - 1) / kBN + (a.num_groups < a.rows ? a.num_groups : a.rows);
}

}  // namespace

void grouped_linear_forward(const GroupedLinearArgs& a, cudaStream_t stream) {
    check(a, 2);
    if (a.rows == 0) return;
    Params p{a, a.n, a.k / kBK, gemm_error_word()};
    launch<kForward, __nv_bfloat16>(bf16_map(a.w, static_cast<int64_t>(a.num_groups) * a.n, a.k, a.ldw, 128),
                                    bf16_map(a.x, a.rows, a.k, a.ldx, 128), p,
                                    most_row_blocks(a) * ((a.n + kBM - 1) / kBM), stream);
}

void grouped_linear_dgrad(const GroupedLinearArgs& a, cudaStream_t stream) {
    check(a, 2);
    if (a.rows == 0) return;
    Params p{a, a.k, a.n / kBK, gemm_error_word()};
    launch<kDgrad, __nv_bfloat16>(bf16_map(a.w, static_cast<int64_t>(a.num_groups) * a.n, a.k, a.ldw, 64),
                                  bf16_map(a.dy, a.rows, a.n, a.lddy, 128), p,
                                  most_row_blocks(a) * ((a.k + kBM - 1) / kBM), stream);
}

void grouped_linear_wgrad(const GroupedLinearArgs& a, cudaStream_t stream) {
    check(a, a.out_fp32 ? 4 : 2);
    Params p{a, a.n, 0, gemm_error_word()};
    const int64_t tiles = static_cast<int64_t>(a.num_groups) * ((a.n + kBM - 1) / kBM) * ((a.k + kBN - 1) / kBN);
    if (tiles > INT32_MAX) throw kiwi::error("grouped_linear: result too large");
    if (a.rows == 0) {  // no contraction and no rows that a tensor map could describe
        const size_t elem = a.out_fp32 ? 4 : 2;
        if (!a.accumulate) {
            KIWI_CUDA_CHECK(cudaMemset2DAsync(a.out, a.ldo * elem, 0, a.k * elem,
                                              static_cast<size_t>(a.num_groups) * a.n, stream));
        }
        return;
    }
    const CUtensorMap tm = bf16_map(a.dy, a.rows, a.n, a.lddy, 64), tn = bf16_map(a.x, a.rows, a.k, a.ldx, 64);
    if (a.out_fp32) launch<kWgrad, float>(tm, tn, p, tiles, stream);
    else launch<kWgrad, __nv_bfloat16>(tm, tn, p, tiles, stream);
}

}  // namespace kiwi::gemm
