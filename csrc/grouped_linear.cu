// The experts' bf16 product with its gradients on sm_100a tensor cores.
//
//   forward  y[r, :]  = w[g] x[r, :]                  for the rows r of group g
//   dgrad    dx[r, :] = w[g]^T dy[r, :]
//   wgrad    dw[g]    = sum over r of dy[r, :] x[r, :]^T
//
// All three are the same kernel over 128 x 256 tiles of the result; they differ
// in which operand runs along the contraction in memory:
//
//            M operand            N operand            contraction
//   forward  x   rows x k (K)     w   n x k (K)        k
//   dgrad    dy  rows x n (K)     w   n x k (MN)       n
//   wgrad    dy  rows x n (MN)    x   rows x k (MN)    the group's rows
//
// (K): the contraction is the contiguous dimension; (MN): it is the row.  The
// tensor core takes either from 128-byte-swizzled shared memory, so no operand
// is ever transposed in memory: an MN operand's tile is loaded as boxes of 64
// contraction rows x 64 columns, and its descriptor says so.
//
// wgrad's contraction ends where the group does, which is anywhere: the last
// 64-row block then also holds rows of the next group, or whatever lies behind
// the last one.  The MMA warp zeroes those rows in both operands' tiles before
// it issues (zero times a stale infinity would not be zero); a group without
// rows gets zeros.
//
// Bound by the power cap where groups are long (1.15 to 1.19 PFLOP/s at 1.25 to
// 1.5 GHz; the tensor pipe is active 75 % of the time), and in wgrad by writing
// dw where they are short: 3.2 TB/s of the 3.95 that a fill reaches.  Measured on
// one B200, 16384 rows over 32 groups, n x k = 4096 x 7168: forward 811 us, dgrad
// 820, wgrad 1046; 4 groups of 4096 rows: wgrad at 1.35 PFLOP/s.  The epilogue
// stores through shared memory: with 16-byte pieces of 32 rows a store, wgrad
// took 1772 us.  wgrad's tiles go down the rows of dw first; along its columns
// first they took 5 to 10 % longer.
//
// Kernel shape (one CTA per SM, persistent): warps 0..7 epilogue (TMEM lane
// quadrant = warp % 4, column half = warp / 4), warp 8 TMA producer, warp 9
// TMEM owner and MMA issuer; 4 stages of 48 KB; two accumulators of 256 columns,
// so the epilogue of one tile runs under the MMAs of the next.  Every wait is
// bounded; one that runs out sets the error word, and the CTA drains its loads,
// frees its TMEM and leaves.
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

constexpr int kBM = 128;
constexpr int kBN = 256;
constexpr int kBK = 64;
constexpr int kStages = 4;
constexpr int kThreads = 320;
constexpr int kEpiThreads = 256;
constexpr int kBox = 64 * 64 * 2;  // one 64 x 64 box of an MN operand

struct Smem {
    static constexpr int kABytes = kBM * kBK * 2;
    static constexpr int kBBytes = kBN * kBK * 2;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kTableOffset = kStages * kStageBytes;
    static constexpr int kStgOffset = kTableOffset + static_cast<int>(round_up(sizeof(GroupTable), 16));
    static constexpr int kBarOffset = kStgOffset + kEpiThreads / 32 * kRowStoreBytes;
    static constexpr int kBytes = kBarOffset + 256 + 1024;  // barriers, TMEM slot, alignment slack
};
static_assert(Smem::kBytes <= 227 * 1024, "exceeds the shared-memory limit");

struct Params {
    GroupedLinearArgs a;
    int m_cols;   // wgrad: rows of one group's result (n)
    int n_cols;   // columns of the result
    int k_blocks; // forward, dgrad: 64-wide blocks of the contraction
    uint32_t* error;
};

template <int MODE, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_linear_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                          const __grid_constant__ Params p) {
    constexpr bool kAMn = MODE == kWgrad;    // M operand stored contraction-row by contraction-row
    constexpr bool kBMn = MODE != kForward;  // N operand
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    GroupTable& table = *reinterpret_cast<GroupTable*>(smem + Smem::kTableOffset);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Smem::kBarOffset);
    uint64_t* empty = full + kStages;
    uint64_t* tmem_full = empty + kStages;
    uint64_t* tmem_empty = tmem_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
    __shared__ int s_abort;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform: the roles' addresses stay in uniform registers
    const int lane = threadIdx.x & 31;
    const int groups = p.a.num_groups;
    const int n_tiles = (p.n_cols + kBN - 1) / kBN;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < kStages; ++s) {
            sm100::mbar_init(&full[s], 1);
            sm100::mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            sm100::mbar_init(&tmem_full[i], 1);
            sm100::mbar_init(&tmem_empty[i], kEpiThreads / 32);
        }
        sm100::fence_mbar_init();
    }
    if (warp == 8 && lane == 0) {
        sm100::tma_prefetch_desc(&tmap_a);
        sm100::tma_prefetch_desc(&tmap_b);
    }
    if (warp == 9) sm100::tmem_alloc(tmem_slot, 2 * kBN);
    build_group_table(table, p.a.counts, groups, p.a.rows, kBM, n_tiles, p.error);
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // wgrad: every group has the same tiles, of a contraction as long as the group.
    const int m_tiles = (p.m_cols + kBM - 1) / kBM;
    const int total_tiles = MODE == kWgrad ? groups * m_tiles * n_tiles : table.tiles[groups];
    auto locate = [&](int tile, int& g, int& mt, int& nt) {
        if constexpr (MODE == kWgrad) {
            g = tile / (m_tiles * n_tiles);
            const int local = tile - g * (m_tiles * n_tiles);
            nt = local / m_tiles;
            mt = local - nt * m_tiles;
        } else {
            find_tile(table, groups, n_tiles, tile, g, mt, nt);
        }
    };
    auto blocks_of = [&](int g) {
        return MODE == kWgrad ? (table.off[g + 1] - table.off[g] + kBK - 1) / kBK : p.k_blocks;
    };

    // A tile with at most 64 rows of its group left runs M = 64 MMAs: half the
    // tensor work, the same sums.  Its row 16 q + i is in TMEM lane 32 q + i.
    auto half_tile = [&](int g, int mt) {
        return MODE != kWgrad && table.off[g + 1] - table.off[g] - mt * kBM <= 64;
    };

    auto aborted = [&]() { return *reinterpret_cast<volatile int*>(&s_abort) != 0; };
    auto fail = [&]() {
        *reinterpret_cast<volatile int*>(&s_abort) = 1;
        atomicOr(p.error, kGemmTimeout);
    };

    if (warp == 8) {
        if (lane == 0) {
            uint32_t issued = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < total_tiles && !aborted(); tile += gridDim.x) {
                int g, mt, nt;
                locate(tile, g, mt, nt);
                const int k_blocks = blocks_of(g);
                const int row0 = table.off[g];
                for (int kb = 0; kb < k_blocks; ++kb) {
                    const uint32_t stage = issued % kStages;
                    if (!sm100::mbar_wait(&empty[stage], ((issued / kStages) & 1) ^ 1)) {
                        fail();
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + stage * Smem::kStageBytes;
                    uint8_t* sb = sa + Smem::kABytes;
                    sm100::mbar_arrive_expect_tx(&full[stage], Smem::kStageBytes);
                    if constexpr (kAMn) {
#pragma unroll
                        for (int j = 0; j < kBM / 64; ++j) {
                            sm100::tma_load_2d(sa + j * kBox, &tmap_a, &full[stage], mt * kBM + j * 64, row0 + kb * kBK);
                        }
                    } else {
                        sm100::tma_load_2d(sa, &tmap_a, &full[stage], kb * kBK, row0 + mt * kBM);
                    }
                    if constexpr (kBMn) {
                        const int krow = MODE == kWgrad ? row0 + kb * kBK : g * p.a.n + kb * kBK;
#pragma unroll
                        for (int j = 0; j < kBN / 64; ++j) {
                            sm100::tma_load_2d(sb + j * kBox, &tmap_b, &full[stage], nt * kBN + j * 64, krow);
                        }
                    } else {
                        sm100::tma_load_2d(sb, &tmap_b, &full[stage], kb * kBK, g * p.a.n + nt * kBN);
                    }
                    ++issued;
                }
            }
            // No load may still be in flight when this CTA's shared memory goes away.
            for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                if (!sm100::mbar_wait(&full[i % kStages], (i / kStages) & 1)) fail();
            }
        }
    } else if (warp == 9) {
        // The whole warp walks the blocks and one elected lane issues, so that
        // descriptors and addresses are warp-uniform.
        constexpr uint32_t majors = (kAMn ? sm100::kIdescAMn : 0u) | (kBMn ? sm100::kIdescBMn : 0u);
        const uint64_t a_desc0 = kAMn ? sm100::sw128_mnmajor_desc(smem) : sm100::sw128_kmajor_desc(smem);
        const uint64_t b_desc0 = (kBMn ? sm100::sw128_mnmajor_desc(smem) : sm100::sw128_kmajor_desc(smem)) +
                                 (Smem::kABytes >> 4);
        const bool issuer = sm100::elect_one();
        uint32_t it = 0, stage = 0, phase = 0;
        uint32_t n_acc = 0;  // accumulators started
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < total_tiles && !aborted(); tile += gridDim.x) {
            int g, mt, nt;
            locate(tile, g, mt, nt);
            const int k_blocks = blocks_of(g);
            if (k_blocks == 0) continue;
            const uint32_t acc = n_acc & 1;
            const uint32_t idesc =
                (half_tile(g, mt) ? sm100::idesc_bf16_f32(64, kBN) : sm100::idesc_bf16_f32(kBM, kBN)) | majors;
            ok = sm100::mbar_wait(&tmem_empty[acc], ((n_acc >> 1) & 1) ^ 1);
            const uint32_t d = tmem_base + acc * kBN;
            for (int kb = 0; ok && kb < k_blocks; ++kb, ++it) {
                ok = sm100::mbar_wait(&full[stage], phase);
                if (!ok) break;
                if constexpr (MODE == kWgrad) {
                    const int left = table.off[g + 1] - table.off[g] - kb * kBK;
                    if (left < kBK) {
                        // Rows past the group's: a box row is 128 contiguous bytes
                        // (the swizzle permutes within it).
                        uint8_t* sa = smem + stage * Smem::kStageBytes;
                        for (int b = 0; b < (kBM + kBN) / 64; ++b) {
                            for (int o = left * 128 + lane * 16; o < kBox; o += 512) {
                                *reinterpret_cast<uint4*>(sa + b * kBox + o) = make_uint4(0, 0, 0, 0);
                            }
                        }
                        sm100::fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                sm100::tc_fence_after();
                const uint64_t ad = a_desc0 + stage * (Smem::kStageBytes >> 4);
                const uint64_t bd = b_desc0 + stage * (Smem::kStageBytes >> 4);
                if (issuer) {
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk) {
                        // 16 of K: 32 bytes along a swizzled row, or 16 rows of 128 bytes.
                        sm100::mma_bf16(d, ad + (kAMn ? 128 : 2) * kk, bd + (kBMn ? 128 : 2) * kk, idesc,
                                        (kb | kk) != 0 ? 1u : 0u);
                    }
                    sm100::mma_commit(&empty[stage]);
                    if (kb == k_blocks - 1) sm100::mma_commit(&tmem_full[acc]);
                }
                __syncwarp();
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok && issuer) fail();
            ++n_acc;
        }
        // Nor may an MMA still write the TMEM that is freed below.
        if (it > 0 && !sm100::mbar_wait(&empty[(it - 1) % kStages], ((it - 1) / kStages) & 1) && issuer) fail();
    } else {
        const int q = warp & 3;
        const int half = warp >> 2;
        T* const out = static_cast<T*>(p.a.out);
        uint8_t* stg = smem + Smem::kStgOffset + warp * kRowStoreBytes;
        uint32_t n_acc = 0;
        for (int tile = blockIdx.x; tile < total_tiles && !aborted(); tile += gridDim.x) {
            int g, mt, nt;
            locate(tile, g, mt, nt);
            // The warp's rows: r0 + lane, `rows` of them in the result.
            const int span = half_tile(g, mt) ? 16 : 32;
            const int64_t r0 = (MODE == kWgrad ? static_cast<int64_t>(g) * p.m_cols : table.off[g]) + mt * kBM + q * span;
            const int64_t r_end = MODE == kWgrad ? static_cast<int64_t>(g + 1) * p.m_cols : table.off[g + 1];
            const int rows = static_cast<int>(r_end - r0 < span ? r_end - r0 : span);
            const int col0 = nt * kBN + half * (kBN / 2);
            const int cols = p.n_cols - col0;  // a multiple of 64
            const bool have = blocks_of(g) != 0;
            const uint32_t acc = n_acc & 1;
            if (have && !sm100::mbar_wait(&tmem_full[acc], (n_acc >> 1) & 1)) {
                fail();
                break;
            }
            sm100::tc_fence_after();
            const uint32_t taddr =
                tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * kBN + static_cast<uint32_t>(half * (kBN / 2));
            // A group without rows has a zero gradient, or adds nothing.
            const bool store = rows > 0 && (have || !p.a.accumulate);
#pragma unroll 1
            for (int c = 0; c < kBN / 2 && c < cols; c += 32) {
                float v[32];
                if (have) {
                    sm100::tmem_ld_32cols(taddr + c, v);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.f;
                }
                if (!store) continue;
                T* dst = out + r0 * p.a.ldo + col0 + c;
                if (sizeof(T) == 2 && !(MODE == kWgrad && p.a.accumulate)) {
                    uint4 w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float f[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = v[8 * j + i];
                        w[j] = ep::f32x8_to_bf16(f);
                    }
                    store_rows64(stg, w, reinterpret_cast<uint8_t*>(dst), p.a.ldo * 2, rows, 64, true);
                } else if constexpr (MODE == kWgrad) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint4 w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float* f = v + 16 * h + 4 * j;
                            w[j] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                              __float_as_uint(f[3]));
                        }
                        if (p.a.accumulate) add_rows16(stg, w, dst + 16 * h, p.a.ldo, rows);
                        else store_rows64(stg, w, reinterpret_cast<uint8_t*>(dst + 16 * h), p.a.ldo * sizeof(T), rows, 64, true);
                    }
                }
            }
            if (have) {
                sm100::tc_fence_before();
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&tmem_empty[acc]);
                ++n_acc;
            }
        }
        if (MODE != kWgrad && p.a.zero_tail) {
            for (int64_t r = table.off[groups] + static_cast<int64_t>(blockIdx.x); r < p.a.rows; r += gridDim.x) {
                for (int c = threadIdx.x * 8; c < p.n_cols; c += kEpiThreads * 8) {
                    *reinterpret_cast<uint4*>(out + r * p.a.ldo + c) = make_uint4(0, 0, 0, 0);
                }
            }
        }
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    if (warp == 9) sm100::tmem_dealloc(tmem_base, 2 * kBN);
}

CUtensorMap bf16_map(const __nv_bfloat16* ptr, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    return make_tmap_2d(ptr, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, cols, ld * 2, box_rows, kBK);
}

void check(const GroupedLinearArgs& a) {
    if (a.num_groups < 1 || a.num_groups > kMaxGroups) throw kiwi::error("grouped_linear: 1..1024 groups");
    if (a.n < 64 || a.n % 64 || a.k < 64 || a.k % 64) throw kiwi::error("grouped_linear: N and K must be multiples of 64");
    if (!a.counts) throw kiwi::error("grouped_linear: counts are required");
    if (a.rows < 0 || a.rows > INT32_MAX - 256 || static_cast<int64_t>(a.num_groups) * a.n > INT32_MAX - 256) {
        throw kiwi::error("grouped_linear: more than 2^31 rows");
    }
    if (a.ldo % 8 || reinterpret_cast<uintptr_t>(a.out) % 16) {
        throw kiwi::error("grouped_linear: the result's rows must start on 16-byte boundaries");
    }
}

template <int MODE, typename T>
void launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int64_t most_tiles, cudaStream_t stream) {
    static std::atomic<uint64_t> attr{0};
    raise_smem_limit(reinterpret_cast<const void*>(grouped_linear_kernel<MODE, T>), Smem::kBytes, attr);
    const int sms = num_sms();
    const int grid = static_cast<int>(most_tiles < sms ? most_tiles : sms);
    grouped_linear_kernel<MODE, T><<<grid, kThreads, Smem::kBytes, stream>>>(ta, tb, p);
    KIWI_CUDA_CHECK(cudaGetLastError());
}

int64_t most_row_tiles(const GroupedLinearArgs& a) { return (a.rows + kBM - 1) / kBM + a.num_groups; }

}  // namespace

void grouped_linear_forward(const GroupedLinearArgs& a, cudaStream_t stream) {
    check(a);
    if (a.rows == 0) return;
    Params p{a, 0, a.n, a.k / kBK, gemm_error_word()};
    launch<kForward, __nv_bfloat16>(bf16_map(a.x, a.rows, a.k, a.ldx, kBM),
                                    bf16_map(a.w, static_cast<int64_t>(a.num_groups) * a.n, a.k, a.ldw, kBN), p,
                                    most_row_tiles(a) * ((a.n + kBN - 1) / kBN), stream);
}

void grouped_linear_dgrad(const GroupedLinearArgs& a, cudaStream_t stream) {
    check(a);
    if (a.rows == 0) return;
    Params p{a, 0, a.k, a.n / kBK, gemm_error_word()};
    launch<kDgrad, __nv_bfloat16>(bf16_map(a.dy, a.rows, a.n, a.lddy, kBM),
                                  bf16_map(a.w, static_cast<int64_t>(a.num_groups) * a.n, a.k, a.ldw, 64), p,
                                  most_row_tiles(a) * ((a.k + kBN - 1) / kBN), stream);
}

void grouped_linear_wgrad(const GroupedLinearArgs& a, cudaStream_t stream) {
    check(a);
    Params p{a, a.n, a.k, 0, gemm_error_word()};
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
    const CUtensorMap ta = bf16_map(a.dy, a.rows, a.n, a.lddy, 64), tb = bf16_map(a.x, a.rows, a.k, a.ldx, 64);
    if (a.out_fp32) launch<kWgrad, float>(ta, tb, p, tiles, stream);
    else launch<kWgrad, __nv_bfloat16>(ta, tb, p, tiles, stream);
}

}  // namespace kiwi::gemm
