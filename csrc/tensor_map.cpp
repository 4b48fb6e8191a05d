// Tensor maps and launch attributes shared by the products' host sides.
#include "kiwi/gemm/tensor_map.hpp"

#include <mutex>

#include "kiwi/common.hpp"
#include "kiwi/p2p/driver.hpp"

namespace kiwi::gemm {

CUtensorMap make_tmap_2d(const void* ptr, CUtensorMapDataType type, int elem, uint64_t rows, uint64_t cols,
                         uint64_t ld_bytes, uint32_t box_rows, uint32_t box_cols) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q{};
        KIWI_CUDA_CHECK(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !fn) throw kiwi::error("cuTensorMapEncodeTiled unavailable");
        encode = reinterpret_cast<Encode>(fn);
    });
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0 || ld_bytes % 16 != 0) {
        throw kiwi::error("make_tmap_2d: base and row stride must be multiples of 16 bytes");
    }
    const uint32_t box_bytes = box_cols * static_cast<uint32_t>(elem);
    if (box_bytes != 128 && box_bytes != 64) throw kiwi::error("make_tmap_2d: box rows must be 128 or 64 bytes");
    // A thread that has made no runtime call yet, such as autograd's worker, has
    // no current context, and the driver call below does not bind one.
    static thread_local bool bound = false;
    if (!bound) {
        int dev = 0;
        KIWI_CUDA_CHECK(cudaGetDevice(&dev));
        KIWI_CUDA_CHECK(cudaSetDevice(dev));
        bound = true;
    }
    CUtensorMap m;
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {ld_bytes};
    const cuuint32_t box[2] = {box_cols, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode(&m, type, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE,
                              box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    p2p::check_cu(r, "cuTensorMapEncodeTiled");
    return m;
}

void raise_smem_limit(const void* kernel, int smem, std::atomic<uint64_t>& done) {
    int dev = 0;
    KIWI_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) throw kiwi::error("device index beyond 64");
    const uint64_t bit = 1ull << dev;
    if (done.load(std::memory_order_acquire) & bit) return;
    KIWI_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done.fetch_or(bit, std::memory_order_acq_rel);
}

}  // namespace kiwi::gemm
