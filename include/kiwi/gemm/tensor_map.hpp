// Tensor maps and launch attributes shared by the products' host sides.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace kiwi::gemm {

/// Tensor map of a row-major [rows, cols] matrix of `elem`-byte elements with a
/// row stride of `ld_bytes`, box [box_rows, box_cols], swizzled over the box
/// rows' 128 or 64 bytes.  Base and row stride are multiples of 16 bytes; what a
/// box covers outside the matrix reads as zero.
CUtensorMap make_tmap_2d(const void* ptr, CUtensorMapDataType type, int elem, uint64_t rows, uint64_t cols,
                         uint64_t ld_bytes, uint32_t box_rows, uint32_t box_cols);

/// Raises a kernel's dynamic shared-memory limit on the current device, once:
/// `done` keeps one bit per device.
void raise_smem_limit(const void* kernel, int smem, std::atomic<uint64_t>& done);

}  // namespace kiwi::gemm
