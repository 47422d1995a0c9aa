// Host-side helpers of the block-128 product kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace ofld {
namespace kern {

extern std::atomic<uint64_t> g_block128_launches;

// Tensor map of a row-major [rows, cols] matrix with `pitch` bytes a row, read
// in tiles of box_rows x box_cols in the 128-byte swizzle; what lies outside
// reads as 0.
cudaError_t tile_map(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, int64_t cols, int64_t rows,
                     int64_t pitch, uint32_t box_cols, uint32_t box_rows);

// This device's error word: host-mapped, 0 until a bounded wait of a kernel
// runs out. block128_error() returns it without waiting for anything.
cudaError_t error_word(uint32_t** word);

// Opts a kernel into `bytes` of dynamic shared memory, once per device.
cudaError_t allow_smem(const void* fn, uint32_t bytes);

int sm_count();  // of the current device

}  // namespace kern
}  // namespace ofld
