// Host-side helpers of the block-128 product kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace ofld {
namespace kern {

extern std::atomic<uint64_t> g_block128_launches;

constexpr int64_t kMostPitch = int64_t(1) << 40;  // bytes: a tensor map's pitch is below this

// Tensor map of a row-major [rows, cols] matrix with `pitch` bytes a row, read
// in tiles of box_rows x box_cols in a swizzle of 128, 64 or 0
// bytes; what lies outside reads as 0.
cudaError_t tile_map(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, int64_t cols, int64_t rows,
                     int64_t pitch, uint32_t box_cols, uint32_t box_rows, int swizzle = 128);

// This device's error word: host-mapped, 0 until a bounded wait of a kernel
// runs out. block128_error() returns it without waiting for anything.
cudaError_t error_word(uint32_t** word);

// Opts a kernel into `bytes` of dynamic shared memory, once per device.
cudaError_t allow_smem(const void* fn, uint32_t bytes);

int sm_count();  // of the current device

// Power-of-two scales as the product kernel wants its column side's: e8m0 in
// byte 0 of a word, the words of a tile's rows (and of each 128 of them: row
// 32 j + i at word 4 i + j) together for each block of the sum.
struct TileScales {
    uint32_t* words = nullptr;
    uint32_t rows = 0;    // of a tile
    uint32_t stride = 0;  // words of a tile and block: rows rounded up to 128
    __host__ __device__ uint64_t at(uint32_t row, uint32_t block, uint32_t nb) const {
        const uint32_t t = row / rows, r = row - t * rows, g = r & 127;
        return (uint64_t(t) * nb + block) * stride + (r & ~127u) + (g & 31) * 4 + (g >> 5);
    }
};

// quantize_block128 that also writes the scales for tiles; out.scales may be null.
struct MatIn;
struct Block128Out;
enum class FloatType : int;
cudaError_t quantize_for_tiles(MatIn x, FloatType type, Block128Out out, TileScales tiles, int64_t rows, int64_t cols,
                               cudaStream_t s);

}  // namespace kern
}  // namespace ofld
