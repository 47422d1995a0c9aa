// Operators on block-128 fp8 tensors.
//
// A block-128 tensor is a pair (q, scales): q e4m3 [rows, cols] with a row
// pitch that is a multiple of 16 bytes from a 16-byte aligned base, scales
// fp32 [rows, ceil(cols / 128)] without gaps. Element (r, c) stands for
// q[r, c] * scales[r, c / 128]. The weights that restore_cast and push write
// (scale amax / 448) have this form when cols is a multiple of 128;
// quantize_block128 writes power-of-two scales.
//
// Every launcher checks pointers, pitches and sizes on the host and returns
// cudaErrorInvalidValue without launching when they do not fit; all launches
// go on the caller's stream and none allocate memory.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace ofld {
namespace kern {

enum class FloatType : int { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

// A row-major matrix: element (r, c) at ptr + r * ld + c (ld in elements).
struct MatIn {
    const void* ptr;
    int64_t ld;
};
struct MatOut {
    void* ptr;
    int64_t ld;
};
struct Block128In {
    const void* q;
    int64_t ld;  // bytes
    const float* scales;
};
struct Block128Out {
    void* q;
    int64_t ld;
    float* scales;
};

cudaError_t quantize_block128(MatIn x, FloatType type, Block128Out out, int64_t rows, int64_t cols, cudaStream_t s);
cudaError_t dequantize_block128(Block128In in, MatOut x, FloatType type, int64_t rows, int64_t cols, cudaStream_t s);

// h = silu(gate) * up; gate and up are also kept as block-128 tensors.
cudaError_t swiglu_forward(MatIn gate, MatIn up, FloatType type, MatOut h, Block128Out kept_gate,
                           Block128Out kept_up, int64_t rows, int64_t cols, cudaStream_t s);
// Gradients at the kept values.
cudaError_t swiglu_backward(MatIn dh, FloatType type, Block128In kept_gate, Block128In kept_up, MatOut dgate,
                            MatOut dup, int64_t rows, int64_t cols, cudaStream_t s);

// y[m, n] = x w^T (+ bias[n], may be null) for x [m, k], quantised on the way
// into `kept` (its scales may be null: then only q is written), and w [n, k]
// block-128. `work` holds at least linear_work_bytes(m, k), 16-byte aligned.
uint64_t linear_work_bytes(int64_t m, int64_t k);
cudaError_t linear_block128(MatIn x, FloatType xtype, Block128Out kept, void* work, uint64_t work_bytes, Block128In w,
                            const void* bias, MatOut y, FloatType type, int64_t m, int64_t n, int64_t k,
                            cudaStream_t s);
// Device memory of a gradient's own for the call (the caller may free or reuse
// it in stream order). Without it the result is the same, but powers of two as
// scales are treated like any others, which takes 16-bit results twice the
// time and fp32 ones three times.
struct GradWork {
    uint32_t* words = nullptr;
    uint32_t count = 0;
};
uint32_t grad_work_words(int64_t ni, int64_t nj);  // for a result of ni x nj; 0 if it needs none
// dx[m, k] = dy w, dy [m, n] bf16, w [n, k] block-128.
cudaError_t matmul_input_grad(MatIn dy, Block128In w, MatOut dx, FloatType type, int64_t m, int64_t n, int64_t k,
                              GradWork work, cudaStream_t s);
// dw[n, k] = dy^T x, dy [m, n] bf16, x [m, k] block-128.
cudaError_t matmul_weight_grad(MatIn dy, Block128In x, MatOut dw, FloatType type, int64_t m, int64_t n, int64_t k,
                               GradWork work, cudaStream_t s);

uint64_t block128_launch_count();

// Code of the first bounded wait that ran out in a product kernel on
// `device` (its result is then incomplete); 0 if none did. Host memory, read
// without waiting for the device.
uint32_t block128_error(int device);
// Sets that word (0: it has been dealt with). No effect before a product has run on the device.
void block128_set_error(int device, uint32_t code);

}  // namespace kern
}  // namespace ofld
