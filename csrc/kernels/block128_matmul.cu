// Matrix products with block-128 operands: y = x w^T and its two gradients.
//
// All three are C[i, j] = sum_t A(i, t) B(t, j) with fp32 sums. A CTA owns a
// 64 x 64 tile of C; its 256 threads load 32 steps of t of both operands as
// fp32 values into shared memory and accumulate 4 x 4 products each.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "block128.h"

namespace ofld {
namespace kern {

extern std::atomic<uint64_t> g_block128_launches;

namespace {

constexpr int kTile = 64, kStep = 32, kThreads = 256;

// Element (r, c) of a block-128 tensor as fp32.
struct QuantAt {
    const uint8_t* q;
    int64_t ld;
    const float* scales;
    int64_t nb;
    __device__ __forceinline__ float operator()(int64_t r, int64_t c) const {
        const __half_raw h = __nv_cvt_fp8_to_halfraw(q[r * ld + c], __NV_E4M3);
        return __half2float(__half(h)) * scales[r * nb + c / 128];
    }
};
struct Bf16At {
    const __nv_bfloat16* p;
    int64_t ld;
    __device__ __forceinline__ float operator()(int64_t r, int64_t c) const { return __bfloat162float(p[r * ld + c]); }
};

template <typename T>
__device__ __forceinline__ float bias_at(const void* b, int64_t j) {
    return b ? float(static_cast<const T*>(b)[j]) : 0.f;
}

// A_T / B_T: the operand is stored with t as its row.
template <typename A, bool A_T, typename B, bool B_T, typename T>
__global__ void __launch_bounds__(kThreads)
    k_product(A a, B b, const void* bias, T* out, int64_t ldo, int64_t ni, int64_t nj, int64_t nt) {
    __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
    const int64_t i0 = int64_t(blockIdx.x) * kTile, j0 = int64_t(blockIdx.y) * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int64_t t0 = 0; t0 < nt; t0 += kStep) {
        for (int e = threadIdx.x; e < kTile * kStep; e += kThreads) {
            const int ai = A_T ? e % kTile : e / kStep, at = A_T ? e / kTile : e % kStep;
            const int bi = B_T ? e % kTile : e / kStep, bt = B_T ? e / kTile : e % kStep;
            const int64_t i = i0 + ai, ta = t0 + at, j = j0 + bi, tb = t0 + bt;
            sa[at][ai] = i < ni && ta < nt ? (A_T ? a(ta, i) : a(i, ta)) : 0.f;
            sb[bt][bi] = j < nj && tb < nt ? (B_T ? b(tb, j) : b(j, tb)) : 0.f;
        }
        __syncthreads();
#pragma unroll 4
        for (int t = 0; t < kStep; ++t)
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[u][v] += sa[t][ty + 16 * u] * sb[t][tx + 16 * v];
        __syncthreads();
    }
    for (int u = 0; u < 4; ++u)
        for (int v = 0; v < 4; ++v) {
            const int64_t i = i0 + ty + 16 * u, j = j0 + tx + 16 * v;
            if (i < ni && j < nj) out[i * ldo + j] = T(acc[u][v] + bias_at<T>(bias, j));
        }
}

bool dims_ok(int64_t a, int64_t b, int64_t c) {
    const int64_t most = 0x7fffff00;
    return a >= 0 && b >= 0 && c >= 0 && a <= most && b <= most && c <= most;
}
bool q_ok(const Block128In& t, int64_t cols) {
    return t.q && t.scales && (reinterpret_cast<uintptr_t>(t.q) & 15) == 0 && t.ld % 16 == 0 && t.ld >= cols;
}

template <bool A_T, bool B_T, typename A, typename B>
cudaError_t launch(A a, B b, const void* bias, MatOut out, FloatType type, int64_t ni, int64_t nj, int64_t nt,
                   cudaStream_t s) {
    const int64_t gi = (ni + kTile - 1) / kTile, gj = (nj + kTile - 1) / kTile;
    if (gj > 65535) return cudaErrorInvalidValue;
    const dim3 g{unsigned(gi), unsigned(gj)};
    if (type == FloatType::kBf16)
        k_product<A, A_T, B, B_T><<<g, kThreads, 0, s>>>(a, b, bias, static_cast<__nv_bfloat16*>(out.ptr), out.ld, ni,
                                                       nj, nt);
    else if (type == FloatType::kFp16)
        k_product<A, A_T, B, B_T><<<g, kThreads, 0, s>>>(a, b, bias, static_cast<__half*>(out.ptr), out.ld, ni, nj, nt);
    else
        k_product<A, A_T, B, B_T><<<g, kThreads, 0, s>>>(a, b, bias, static_cast<float*>(out.ptr), out.ld, ni, nj, nt);
    g_block128_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaGetLastError();
}

QuantAt quant_at(const Block128In& t, int64_t cols) {
    return QuantAt{static_cast<const uint8_t*>(t.q), t.ld, t.scales, (cols + 127) / 128};
}

}  // namespace

cudaError_t matmul_input_grad(MatIn dy, Block128In w, MatOut dx, FloatType type, int64_t m, int64_t n, int64_t k,
                              cudaStream_t s) {
    if (!dims_ok(m, n, k) || n == 0) return cudaErrorInvalidValue;
    if (m == 0 || k == 0) return cudaSuccess;
    if (!dy.ptr || dy.ld < n || !q_ok(w, k) || !dx.ptr || dx.ld < k) return cudaErrorInvalidValue;
    return launch<false, true>(Bf16At{static_cast<const __nv_bfloat16*>(dy.ptr), dy.ld}, quant_at(w, k), nullptr, dx,
                               type, m, k, n, s);
}

cudaError_t matmul_weight_grad(MatIn dy, Block128In x, MatOut dw, FloatType type, int64_t m, int64_t n, int64_t k,
                               cudaStream_t s) {
    if (!dims_ok(m, n, k) || m == 0) return cudaErrorInvalidValue;
    if (n == 0 || k == 0) return cudaSuccess;
    if (!dy.ptr || dy.ld < n || !q_ok(x, k) || !dw.ptr || dw.ld < k) return cudaErrorInvalidValue;
    return launch<true, true>(Bf16At{static_cast<const __nv_bfloat16*>(dy.ptr), dy.ld}, quant_at(x, k), nullptr, dw,
                              type, n, k, m, s);
}

}  // namespace kern
}  // namespace ofld
