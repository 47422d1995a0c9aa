// Block-128 quantisation and the gated activation that keeps its inputs in
// 8 bits.
//
// Sixteen lanes own one block of 128 values, eight consecutive values each,
// so a block's amax is four shuffles and every access of a 16-bit type is one
// 16-byte vector. All kernels are bound by HBM: each value is read once and
// written once.
//
// The scale is the smallest power of two 2^e, e >= -117, with
// amax <= 448 * 2^e. Dividing by it is exact, so the only rounding is the one
// to e4m3 (to nearest, ties to even, at most 2^-4 of the value), and q * 2^e
// is exact in bf16: a product that reads the checkpoint as bf16 sees just
// what the forward pass kept. An amax / 448 scale would add a rounding on
// either side for the one binade of range that it gains. e >= -117 keeps the
// smallest product 2^-9 * 2^-117 normal. Values that are not finite become
// NaN and do not count in amax, so one of them does not spoil its block.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>

#include "block128.h"
#include "block128_host.h"

namespace ofld {
namespace kern {

std::atomic<uint64_t> g_block128_launches{0};
uint64_t block128_launch_count() { return g_block128_launches.load(std::memory_order_relaxed); }

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;  // blocks in flight per CTA and step
constexpr int kMinExp = -117;

struct Shape {
    uint32_t rows, cols, nb, total;  // total = rows * nb blocks
};

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_float(float v) { return v; }

template <typename T>
struct alignas(16) Pack8 {
    T v[8];
};

// Eight values from column c of a row (n of them inside the row, the rest 0).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, uint32_t c, uint32_t n, float f[8]) {
    if (VEC && n == 8) {
        Pack8<T> p;
        const uint4* src = reinterpret_cast<const uint4*>(row + c);
        uint4* dst = reinterpret_cast<uint4*>(&p);
#pragma unroll
        for (int i = 0; i < int(sizeof(p) / 16); ++i) dst[i] = __ldcs(src + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_float(p.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = uint32_t(i) < n ? to_float(row[c + i]) : 0.f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, uint32_t c, uint32_t n, const float f[8]) {
    if (VEC && n == 8) {
        Pack8<T> p;
#pragma unroll
        for (int i = 0; i < 8; ++i) p.v[i] = from_float<T>(f[i]);
        uint4* dst = reinterpret_cast<uint4*>(row + c);
        const uint4* src = reinterpret_cast<const uint4*>(&p);
#pragma unroll
        for (int i = 0; i < int(sizeof(p) / 16); ++i) dst[i] = src[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (uint32_t(i) < n) row[c + i] = from_float<T>(f[i]);
    }
}

__device__ __forceinline__ void store_q(uint8_t* row, uint32_t c, uint32_t n, uint2 q) {
    if (n == 8) {
        *reinterpret_cast<uint2*>(row + c) = q;
    } else {
        for (uint32_t i = 0; i < n; ++i) row[c + i] = uint8_t((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    }
}

__device__ __forceinline__ uint2 load_q(const uint8_t* row, uint32_t c, uint32_t n) {
    if (n == 8) return __ldcs(reinterpret_cast<const uint2*>(row + c));
    uint2 q = make_uint2(0, 0);
    for (uint32_t i = 0; i < n; ++i) (i < 4 ? q.x : q.y) |= uint32_t(row[c + i]) << (8 * (i & 3));
    return q;
}

__device__ __forceinline__ uint32_t fp8x2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ void fp8_to_float(uint32_t w, float f[4]) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w & 0xffff), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w >> 16), __NV_E4M3);
    const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

// Quantises the eight values that this lane holds of its group's block.
__device__ __forceinline__ uint2 quantize8(const float f[8], float* scale) {
    float v[8], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = fabsf(f[i]) <= 3.402823466e38f ? f[i] : __int_as_float(0x7fffffff);
        amax = fmaxf(amax, fabsf(v[i]));  // fmaxf drops a NaN
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    // amax = 1.f * 2^E and 448 = 1.75 * 2^8: e = E - 8, one more where 1.f > 1.75
    const uint32_t u = __float_as_uint(amax);
    int e = int(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
    e = amax > 0.f ? max(e, kMinExp) : 0;
    *scale = __uint_as_float(uint32_t(e + 127) << 23);
    const float inv = __uint_as_float(uint32_t(127 - e) << 23);
    return make_uint2(fp8x2(v[0] * inv, v[1] * inv) | fp8x2(v[2] * inv, v[3] * inv) << 16,
                      fp8x2(v[4] * inv, v[5] * inv) | fp8x2(v[6] * inv, v[7] * inv) << 16);
}

struct Pos {
    uint32_t row, b, c, n;  // row, block in the row, this lane's first column, its columns inside the row
};
__device__ __forceinline__ Pos locate(const Shape& sh, uint32_t blk) {
    Pos p;
    p.row = blk / sh.nb;
    p.b = blk - p.row * sh.nb;
    p.c = p.b * 128 + (threadIdx.x & 15) * 8;
    p.n = blk >= sh.total || p.c >= sh.cols ? 0u : min(8u, sh.cols - p.c);
    return p;
}

// Every warp holds two blocks a step; both halves take the same number of
// steps so that the shuffles see whole warps.
#define FOR_BLOCKS(blk)                                                                          \
    for (uint32_t first_ = blockIdx.x * kGroups; first_ < sh.total; first_ += gridDim.x * kGroups) \
        if (const uint32_t blk = first_ + threadIdx.x / 16; true)

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_quantize(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq,
               float* __restrict__ scales, TileScales tiles, Shape sh) {
    FOR_BLOCKS(blk) {
        const Pos p = locate(sh, blk);
        float f[8], s;
        load8<T, VEC>(x + p.row * ldx, p.c, p.n, f);
        const uint2 v = quantize8(f, &s);
        store_q(q + p.row * ldq, p.c, p.n, v);
        if ((threadIdx.x & 15) == 0 && blk < sh.total) {
            if (scales) scales[blk] = s;
            if (tiles.words) tiles.words[tiles.at(p.row, p.b, sh.nb)] = __float_as_uint(s) >> 23;
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_dequantize(const uint8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scales, T* __restrict__ x,
                 int64_t ldx, Shape sh) {
    FOR_BLOCKS(blk) {
        const Pos p = locate(sh, blk);
        if (p.n == 0) continue;
        const uint2 v = load_q(q + p.row * ldq, p.c, p.n);
        const float s = __ldg(scales + blk);
        float f[8];
        fp8_to_float(v.x, f);
        fp8_to_float(v.y, f + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= s;
        store8<T, VEC>(x + p.row * ldx, p.c, p.n, f);
    }
}

// exp of the negative side alone: 1 / (1 + exp(-g)) would be 0 below g = -88.7, where g s(g) is still in range.
// Results in 16 bits take the hardware's exp and reciprocal, whose errors (2^-22 and a unit for each of g's) are far
// under half a step of theirs, 2^-12 and more; in fp32 they would be the largest error, so fp32 takes the exact forms.
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
    if (sizeof(T) == 2) {
        const float e = __expf(-fabsf(g));
        return __fdividef(g >= 0.f ? 1.f : e, 1.f + e);
    }
    const float e = expf(-fabsf(g));
    return (g >= 0.f ? 1.f : e) / (1.f + e);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_swiglu_forward(const T* __restrict__ gate, int64_t ldg, const T* __restrict__ up, int64_t ldu,
                     T* __restrict__ h, int64_t ldh, uint8_t* __restrict__ qg, int64_t ldqg, float* __restrict__ sg,
                     uint8_t* __restrict__ qu, int64_t ldqu, float* __restrict__ su, Shape sh) {
    FOR_BLOCKS(blk) {
        const Pos p = locate(sh, blk);
        float g[8], u[8], o[8], s;
        load8<T, VEC>(gate + p.row * ldg, p.c, p.n, g);
        load8<T, VEC>(up + p.row * ldu, p.c, p.n, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = g[i] * sigmoid<T>(g[i]) * u[i];
        store8<T, VEC>(h + p.row * ldh, p.c, p.n, o);
        const bool first = (threadIdx.x & 15) == 0 && blk < sh.total;
        uint2 v = quantize8(g, &s);
        store_q(qg + p.row * ldqg, p.c, p.n, v);
        if (first) sg[blk] = s;
        v = quantize8(u, &s);
        store_q(qu + p.row * ldqu, p.c, p.n, v);
        if (first) su[blk] = s;
    }
}

// h = g s(g) u: du = dh g s(g), dg = dh u s(g) (1 + g (1 - s(g))).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_swiglu_backward(const T* __restrict__ dh, int64_t lddh, const uint8_t* __restrict__ qg, int64_t ldqg,
                      const float* __restrict__ sg, const uint8_t* __restrict__ qu, int64_t ldqu,
                      const float* __restrict__ su, T* __restrict__ dg, int64_t lddg, T* __restrict__ du,
                      int64_t lddu, Shape sh) {
    FOR_BLOCKS(blk) {
        const Pos p = locate(sh, blk);
        if (p.n == 0) continue;
        float d[8], g[8], u[8], a[8], b[8];
        load8<T, VEC>(dh + p.row * lddh, p.c, p.n, d);
        const uint2 vg = load_q(qg + p.row * ldqg, p.c, p.n), vu = load_q(qu + p.row * ldqu, p.c, p.n);
        const float fg = __ldg(sg + blk), fu = __ldg(su + blk);
        fp8_to_float(vg.x, g);
        fp8_to_float(vg.y, g + 4);
        fp8_to_float(vu.x, u);
        fp8_to_float(vu.y, u + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float gi = g[i] * fg, ui = u[i] * fu, s = sigmoid<T>(gi);
            b[i] = d[i] * gi * s;
            a[i] = d[i] * ui * s * (1.f + gi * (1.f - s));
        }
        store8<T, VEC>(dg + p.row * lddg, p.c, p.n, a);
        store8<T, VEC>(du + p.row * lddu, p.c, p.n, b);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t size_of(FloatType t) { return t == FloatType::kFp32 ? 4 : 2; }
bool type_ok(FloatType t) { return t == FloatType::kBf16 || t == FloatType::kFp16 || t == FloatType::kFp32; }
bool vec_ok(const void* p, int64_t ld, FloatType t) { return aligned16(p) && (ld * int64_t(size_of(t))) % 16 == 0; }
bool mat_ok(const void* p, int64_t ld, int64_t cols) { return p && ld >= cols; }
bool q_ptr_ok(const void* q, int64_t ld, int64_t cols) { return q && aligned16(q) && ld % 16 == 0 && ld >= cols; }
bool q_ok(const void* q, int64_t ld, const float* s, int64_t cols) { return s && q_ptr_ok(q, ld, cols); }

// False when the sizes are out of range; an empty shape has total 0.
bool make_shape(int64_t rows, int64_t cols, Shape* sh) {
    if (rows < 0 || cols < 0 || rows > 0x7fffffff || cols > 0x7fffff00) return false;
    const int64_t nb = (cols + 127) / 128;
    if (nb > 0 && rows > 0x7fffffff / nb) return false;
    *sh = Shape{uint32_t(rows), uint32_t(cols), uint32_t(nb), uint32_t(rows * nb)};
    return true;
}

int grid(const Shape& sh) { return int(std::min<uint32_t>((sh.total + kGroups - 1) / kGroups, 148 * 8)); }

cudaError_t launched() {
    g_block128_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaGetLastError();
}

template <typename F>
void by_type(FloatType t, F f) {
    if (t == FloatType::kBf16)
        f(__nv_bfloat16{});
    else if (t == FloatType::kFp16)
        f(__half{});
    else
        f(float{});
}

}  // namespace

cudaError_t quantize_block128(MatIn x, FloatType type, Block128Out out, int64_t rows, int64_t cols, cudaStream_t s) {
    if (rows > 0 && cols > 0 && !out.scales) return cudaErrorInvalidValue;
    return quantize_for_tiles(x, type, out, TileScales{}, rows, cols, s);
}

cudaError_t quantize_for_tiles(MatIn x, FloatType type, Block128Out out, TileScales tiles, int64_t rows, int64_t cols,
                               cudaStream_t s) {
    Shape sh;
    if (!make_shape(rows, cols, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(x.ptr, x.ld, cols) || !q_ptr_ok(out.q, out.ld, cols)) return cudaErrorInvalidValue;
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec_ok(x.ptr, x.ld, type) ? k_quantize<T, true> : k_quantize<T, false>;
        fn<<<grid(sh), kThreads, 0, s>>>(static_cast<const T*>(x.ptr), x.ld, static_cast<uint8_t*>(out.q), out.ld,
                                         out.scales, tiles, sh);
    });
    return launched();
}

cudaError_t dequantize_block128(Block128In in, MatOut x, FloatType type, int64_t rows, int64_t cols, cudaStream_t s) {
    Shape sh;
    if (!make_shape(rows, cols, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(x.ptr, x.ld, cols) || !q_ok(in.q, in.ld, in.scales, cols)) return cudaErrorInvalidValue;
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec_ok(x.ptr, x.ld, type) ? k_dequantize<T, true> : k_dequantize<T, false>;
        fn<<<grid(sh), kThreads, 0, s>>>(static_cast<const uint8_t*>(in.q), in.ld, in.scales, static_cast<T*>(x.ptr),
                                         x.ld, sh);
    });
    return launched();
}

cudaError_t swiglu_forward(MatIn gate, MatIn up, FloatType type, MatOut h, Block128Out kg, Block128Out ku,
                           int64_t rows, int64_t cols, cudaStream_t s) {
    Shape sh;
    if (!make_shape(rows, cols, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(gate.ptr, gate.ld, cols) || !mat_ok(up.ptr, up.ld, cols) || !mat_ok(h.ptr, h.ld, cols) ||
        !q_ok(kg.q, kg.ld, kg.scales, cols) || !q_ok(ku.q, ku.ld, ku.scales, cols))
        return cudaErrorInvalidValue;
    const bool vec = vec_ok(gate.ptr, gate.ld, type) && vec_ok(up.ptr, up.ld, type) && vec_ok(h.ptr, h.ld, type);
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec ? k_swiglu_forward<T, true> : k_swiglu_forward<T, false>;
        fn<<<grid(sh), kThreads, 0, s>>>(static_cast<const T*>(gate.ptr), gate.ld, static_cast<const T*>(up.ptr),
                                         up.ld, static_cast<T*>(h.ptr), h.ld, static_cast<uint8_t*>(kg.q), kg.ld,
                                         kg.scales, static_cast<uint8_t*>(ku.q), ku.ld, ku.scales, sh);
    });
    return launched();
}

cudaError_t swiglu_backward(MatIn dh, FloatType type, Block128In kg, Block128In ku, MatOut dg, MatOut du,
                            int64_t rows, int64_t cols, cudaStream_t s) {
    Shape sh;
    if (!make_shape(rows, cols, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(dh.ptr, dh.ld, cols) || !mat_ok(dg.ptr, dg.ld, cols) || !mat_ok(du.ptr, du.ld, cols) ||
        !q_ok(kg.q, kg.ld, kg.scales, cols) || !q_ok(ku.q, ku.ld, ku.scales, cols))
        return cudaErrorInvalidValue;
    const bool vec = vec_ok(dh.ptr, dh.ld, type) && vec_ok(dg.ptr, dg.ld, type) && vec_ok(du.ptr, du.ld, type);
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec ? k_swiglu_backward<T, true> : k_swiglu_backward<T, false>;
        fn<<<grid(sh), kThreads, 0, s>>>(static_cast<const T*>(dh.ptr), dh.ld, static_cast<const uint8_t*>(kg.q),
                                         kg.ld, kg.scales, static_cast<const uint8_t*>(ku.q), ku.ld, ku.scales,
                                         static_cast<T*>(dg.ptr), dg.ld, static_cast<T*>(du.ptr), du.ld, sh);
    });
    return launched();
}

}  // namespace kern
}  // namespace ofld
