// What one lane does of a block-128 quantisation: eight lanes own a block of
// 128 values, sixteen consecutive ones each.
//
// The scale is the smallest power of two 2^e, e >= -117, with
// amax <= 448 * 2^e. Dividing by it is exact, so the only rounding is the one
// to e4m3 (to nearest, ties to even, at most 2^-4 of the value), and q * 2^e
// is exact in bf16: a product that reads the checkpoint as bf16 sees just
// what the forward pass kept. An amax / 448 scale would add a rounding on
// either side for the one binade of range that it gains. e >= -117 keeps the
// smallest product 2^-9 * 2^-117 normal. Values that are not finite become
// NaN and do not count in amax, so one of them does not spoil its block.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace ofld {
namespace kern {
namespace lane128 {

constexpr int kVals = 16;            // of a lane
constexpr int kLanes = 128 / kVals;  // of a block
constexpr int kMinExp = -117;

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

// A lane's consecutive values as they are in memory.
template <typename T>
struct alignas(16) Pack {
    T v[kVals];
    __device__ __forceinline__ void floats(float f[kVals]) const {
#pragma unroll
        for (int i = 0; i < kVals; ++i) f[i] = to_float(v[i]);
    }
};

// A lane's values from column c of a row on (n of them inside the row, the rest 0).
template <typename T, bool VEC>
__device__ __forceinline__ Pack<T> load(const T* row, uint32_t c, uint32_t n) {
    Pack<T> p;
    if (VEC && n == kVals) {
        const uint4* src = reinterpret_cast<const uint4*>(row + c);
        uint4* dst = reinterpret_cast<uint4*>(&p);
#pragma unroll
        for (int i = 0; i < int(sizeof(p) / 16); ++i) dst[i] = __ldg(src + i);
    } else {
#pragma unroll
        for (int i = 0; i < kVals; ++i) p.v[i] = uint32_t(i) < n ? row[c + i] : from_float<T>(0.f);
    }
    return p;
}

template <typename T, bool VEC>
__device__ __forceinline__ void store(T* row, uint32_t c, uint32_t n, const float f[kVals]) {
    if (VEC && n == kVals) {
        Pack<T> p;
#pragma unroll
        for (int i = 0; i < kVals; ++i) p.v[i] = from_float<T>(f[i]);
        uint4* dst = reinterpret_cast<uint4*>(row + c);
        const uint4* src = reinterpret_cast<const uint4*>(&p);
#pragma unroll
        for (int i = 0; i < int(sizeof(p) / 16); ++i) dst[i] = src[i];
    } else {
#pragma unroll
        for (int i = 0; i < kVals; ++i)
            if (uint32_t(i) < n) row[c + i] = from_float<T>(f[i]);
    }
}

__device__ __forceinline__ uint32_t byte_of(uint4 q, uint32_t i) {
    return (i < 8 ? (i < 4 ? q.x : q.y) : (i < 12 ? q.z : q.w)) >> (8 * (i & 3)) & 0xff;
}
__device__ __forceinline__ void store_q(uint8_t* row, uint32_t c, uint32_t n, uint4 q) {
    if (n == kVals) {
        *reinterpret_cast<uint4*>(row + c) = q;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kVals; ++i)
            if (i < n) row[c + i] = uint8_t(byte_of(q, i));
    }
}

__device__ __forceinline__ uint4 load_q(const uint8_t* row, uint32_t c, uint32_t n) {
    if (n == kVals) return __ldg(reinterpret_cast<const uint4*>(row + c));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < kVals; ++i)
        if (i < n) w[i / 4] |= uint32_t(row[c + i]) << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint32_t fp8x2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ void fp8_to_float(uint32_t w, float* f) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w & 0xffff), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w >> 16), __NV_E4M3);
    const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

__device__ __forceinline__ void unpack(uint4 q, float f[kVals]) {
    fp8_to_float(q.x, f);
    fp8_to_float(q.y, f + 4);
    fp8_to_float(q.z, f + 8);
    fp8_to_float(q.w, f + 12);
}

// The largest of a lane's magnitudes; a value that is not finite becomes
// NaN in f and does not count.
__device__ __forceinline__ float lane_amax(const Pack<float>& p, float f[kVals]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kVals; ++i) {
        f[i] = fabsf(p.v[i]) <= 3.402823466e38f ? p.v[i] : __int_as_float(0x7fffffff);
        m = fmaxf(m, fabsf(f[i]));  // fmaxf drops a NaN
    }
    return m;
}
// 16-bit types: magnitudes order like their bits, so two go at a time, and one
// comparison finds what is not finite.
template <typename T>
__device__ __forceinline__ float lane_amax(const Pack<T>& p, float f[kVals]) {
    constexpr uint32_t kInf = sizeof(T) == 2 && __is_same(T, __half) ? 0x7c00u : 0x7f80u;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&p);
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < kVals / 2; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    p.floats(f);
    if (m >= kInf) {
        Pack<float> q;
#pragma unroll
        for (int i = 0; i < kVals; ++i) q.v[i] = f[i];
        return lane_amax(q, f);
    }
    const uint16_t bits = uint16_t(m);
    return to_float(*reinterpret_cast<const T*>(&bits));
}

// Quantises the values that this lane holds of its group's block and leaves
// them in f as fp32.
template <typename T>
__device__ __forceinline__ uint4 quantize_lane(const Pack<T>& p, float f[kVals], float* scale) {
    float amax = lane_amax(p, f);
#pragma unroll
    for (int o = 64 / kVals; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    // amax = 1.f * 2^E and 448 = 1.75 * 2^8: e = E - 8, one more where 1.f > 1.75
    const uint32_t u = __float_as_uint(amax);
    int e = int(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
    e = amax > 0.f ? max(e, kMinExp) : 0;
    *scale = __uint_as_float(uint32_t(e + 127) << 23);
    const float inv = __uint_as_float(uint32_t(127 - e) << 23);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = fp8x2(f[4 * i] * inv, f[4 * i + 1] * inv) | fp8x2(f[4 * i + 2] * inv, f[4 * i + 3] * inv) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace lane128
}  // namespace kern
}  // namespace ofld
