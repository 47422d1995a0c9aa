// Block-128 quantisation and the gated activation that keeps its inputs in
// 8 bits.
//
// Eight lanes own one block of 128 values, sixteen consecutive values each: a
// block's amax is three shuffles, and the scale and the addresses, which each
// lane works out for itself, are shared by sixteen values (with eight a lane
// the passes were bound by issue: 64 us instead of 41 for 16384 x 5120 bf16).
// Each value is read once and written once, 16 bytes at a time, and HBM bounds
// all four: swiglu of 8192 x 14336 bf16 forward 158 us and backward 150 (6.0
// and 6.3 TB/s), quantise 16384 x 5120 bf16 40 us, back 43 (6.4, 5.9 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>

#include "block128.h"
#include "block128_host.h"
#include "block128_lane.cuh"

namespace ofld {
namespace kern {

std::atomic<uint64_t> g_block128_launches{0};
uint64_t block128_launch_count() { return g_block128_launches.load(std::memory_order_relaxed); }

namespace {

using namespace lane128;

constexpr int kThreads = 128;
constexpr int kGroups = kThreads * kVals / 128;  // blocks in flight per CTA and step

struct Shape {
    uint32_t rows, cols, nb, total;    // total = rows * nb blocks
    uint32_t grid;
    uint32_t step, step_rows, step_b;  // from a group's block to its next: in blocks, and as rows and blocks of a row
};

// A group's walk over its blocks. The groups of a warp take the same number of
// steps, past the last block too, so that the shuffles see whole warps.
struct Walk {
    uint32_t blk, row, b;
    __device__ __forceinline__ explicit Walk(const Shape& sh) {
        blk = blockIdx.x * kGroups + threadIdx.x / kLanes;
        row = blk / sh.nb;
        b = blk - row * sh.nb;
    }
    __device__ __forceinline__ bool more(const Shape& sh) const { return (blk & ~(32u / kLanes - 1)) < sh.total; }
    __device__ __forceinline__ void next(const Shape& sh) {
        blk += sh.step;
        row += sh.step_rows;
        b += sh.step_b;
        if (b >= sh.nb) b -= sh.nb, ++row;
    }
    __device__ __forceinline__ uint32_t col() const { return b * 128 + threadIdx.x % kLanes * kVals; }
    // this lane's columns inside the row
    __device__ __forceinline__ uint32_t count(const Shape& sh) const {
        return blk >= sh.total || col() >= sh.cols ? 0u : min(uint32_t(kVals), sh.cols - col());
    }
    __device__ __forceinline__ bool first(const Shape& sh) const { return threadIdx.x % kLanes == 0 && blk < sh.total; }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_quantize(const T* __restrict__ x, uint32_t ldx, uint8_t* __restrict__ q, uint32_t ldq,
               float* __restrict__ scales, TileScales tiles, Shape sh) {
    // a product that waits for the tiles may start its own preparations
    if (tiles.words) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (Walk w(sh); w.more(sh); w.next(sh)) {
        const uint32_t c = w.col(), n = w.count(sh);
        const Pack<T> p = load<T, VEC>(x + uint64_t(w.row) * ldx, c, n);
        float f[kVals], s;
        const uint4 v = quantize_lane(p, f, &s);
        store_q(q + uint64_t(w.row) * ldq, c, n, v);
        if (w.first(sh)) {
            if (scales) scales[w.blk] = s;
            if (tiles.words) tiles.words[tiles.at(w.row, w.b, sh.nb)] = __float_as_uint(s) >> 23;
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_dequantize(const uint8_t* __restrict__ q, uint32_t ldq, const float* __restrict__ scales, T* __restrict__ x,
                 uint32_t ldx, Shape sh) {
    for (Walk w(sh); w.more(sh); w.next(sh)) {
        const uint32_t c = w.col(), n = w.count(sh);
        if (n == 0) continue;
        const uint4 v = load_q(q + uint64_t(w.row) * ldq, c, n);
        const float s = __ldg(scales + w.blk);
        float f[kVals];
        unpack(v, f);
#pragma unroll
        for (int i = 0; i < kVals; ++i) f[i] *= s;
        store<T, VEC>(x + uint64_t(w.row) * ldx, c, n, f);
    }
}

// exp of the negative side alone: 1 / (1 + exp(-g)) would be 0 below g = -88.7, where g s(g) is still in range.
// Results in 16 bits take the hardware's exp2 and reciprocal, whose errors (2^-22 and a unit for each of g's) are far
// under half a step of theirs, 2^-12 and more; in fp32 they would be the largest error, so fp32 takes the exact forms.
// The flushing exp2 is kept off subnormal results by a factor of 2^8, taken back after it: below e^-92 nothing is left
// of g s(g) in any case.
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
    if (sizeof(T) == 2) {
        float e, r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(fabsf(g), -1.4426950408889634f, 8.f)));
        e *= 0.00390625f;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
        return g >= 0.f ? r : e * r;
    }
    const float e = expf(-fabsf(g));
    return (g >= 0.f ? 1.f : e) / (1.f + e);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_swiglu_forward(const T* __restrict__ gate, uint32_t ldg, const T* __restrict__ up, uint32_t ldu,
                     T* __restrict__ h, uint32_t ldh, uint8_t* __restrict__ qg, uint32_t ldqg, float* __restrict__ sg,
                     uint8_t* __restrict__ qu, uint32_t ldqu, float* __restrict__ su, Shape sh) {
    for (Walk w(sh); w.more(sh); w.next(sh)) {
        const uint32_t c = w.col(), n = w.count(sh);
        const Pack<T> pg = load<T, VEC>(gate + uint64_t(w.row) * ldg, c, n);
        const Pack<T> pu = load<T, VEC>(up + uint64_t(w.row) * ldu, c, n);
        const bool first = w.first(sh);
        float g[kVals], u[kVals], s;
        uint4 v = quantize_lane(pg, g, &s);
        store_q(qg + uint64_t(w.row) * ldqg, c, n, v);
        if (first) sg[w.blk] = s;
        v = quantize_lane(pu, u, &s);
        store_q(qu + uint64_t(w.row) * ldqu, c, n, v);
        if (first) su[w.blk] = s;
        pg.floats(g);  // what is not finite goes into h as it is
        pu.floats(u);
#pragma unroll
        for (int i = 0; i < kVals; ++i) g[i] = g[i] * sigmoid<T>(g[i]) * u[i];
        store<T, VEC>(h + uint64_t(w.row) * ldh, c, n, g);
    }
}

// h = g s(g) u: du = dh g s(g), dg = dh u s(g) (1 + g (1 - s(g))).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    k_swiglu_backward(const T* __restrict__ dh, uint32_t lddh, const uint8_t* __restrict__ qg, uint32_t ldqg,
                      const float* __restrict__ sg, const uint8_t* __restrict__ qu, uint32_t ldqu,
                      const float* __restrict__ su, T* __restrict__ dg, uint32_t lddg, T* __restrict__ du,
                      uint32_t lddu, Shape sh) {
    for (Walk w(sh); w.more(sh); w.next(sh)) {
        const uint32_t c = w.col(), n = w.count(sh);
        if (n == 0) continue;
        const Pack<T> pd = load<T, VEC>(dh + uint64_t(w.row) * lddh, c, n);
        const uint4 vg = load_q(qg + uint64_t(w.row) * ldqg, c, n), vu = load_q(qu + uint64_t(w.row) * ldqu, c, n);
        const float fg = __ldg(sg + w.blk), fu = __ldg(su + w.blk);
        float d[kVals], g[kVals], u[kVals];
        pd.floats(d);
        unpack(vg, g);
        unpack(vu, u);
#pragma unroll
        for (int i = 0; i < kVals; ++i) {
            const float gi = g[i] * fg, s = sigmoid<T>(gi), ds = d[i] * s;
            g[i] = ds * (u[i] * fu) * (1.f + gi * (1.f - s));
            u[i] = ds * gi;
        }
        store<T, VEC>(dg + uint64_t(w.row) * lddg, c, n, g);
        store<T, VEC>(du + uint64_t(w.row) * lddu, c, n, u);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t size_of(FloatType t) { return t == FloatType::kFp32 ? 4 : 2; }
bool type_ok(FloatType t) { return t == FloatType::kBf16 || t == FloatType::kFp16 || t == FloatType::kFp32; }
bool vec_ok(const void* p, int64_t ld, FloatType t) { return aligned16(p) && (ld * int64_t(size_of(t))) % 16 == 0; }
bool mat_ok(const void* p, int64_t ld, int64_t cols) { return p && ld >= cols && ld <= 0xffffffff; }
bool q_ptr_ok(const void* q, int64_t ld, int64_t cols) {
    return q && aligned16(q) && ld % 16 == 0 && ld >= cols && ld <= 0xffffffff;
}
bool q_ok(const void* q, int64_t ld, const float* s, int64_t cols) { return s && q_ptr_ok(q, ld, cols); }


// False when the sizes are out of range; an empty shape has total 0.
// `per_sm`: CTAs of the grid for each SM, many times what fits at once: CTAs
// that start as others end keep loads in flight, where a few long ones (5 to
// 16 an SM) took 10 to 30 % more time.
bool make_shape(int64_t rows, int64_t cols, int per_sm, Shape* sh) {
    if (rows < 0 || cols < 0 || rows > 0x7fffffff || cols > 0x7fffff00) return false;
    const int64_t nb = (cols + 127) / 128;
    if (nb > 0 && rows > 0x7ff00000 / nb) return false;  // room to step past the end
    *sh = Shape{uint32_t(rows), uint32_t(cols), uint32_t(nb), uint32_t(rows * nb), 0, 0, 0, 0};
    if (sh->total) {
        sh->grid = std::min<uint32_t>((sh->total + kGroups - 1) / kGroups, uint32_t(sm_count() * per_sm));
        sh->step = sh->grid * kGroups;
        sh->step_rows = sh->step / sh->nb;
        sh->step_b = sh->step % sh->nb;
    }
    return true;
}

cudaError_t launched() {
    g_block128_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaGetLastError();
}

uint32_t u32(int64_t v) { return uint32_t(v); }
const uint8_t* q8(const void* p) { return static_cast<const uint8_t*>(p); }
uint8_t* q8(void* p) { return static_cast<uint8_t*>(p); }

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
    if (!make_shape(rows, cols, 160, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(x.ptr, x.ld, cols) || !q_ptr_ok(out.q, out.ld, cols)) return cudaErrorInvalidValue;
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec_ok(x.ptr, x.ld, type) ? k_quantize<T, true> : k_quantize<T, false>;
        fn<<<sh.grid, kThreads, 0, s>>>(static_cast<const T*>(x.ptr), u32(x.ld), q8(out.q),
                                         u32(out.ld), out.scales, tiles, sh);
    });
    return launched();
}

cudaError_t dequantize_block128(Block128In in, MatOut x, FloatType type, int64_t rows, int64_t cols, cudaStream_t s) {
    Shape sh;
    if (!make_shape(rows, cols, 160, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(x.ptr, x.ld, cols) || !q_ok(in.q, in.ld, in.scales, cols)) return cudaErrorInvalidValue;
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec_ok(x.ptr, x.ld, type) ? k_dequantize<T, true> : k_dequantize<T, false>;
        fn<<<sh.grid, kThreads, 0, s>>>(q8(in.q), u32(in.ld), in.scales, static_cast<T*>(x.ptr),
                                         u32(x.ld), sh);
    });
    return launched();
}

cudaError_t swiglu_forward(MatIn gate, MatIn up, FloatType type, MatOut h, Block128Out kg, Block128Out ku,
                           int64_t rows, int64_t cols, cudaStream_t s) {
    Shape sh;
    if (!make_shape(rows, cols, 160, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(gate.ptr, gate.ld, cols) || !mat_ok(up.ptr, up.ld, cols) || !mat_ok(h.ptr, h.ld, cols) ||
        !q_ok(kg.q, kg.ld, kg.scales, cols) || !q_ok(ku.q, ku.ld, ku.scales, cols))
        return cudaErrorInvalidValue;
    const bool vec = vec_ok(gate.ptr, gate.ld, type) && vec_ok(up.ptr, up.ld, type) && vec_ok(h.ptr, h.ld, type);
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec ? k_swiglu_forward<T, true> : k_swiglu_forward<T, false>;
        fn<<<sh.grid, kThreads, 0, s>>>(static_cast<const T*>(gate.ptr), u32(gate.ld), static_cast<const T*>(up.ptr),
                                         u32(up.ld), static_cast<T*>(h.ptr), u32(h.ld), q8(kg.q), u32(kg.ld),
                                         kg.scales, q8(ku.q), u32(ku.ld), ku.scales, sh);
    });
    return launched();
}

cudaError_t swiglu_backward(MatIn dh, FloatType type, Block128In kg, Block128In ku, MatOut dg, MatOut du,
                            int64_t rows, int64_t cols, cudaStream_t s) {
    Shape sh;
    if (!make_shape(rows, cols, 20, &sh) || !type_ok(type)) return cudaErrorInvalidValue;
    if (sh.total == 0) return cudaSuccess;
    if (!mat_ok(dh.ptr, dh.ld, cols) || !mat_ok(dg.ptr, dg.ld, cols) || !mat_ok(du.ptr, du.ld, cols) ||
        !q_ok(kg.q, kg.ld, kg.scales, cols) || !q_ok(ku.q, ku.ld, ku.scales, cols))
        return cudaErrorInvalidValue;
    const bool vec = vec_ok(dh.ptr, dh.ld, type) && vec_ok(dg.ptr, dg.ld, type) && vec_ok(du.ptr, du.ld, type);
    by_type(type, [&](auto t) {
        using T = decltype(t);
        auto* fn = vec ? k_swiglu_backward<T, true> : k_swiglu_backward<T, false>;
        fn<<<sh.grid, kThreads, 0, s>>>(static_cast<const T*>(dh.ptr), u32(dh.ld), q8(kg.q),
                                         u32(kg.ld), kg.scales, q8(ku.q), u32(ku.ld), ku.scales,
                                         static_cast<T*>(dg.ptr), u32(dg.ld), static_cast<T*>(du.ptr), u32(du.ld), sh);
    });
    return launched();
}

}  // namespace kern
}  // namespace ofld
