// The two gradients of y = x w^T, each a bf16 matrix times a block-128 one:
//
//   input:  dx[m, k] = sum_n dy[m, n] w[n, k]       weight:  dw[n, k] = sum_m dy[m, n] x[m, k]
//
// Both are out[i, j] = sum_t A(i, t) Q[t, j] s[t, j / 128]: the 8-bit operand
// is stored with the summed index as its row, and its scale changes with the
// row, so it cannot leave the sum. Converter warps bring each tile of Q from
// 8 bits to bf16 in shared memory, times its scale, and the tensor core
// multiplies it with dy as it is (tcgen05.mma kind::f16, fp32 accumulators in
// tensor memory). The converted tile and, for the weight gradient, dy's are
// read "MN-major": their rows run along the output, not along the sum, so
// nothing is transposed.
//
// A value times a power of two, as in everything that quantize made, is exact
// in bf16. Any other scale leaves up to 28 bits, of which one bf16 rounding
// would drop 20: the gradient would be 2.3e-3 off the exact one where rounding
// it to bf16 costs 1.7e-3. So where there is such a scale, each tile of Q goes
// to the tensor core in parts, each the bf16 rounding of what the parts before
// left over: two (2^-16 of a value) for results in 16 bits, three (2^-24) for
// fp32. 4096 x 4096 x 14336, bf16 results: 369 us with powers of two, 727 us
// with other scales.
//
// Which of the two it is, is found on the device: a CTA with a tile of its own
// looks at the scales that it will use; for pairs, which use each scale many
// times, a kernel ahead reads them all once (2 us).
//
// A pair of CTAs owns 256 x 256 outputs; each loads 128 rows of A and 128
// columns of Q for 64 steps of t, and converts its 8192 values while the
// tensor core spends 512 cycles on the step before. Few outputs: one CTA owns
// 128 x 128, and the sum is split over a cluster of up to 8.
//
// 8192 tokens, 14336 x 4096, bf16 results: 670 us (1.44 PFLOP/s, the tensor
// pipe active 76 % of the cycles; cuBLAS bf16 reaches 1.65 in bursts and 1.38
// in a loop of seconds, under the power cap that bounds this kernel too). What
// it took: a converter that arrives without a release to the cluster (746 us
// to 357 for 4096 x 4096 x 14336), a ring for each kind of tile, and results
// stored as tiles (1.35 to 1.45 PFLOP/s).
//
// Warps: 0 loads A, 1 issues the products, 2 loads Q and its scales, 3 owns
// the tensor memory, 4-7 store the results (of the last tile, while the next
// one's sum runs in the other half of tensor memory), 8-15 convert.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "block128.h"
#include "block128_host.h"
#include "sm100.cuh"

namespace ofld {
namespace kern {

namespace {

using namespace sm100;

constexpr uint32_t kSide = 128;  // rows of A and columns of Q of one CTA
constexpr uint32_t kStep = 64;   // of t
// The tensor core's fp32 additions round towards zero, so their error grows
// with their number: 8192 steps of t, 512 additions, leave a result of normal
// values 3e-6 off, 70000 5e-5. Longer sums are taken in runs of 8192 terms,
// 2048 for results in fp32 (1e-6 off; terms in three parts 640). The storing
// warps add the runs up in tensor memory, rounding to nearest. In fp32 they
// add each to the output as it is stored, if it can be stored in tiles and the
// sum is not split: one tile has one owner, which waits for a run's stores
// before it sends the next, so the order of the additions never changes.
constexpr uint32_t kRun = 8192 / kStep, kRunFp32 = 2048 / kStep;
constexpr uint32_t kGroups = 2, kGroupWarps = 4;  // of converters: a group takes every second step
constexpr uint32_t kThreads = 512;

// Codes of waits that ran out.
enum : uint32_t {
    kWaitAEmpty = 201,
    kWaitQEmpty,
    kWaitBEmpty,
    kWaitAFull,
    kWaitQFull,
    kWaitBFull,
    kWaitTmemEmpty,
    kWaitTmemFull
};

constexpr uint32_t kOddThreads = 1024;

struct Args {
    const float* scales;
    void* out;
    int64_t ld;
    uint32_t ni, nj, nt, nb;
    uint32_t tiles_i, tiles_j, split;
    int type;  // FloatType
    bool tiled;  // the output can be stored in tiles (16-byte rows)
    const uint32_t* odd;  // pairs: words of k_odd, any of them not 0 where a scale is no power of two; null: assume so
    uint32_t odd_words;
    uint32_t* error;
};

// A_T: A is stored with t as its row. CG: CTAs on one tile.
template <bool A_T_, int CG_>
struct Config {
    static constexpr bool A_T = A_T_;
    static constexpr int CG = CG_;
    static constexpr uint32_t BN = kSide * CG;
    static constexpr uint32_t a_bytes = kSide * kStep * 2, q_bytes = kSide * kStep, b_bytes = kSide * kStep * 2;
    // Tiles in flight. From its load to the end of its product a tile of A
    // lives about 3700 cycles, one of Q (until it is converted) 2500, a
    // converted one 2000; a step takes 512.
    static constexpr uint32_t NA = 6, NQ = 6, NB = 4;
    static constexpr uint32_t off_q = NA * a_bytes, off_b = off_q + NQ * q_bytes, off_out = off_b + NB * b_bytes;
    static constexpr uint32_t out_bytes = 32 * 64;  // of one storing warp: 32 rows of 64 bytes, twice
    static constexpr uint32_t off_scale = off_out + 4 * 2 * out_bytes;
    static constexpr uint32_t off_bar = off_scale + NQ * kStep * 4;
    static constexpr uint32_t off_misc = off_bar + (2 * (NA + NQ + NB) + 4) * 8;
    static_assert(off_misc % 8 == 0, "a barrier there");
    static constexpr uint32_t smem = off_misc + 16 + 1024;
    static constexpr uint32_t tmem_cols = 2 * BN;
    static_assert(smem <= 227 * 1024 && tmem_cols <= 512, "");
    static_assert(off_out % (2 * out_bytes) == 0, "turns by one bit");
    static_assert(a_bytes % 1024 == 0 && q_bytes % 1024 == 0 && b_bytes % 1024 == 0 && out_bytes % 1024 == 0, "");
    // A slot always belongs to one group of converters: a group that saw only
    // some uses of a slot could take one phase of its barrier for another. With
    // several parts to a step that takes a ring for each group.
    static_assert(NQ % kGroups == 0 && NB % kGroups == 0, "");
    static constexpr uint32_t NBG = NB / kGroups;
    static constexpr uint32_t part_pitch = BN + 4;  // words of a row of partial sums: rows on different banks
    static_assert(off_out >= kSide * part_pitch * 4, "the split reduction's tile");
};

// Position in a ring of N.
template <uint32_t N>
struct Ring {
    uint32_t at = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) at = 0, phase ^= 1;
    }
};

__device__ __forceinline__ uint32_t pack16(int type, float lo, float hi) {
    if (type == 0) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_one(const Args& a, int64_t at, float v) {
    if (a.type == 0)
        static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
    else if (a.type == 1)
        static_cast<__half*>(a.out)[at] = __float2half_rn(v);
    else
        static_cast<float*>(a.out)[at] = v;
}
// The runs of a part of the sum, and the buffers of tensor memory that take
// them in turn: both, or where the runs are added up there, the first, with
// the second for their total.
struct Runs {
    bool added, total;
    uint32_t length, at = 0, phase = 0;
    __device__ __forceinline__ Runs(const Args& a, uint32_t steps, uint32_t parts) {
        added = a.type == 2 && a.tiled && a.split == 1;
        length = a.type == 2 ? kRunFp32 / parts : kRun;
        total = !added && steps > length;
    }
    __device__ __forceinline__ void next() {
        if (++at == (total ? 1 : 2)) at = 0, phase ^= 1;
    }
};

// A scale that is no power of two (or 0, or infinite).
__device__ __forceinline__ bool is_odd(float s) { return (__float_as_uint(s) & 0x7fffffu) != 0; }

// Whether any of `count` scales is odd, one word for each CTA.
__global__ void __launch_bounds__(kOddThreads)
    k_odd(const float* __restrict__ scales, uint64_t count, uint32_t* words) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    bool any = false;
#pragma unroll 8
    for (uint64_t i = blockIdx.x * kOddThreads + threadIdx.x; i < count; i += uint64_t(gridDim.x) * kOddThreads)
        any |= is_odd(__ldg(scales + i));
    any = __syncthreads_or(any);
    if (threadIdx.x == 0) words[blockIdx.x] = any;
}

// bf16 of two values. What is too large becomes the largest finite value, so
// that there is something left for the next part.
__device__ __forceinline__ uint32_t pack_finite(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
// Part AT of two values: the rounding of what AT parts have left over; the LAST one may be infinite.
template <int AT, bool LAST>
__device__ __forceinline__ uint32_t part2(float lo, float hi) {
#pragma unroll
    for (int i = 0; i < AT; ++i) {
        const uint32_t w = pack_finite(lo, hi);
        lo -= __uint_as_float(w << 16);
        hi -= __uint_as_float(w & 0xffff0000u);
    }
    return LAST ? pack16(0, lo, hi) : pack_finite(lo, hi);
}
// Four e4m3 values times a scale, as bf16.
template <int AT, bool LAST>
__device__ __forceinline__ uint2 convert4(uint32_t w, float s) {
    const __half2 lo(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w & 0xffff), __NV_E4M3));
    const __half2 hi(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w >> 16), __NV_E4M3));
    const float2 a = __half22float2(lo), b = __half22float2(hi);
    return make_uint2(part2<AT, LAST>(a.x * s, a.y * s), part2<AT, LAST>(b.x * s, b.y * s));
}
template <int AT, bool LAST>
__device__ __forceinline__ void convert16(uint4 w, float s, uint4* o) {
    const uint2 c0 = convert4<AT, LAST>(w.x, s), c1 = convert4<AT, LAST>(w.y, s);
    const uint2 c2 = convert4<AT, LAST>(w.z, s), c3 = convert4<AT, LAST>(w.w, s);
    o[0] = make_uint4(c0.x, c0.y, c1.x, c1.y);
    o[1] = make_uint4(c2.x, c2.y, c3.x, c3.y);
}
// Half a row, 64 columns: four chunks of 16 bytes of Q that become eight of
// the operand, each at its place in the 128-byte swizzle. The two halves take
// the chunks in different order, which keeps eight lanes on eight banks.
struct HalfRow {
    uint32_t h, swz;
    __device__ __forceinline__ uint4 load(const uint8_t* q, uint32_t i) const {
        return *reinterpret_cast<const uint4*>(q + (((i ^ 2 * h) + 4 * h) ^ swz) * 16);
    }
    __device__ __forceinline__ void store(uint8_t* d, uint32_t i, uint4 v) const {
        *reinterpret_cast<uint4*>(d + ((i ^ 4 * h) ^ swz) * 16) = v;
    }
    template <int AT, bool LAST>
    __device__ __forceinline__ void convert(const uint8_t* q, float s, uint8_t* d) const {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            uint4 o[2];
            convert16<AT, LAST>(load(q, i), s, o);
            store(d, 2 * i, o[0]);
            store(d, 2 * i + 1, o[1]);
        }
    }
};

template <typename C>
__global__ void __launch_bounds__(kThreads, 1)
    k_grad(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_q,
           const __grid_constant__ CUtensorMap map_out, const Args a) {
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    uint8_t* const sm = raw + (base - smem_addr(raw));
    const uint32_t bar = base + C::off_bar;
    auto a_full = [&](uint32_t s) { return bar + 8 * s; };  // in a pair: both CTAs' tiles, on the first one's barrier
    auto a_empty = [&](uint32_t s) { return bar + 8 * (C::NA + s); };
    auto q_full = [&](uint32_t s) { return bar + 8 * (2 * C::NA + s); };  // with its scales
    auto q_empty = [&](uint32_t s) { return bar + 8 * (2 * C::NA + C::NQ + s); };
    // converted, in every CTA of the tile
    auto b_full = [&](uint32_t s) { return bar + 8 * (2 * (C::NA + C::NQ) + s); };
    auto b_empty = [&](uint32_t s) { return bar + 8 * (2 * (C::NA + C::NQ) + C::NB + s); };
    auto tfull = [&](uint32_t b) { return bar + 8 * (2 * (C::NA + C::NQ + C::NB) + b); };
    auto tempty = [&](uint32_t b) { return bar + 8 * (2 * (C::NA + C::NQ + C::NB) + 2 + b); };
    // tensor memory, abort, a barrier for the end of an aborted launch
    volatile uint32_t* const misc = reinterpret_cast<volatile uint32_t*>(sm + C::off_misc);
    const uint32_t drained = base + C::off_misc + 8;
    const Guard guard{misc + 1, a.error};

    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t in_cluster = C::CG == 2 || a.split > 1 ? cluster_rank() : 0;
    const uint32_t half = C::CG == 2 ? in_cluster : 0;  // which CTA of the pair
    const uint32_t part = C::CG == 1 ? in_cluster : 0;  // which part of the sum
    const uint32_t group = C::CG == 2 ? 2 : a.split;
    const uint32_t first_tile = blockIdx.x / group, step = gridDim.x / group, tiles = a.tiles_i * a.tiles_j;
    const uint32_t steps = (a.nt + kStep - 1) / kStep;
    const uint32_t t0 = uint32_t(uint64_t(steps) * part / a.split);
    const uint32_t t1 = uint32_t(uint64_t(steps) * (part + 1) / a.split);

    // Tiles in groups of 8 row tiles, those fastest: what is in flight shares
    // its rows of A and columns of Q through L2.
    auto place = [&](uint32_t t, uint32_t* i0, uint32_t* j0) {
        const uint32_t per = 8 * a.tiles_j, g = t / per, first = g * 8, in = t - g * per;
        const uint32_t wide = min(8u, a.tiles_i - first);
        *i0 = (first + in % wide) * kSide * C::CG + half * kSide;  // this CTA's rows
        *j0 = in / wide * C::BN;                                   // the tile's columns
    };

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < C::NA; ++s) mbar_init(a_full(s), 1), mbar_init(a_empty(s), 1);
        // the load's thread, and each lane that fetches scales
        for (uint32_t s = 0; s < C::NQ; ++s) mbar_init(q_full(s), 1 + 32), mbar_init(q_empty(s), kGroupWarps);
        for (uint32_t s = 0; s < C::NB; ++s) mbar_init(b_full(s), kGroupWarps * C::CG), mbar_init(b_empty(s), 1);
        for (uint32_t b = 0; b < 2; ++b) mbar_init(tfull(b), 1), mbar_init(tempty(b), 4 * C::CG);
        mbar_init(drained, 1);
        mbar_init_fence();
        misc[1] = 0;
    }
    if (warp == 3) tmem_alloc<C::CG>(base + C::off_misc, C::tmem_cols);
    bool odd = false;
    if (C::CG == 1 && first_tile < tiles) {  // its one tile: a part of a column of scales
        uint32_t i0, j0;
        place(first_tile, &i0, &j0);
#pragma unroll 4
        for (uint32_t row = t0 * kStep + threadIdx.x; row < min(t1 * kStep, a.nt); row += kThreads)
            odd |= is_odd(__ldg(a.scales + uint64_t(row) * a.nb + j0 / 128));
    }
    if (C::CG == 2) {
        odd = !a.odd;
        grid_wait();
        if (threadIdx.x < a.odd_words) odd |= *reinterpret_cast<const volatile uint32_t*>(a.odd + threadIdx.x) != 0;
    }
    tc_fence_before();
    // one value for a warp, as for `warp` above: 688 us for 8192 x 4096 x 14336, else 780
    odd = __shfl_sync(0xffffffffu, __syncthreads_or(odd), 0);
    if (C::CG == 2)
        cluster_sync();
    else if (a.split > 1)
        cluster_arrive();  // waited for where the parts meet
    tc_fence_after();
    const uint32_t tmem = misc[0];

    // of a step's tile of Q, where there are several
    const uint32_t parts = a.type == 2 ? 3 : 2;

    if (warp == 0) {
        const bool leader = elect_one();
        if (leader) prefetch_map(&map_a);
        Ring<C::NA> r;
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t i0, j0;
            place(t, &i0, &j0);
            for (uint32_t k = t0; k < t1; ++k, ++it, r.next()) {
                ok = __all_sync(0xffffffffu, mbar_wait(a_empty(r.at), r.phase ^ 1, guard, kWaitAEmpty));
                if (!ok) break;
                if (leader) {
                    const uint32_t dst = base + r.at * C::a_bytes;
                    if (half == 0) mbar_expect(a_full(r.at), C::a_bytes * C::CG);
                    const uint32_t b = C::CG == 2 ? map_to_rank(a_full(r.at), 0) : a_full(r.at);
                    auto load = [&](uint32_t to, int32_t x, int32_t y) {
                        if (C::CG == 2)
                            tma_load_pair(to, &map_a, x, y, b);
                        else
                            tma_load(to, &map_a, x, y, b);
                    };
                    if (C::A_T) {
                        load(dst, i0, k * kStep);
                        load(dst + C::a_bytes / 2, i0 + 64, k * kStep);
                    } else {
                        load(dst, k * kStep, i0);
                    }
                }
                __syncwarp();
            }
        }
        if (*guard.abort && leader && half == 0) {  // let copies in flight land before the block retires
            const long long c0 = clock64();
            for (uint32_t i = it > C::NA ? it - C::NA : 0; i < it; ++i)
                while (!mbar_test(a_full(i % C::NA), i / C::NA & 1) && clock64() - c0 < kWaitCycles / 8) {
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        auto issue = [&](auto in_parts) {
            constexpr bool PARTS = decltype(in_parts)::value;
            constexpr uint32_t idesc = instr_desc(kSide * C::CG, C::BN, 1, C::A_T, true);
            // 16 steps of t: 32 bytes of a row, or 16 rows of 128 bytes
            constexpr uint32_t a_next = C::A_T ? 2048 >> 4 : 32 >> 4, b_next = 2048 >> 4;
            const bool leader = elect_one();
            Ring<C::NA> ra;
            Ring<PARTS ? C::NBG : C::NB> rb, rb_other;  // of the group whose turn it is, and of the other
            uint32_t turn = 0;
            Runs rt(a, t1 - t0, PARTS ? parts : 1);
            bool ok = true;
            for (uint32_t t = first_tile; ok && t < tiles; t += step) {
                uint32_t in_run = 0;
                for (uint32_t k = t0; k < t1; ++k, ra.next()) {
                    const bool first = in_run == 0, last = k + 1 == t1 || in_run + 1 == rt.length;
                    in_run = last ? 0 : in_run + 1;
                    ok = (!first || mbar_wait<C::CG == 2>(tempty(rt.at), rt.phase ^ 1, guard, kWaitTmemEmpty)) &&
                         mbar_wait(a_full(ra.at), ra.phase, guard, kWaitAFull);
#pragma unroll 1
                    for (uint32_t p = 0; p < (PARTS ? parts : 1); ++p, rb.next()) {
                        const uint32_t slot = PARTS ? rb.at * kGroups + turn : rb.at;
                        ok = ok && mbar_wait<C::CG == 2>(b_full(slot), rb.phase, guard, kWaitBFull);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
                            const uint64_t da = operand_desc(base + ra.at * C::a_bytes, C::A_T ? C::a_bytes / 2 : 16);
                            const uint64_t db = operand_desc(base + C::off_b + slot * C::b_bytes, C::b_bytes / 2);
#pragma unroll
                            for (uint32_t i = 0; i < kStep / 16; ++i)
                                mma_f16<C::CG>(tmem + rt.at * C::BN, da + i * a_next, db + i * b_next, idesc,
                                               !first || p > 0 || i > 0);
                            const bool whole = !PARTS || p + 1 == parts;
                            if (whole) mma_commit<C::CG>(a_empty(ra.at));
                            mma_commit<C::CG>(b_empty(slot));
                            if (last && whole) mma_commit<C::CG>(tfull(rt.at));
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (last) rt.next();
                    if constexpr (PARTS) {
                        const auto r = rb;
                        rb = rb_other;
                        rb_other = r;
                        turn = (turn + 1) % kGroups;
                    }
                }
            }
            if (*guard.abort && leader) mma_drain<C::CG>(drained);
        };
        if (half == 0) {
            if (__builtin_expect(odd, 0))
                issue(std::true_type{});
            else
                issue(std::false_type{});
            __syncwarp();
        }
    } else if (warp == 2) {
        const bool leader = elect_one();
        if (leader) prefetch_map(&map_q);
        Ring<C::NQ> r;
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t i0, j0;
            place(t, &i0, &j0);
            const uint32_t j = j0 + half * kSide, jb = j / 128;
            for (uint32_t k = t0; k < t1; ++k, ++it, r.next()) {
                ok = __all_sync(0xffffffffu, mbar_wait(q_empty(r.at), r.phase ^ 1, guard, kWaitQEmpty));
                if (!ok) break;
                if (leader) {
                    mbar_expect(q_full(r.at), C::q_bytes);
                    tma_load(base + C::off_q + r.at * C::q_bytes, &map_q, j, k * kStep, q_full(r.at));
                }
                __syncwarp();
                const uint32_t dst = base + C::off_scale + r.at * kStep * 4;
#pragma unroll
                for (uint32_t i = 0; i < kStep; i += 32) {
                    const uint32_t row = k * kStep + i + lane;
                    const bool valid = row < a.nt && jb < a.nb;
                    cp_async4(dst + (i + lane) * 4, valid ? a.scales + uint64_t(row) * a.nb + jb : a.scales, valid);
                }
                cp_async_arrive(q_full(r.at));
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (*guard.abort && leader) {
            const long long c0 = clock64();
            for (uint32_t i = it > C::NQ ? it - C::NQ : 0; i < it; ++i)
                while (!mbar_test(q_full(i % C::NQ), i / C::NQ & 1) && clock64() - c0 < kWaitCycles / 8) {
                }
        }
        __syncwarp();
    } else if (warp >= 8) {
        const uint32_t mine = (warp - 8) / kGroupWarps, id = threadIdx.x % (kGroupWarps * 32);
        const uint32_t row = id / 2;
        const HalfRow at{id % 2, row % 8};
        auto convert = [&](auto in_parts) {
            constexpr bool PARTS = decltype(in_parts)::value;
            Ring<C::NQ> rq;
            Ring<PARTS ? C::NBG : C::NB> rb;
            uint32_t turn = 0;
            bool ok = true;
            auto slot = [&] { return PARTS ? rb.at * kGroups + mine : rb.at; };
            auto room = [&] {
                ok = mbar_wait(b_empty(slot()), rb.phase ^ 1, guard, kWaitBEmpty);
                return ok = __all_sync(0xffffffffu, ok);
            };
            auto written = [&] {
                fence_async_smem();
                __syncwarp();
                // The tensor core of this SM reads what was written here,
                // from this SM's shared memory: the fence above has put it
                // there, and the arrival at the first CTA of a pair, where
                // the product is issued, only has to come after it. A
                // release to the cluster would also wait for this SM's
                // global memory, 1300 to 1900 cycles a step.
                if (lane == 0) {
                    if (C::CG == 2)
                        mbar_arrive_remote(map_to_rank(b_full(slot()), 0));
                    else
                        mbar_arrive(b_full(slot()));
                }
            };
            for (uint32_t t = first_tile; ok && t < tiles; t += step) {
                for (uint32_t k = t0; k < t1; ++k, rq.next()) {
                    if (turn == mine) {
                        ok = mbar_wait(q_full(rq.at), rq.phase, guard, kWaitQFull);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        const uint8_t* q = sm + C::off_q + rq.at * C::q_bytes + row * 128;
                        const float f = reinterpret_cast<const float*>(sm + C::off_scale)[rq.at * kStep + row];
                        auto to = [&] {
                            return sm + C::off_b + slot() * C::b_bytes + at.h * (C::b_bytes / 2) + row * 128;
                        };
                        if constexpr (!PARTS) {  // converted before there is room for it
                            uint4 w[4], o[8];
#pragma unroll
                            for (uint32_t i = 0; i < 4; ++i) w[i] = at.load(q, i);
#pragma unroll
                            for (uint32_t i = 0; i < 4; ++i) convert16<0, true>(w[i], f, o + 2 * i);
                            if (!room()) break;
                            if (lane == 0) mbar_arrive(q_empty(rq.at));
                            uint8_t* d = to();
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) at.store(d, i, o[i]);
                            written();
                        } else {
#pragma unroll 1
                            for (uint32_t p = 0; p < parts; ++p, rb.next()) {
                                if (!room()) break;
                                if (p == 0)
                                    at.convert<0, false>(q, f, to());
                                else if (p + 1 < parts)
                                    at.convert<1, false>(q, f, to());
                                else if (p == 1)
                                    at.convert<1, true>(q, f, to());
                                else
                                    at.convert<2, true>(q, f, to());
                                written();
                            }
                            if (!ok) break;
                            if (lane == 0) mbar_arrive(q_empty(rq.at));
                        }
                    }
                    if constexpr (!PARTS) rb.next();
                    turn = turn + 1 == kGroups ? 0 : turn + 1;
                }
            }
        };
        if (__builtin_expect(odd, 0))
            convert(std::true_type{});
        else
            convert(std::false_type{});
    } else if (warp >= 4) {
        const uint32_t quad = warp % 4, my_lane = quad * 32 + lane;
        uint32_t stage = C::off_out + quad * 2 * C::out_bytes;  // the two take turns
        Runs rt(a, t1 - t0, odd ? parts : 1);
        bool ok = true;
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (C::CG == 2)
                    mbar_arrive_remote(map_to_rank(tempty(rt.at), 0));
                else
                    mbar_arrive(tempty(rt.at));
            }
            rt.next();
        };
        const uint32_t lanes = quad * 32 << 16;
        const bool share = C::CG == 1 && a.split > 1;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t i0, j0;
            place(t, &i0, &j0);
            const uint32_t row0 = i0 + quad * 32;
            auto store = [&](uint32_t from, bool add) {
                if (add && lane == 0) tma_store_wait();  // for the run before
#pragma unroll 1
                for (uint32_t c = 0; c < C::BN; c += 32) {
                    uint32_t v[32];
                    tmem_ld(from + c, v);
                    tmem_ld_keep(v);
                    if (share) {
                        // Partial sums meet in shared memory: the rings are free
                        // (the last product is done, one tile to a CTA).
                        uint32_t* to = reinterpret_cast<uint32_t*>(sm) + my_lane * C::part_pitch + c;
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4*>(to + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    } else if (row0 >= a.ni || j0 + c >= a.nj) {
                        // nothing of this piece is inside
                    } else if (a.tiled) {
                        // Through shared memory (in the 64-byte swizzle) and out as
                        // tiles: a lane's own stores would each touch a line of
                        // their own, and hold up the converters' traffic.
                        const uint32_t at = lane * 64, swz = lane / 2 % 4;
                        if (a.type == 2) {
#pragma unroll
                            for (int p = 0; p < 2; ++p) {
                                // nothing to send must not take a turn: the wait counts what was sent
                                if (j0 + c + 16 * p >= a.nj) break;
                                if (lane == 0) tma_store_wait_read();
                                __syncwarp();
#pragma unroll
                                for (uint32_t i = 0; i < 4; ++i)
                                    *reinterpret_cast<uint4*>(sm + stage + at + (i ^ swz) * 16) =
                                        make_uint4(v[16 * p + 4 * i], v[16 * p + 4 * i + 1], v[16 * p + 4 * i + 2],
                                                   v[16 * p + 4 * i + 3]);
                                fence_async_smem();
                                __syncwarp();
                                if (lane == 0) {
                                    if (add)
                                        tma_add(&map_out, base + stage, j0 + c + 16 * p, row0);
                                    else
                                        tma_store(&map_out, base + stage, j0 + c + 16 * p, row0);
                                }
                                stage ^= C::out_bytes;
                            }
                        } else {
                            if (lane == 0) tma_store_wait_read();
                            __syncwarp();
#pragma unroll
                            for (uint32_t i = 0; i < 4; ++i) {
                                uint32_t w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    w[k] = pack16(a.type, __uint_as_float(v[8 * i + 2 * k]),
                                                  __uint_as_float(v[8 * i + 2 * k + 1]));
                                *reinterpret_cast<uint4*>(sm + stage + at + (i ^ swz) * 16) =
                                    make_uint4(w[0], w[1], w[2], w[3]);
                            }
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0) tma_store(&map_out, base + stage, j0 + c, row0);
                            stage ^= C::out_bytes;
                        }
                    } else {
                        // Rows that start anywhere: turned around in shared memory,
                        // 16 columns at a time, so that lanes store neighbours.
                        float* turn = reinterpret_cast<float*>(sm + stage);
#pragma unroll
                        for (uint32_t p = 0; p < 2; ++p) {
                            __syncwarp();
#pragma unroll
                            for (uint32_t i = 0; i < 16; ++i)
                                turn[i * 32 + (lane ^ i)] = __uint_as_float(v[16 * p + i]);
                            __syncwarp();
                            const uint32_t i = lane % 16, col = j0 + c + 16 * p + i;
#pragma unroll 4
                            for (uint32_t r = lane / 16; r < 32; r += 2)
                                if (row0 + r < a.ni && col < a.nj)
                                    store_one(a, int64_t(row0 + r) * a.ld + col, turn[i * 32 + (r ^ i)]);
                        }
                    }
                    __syncwarp();
                }
            };
            for (uint32_t k = t0; k < t1; k += rt.length) {
                ok = __all_sync(0xffffffffu, mbar_wait(tfull(rt.at), rt.phase, guard, kWaitTmemFull));
                __syncwarp();
                if (!ok) break;
                tc_fence_after();
                if (!rt.total) {
                    store(tmem + rt.at * C::BN + lanes, k > t0);
                    release();
                    continue;
                }
#pragma unroll 1
                for (uint32_t c = 0; c < C::BN; c += 32) {  // total = run, or total + run
                    uint32_t v[32];
                    if (k > t0) {
                        uint32_t w[32];
                        tmem_ld(tmem + C::BN + c + lanes, w);
                        tmem_ld(tmem + c + lanes, v);
                        tmem_ld_keep(v);
                        tmem_ld_keep(w);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(w[i]));
                    } else {
                        tmem_ld(tmem + c + lanes, v);
                        tmem_ld_keep(v);
                    }
                    tmem_st(tmem + C::BN + c + lanes, v);
                }
                tmem_st_wait();
                release();
            }
            if (!ok) break;
            if (rt.total) {
                tc_fence_after();
                store(tmem + C::BN + lanes, false);
            }
        }
        if (lane == 0) tma_store_wait();
    }
    __syncwarp();
    if (C::CG == 1 && a.split > 1) {
        __syncthreads();
        cluster_wait();
        cluster_sync();
        uint32_t i0, j0;
        place(first_tile, &i0, &j0);
        // every CTA of the cluster adds its share of the rows, in the order of the parts
        const uint32_t from = kSide * part / a.split, rows = kSide * (part + 1) / a.split - from;
        for (uint32_t e = threadIdx.x; e < rows * (C::BN / 4); e += kThreads) {
            const uint32_t r = from + e / (C::BN / 4), c = e % (C::BN / 4) * 4;
            if (i0 + r >= a.ni || j0 + c >= a.nj) continue;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            for (uint32_t p = 0; p < a.split; ++p) {
                const float4 v = ld_cluster4(map_to_rank(base + (r * C::part_pitch + c) * 4, p));
                sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
            }
            const int64_t at = int64_t(i0 + r) * a.ld + j0 + c;
            if (a.tiled && j0 + c + 4 <= a.nj) {  // four columns start on 8 or 16 bytes
                if (a.type == 2)
                    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
                        make_float4(sum[0], sum[1], sum[2], sum[3]);
                else
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
                        make_uint2(pack16(a.type, sum[0], sum[1]), pack16(a.type, sum[2], sum[3]));
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (j0 + c + i < a.nj) store_one(a, at + i, sum[i]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (C::CG == 2 || a.split > 1) cluster_sync();
    if (warp == 3) {
        tc_fence_after();
        tmem_free<C::CG>(tmem, C::tmem_cols);
    }
}

template <typename C>
cudaError_t run(MatIn dy, int64_t dy_rows, int64_t dy_cols, const Block128In& q, MatOut out, FloatType type, int64_t ni,
                int64_t nj, int64_t nt, uint32_t split, GradWork work, cudaStream_t s) {
    Args a{};
    cudaError_t e = error_word(&a.error);
    if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(k_grad<C>), C::smem);
    CUtensorMap ma, mq, mo;
    if (e == cudaSuccess)
        e = tile_map(&ma, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dy.ptr, dy_cols, dy_rows, dy.ld * 2, 64,
                     C::A_T ? kStep : kSide);
    const int64_t esz = type == FloatType::kFp32 ? 4 : 2;
    a.tiled = reinterpret_cast<uintptr_t>(out.ptr) % 16 == 0 && out.ld * esz % 16 == 0;
    mo = ma;
    if (e == cudaSuccess && a.tiled)
        e = tile_map(&mo, type == FloatType::kBf16   ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                          : type == FloatType::kFp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                     out.ptr, nj, ni, out.ld * esz, uint32_t(64 / esz), 32, 64);
    if (e == cudaSuccess) e = tile_map(&mq, CU_TENSOR_MAP_DATA_TYPE_UINT8, q.q, nj, nt, q.ld, kSide, kStep);
    if (e != cudaSuccess) return e;
    a.scales = q.scales;
    a.out = out.ptr;
    a.ld = out.ld;
    a.ni = uint32_t(ni);
    a.nj = uint32_t(nj);
    a.nt = uint32_t(nt);
    a.nb = uint32_t((nj + 127) / 128);
    a.tiles_i = uint32_t((ni + kSide * C::CG - 1) / (kSide * C::CG));
    a.tiles_j = uint32_t((nj + C::BN - 1) / C::BN);
    const uint64_t scales = uint64_t(a.nb) * a.nt;
    if (C::CG == 2 && work.words && work.count) {
        a.odd = work.words;
        a.odd_words = uint32_t(std::min<uint64_t>(
            {work.count, uint64_t(sm_count()), kThreads, (scales + kOddThreads - 1) / kOddThreads}));
    }
    a.split = C::CG == 2 ? 1 : split;
    a.type = int(type);
    const uint64_t tiles = uint64_t(a.tiles_i) * a.tiles_j;
    if (tiles * a.split > 0x7fffffff) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::smem;
    cfg.stream = s;
    cfg.attrs = at;
    const uint32_t group = C::CG == 2 ? 2 : a.split;
    if (group > 1) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = group;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    if (a.odd) {  // starts while the scales are being read
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    const uint64_t units = a.split > 1 ? tiles : std::min<uint64_t>(tiles, uint64_t(sm_count()) / group);
    cfg.gridDim = dim3(uint32_t(units * group));
    if (a.odd) {
        k_odd<<<a.odd_words, kOddThreads, 0, s>>>(q.scales, scales, work.words);
        g_block128_launches.fetch_add(1, std::memory_order_relaxed);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    e = cudaLaunchKernelEx(&cfg, k_grad<C>, ma, mq, mo, a);
    g_block128_launches.fetch_add(1, std::memory_order_relaxed);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// A step takes a pair and a single CTA the same 0.45 us, and a pair does four
// times the work. So pairs, unless even the single CTAs' tiles leave half of
// the SMs idle: then single CTAs, and the sum in as many parts (of at least
// eight steps, under which joining them costs more than it saves) as there are
// SMs for. Microseconds with pairs / single / the rule's split:
//   32 single tiles x 224 steps  78 / 86 / 28 (4)     64 x 128  47 / 51 / 31 (2)
//   40 x 80  33 / 34 / 19 (3)   40 x 2  8.3 / 6.6 / -   112 x 64  37 / 42 / -   320 x 32  29 / 41 / -
int64_t single_tiles(int64_t ni, int64_t nj) { return (ni + 127) / 128 * ((nj + 127) / 128); }
bool in_pairs(int64_t ni, int64_t nj) { return single_tiles(ni, nj) * 2 > sm_count(); }
template <bool A_T>
cudaError_t choose(MatIn dy, int64_t dy_rows, int64_t dy_cols, const Block128In& q, MatOut out, FloatType type,
                   int64_t ni, int64_t nj, int64_t nt, GradWork work, cudaStream_t s) {
    const int64_t sms = sm_count(), tiles = single_tiles(ni, nj), steps = (nt + kStep - 1) / kStep;
    if (in_pairs(ni, nj)) return run<Config<A_T, 2>>(dy, dy_rows, dy_cols, q, out, type, ni, nj, nt, 1, work, s);
    const int64_t split = std::max<int64_t>(1, std::min<int64_t>({8, sms / tiles, steps / 8}));
    return run<Config<A_T, 1>>(dy, dy_rows, dy_cols, q, out, type, ni, nj, nt, uint32_t(split), work, s);
}

bool args_ok(const MatIn& dy, int64_t n, const Block128In& q, const MatOut& out, int64_t k, FloatType type) {
    auto aligned = [](const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    return aligned(dy.ptr) && dy.ld >= n && dy.ld % 8 == 0 && dy.ld < kMostPitch / 2 && aligned(q.q) && q.scales &&
           q.ld % 16 == 0 && q.ld >= k && q.ld < kMostPitch && out.ptr && out.ld >= k && int(type) >= 0 && int(type) <= 2;
}
bool work_ok(const GradWork& w) { return reinterpret_cast<uintptr_t>(w.words) % 4 == 0; }
bool dims_ok(int64_t a, int64_t b, int64_t c) {
    const int64_t most = 0x7fffff00;
    return a >= 0 && b >= 0 && c >= 0 && a <= most && b <= most && c <= most;
}

}  // namespace

uint32_t grad_work_words(int64_t ni, int64_t nj) {
    return ni > 0 && nj > 0 && in_pairs(ni, nj) ? uint32_t(sm_count()) : 0;
}

cudaError_t matmul_input_grad(MatIn dy, Block128In w, MatOut dx, FloatType type, int64_t m, int64_t n, int64_t k,
                              GradWork work, cudaStream_t s) {
    if (!dims_ok(m, n, k) || n == 0) return cudaErrorInvalidValue;
    if (m == 0 || k == 0) return cudaSuccess;
    if (!args_ok(dy, n, w, dx, k, type) || !work_ok(work)) return cudaErrorInvalidValue;
    return choose<false>(dy, m, n, w, dx, type, m, k, n, work, s);
}

cudaError_t matmul_weight_grad(MatIn dy, Block128In x, MatOut dw, FloatType type, int64_t m, int64_t n, int64_t k,
                               GradWork work, cudaStream_t s) {
    if (!dims_ok(m, n, k) || m == 0) return cudaErrorInvalidValue;
    if (n == 0 || k == 0) return cudaSuccess;
    if (!args_ok(dy, n, x, dw, k, type) || !work_ok(work)) return cudaErrorInvalidValue;
    return choose<true>(dy, m, n, x, dw, type, n, k, m, work, s);
}

}  // namespace kern
}  // namespace ofld
