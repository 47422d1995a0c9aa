// The two gradients of y = x w^T, each a bf16 matrix times a block-128 one:
//
//   input:  dx[m, k] = sum_n dy[m, n] w[n, k]       weight:  dw[n, k] = sum_m dy[m, n] x[m, k]
//
// Both are out[i, j] = sum_t A(i, t) Q[t, j] s[t, j / 128]: the 8-bit operand
// is stored with the summed index as its row, and its scale changes with the
// row, so it cannot leave the sum. Converter warps bring each tile of Q from
// 8 bits to bf16 in shared memory, times its scale (fp32 product, one rounding
// to bf16; none when the scale is a power of two, as in everything that
// quantize made), and the tensor core multiplies it with dy as it is
// (tcgen05.mma kind::f16, fp32 accumulators in tensor memory). The converted
// tile and, for the weight gradient, dy's are read "MN-major": their rows run
// along the output, not along the sum, so nothing is transposed.
//
// A pair of CTAs owns 256 x 256 outputs; each loads 128 rows of A and 128
// columns of Q for 64 steps of t, and converts its 8192 values while the
// tensor core spends 512 cycles on the step before. Few outputs: one CTA owns
// 128 x 128, and the sum is split over a cluster of up to 8.
//
// Warps: 0 loads, 1 issues the products, 2 fetches the scales, 3 owns the
// tensor memory, 4-7 store the results (of the last tile, while the next one's
// sum runs in the other half of tensor memory), 8-15 convert.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>

#include "block128.h"
#include "block128_host.h"
#include "sm100.cuh"

namespace ofld {
namespace kern {

namespace {

using namespace sm100;

constexpr uint32_t kSide = 128;  // rows of A and columns of Q of one CTA
constexpr uint32_t kStep = 64;   // of t
constexpr uint32_t kGroups = 2, kGroupWarps = 4;  // of converters: a group takes every second step
constexpr uint32_t kThreads = 512;

enum : uint32_t { kWaitEmpty = 201, kWaitFull, kWaitConverted, kWaitTmemEmpty, kWaitTmemFull };

struct Args {
    const float* scales;
    void* out;
    int64_t ld;
    uint32_t ni, nj, nt, nb;
    uint32_t tiles_i, tiles_j, split;
    int type;  // FloatType
    bool vec;  // 16-byte stores are aligned
    uint32_t* error;
};

// A_T: A is stored with t as its row. CG: CTAs on one tile.
template <bool A_T_, int CG_>
struct Config {
    static constexpr bool A_T = A_T_;
    static constexpr int CG = CG_, ST = 5;
    static constexpr uint32_t BN = kSide * CG;
    static constexpr uint32_t a_bytes = kSide * kStep * 2, q_bytes = kSide * kStep, b_bytes = kSide * kStep * 2;
    static constexpr uint32_t off_q = a_bytes, off_b = off_q + q_bytes, stage = off_b + b_bytes;
    static constexpr uint32_t off_scale = ST * stage;
    static constexpr uint32_t off_bar = off_scale + ST * kStep * 4;
    static constexpr uint32_t off_misc = off_bar + (3 * ST + 4) * 8;
    static constexpr uint32_t smem = off_misc + 16 + 1024;
    static constexpr uint32_t tmem_cols = 2 * BN;
    static_assert(smem <= 227 * 1024 && tmem_cols <= 512, "");
    static_assert(a_bytes % 1024 == 0 && q_bytes % 1024 == 0 && b_bytes % 1024 == 0, "");
    static_assert(ST * stage >= kSide * BN * 4 || CG == 2, "the split reduction's tile");
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
// Results of one row from column j on.
template <int N>
__device__ __forceinline__ void store_row(const Args& a, uint32_t row, uint32_t j, const uint32_t (&v)[N]) {
    const int64_t at = int64_t(row) * a.ld + j;
    if (a.vec && j + N <= a.nj) {
        if (a.type == 2) {
            uint4* p = reinterpret_cast<uint4*>(static_cast<float*>(a.out) + at);
#pragma unroll
            for (int i = 0; i < N; i += 4) p[i / 4] = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
            uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at);
#pragma unroll
            for (int i = 0; i < N; i += 8) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = pack16(a.type, __uint_as_float(v[i + 2 * k]), __uint_as_float(v[i + 2 * k + 1]));
                p[i / 8] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (j + i < a.nj) store_one(a, at + i, __uint_as_float(v[i]));
    }
}

// Four e4m3 values times a scale, as bf16.
__device__ __forceinline__ uint2 convert4(uint32_t w, float s) {
    const __half2 lo(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w & 0xffff), __NV_E4M3));
    const __half2 hi(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w >> 16), __NV_E4M3));
    const float2 a = __half22float2(lo), b = __half22float2(hi);
    return make_uint2(pack16(0, a.x * s, a.y * s), pack16(0, b.x * s, b.y * s));
}

template <typename C>
__global__ void __launch_bounds__(kThreads, 1)
    k_grad(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_q, const Args a) {
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    uint8_t* const sm = raw + (base - smem_addr(raw));
    const uint32_t bar = base + C::off_bar;
    auto full = [&](uint32_t s) { return bar + 8 * s; };                 // A, Q and the scales have landed
    auto ready = [&](uint32_t s) { return bar + 8 * (C::ST + s); };      // converted, in every CTA of the tile
    auto empty = [&](uint32_t s) { return bar + 8 * (2 * C::ST + s); };  // multiplied
    auto tfull = [&](uint32_t b) { return bar + 8 * (3 * C::ST + b); };
    auto tempty = [&](uint32_t b) { return bar + 8 * (3 * C::ST + 2 + b); };
    volatile uint32_t* const misc = reinterpret_cast<volatile uint32_t*>(sm + C::off_misc);  // tensor memory, abort
    const Guard guard{misc + 1, a.error};

    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t in_cluster = C::CG == 2 || a.split > 1 ? cluster_rank() : 0;
    const uint32_t half = C::CG == 2 ? in_cluster : 0;  // which CTA of the pair
    const uint32_t part = C::CG == 1 ? in_cluster : 0;  // which part of the sum
    const uint32_t group = C::CG == 2 ? 2 : a.split;
    const uint32_t first_tile = blockIdx.x / group, step = gridDim.x / group, tiles = a.tiles_i * a.tiles_j;
    const uint32_t steps = (a.nt + kStep - 1) / kStep;
    const uint32_t t0 = uint32_t(uint64_t(steps) * part / a.split), t1 = uint32_t(uint64_t(steps) * (part + 1) / a.split);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < C::ST; ++s) {
            mbar_init(full(s), 1 + 32);  // the loads' thread, and each lane that fetches scales
            mbar_init(ready(s), kGroupWarps * C::CG);
            mbar_init(empty(s), 1);
        }
        for (uint32_t b = 0; b < 2; ++b) mbar_init(tfull(b), 1), mbar_init(tempty(b), 4 * C::CG);
        mbar_init_fence();
        misc[1] = 0;
    }
    if (warp == 3) tmem_alloc<C::CG>(base + C::off_misc, C::tmem_cols);
    tc_fence_before();
    __syncthreads();
    if (C::CG == 2 || a.split > 1) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = misc[0];

    // Tiles in groups of 8 row tiles, those fastest: what is in flight shares
    // its rows of A and columns of Q through L2.
    auto place = [&](uint32_t t, uint32_t* i0, uint32_t* j0) {
        const uint32_t per = 8 * a.tiles_j, g = t / per, first = g * 8, in = t - g * per;
        const uint32_t wide = min(8u, a.tiles_i - first);
        *i0 = (first + in % wide) * kSide * C::CG + half * kSide;  // this CTA's rows
        *j0 = in / wide * C::BN;                                   // the tile's columns
    };

    if (warp == 0) {
        const bool leader = elect_one();
        if (leader) {
            prefetch_map(&map_a);
            prefetch_map(&map_q);
        }
        uint32_t it = 0, s = 0, phase = 1;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t i0, j0;
            place(t, &i0, &j0);
            for (uint32_t k = t0; k < t1; ++k, ++it) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty(s), phase, guard, kWaitEmpty));
                if (!ok) break;
                if (leader) {
                    const uint32_t dst = base + s * C::stage;
                    mbar_expect(full(s), C::a_bytes + C::q_bytes);
                    if (C::A_T) {
                        tma_load(dst, &map_a, i0, k * kStep, full(s));
                        tma_load(dst + C::a_bytes / 2, &map_a, i0 + 64, k * kStep, full(s));
                    } else {
                        tma_load(dst, &map_a, k * kStep, i0, full(s));
                    }
                    tma_load(dst + C::off_q, &map_q, j0 + half * kSide, k * kStep, full(s));
                }
                __syncwarp();
                if (++s == C::ST) s = 0, phase ^= 1;
            }
        }
        if (*guard.abort && leader) {  // let copies in flight land before the block retires
            const long long c0 = clock64();
            for (uint32_t i = it > C::ST ? it - C::ST : 0; i < it; ++i)
                while (!mbar_test(full(i % C::ST), i / C::ST & 1) && clock64() - c0 < kWaitCycles / 8) {
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (half == 0) {
            constexpr uint32_t idesc = instr_desc(kSide * C::CG, C::BN, 1, C::A_T, true);
            // 16 steps of t: 32 bytes of a row, or 16 rows of 128 bytes
            constexpr uint32_t a_next = C::A_T ? 2048 >> 4 : 32 >> 4, b_next = 2048 >> 4;
            const bool leader = elect_one();
            uint32_t s = 0, phase = 0, b = 0, bphase = 1;
            bool ok = true;
            for (uint32_t t = first_tile; ok && t < tiles; t += step) {
                ok = __all_sync(0xffffffffu, mbar_wait<C::CG == 2>(tempty(b), bphase, guard, kWaitTmemEmpty));
                if (!ok) break;
                for (uint32_t k = t0; k < t1; ++k) {
                    ok = __all_sync(0xffffffffu, mbar_wait<C::CG == 2>(ready(s), phase, guard, kWaitConverted));
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
                        const uint32_t src = base + s * C::stage;
                        const uint64_t da = operand_desc(src, C::A_T ? C::a_bytes / 2 : 16);
                        const uint64_t db = operand_desc(src + C::off_b, C::b_bytes / 2);
#pragma unroll
                        for (uint32_t i = 0; i < kStep / 16; ++i)
                            mma_f16<C::CG>(tmem + b * C::BN, da + i * a_next, db + i * b_next, idesc, k > t0 || i > 0);
                        mma_commit<C::CG>(empty(s));
                        if (k + 1 == t1) mma_commit<C::CG>(tfull(b));
                    }
                    __syncwarp();
                    if (++s == C::ST) s = 0, phase ^= 1;
                }
                b ^= 1;
                if (b == 0) bphase ^= 1;
            }
        }
    } else if (warp == 2) {
        uint32_t s = 0, phase = 1;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t i0, j0;
            place(t, &i0, &j0);
            const uint32_t jb = j0 / 128 + half;
            for (uint32_t k = t0; k < t1; ++k) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty(s), phase, guard, kWaitEmpty));
                if (!ok) break;
                const uint32_t dst = base + C::off_scale + s * kStep * 4;
#pragma unroll
                for (uint32_t i = 0; i < kStep; i += 32) {
                    const uint32_t r = k * kStep + i + lane;
                    const bool valid = r < a.nt && jb < a.nb;
                    cp_async4(dst + (i + lane) * 4, valid ? a.scales + uint64_t(r) * a.nb + jb : a.scales, valid);
                }
                cp_async_arrive(full(s));
                if (++s == C::ST) s = 0, phase ^= 1;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= 8) {
        const uint32_t mine = (warp - 8) / kGroupWarps, id = threadIdx.x % (kGroupWarps * 32);
        const uint32_t row = id / 2, h = id % 2, swz = row % 8;
        uint32_t s = 0, phase = 0, turn = 0;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            for (uint32_t k = t0; k < t1; ++k) {
                if (turn == mine) {
                    ok = __all_sync(0xffffffffu, mbar_wait(full(s), phase, guard, kWaitFull));
                    if (!ok) break;
                    // Half a row: 64 columns, four chunks of 16 bytes of Q that
                    // become eight of the operand, each at its place in the
                    // 128-byte swizzle. The two halves take the chunks in
                    // different order, which keeps eight lanes on eight banks.
                    const uint8_t* q = sm + s * C::stage + C::off_q + row * 128;
                    uint8_t* d = sm + s * C::stage + C::off_b + h * (C::b_bytes / 2) + row * 128;
                    const float f = reinterpret_cast<const float*>(sm + C::off_scale)[s * kStep + row];
                    uint4 w[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        w[i] = *reinterpret_cast<const uint4*>(q + (((i ^ 2 * h) + 4 * h) ^ swz) * 16);
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t c = 2 * (i ^ 2 * h);
                        const uint2 c0 = convert4(w[i].x, f), c1 = convert4(w[i].y, f);
                        const uint2 c2 = convert4(w[i].z, f), c3 = convert4(w[i].w, f);
                        *reinterpret_cast<uint4*>(d + (c ^ swz) * 16) = make_uint4(c0.x, c0.y, c1.x, c1.y);
                        *reinterpret_cast<uint4*>(d + ((c + 1) ^ swz) * 16) = make_uint4(c2.x, c2.y, c3.x, c3.y);
                    }
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
                            mbar_arrive_remote(map_to_rank(ready(s), 0));
                        else
                            mbar_arrive(ready(s));
                    }
                }
                turn = turn + 1 == kGroups ? 0 : turn + 1;
                if (++s == C::ST) s = 0, phase ^= 1;
            }
        }
    } else if (warp >= 4) {
        const uint32_t quad = warp % 4, my_lane = quad * 32 + lane;
        uint32_t b = 0, bphase = 0;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t i0, j0;
            place(t, &i0, &j0);
            ok = __all_sync(0xffffffffu, mbar_wait(tfull(b), bphase, guard, kWaitTmemFull));
            __syncwarp();
            if (!ok) break;
            tc_fence_after();
            const uint32_t row = i0 + my_lane;
            const bool share = C::CG == 1 && a.split > 1;
#pragma unroll 1
            for (uint32_t c = 0; c < C::BN; c += 32) {
                uint32_t v[32];
                tmem_ld(tmem + b * C::BN + c + (quad * 32 << 16), v);
                tmem_ld_keep(v);
                if (share) {
                    // Partial sums meet in shared memory: the stages are free
                    // (the last product is done, one tile to a CTA).
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        reinterpret_cast<uint32_t*>(sm)[(c + i) * kSide + my_lane] = v[i];
                } else if (row < a.ni && j0 + c < a.nj) {
                    store_row(a, row, j0 + c, v);
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (C::CG == 2)
                    mbar_arrive_remote(map_to_rank(tempty(b), 0));
                else
                    mbar_arrive(tempty(b));
            }
            b ^= 1;
            if (b == 0) bphase ^= 1;
        }
    }
    __syncwarp();
    if (C::CG == 1 && a.split > 1) {
        __syncthreads();
        cluster_sync();
        uint32_t i0, j0;
        place(first_tile, &i0, &j0);
        // every CTA of the cluster adds its share of the rows, in the order of the parts
        const uint32_t from = kSide * part / a.split, rows = kSide * (part + 1) / a.split - from;
        for (uint32_t e = threadIdx.x; e < rows * C::BN; e += kThreads) {
            const uint32_t r = from + e / C::BN, c = e % C::BN;
            if (i0 + r >= a.ni || j0 + c >= a.nj) continue;
            float sum = 0.f;
            for (uint32_t p = 0; p < a.split; ++p) sum += ld_cluster(map_to_rank(base + (c * kSide + r) * 4, p));
            store_one(a, int64_t(i0 + r) * a.ld + j0 + c, sum);
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
                int64_t nj, int64_t nt, uint32_t split, cudaStream_t s) {
    Args a{};
    cudaError_t e = error_word(&a.error);
    if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(k_grad<C>), C::smem);
    CUtensorMap ma, mq;
    if (e == cudaSuccess)
        e = tile_map(&ma, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dy.ptr, dy_cols, dy_rows, dy.ld * 2, 64,
                     C::A_T ? kStep : kSide);
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
    a.split = C::CG == 2 ? 1 : split;
    a.type = int(type);
    const int64_t esz = type == FloatType::kFp32 ? 4 : 2;
    a.vec = reinterpret_cast<uintptr_t>(out.ptr) % 16 == 0 && out.ld * esz % 16 == 0;
    const uint64_t tiles = uint64_t(a.tiles_i) * a.tiles_j;
    if (tiles * a.split > 0x7fffffff) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
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
    const uint64_t units = a.split > 1 ? tiles : std::min<uint64_t>(tiles, uint64_t(sm_count()) / group);
    cfg.gridDim = dim3(uint32_t(units * group));
    e = cudaLaunchKernelEx(&cfg, k_grad<C>, ma, mq, a);
    g_block128_launches.fetch_add(1, std::memory_order_relaxed);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// Pairs of CTAs once their tiles fill the GPU, else single CTAs with the sum
// in as many parts as there are SMs for, of two steps at least.
template <bool A_T>
cudaError_t choose(MatIn dy, int64_t dy_rows, int64_t dy_cols, const Block128In& q, MatOut out, FloatType type,
                   int64_t ni, int64_t nj, int64_t nt, cudaStream_t s) {
    const int64_t sms = sm_count(), pairs = (ni + 255) / 256 * ((nj + 255) / 256);
    if (pairs * 2 >= sms) return run<Config<A_T, 2>>(dy, dy_rows, dy_cols, q, out, type, ni, nj, nt, 1, s);
    const int64_t tiles = (ni + 127) / 128 * ((nj + 127) / 128), steps = (nt + kStep - 1) / kStep;
    uint32_t split = 1;
    while (split < 8 && tiles * split * 2 <= sms && steps >= split * 4) split *= 2;
    return run<Config<A_T, 1>>(dy, dy_rows, dy_cols, q, out, type, ni, nj, nt, split, s);
}

bool args_ok(const MatIn& dy, int64_t n, const Block128In& q, const MatOut& out, int64_t k, FloatType type) {
    auto aligned = [](const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    return aligned(dy.ptr) && dy.ld >= n && dy.ld % 8 == 0 && aligned(q.q) && q.scales && q.ld % 16 == 0 &&
           q.ld >= k && out.ptr && out.ld >= k && int(type) >= 0 && int(type) <= 2;
}
bool dims_ok(int64_t a, int64_t b, int64_t c) {
    const int64_t most = 0x7fffff00;
    return a >= 0 && b >= 0 && c >= 0 && a <= most && b <= most && c <= most;
}

}  // namespace

cudaError_t matmul_input_grad(MatIn dy, Block128In w, MatOut dx, FloatType type, int64_t m, int64_t n, int64_t k,
                              cudaStream_t s) {
    if (!dims_ok(m, n, k) || n == 0) return cudaErrorInvalidValue;
    if (m == 0 || k == 0) return cudaSuccess;
    if (!args_ok(dy, n, w, dx, k, type)) return cudaErrorInvalidValue;
    return choose<false>(dy, m, n, w, dx, type, m, k, n, s);
}

cudaError_t matmul_weight_grad(MatIn dy, Block128In x, MatOut dw, FloatType type, int64_t m, int64_t n, int64_t k,
                               cudaStream_t s) {
    if (!dims_ok(m, n, k) || m == 0) return cudaErrorInvalidValue;
    if (n == 0 || k == 0) return cudaSuccess;
    if (!args_ok(dy, n, x, dw, k, type)) return cudaErrorInvalidValue;
    return choose<true>(dy, m, n, x, dw, type, n, k, m, s);
}

}  // namespace kern
}  // namespace ofld
