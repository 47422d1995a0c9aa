// y = x w^T on the fp8 tensor cores, both operands block-128.
//
//   y[m, n] = sum_b sw[n, b] P_b[m, n],   P_b[m, n] = sx[m, b] sum_{k in b} qx[m, k] qw[n, k]
//
// x's scales are powers of two (the call quantises x itself), so they go into
// the tensor core as e8m0 factors (kind::mxf8f6f4). w's are any fp32 numbers
// and change with every block of the sum: each P_b (four tcgen05.mma of 32
// values) goes to one of several buffers of tensor memory, and the epilogue
// warps add sw P_b to fp32 registers while the next block's product runs.
//
// A P_b can be far larger than what it adds to y, since the weight's scale is
// not in it: activations of 2^128 times 448, 128 of them, would overflow. So
// the factor of all weights is 2^-16 and not 1, which keeps every P_b in range
// (subnormal ones lose nothing: the tensor core keeps them), and the sum gets
// 2^16 back as it is stored. Results under 2^-110 give bits for that. (2^16 in
// sw instead, with a way out for scales over 2^111, took 5 % more time.)
//
// The rows of w lie on the 128 lanes of tensor memory, so that sw is one
// register of each epilogue thread and the addition one multiply-add for a
// result; the tokens lie on its BN columns. With few tokens the tile then
// holds little but weights.
//
// Many tokens: a pair of CTAs owns 256 x 224 results. A block of the sum takes
// the tensor core 448 cycles and the epilogue 112 multiply-adds a lane, 224
// issue slots of each scheduler. 4096 x 5120 x 27648: 540 us (2.1 PFLOP/s); with
// x's quantisation 567, in a loop of seconds 666. A block takes about 800
// cycles: the issuing warp is busy for 690 of them (two in turn were no
// faster), the epilogue for all. At 1000 W the SMs run at 1.6 GHz; without the
// epilogue's arithmetic they run at 1.48 GHz and need 416 us, so the power cap
// would take most of what fewer cycles gave.
// Few tokens: the bytes of w, in tiles of 128 rows x 16, 32 or 64 tokens, the
// sum in parts over a cluster. 16 tokens x 4096 x 14336: 14.9 us (4 TB/s), one
// token x 5120 x 5120: 10.2 us, of which 3 to 4 are starting and joining.
//
// Warps: 0 loads (TMA in the 128-byte swizzle), 1 issues the products, 2 owns
// the tensor memory, 3 idles, the rest are the epilogue.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "block128.h"
#include "block128_host.h"
#include "sm100.cuh"

namespace ofld {
namespace kern {

namespace {

using namespace sm100;

constexpr uint32_t kLanes = 128, kBlock = 128;
constexpr uint32_t kDown = 0x6f6f6f6fu;  // e8m0 of 2^-16
constexpr float kUp = 65536.f;

// Codes of waits that ran out.
enum : uint32_t { kWaitEmpty = 101, kWaitFull, kWaitTmemEmpty, kWaitTmemFull };

struct Args {
    const float* scale_w;
    const void* bias;
    void* out;
    int64_t ld;
    uint32_t m, n, nb;
    uint32_t tiles_n, tiles_m, split;
    int type;  // FloatType
    uint32_t* error;
};

// BN columns, CG CTAs on one tile (2: 256 rows of w, each CTA loads its own
// and half of the tokens), EW epilogue warps, ST stages, NBUF buffers of
// tensor memory.
template <int BN_, int CG_, int EW_, int ST_, int NBUF_, int PER_SM_>
struct Config {
    static constexpr int BN = BN_, CG = CG_, EW = EW_, ST = ST_, NBUF = NBUF_, per_sm = PER_SM_;
    static constexpr int threads = 128 + 32 * EW;
    static constexpr uint32_t w_bytes = kLanes * kBlock, x_bytes = BN / CG * kBlock;
    static constexpr uint32_t sx_words = (BN + 127) / 128 * 128;
    static constexpr uint32_t stage_bytes = w_bytes + x_bytes + sx_words * 4;
    static constexpr uint32_t stage_pitch = (stage_bytes + 1023) / 1024 * 1024;
    static constexpr uint32_t tmem_sx = NBUF * BN;             // factors of x: four columns for 128 tokens
    static constexpr uint32_t tmem_sw = tmem_sx + sx_words / 32;  // factors of w: all 2^-16
    static constexpr uint32_t tmem_used = tmem_sw + 4;
    static constexpr uint32_t tmem_cols = tmem_used <= 64 ? 64 : tmem_used <= 128 ? 128 : tmem_used <= 256 ? 256 : 512;
    static constexpr uint32_t off_bar = ST * stage_pitch;
    static constexpr uint32_t off_misc = off_bar + (2 * ST + 2 * NBUF) * 8;
    static_assert(off_misc % 8 == 0, "a barrier there");
    static constexpr uint32_t smem = off_misc + 16 + 1024;  // + alignment of the base
    static constexpr int CPT = BN / (EW / 4);                  // columns of one epilogue thread
    static constexpr int CH = CPT % 32 ? 16 : 32;            // columns of one tensor-memory load
    // The epilogue reads all its columns of a product before the arithmetic, so
    // that the buffer is free early.
    // 224 columns a pair take more registers for that than an even share: the
    // four warps that are not the epilogue give up theirs.
    static constexpr bool SHIFT = CPT > 64;
    static_assert(!SHIFT || EW == 8, "");
    static constexpr int kEven = 168, kFew = 40, kMany = 232;
    static_assert(!SHIFT || 128 * kFew + 256 * kMany <= 384 * kEven, "a split that the block has registers for");
    static_assert(tmem_used <= 512 && tmem_cols * per_sm <= 512, "tensor memory");
    static_assert(smem * per_sm <= 227 * 1024, "shared memory");
    static_assert(CPT % CH == 0 && BN % 16 == 0 && (CG == 1 || BN % 32 == 0), "");
    static_assert(x_bytes % 1024 == 0 && w_bytes % 1024 == 0, "operands start on the swizzle's 1024 bytes");
    // the split reduction keeps a 128 x BN fp32 tile in the stages
    static_assert(CG == 2 || ST * stage_pitch >= kLanes * BN * 4, "");
};

template <typename T>
__device__ __forceinline__ float as_float(const void* p, uint32_t i) {
    return float(static_cast<const T*>(p)[i]);
}
__device__ __forceinline__ float bias_at(const Args& a, uint32_t i) {
    return a.type == 0 ? as_float<__nv_bfloat16>(a.bias, i) : a.type == 1 ? as_float<__half>(a.bias, i)
                                                                        : as_float<float>(a.bias, i);
}
template <typename T>
__device__ __forceinline__ T rounded(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 rounded(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half rounded(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float rounded(float v) { return v; }

__device__ __forceinline__ void store_one(const Args& a, int64_t at, float v) {
    if (a.type == 0)
        static_cast<__nv_bfloat16*>(a.out)[at] = rounded<__nv_bfloat16>(v);
    else if (a.type == 1)
        static_cast<__half*>(a.out)[at] = rounded<__half>(v);
    else
        static_cast<float*>(a.out)[at] = v;
}
// One lane's results: output `row` for tokens c0 and on.
template <typename T, int N>
__device__ __forceinline__ void store_column(const Args& a, uint32_t row, uint32_t c0, const float (&acc)[N],
                                             float add) {
    T* p = static_cast<T*>(a.out) + int64_t(c0) * a.ld + row;
    const uint32_t left = a.m > c0 ? a.m - c0 : 0;
#pragma unroll
    for (int i = 0; i < N; ++i, p += a.ld)
        if (uint32_t(i) < left) *p = rounded<T>(fmaf(acc[i], kUp, add));
}

template <typename C>
__global__ void __launch_bounds__(C::threads, C::per_sm)
    k_linear(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
             const __grid_constant__ CUtensorMap map_sx, const Args a) {
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    uint8_t* const sm = raw + (base - smem_addr(raw));
    const uint32_t bar = base + C::off_bar;
    auto full = [&](uint32_t s) { return bar + 8 * s; };
    auto empty = [&](uint32_t s) { return bar + 8 * (C::ST + s); };
    auto tfull = [&](uint32_t b) { return bar + 8 * (2 * C::ST + b); };
    auto tempty = [&](uint32_t b) { return bar + 8 * (2 * C::ST + C::NBUF + b); };
    // tensor memory, abort, a barrier for the end of an aborted launch
    volatile uint32_t* const misc = reinterpret_cast<volatile uint32_t*>(sm + C::off_misc);
    const uint32_t drained = base + C::off_misc + 8;
    const Guard guard{misc + 1, a.error};

    // one value for a warp, so that what the issuing warps compute stays in uniform registers
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t in_cluster = C::CG == 2 || a.split > 1 ? cluster_rank() : 0;
    const uint32_t half = C::CG == 2 ? in_cluster : 0;  // which CTA of the pair
    const uint32_t part = C::CG == 1 ? in_cluster : 0;  // which part of the sum
    const uint32_t group = C::CG == 2 ? 2 : a.split;
    const uint32_t first_tile = blockIdx.x / group, step = gridDim.x / group, tiles = a.tiles_n * a.tiles_m;
    const uint32_t kb0 = uint32_t(uint64_t(a.nb) * part / a.split);
    const uint32_t kb1 = uint32_t(uint64_t(a.nb) * (part + 1) / a.split);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < C::ST; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
        for (uint32_t b = 0; b < C::NBUF; ++b) mbar_init(tfull(b), 1), mbar_init(tempty(b), C::EW * C::CG);
        mbar_init(drained, 1);
        mbar_init_fence();
        misc[1] = 0;
    }
    if (warp == 2) tmem_alloc<C::CG>(base + C::off_misc, C::tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    if (warp >= 4 && warp < 8) tmem_fill4(tmem + C::tmem_sw + (warp % 4 * 32 << 16), kDown);
    tc_fence_before();
    __syncthreads();
    if (C::CG == 2)
        cluster_sync();
    else if (a.split > 1)
        cluster_arrive();  // waited for where the parts meet
    tc_fence_after();

    // Tiles in groups of 16 row tiles of w, those fastest: what is in flight
    // shares few token tiles and at most 16 of w through L2.
    auto place = [&](uint32_t t, uint32_t* n0, uint32_t* tm) {
        const uint32_t per = 16 * a.tiles_m, g = t / per, first = g * 16, in = t - g * per;
        const uint32_t wide = min(16u, a.tiles_n - first);
        *n0 = (first + in % wide) * kLanes * C::CG + half * kLanes;
        *tm = in / wide;
    };

    if (warp < 4) {
        if (C::SHIFT) regs_less<C::kFew>();
        if (warp == 0) {
            const bool leader = elect_one();
            uint32_t it = 0, s = 0, phase = 1;
            bool ok = true;
            auto load_w = [&](uint32_t s, uint32_t kb, uint32_t n0) {
                const uint32_t dst = base + s * C::stage_pitch;
                if (C::CG == 1) {
                    mbar_expect(full(s), C::stage_bytes);
                    tma_load(dst, &map_w, kb * kBlock, n0, full(s));
                } else {
                    // The tiles of both CTAs count on the first one's barrier,
                    // where the products wait.
                    if (half == 0) mbar_expect(full(s), 2 * C::stage_bytes);
                    tma_load_pair(dst, &map_w, kb * kBlock, n0, map_to_rank(full(s), 0));
                }
            };
            // The first tiles of w do not wait for x's quantisation.
            uint32_t ahead = 0;
            if (first_tile < tiles) {
                uint32_t n0, tm;
                place(first_tile, &n0, &tm);
                ahead = min(kb1 - kb0, uint32_t(C::ST));
                if (leader) {
                    prefetch_map(&map_w);
                    prefetch_map(&map_x);
                    prefetch_map(&map_sx);
                    for (uint32_t i = 0; i < ahead; ++i) load_w(i, kb0 + i, n0);
                }
                __syncwarp();
            }
            grid_wait();
            for (uint32_t t = first_tile; ok && t < tiles; t += step) {
                uint32_t n0, tm;
                place(t, &n0, &tm);
                for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                    ok = __all_sync(0xffffffffu, mbar_wait(empty(s), phase, guard, kWaitEmpty));
                    if (!ok) break;
                    if (leader) {
                        if (it >= ahead) load_w(s, kb, n0);
                        const uint32_t dst = base + s * C::stage_pitch + C::w_bytes, dst_sx = dst + C::x_bytes;
                        if (C::CG == 1) {
                            tma_load(dst, &map_x, kb * kBlock, tm * C::BN, full(s));
                            tma_load(dst_sx, &map_sx, 0, tm * a.nb + kb, full(s));
                        } else {
                            // Both CTAs need all of the factors, which go from
                            // each one's shared memory to its tensor memory.
                            const uint32_t b = map_to_rank(full(s), 0);
                            tma_load_pair(dst, &map_x, kb * kBlock, tm * C::BN + half * (C::BN / 2), b);
                            tma_load_pair(dst_sx, &map_sx, 0, tm * a.nb + kb, b);
                        }
                    }
                    __syncwarp();
                    if (++s == C::ST) s = 0, phase ^= 1;
                }
            }
            if (*guard.abort && half == 0 && leader) {  // let copies in flight land before the block retires
                const long long t0 = clock64();
                const uint32_t end = max(it, ahead);
                for (uint32_t i = end > C::ST ? end - C::ST : 0; i < end; ++i)
                    while (!mbar_test(full(i % C::ST), i / C::ST & 1) && clock64() - t0 < kWaitCycles / 8) {
                    }
            }
            __syncwarp();
        }
        if (warp == 1 && half == 0) {
            constexpr uint32_t idesc = instr_desc_mxf8(kLanes * C::CG, C::BN);
            const bool leader = elect_one();
            uint32_t it = 0, s = 0, b = 0, sphase = 0, bphase = 1;
            bool ok = true;
            for (uint32_t t = first_tile; ok && t < tiles; t += step)
                for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                    // the factors go ahead of the wait for a buffer: copies and products run in order
                    const uint32_t src = base + s * C::stage_pitch;
                    ok = __all_sync(0xffffffffu, mbar_wait(full(s), sphase, guard, kWaitFull));
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (uint32_t i = 0; i < C::sx_words; i += 128)
                            scales_to_tmem<C::CG>(tmem + C::tmem_sx + i / 32, src + C::w_bytes + C::x_bytes + i * 4);
                    }
                    __syncwarp();
                    ok = __all_sync(0xffffffffu, mbar_wait<C::CG == 2>(tempty(b), bphase, guard, kWaitTmemEmpty));
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
                        const uint32_t d = tmem + b * C::BN;
                        const uint64_t dw = operand_desc(src), dx = operand_desc(src + C::w_bytes);
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)  // 32 values, 32 bytes, a step
                            mma_mxf8<C::CG>(d, dw + 2 * k, dx + 2 * k, idesc, tmem + C::tmem_sw, tmem + C::tmem_sx,
                                            k > 0);
                        mma_commit<C::CG>(empty(s));
                        mma_commit<C::CG>(tfull(b));
                    }
                    __syncwarp();
                    if (++s == C::ST) s = 0, sphase ^= 1;
                    if (++b == C::NBUF) b = 0, bphase ^= 1;
                }
            if (*guard.abort && leader) mma_drain<C::CG>(drained);
            __syncwarp();
        }
        // Even shares of registers again, for the code that all warps run; not
        // before every warp is done with its own.
        __syncwarp();
        if (C::SHIFT) {
            __syncthreads();
            regs_more<C::kEven>();
        }
    } else {
        if (C::SHIFT) regs_more<C::kMany>();
        const uint32_t quad = warp % 4, mine = (warp - 4) / 4 * C::CPT;  // lanes, first column
        const uint32_t my_lane = quad * 32 + lane;
        uint32_t b = 0, bphase = 0;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t n0, tm;
            place(t, &n0, &tm);
            const uint32_t row = n0 + my_lane;
            const float* sw = a.scale_w + uint64_t(min(row, a.n - 1)) * a.nb;
            float next = __ldg(sw + kb0);
            float acc[C::CPT];
#pragma unroll
            for (int i = 0; i < C::CPT; ++i) acc[i] = 0.f;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                const float scale = next;
                ok = mbar_wait(tfull(b), bphase, guard, kWaitTmemFull);
                ok = __all_sync(0xffffffffu, ok);
                __syncwarp();
                if (!ok) break;
                tc_fence_after();
                const uint32_t from = tmem + b * C::BN + mine + (quad * 32 << 16);
                constexpr int NC = C::CPT / C::CH;
                uint32_t v[NC][C::CH];
#pragma unroll
                for (int c = 0; c < NC; ++c) tmem_ld(from + c * C::CH, v[c]);
                if (kb + 1 < kb1) next = __ldg(sw + kb + 1);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (C::CG == 2)
                        mbar_arrive_remote(map_to_rank(tempty(b), 0));
                    else
                        mbar_arrive(tempty(b));
                }
#pragma unroll
                for (int i = 0; i < C::CPT; ++i) add_scaled(acc[i], v[i / C::CH][i % C::CH], scale);
                if (++b == C::NBUF) b = 0, bphase ^= 1;
            }
            if (C::CG == 1 && a.split > 1) {
                // Partial sums meet in shared memory: the stages are free (the
                // last product of this CTA has been read, and there is one
                // tile to a CTA). Every CTA of the cluster adds its share of
                // the columns, in the order of the parts.
                float* part_sum = reinterpret_cast<float*>(sm);
#pragma unroll
                for (int i = 0; i < C::CPT; ++i) part_sum[(mine + i) * kLanes + my_lane] = acc[i];
                break;
            }
            // The lanes past the last row take no other way through the loop:
            // the loads of tensor memory need whole warps.
            if (ok && row < a.n) {
                const float add = a.bias ? bias_at(a, row) : 0.f;
                const uint32_t c0 = tm * C::BN + mine;
                if (a.type == 0)
                    store_column<__nv_bfloat16, C::CPT>(a, row, c0, acc, add);
                else if (a.type == 1)
                    store_column<__half, C::CPT>(a, row, c0, acc, add);
                else
                    store_column<float, C::CPT>(a, row, c0, acc, add);
            }
            __syncwarp();
        }
        __syncwarp();
        if (C::SHIFT) {
            __syncthreads();
            regs_less<C::kEven>();
        }
    }
    if (C::CG == 1 && a.split > 1) {
        __syncthreads();
        cluster_wait();
        cluster_sync();
        uint32_t n0, tm;
        place(first_tile, &n0, &tm);
        const uint32_t from = C::BN * part / a.split, to = C::BN * (part + 1) / a.split;
        for (uint32_t e = from * kLanes + threadIdx.x; e < to * kLanes; e += C::threads) {
            const uint32_t row = n0 + e % kLanes, c = tm * C::BN + e / kLanes;
            if (row >= a.n || c >= a.m) continue;
            float sum = 0.f;
            for (uint32_t r = 0; r < a.split; ++r) sum += ld_cluster(map_to_rank(base + e * 4, r));
            store_one(a, int64_t(c) * a.ld + row, fmaf(sum, kUp, a.bias ? bias_at(a, row) : 0.f));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (C::CG == 2 || a.split > 1) cluster_sync();
    if (warp == 2) {
        tc_fence_after();
        tmem_free<C::CG>(tmem, C::tmem_cols);
    }
}

bool q_ok(const Block128In& t, int64_t cols) {
    return t.q && t.scales && (reinterpret_cast<uintptr_t>(t.q) & 15) == 0 && t.ld % 16 == 0 && t.ld >= cols &&
           t.ld < kMostPitch;
}

struct Problem {
    MatIn x;
    FloatType xtype;
    Block128Out kept;
    uint32_t* work;
    uint64_t work_bytes;
    Block128In w;
    const void* bias;
    MatOut y;
    FloatType type;
    int64_t m, n, k;
    cudaStream_t s;
};

template <typename C>
cudaError_t run(const Problem& p, uint32_t split) {
    Args a{};
    a.nb = uint32_t((p.k + 127) / 128);
    a.tiles_n = uint32_t((p.n + kLanes * C::CG - 1) / (kLanes * C::CG));
    a.tiles_m = uint32_t((p.m + C::BN - 1) / C::BN);
    TileScales ts;
    ts.words = p.work;
    ts.rows = C::BN;
    ts.stride = C::sx_words;
    if (uint64_t(a.tiles_m) * a.nb * ts.stride * 4 > p.work_bytes) return cudaErrorInvalidValue;
    cudaError_t e = error_word(&a.error);
    if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(k_linear<C>), C::smem);
    CUtensorMap mw, mx, msx;
    if (e == cudaSuccess) e = tile_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w.q, p.k, p.n, p.w.ld, kBlock, kLanes);
    if (e == cudaSuccess)
        e = tile_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.kept.q, p.k, p.m, p.kept.ld, kBlock, C::BN / C::CG);
    if (e == cudaSuccess)
        e = tile_map(&msx, CU_TENSOR_MAP_DATA_TYPE_UINT32, p.work, ts.stride, int64_t(a.tiles_m) * a.nb,
                     int64_t(ts.stride) * 4, ts.stride, 1, 0);
    if (e == cudaSuccess) e = quantize_for_tiles(p.x, p.xtype, p.kept, ts, p.m, p.k, p.s);
    if (e != cudaSuccess) return e;
    a.scale_w = p.w.scales;
    a.bias = p.bias;
    a.out = p.y.ptr;
    a.ld = p.y.ld;
    a.m = uint32_t(p.m);
    a.n = uint32_t(p.n);
    a.split = C::CG == 2 ? 1 : split;
    a.type = int(p.type);
    const uint64_t tiles = uint64_t(a.tiles_n) * a.tiles_m;
    if (tiles * a.split > 0x7fffffff) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    cfg.blockDim = dim3(C::threads);
    cfg.dynamicSmemBytes = C::smem;
    cfg.stream = p.s;
    cfg.attrs = at;
    const uint32_t group = C::CG == 2 ? 2 : a.split;
    if (group > 1) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = group;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    // starts while x is being quantised, with what does not need it (3 us of a decode step)
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
    // a split tile has a cluster of its own; else the CTAs (or pairs) walk the tiles
    const uint64_t units = a.split > 1 ? tiles : std::min<uint64_t>(tiles, uint64_t(sm_count()) * C::per_sm / group);
    cfg.gridDim = dim3(uint32_t(units * group));
    e = cudaLaunchKernelEx(&cfg, k_linear<C>, mw, mx, msx, a);
    g_block128_launches.fetch_add(1, std::memory_order_relaxed);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// Parts of the sum while they reach SMs that have nothing to do, of two blocks
// at least: n = 5120 (40 tiles), one token, 1 / 2 / 4 / 8 parts 16.3 / 13.5 /
// 12.7 / 16.6 us; n = 14336 (112 tiles), 16 tokens, 1 / 2 parts 16.7 / 18.6.
uint32_t parts(int64_t tiles, int64_t nb, int64_t room) {
    const int64_t sms = sm_count();
    uint32_t s = 1;
    while (s < 8 && tiles * s * 4 < sms * 3 && tiles * s * 2 <= room && nb >= s * 4) s *= 2;
    return s;
}

}  // namespace

uint64_t linear_work_bytes(int64_t m, int64_t k) {
    // tiles of 224 rows take 256 words a block, those of 128 and fewer 128
    return m <= 0 || k <= 0 ? 0 : uint64_t((m + 111) / 112 + 1) * 128 * 4 * uint64_t((k + 127) / 128);
}

cudaError_t linear_block128(MatIn x, FloatType xtype, Block128Out kept, void* work, uint64_t work_bytes, Block128In w,
                            const void* bias, MatOut y, FloatType type, int64_t m, int64_t n, int64_t k,
                            cudaStream_t s) {
    const int64_t most = 0x7fffff00;
    if (m < 0 || n < 0 || k <= 0 || m > most || n > most || k > most || int(type) < 0 || int(type) > 2)
        return cudaErrorInvalidValue;
    if (m == 0) return cudaSuccess;
    if (n == 0) return kept.scales ? quantize_block128(x, xtype, kept, m, k, s) : cudaSuccess;
    if (!x.ptr || x.ld < k || x.ld > 0xffffffff || kept.ld < k || kept.ld % 16 != 0 || kept.ld >= kMostPitch ||
        !kept.q || int(xtype) < 0 || int(xtype) > 2 || !q_ok(w, k) || !y.ptr || y.ld < n || !work ||
        (reinterpret_cast<uintptr_t>(work) & 15))
        return cudaErrorInvalidValue;
    const Problem p{x, xtype, kept, static_cast<uint32_t*>(work), work_bytes, w, bias, y, type, m, n, k, s};
    const int64_t nb = (k + 127) / 128, nt = (n + 127) / 128;
    // Few tokens: the fewest columns that hold them (the rest of the columns
    // costs time too: 24 tokens x 5120 x 5120 take 14.5 us with 32 columns, 16.7
    // with 64), two CTAs an SM where they fit.
    const int64_t sms = sm_count();
    if (m <= 16) return run<Config<16, 1, 4, 5, 4, 2>>(p, parts(nt, nb, sms * 2));
    if (m <= 32) return run<Config<32, 1, 4, 5, 4, 2>>(p, parts(nt, nb, sms * 2));
    if (m <= 64) {
        const int64_t split = std::max<int64_t>(1, std::min<int64_t>({8, sms / nt, nb / 2}));
        return run<Config<64, 1, 8, 8, 4, 1>>(p, uint32_t(split));
    }
    // Else by the number of rounds of tiles, of 224 x 256 for a pair of CTAs
    // or 128 x 128 for each: a block of the sum takes a round 0.47 or 0.385 us.
    // 1531 x 3456 x 5001: 36.1 us in pairs, 46.5 in 128s; 1024 x 4096 x 4096 37.0, 30.6.
    const int64_t pairs = (m + 223) / 224 * ((n + 255) / 256), tiles = (m + 127) / 128 * nt;
    const int64_t rounds2 = (pairs * 2 + sms - 1) / sms, rounds1 = (tiles + sms - 1) / sms;
    if (rounds2 * 11 < rounds1 * 9) return run<Config<224, 2, 8, 6, 2, 1>>(p, 1);
    // the parts of a 128 x 128 tile are 64 KiB each to join: not for two of them
    return run<Config<128, 1, 8, 6, 3, 1>>(p, tiles * 4 <= sms ? parts(tiles, nb, sms) : 1);
}

}  // namespace kern
}  // namespace ofld
