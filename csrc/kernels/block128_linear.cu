// y = x w^T on the fp8 tensor cores, both operands block-128.
//
//   y[m, n] = sum_b sx[m, b] sw[n, b] P_b[m, n],   P_b = the e4m3 product over the 128 values of block b
//
// The scales change with every block of the sum and are any fp32 numbers, so
// they cannot go into the tensor core's accumulator: each P_b (four
// tcgen05.mma of 32 values) is written to tensor memory on its own, in one of
// several buffers, and the epilogue warps add sx sw P_b to fp32 registers
// while the next block's product runs. Per 128 x BN tile and block that is
// 2 BN cycles of tensor core against BN fp32 multiplies and BN multiply-adds
// on each of 128 lanes, done as packed pairs.
//
// One operand's rows lie on the 128 lanes of tensor memory ("lane side"), the
// other's on its columns ("column side", BN of them). With many tokens the
// lane side is x; with few it is w, so that the tile holds little but weights
// and the 128 lanes are never empty.
//
// Warps: 0 loads the tiles (TMA, 128-byte swizzle), 1 issues the products, 2
// fetches the scales (cp.async, rows of different blocks are far apart), 3
// owns the tensor memory, the rest are the epilogue.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "block128.h"
#include "block128_host.h"
#include "sm100.cuh"

namespace ofld {
namespace kern {

namespace {

using namespace sm100;

constexpr uint32_t kLanes = 128, kBlock = 128;
constexpr uint32_t kScaleSlots = 8;

// Codes of waits that ran out.
enum : uint32_t { kWaitEmpty = 101, kWaitFull, kWaitTmemEmpty, kWaitTmemFull, kWaitScaleEmpty, kWaitScaleFull };

struct Args {
    const float* scale_lane;
    const float* scale_col;
    const void* bias;
    void* out;
    int64_t ld;
    uint32_t rows_lane, rows_col, nb;
    uint32_t tiles_lane, tiles_col, split;
    int type;    // FloatType
    bool vec;    // 16-byte stores are aligned
    uint32_t* error;
};

// BN columns, CG CTAs on one tile (2: 256 lane rows, each CTA loads half of
// the column side), EW epilogue warps, ST stages, SWAP: the lane side is w.
template <int BN_, int CG_, int EW_, int ST_, bool SWAP_>
struct Config {
    static constexpr int BN = BN_, CG = CG_, EW = EW_, ST = ST_;
    static constexpr bool SWAP = SWAP_;
    static constexpr int threads = 128 + 32 * EW;
    static constexpr int NBUF = BN >= 128 ? 2 : 4;
    static constexpr uint32_t tmem_cols = NBUF * BN;
    static constexpr uint32_t lane_bytes = kLanes * kBlock, col_bytes = BN / CG * kBlock;
    static constexpr uint32_t stage_bytes = lane_bytes + col_bytes;
    static constexpr uint32_t scale_floats = kLanes + BN;
    static constexpr uint32_t bars = 2 * ST + 2 * NBUF + 2 * kScaleSlots;
    static constexpr uint32_t off_scale = ST * stage_bytes;
    static constexpr uint32_t off_bar = off_scale + kScaleSlots * scale_floats * 4;
    static constexpr uint32_t off_misc = off_bar + bars * 8;
    static constexpr uint32_t smem = off_misc + 16 + 1024;  // + alignment of the base
    static constexpr int per_sm = EW == 4 && BN <= 64 ? 2 : 1;
    static constexpr int CPT = BN / (EW / 4);   // columns of one epilogue thread
    static constexpr int CH = BN < 32 || BN == 256 ? 16 : 32;  // columns of one tensor-memory load (registers)
    static_assert(tmem_cols >= 32 && tmem_cols * per_sm <= 512, "tensor memory");
    static_assert(smem * per_sm <= 227 * 1024, "shared memory");
    static_assert(CPT % CH == 0, "");
    // the split reduction keeps a 128 x BN fp32 tile in the stages
    static_assert(CG == 2 || ST * stage_bytes >= kLanes * BN * 4, "");
};

template <typename T>
__device__ __forceinline__ float as_float(const void* p, uint32_t i) {
    return float(static_cast<const T*>(p)[i]);
}
__device__ __forceinline__ float bias_at(const Args& a, uint32_t i) {
    return a.type == 0 ? as_float<__nv_bfloat16>(a.bias, i) : a.type == 1 ? as_float<__half>(a.bias, i)
                                                                        : as_float<float>(a.bias, i);
}
__device__ __forceinline__ void store_one(const Args& a, int64_t at, float v) {
    if (a.type == 0)
        static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
    else if (a.type == 1)
        static_cast<__half*>(a.out)[at] = __float2half_rn(v);
    else
        static_cast<float*>(a.out)[at] = v;
}
__device__ __forceinline__ uint32_t pack16(int type, float lo, float hi) {
    if (type == 0) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Eight consecutive results of one row.
__device__ __forceinline__ void store_eight(const Args& a, int64_t row, uint32_t c, const float v[8]) {
    const int64_t at = row * a.ld + c;
    if (a.vec && c + 8 <= a.rows_col) {
        if (a.type == 2) {
            float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint4 w;
            w.x = pack16(a.type, v[0], v[1]);
            w.y = pack16(a.type, v[2], v[3]);
            w.z = pack16(a.type, v[4], v[5]);
            w.w = pack16(a.type, v[6], v[7]);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < a.rows_col) store_one(a, at + i, v[i]);
    }
}

template <typename C>
__global__ void __launch_bounds__(C::threads, C::per_sm)
    k_linear(const __grid_constant__ CUtensorMap map_lane, const __grid_constant__ CUtensorMap map_col, const Args a) {
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    uint8_t* const sm = raw + (base - smem_addr(raw));
    const uint32_t bar = base + C::off_bar;
    auto full = [&](uint32_t s) { return bar + 8 * s; };
    auto empty = [&](uint32_t s) { return bar + 8 * (C::ST + s); };
    auto tfull = [&](uint32_t b) { return bar + 8 * (2 * C::ST + b); };
    auto tempty = [&](uint32_t b) { return bar + 8 * (2 * C::ST + C::NBUF + b); };
    auto sfull = [&](uint32_t s) { return bar + 8 * (2 * C::ST + 2 * C::NBUF + s); };
    auto sempty = [&](uint32_t s) { return bar + 8 * (2 * C::ST + 2 * C::NBUF + kScaleSlots + s); };
    volatile uint32_t* const misc = reinterpret_cast<volatile uint32_t*>(sm + C::off_misc);  // tensor memory, abort
    const Guard guard{misc + 1, a.error};

    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t in_cluster = C::CG == 2 || a.split > 1 ? cluster_rank() : 0;
    const uint32_t half = C::CG == 2 ? in_cluster : 0;  // which CTA of the pair
    const uint32_t part = C::CG == 1 ? in_cluster : 0;  // which part of the sum
    const uint32_t group = C::CG == 2 ? 2 : a.split;
    const uint32_t first_tile = blockIdx.x / group, step = gridDim.x / group, tiles = a.tiles_lane * a.tiles_col;
    const uint32_t kb0 = uint32_t(uint64_t(a.nb) * part / a.split), kb1 = uint32_t(uint64_t(a.nb) * (part + 1) / a.split);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < C::ST; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
        for (uint32_t b = 0; b < C::NBUF; ++b) mbar_init(tfull(b), 1), mbar_init(tempty(b), C::EW * C::CG);
        for (uint32_t s = 0; s < kScaleSlots; ++s) mbar_init(sfull(s), 32), mbar_init(sempty(s), C::EW);
        mbar_init_fence();
        misc[1] = 0;
    }
    if (warp == 3) tmem_alloc<C::CG>(base + C::off_misc, C::tmem_cols);
    tc_fence_before();
    __syncthreads();
    if (C::CG == 2 || a.split > 1) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = misc[0];

    // Tiles in groups of 16 lane tiles, lane tiles fastest: the tiles in
    // flight share few column tiles and at most 16 lane tiles through L2.
    auto place = [&](uint32_t t, uint32_t* l0, uint32_t* c0) {
        const uint32_t per = 16 * a.tiles_col, g = t / per, first = g * 16, in = t - g * per;
        const uint32_t wide = min(16u, a.tiles_lane - first);
        *l0 = (first + in % wide) * kLanes * C::CG + half * kLanes;
        *c0 = in / wide * C::BN;
    };

    if (warp == 0) {
        if (lane == 0) {
            prefetch_map(&map_lane);
            prefetch_map(&map_col);
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t t = first_tile; ok && t < tiles; t += step) {
                uint32_t l0, c0;
                place(t, &l0, &c0);
                for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                    const uint32_t s = it % C::ST;
                    if (!(ok = mbar_wait(empty(s), (it / C::ST & 1) ^ 1, guard, kWaitEmpty))) break;
                    const uint32_t dst = base + s * C::stage_bytes;
                    if (C::CG == 1) {
                        mbar_expect(full(s), C::stage_bytes);
                        tma_load(dst, &map_lane, kb * kBlock, l0, full(s));
                        tma_load(dst + C::lane_bytes, &map_col, kb * kBlock, c0, full(s));
                    } else {  // both CTAs' tiles count on the first one's barrier
                        if (half == 0) mbar_expect(full(s), 2 * C::stage_bytes);
                        const uint32_t b = map_to_rank(full(s), 0);
                        tma_load_pair(dst, &map_lane, kb * kBlock, l0, b);
                        tma_load_pair(dst + C::lane_bytes, &map_col, kb * kBlock, c0 + half * (C::BN / 2), b);
                    }
                }
            }
            if (*guard.abort && half == 0) {  // let copies in flight land before the block retires
                const long long t0 = clock64();
                for (uint32_t i = it > C::ST ? it - C::ST : 0; i < it; ++i)
                    while (!mbar_test(full(i % C::ST), i / C::ST & 1) && clock64() - t0 < kWaitCycles / 8) {
                    }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && half == 0) {
            constexpr uint32_t idesc = instr_desc(kLanes * C::CG, C::BN, 0, false, false);
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t t = first_tile; ok && t < tiles; t += step)
                for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                    const uint32_t s = it % C::ST, b = it % C::NBUF;
                    ok = mbar_wait<C::CG == 2>(tempty(b), (it / C::NBUF & 1) ^ 1, guard, kWaitTmemEmpty) &&
                         mbar_wait(full(s), it / C::ST & 1, guard, kWaitFull);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t src = base + s * C::stage_bytes;
                    const uint64_t da = operand_desc(src), db = operand_desc(src + C::lane_bytes);
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)  // 32 values, 32 bytes, a step
                        mma_f8<C::CG>(tmem + b * C::BN, da + 2 * k, db + 2 * k, idesc, k > 0);
                    mma_commit<C::CG>(empty(s));
                    mma_commit<C::CG>(tfull(b));
                }
        }
    } else if (warp == 2) {
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint32_t l0, c0;
            place(t, &l0, &c0);
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                const uint32_t s = it % kScaleSlots;
                if (!(ok = mbar_wait(sempty(s), (it / kScaleSlots & 1) ^ 1, guard, kWaitScaleEmpty))) break;
                const uint32_t dst = base + C::off_scale + s * C::scale_floats * 4;
#pragma unroll
                for (uint32_t i = 0; i < C::scale_floats; i += 32) {
                    const bool lanes = i < kLanes;
                    const uint32_t r = lanes ? l0 + i + lane : c0 + i - kLanes + lane;
                    const bool valid = r < (lanes ? a.rows_lane : a.rows_col) && i + lane < C::scale_floats;
                    const float* src = lanes ? a.scale_lane : a.scale_col;
                    if (i + lane < C::scale_floats)
                        cp_async4(dst + (i + lane) * 4, valid ? src + uint64_t(r) * a.nb + kb : src, valid);
                }
                cp_async_arrive(sfull(s));
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= 4) {
        const uint32_t quad = warp % 4, mine = (warp - 4) / 4 * C::CPT;  // lanes, first column
        const uint32_t my_lane = quad * 32 + lane;
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = first_tile; ok && t < tiles; t += step) {
            uint64_t acc[C::CPT / 2];
#pragma unroll
            for (int i = 0; i < C::CPT / 2; ++i) acc[i] = 0;
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                const uint32_t b = it % C::NBUF, s = it % kScaleSlots;
                ok = mbar_wait(sfull(s), it / kScaleSlots & 1, guard, kWaitScaleFull) &&
                     mbar_wait(tfull(b), it / C::NBUF & 1, guard, kWaitTmemFull);
                ok = __all_sync(0xffffffffu, ok);
                __syncwarp();
                if (!ok) break;
                tc_fence_after();
                const float* sc = reinterpret_cast<const float*>(sm + C::off_scale) + s * C::scale_floats;
                const uint32_t sl = __float_as_uint(sc[my_lane]);
                const uint64_t sl2 = pack2(sl, sl);
                const uint32_t from = tmem + b * C::BN + mine + (quad * 32 << 16);
                uint32_t v[2][C::CH];
                tmem_ld(from, v[0]);
                tmem_ld_wait(v[0]);
#pragma unroll
                for (int c = 0; c < C::CPT / C::CH; ++c) {
                    if (c + 1 < C::CPT / C::CH) tmem_ld(from + (c + 1) * C::CH, v[(c + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < C::CH; i += 4) {
                        const ulonglong2 sr = *reinterpret_cast<const ulonglong2*>(sc + kLanes + mine + c * C::CH + i);
                        uint64_t* d = acc + (c * C::CH + i) / 2;
                        d[0] = fma2(pack2(v[c & 1][i], v[c & 1][i + 1]), mul2(sl2, sr.x), d[0]);
                        d[1] = fma2(pack2(v[c & 1][i + 2], v[c & 1][i + 3]), mul2(sl2, sr.y), d[1]);
                    }
                    if (c + 1 < C::CPT / C::CH) tmem_ld_wait(v[(c + 1) & 1]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (C::CG == 2)
                        mbar_arrive_remote(map_to_rank(tempty(b), 0));
                    else
                        mbar_arrive(tempty(b));
                    mbar_arrive(sempty(s));
                }
            }
            uint32_t l0, c0;
            place(t, &l0, &c0);
            const uint32_t row = l0 + my_lane;
            if (C::CG == 1 && a.split > 1) {
                // Partial sums meet in shared memory: the stages are free (the
                // last product of this CTA has been read, and there is one
                // tile to a CTA). Every CTA of the cluster adds its share of
                // the columns, in the order of the parts.
                float* part_sum = reinterpret_cast<float*>(sm);
#pragma unroll
                for (int i = 0; i < C::CPT / 2; ++i) {
                    const float2 f = unpack2(acc[i]);
                    part_sum[(2 * i) * kLanes + my_lane] = f.x;
                    part_sum[(2 * i + 1) * kLanes + my_lane] = f.y;
                }
                break;
            }
            // The lanes past the last row take no other way through the loop:
            // the loads of tensor memory need whole warps.
            if (ok && row < a.rows_lane) {
                if (C::SWAP) {
                    const float add = a.bias ? bias_at(a, row) : 0.f;
#pragma unroll
                    for (int i = 0; i < C::CPT; ++i) {
                        const float2 f = unpack2(acc[i / 2]);
                        const uint32_t r = c0 + mine + i;
                        if (r < a.rows_col) store_one(a, int64_t(r) * a.ld + row, (i & 1 ? f.y : f.x) + add);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < C::CPT; i += 8) {
                        const uint32_t c = c0 + mine + i;
                        if (c >= a.rows_col) break;
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const float2 f = unpack2(acc[(i + j) / 2]);
                            v[j] = f.x, v[j + 1] = f.y;
                        }
                        if (a.bias) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (c + j < a.rows_col) v[j] += bias_at(a, c + j);
                        }
                        store_eight(a, row, c, v);
                    }
                }
            }
            __syncwarp();
        }
    }
    __syncwarp();
    if (C::CG == 1 && a.split > 1) {
        __syncthreads();
        cluster_sync();
        uint32_t l0, c0;
        place(first_tile, &l0, &c0);
        const uint32_t from = C::BN * part / a.split, to = C::BN * (part + 1) / a.split;
        for (uint32_t e = from * kLanes + threadIdx.x; e < to * kLanes; e += C::threads) {
            const uint32_t l = l0 + e % kLanes, c = c0 + e / kLanes;
            if (l >= a.rows_lane || c >= a.rows_col) continue;
            float sum = 0.f;
            for (uint32_t r = 0; r < a.split; ++r) sum += ld_cluster(map_to_rank(base + e * 4, r));
            const uint32_t n = C::SWAP ? l : c;
            if (a.bias) sum += bias_at(a, n);
            store_one(a, int64_t(C::SWAP ? c : l) * a.ld + n, sum);
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
cudaError_t run(const Block128In& x, const Block128In& w, const void* bias, MatOut y, FloatType type, int64_t m,
                int64_t n, int64_t k, uint32_t split, cudaStream_t s) {
    const Block128In& lane = C::SWAP ? w : x;
    const Block128In& col = C::SWAP ? x : w;
    const int64_t nl = C::SWAP ? n : m, nc = C::SWAP ? m : n;
    CUtensorMap ml, mc;
    cudaError_t e = tile_map(&ml, CU_TENSOR_MAP_DATA_TYPE_UINT8, lane.q, k, nl, lane.ld, kBlock, kLanes);
    if (e == cudaSuccess) e = tile_map(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT8, col.q, k, nc, col.ld, kBlock, C::BN / C::CG);
    Args a{};
    if (e == cudaSuccess) e = error_word(&a.error);
    if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(k_linear<C>), C::smem);
    if (e != cudaSuccess) return e;
    const size_t esz = type == FloatType::kFp32 ? 4 : 2;
    a.scale_lane = lane.scales;
    a.scale_col = col.scales;
    a.bias = bias;
    a.out = y.ptr;
    a.ld = y.ld;
    a.rows_lane = uint32_t(nl);
    a.rows_col = uint32_t(nc);
    a.nb = uint32_t((k + 127) / 128);
    a.tiles_lane = uint32_t((nl + kLanes * C::CG - 1) / (kLanes * C::CG));
    a.tiles_col = uint32_t((nc + C::BN - 1) / C::BN);
    a.split = C::CG == 2 ? 1 : split;
    a.type = int(type);
    a.vec = reinterpret_cast<uintptr_t>(y.ptr) % 16 == 0 && y.ld * int64_t(esz) % 16 == 0;
    const uint64_t tiles = uint64_t(a.tiles_lane) * a.tiles_col;
    if (tiles * a.split > 0x7fffffff) return cudaErrorInvalidValue;
    const uint32_t sms = uint32_t(sm_count());
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    cfg.blockDim = dim3(C::threads);
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
    // a split tile has a cluster of its own; else the CTAs (or pairs) walk the tiles
    const uint64_t units = a.split > 1 ? tiles : std::min<uint64_t>(tiles, sms * C::per_sm / group);
    cfg.gridDim = dim3(uint32_t(units * group));
    e = cudaLaunchKernelEx(&cfg, k_linear<C>, ml, mc, a);
    g_block128_launches.fetch_add(1, std::memory_order_relaxed);
    return e != cudaSuccess ? e : cudaGetLastError();
}

bool q_ok(const Block128In& t, int64_t cols) {
    return t.q && t.scales && (reinterpret_cast<uintptr_t>(t.q) & 15) == 0 && t.ld % 16 == 0 && t.ld >= cols;
}

// Parts of the sum: enough to give every SM work, at least two blocks each.
uint32_t parts(int64_t tiles, int64_t nb, int per_sm) {
    uint32_t s = 1;
    while (s < 8 && tiles * s * 2 <= int64_t(sm_count()) * per_sm && nb >= s * 4) s *= 2;
    return s;
}

}  // namespace

cudaError_t matmul_block128(Block128In x, Block128In w, const void* bias, MatOut y, FloatType type, int64_t m,
                            int64_t n, int64_t k, cudaStream_t s) {
    const int64_t most = 0x7fffff00;
    if (m < 0 || n < 0 || k <= 0 || m > most || n > most || k > most || int(type) < 0 || int(type) > 2)
        return cudaErrorInvalidValue;
    if (m == 0 || n == 0) return cudaSuccess;
    if (!q_ok(x, k) || !q_ok(w, k) || !y.ptr || y.ld < n) return cudaErrorInvalidValue;
    const int64_t nb = (k + 127) / 128, wt = (n + 127) / 128;
    if (m <= 16) return run<Config<16, 1, 4, 5, true>>(x, w, bias, y, type, m, n, k, parts(wt, nb, 2), s);
    if (m <= 32) return run<Config<32, 1, 4, 4, true>>(x, w, bias, y, type, m, n, k, parts(wt, nb, 2), s);
    if (m <= 64) return run<Config<64, 1, 4, 4, true>>(x, w, bias, y, type, m, n, k, parts(wt, nb, 2), s);
    const int64_t pairs = ((m + 255) / 256) * ((n + 255) / 256);
    if (pairs >= 74) return run<Config<256, 2, 8, 5, false>>(x, w, bias, y, type, m, n, k, 1, s);
    if (m <= 128) return run<Config<128, 1, 4, 6, true>>(x, w, bias, y, type, m, n, k, parts(wt, nb, 1), s);
    return run<Config<128, 1, 4, 6, false>>(x, w, bias, y, type, m, n, k, parts((m + 127) / 128 * wt, nb, 1), s);
}

}  // namespace kern
}  // namespace ofld
