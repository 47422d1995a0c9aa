#include "block128_host.h"

#include <map>
#include <mutex>
#include <set>

#include "block128.h"

namespace ofld {
namespace kern {

namespace {

std::mutex g_mu;

struct PerDevice {
    uint32_t* host = nullptr;
    uint32_t* dev = nullptr;
    int sms = 0;
};
constexpr int kDevices = 64;
PerDevice g_dev[kDevices];
std::atomic<bool> g_ready[kDevices];

// Set up on a device's first use, which may be inside a graph capture: the
// allocation is not a stream operation, so the capture is told to let it pass.
cudaError_t per_device(PerDevice** out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kDevices) return cudaErrorInvalidDevice;
    *out = &g_dev[dev];
    if (g_ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
    std::lock_guard<std::mutex> g(g_mu);
    if (g_ready[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    PerDevice& d = g_dev[dev];
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return e;
    void* p = nullptr;
    void* q = nullptr;
    e = cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable);
    if (e == cudaSuccess) e = cudaHostGetDevicePointer(&q, p, 0);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
        if (p) cudaFreeHost(p);
        return e;
    }
    d.host = static_cast<uint32_t*>(p);
    d.dev = static_cast<uint32_t*>(q);
    *d.host = 0;
    g_ready[dev].store(true, std::memory_order_release);
    return cudaSuccess;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

void* driver_entry(const char* name) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? p : nullptr;
}
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = reinterpret_cast<EncodeTiled>(driver_entry("cuTensorMapEncodeTiled"));
    return fn;
}

// A driver call needs a current context. A thread gets one with its first call
// to the runtime that needs it, and an autograd thread's or a user's own may
// have made none yet: its results came from torch's cache of memory.
cudaError_t bind_thread() {
    static const auto current = reinterpret_cast<CUresult (*)(CUcontext*)>(driver_entry("cuCtxGetCurrent"));
    CUcontext ctx = nullptr;
    if (current && current(&ctx) == CUDA_SUCCESS && ctx) return cudaSuccess;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    return e == cudaSuccess ? cudaSetDevice(dev) : e;
}

}  // namespace

cudaError_t tile_map(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, int64_t cols, int64_t rows,
                     int64_t pitch, uint32_t box_cols, uint32_t box_rows, int swizzle) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return cudaErrorNotSupported;
    if (const cudaError_t e = bind_thread()) return e;
    const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
    const cuuint64_t strides[1] = {cuuint64_t(pitch)};
    const cuuint32_t box[2] = {box_cols, box_rows}, step[2] = {1, 1};
    const CUresult r = fn(map, type, 2, const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          swizzle == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                          : swizzle == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t error_word(uint32_t** word) {
    PerDevice* d = nullptr;
    const cudaError_t e = per_device(&d);
    if (e == cudaSuccess) *word = d->dev;
    return e;
}

uint32_t block128_error(int device) {
    if (device < 0 || device >= kDevices || !g_ready[device].load(std::memory_order_acquire)) return 0;
    return *static_cast<volatile uint32_t*>(g_dev[device].host);
}

void block128_set_error(int device, uint32_t code) {
    if (device < 0 || device >= kDevices || !g_ready[device].load(std::memory_order_acquire)) return;
    *static_cast<volatile uint32_t*>(g_dev[device].host) = code;
}

cudaError_t allow_smem(const void* fn, uint32_t bytes) {
    static std::mutex mu;
    static std::set<std::pair<const void*, int>> done;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> g(mu);
    if (done.count({fn, dev})) return cudaSuccess;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    if (e == cudaSuccess) done.insert({fn, dev});
    return e;
}

int sm_count() {
    PerDevice* d = nullptr;
    return per_device(&d) == cudaSuccess ? d->sms : 1;
}

}  // namespace kern
}  // namespace ofld
