// fg_host.cu — host helpers shared by the library's translation units.
#include <atomic>

#include "fg_internal.h"
#include "fg_tma.h"

namespace fg {
namespace host {

std::mutex g_mu;

namespace {
DevInfo g_dev[kMaxDevices];
}  // namespace

int device_info(DevInfo** out) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return FG_EDEVICE;
    std::lock_guard<std::mutex> lk(g_mu);
    DevInfo& d = g_dev[dev];
    if (!d.ok) {
        if (cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return FG_EDEVICE;
        if (cudaDeviceGetAttribute(&d.smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) != cudaSuccess)
            return FG_EDEVICE;
        if (cudaDeviceGetAttribute(&d.smem_per_sm, cudaDevAttrMaxSharedMemoryPerMultiprocessor, dev) != cudaSuccess)
            return FG_EDEVICE;
        d.ok = true;
    }
    *out = &d;
    return FG_OK;
}

namespace {
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder, through the runtime (the library links no libcuda).
EncodeTiledFn encoder() {
    static std::atomic<EncodeTiledFn> fn{nullptr};
    EncodeTiledFn f = fn.load(std::memory_order_acquire);
    if (f == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) !=
                cudaSuccess || q != cudaDriverEntryPointSuccess)
            return nullptr;
        f = reinterpret_cast<EncodeTiledFn>(p);
        fn.store(f, std::memory_order_release);
    }
    return f;
}

}  // namespace

bool encode_rows(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t dim, int64_t stride,
                 int box_rows) {
    EncodeTiledFn f = encoder();
    if (f == nullptr) return false;
    const cuuint64_t extent[2] = {cuuint64_t(dim), cuuint64_t(rows)};
    const cuuint64_t pitch[1] = {cuuint64_t(stride) * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(box_rows)};
    const cuuint32_t step[2] = {1, 1};
    auto encode = [&]() {
        return f(map, dtype == FG_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                 const_cast<void*>(base), extent, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (encode()) return true;
    // a thread that has made no runtime call that needs the device (a backward pass's) has no
    // current context, which the driver wants here: make the device's own one current
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess && encode();
}

}  // namespace host
}  // namespace fg
