// fg_clip.cu — C ABI entry points of the gradient norm and clipping: argument checks
// and launches.
#include <algorithm>
#include <vector>

#include "fg_clip.cuh"
#include "fg_internal.h"

namespace {

using fg::host::DevInfo;
using fg::host::elem_size;

constexpr int32_t kMaxTensors = 1 << 20;

int64_t launches_for(int64_t count) { return (count + fg::clip::MAX_TENSORS - 1) / fg::clip::MAX_TENSORS; }

// A launch that may begin while the stream's previous kernel ends: the kernel itself
// waits for that one before it touches memory.
template <class... Params, class... Args>
int launch_early(void (*kern)(Params...), unsigned grid, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(fg::clip::THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? FG_OK : FG_ELAUNCH;
}

struct Span {
    uintptr_t lo, hi;
    int32_t tensor;
    bool operator<(const Span& o) const { return lo < o.lo; }
};

// Whether a result shares memory with another tensor's result or gradients, or with a
// part of its own gradients.
bool results_meet(const FgGradTensor* t, int32_t n) {
    std::vector<Span> outs;
    outs.reserve(n);
    for (int32_t i = 0; i < n; ++i)
        if (t[i].out && t[i].count > 0) {
            const uintptr_t lo = reinterpret_cast<uintptr_t>(t[i].out);
            outs.push_back({lo, lo + uintptr_t(t[i].count) * elem_size(t[i].out_dtype), i});
        }
    if (outs.empty()) return false;
    std::sort(outs.begin(), outs.end());
    for (size_t i = 1; i < outs.size(); ++i)
        if (outs[i].lo < outs[i - 1].hi) return true;
    for (int32_t i = 0; i < n; ++i) {
        if (t[i].count == 0) continue;
        const uintptr_t lo = reinterpret_cast<uintptr_t>(t[i].grad);
        const uintptr_t hi = lo + uintptr_t(t[i].count) * elem_size(t[i].dtype);
        // results are apart from each other: those that meet [lo, hi) are neighbours
        auto it = std::lower_bound(outs.begin(), outs.end(), Span{hi, 0, 0});
        while (it != outs.begin()) {
            --it;
            if (it->hi <= lo) break;
            if (!(it->tensor == i && it->lo == lo && t[i].dtype == t[i].out_dtype)) return true;
        }
    }
    return false;
}

}  // namespace

extern "C" {

size_t fg_clip_workspace_size(int32_t count) {
    if (count < 0 || count > kMaxTensors) return 0;
    return sizeof(double) * (1 + size_t(launches_for(std::max(count, 1))) * fg::clip::MAX_GRID);
}

int fg_clip_grad_norm(const FgClipArgs* a, void* stream) {
    if (a == nullptr || a->reserved != 0 || a->count < 0 || (a->count > 0 && a->tensors == nullptr)) return FG_EINVAL;
    if (a->out_norm == nullptr || reinterpret_cast<uintptr_t>(a->out_norm) % 4 != 0) return FG_EINVAL;
    if (!(a->max_norm >= 0.0f) || !(a->scale > 0.0f && a->scale < INFINITY)) return FG_EINVAL;
    if (a->count > kMaxTensors) return FG_ENOTSUP;
    for (int32_t i = 0; i < a->count; ++i) {
        const FgGradTensor& t = a->tensors[i];
        const int esz = elem_size(t.dtype), osz = elem_size(t.out_dtype);
        if (esz == 0 || t.count < 0) return FG_EINVAL;
        if (t.count > (int64_t(1) << 40)) return FG_ENOTSUP;
        if (t.count > 0 && (t.grad == nullptr || reinterpret_cast<uintptr_t>(t.grad) % esz != 0)) return FG_EINVAL;
        if (t.out != nullptr && (osz == 0 || reinterpret_cast<uintptr_t>(t.out) % osz != 0)) return FG_EINVAL;
    }
    if (a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 8 != 0 ||
        a->workspace_bytes < fg_clip_workspace_size(a->count))
        return FG_EINVAL;
    try {
        if (results_meet(a->tensors, a->count)) return FG_EINVAL;
    } catch (...) {   // no host memory for the check
        return FG_ENOTSUP;
    }
    DevInfo* d = nullptr;
    const int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    double* total = reinterpret_cast<double*>(a->workspace);
    double* partial = total + 1;
    const int64_t cap = std::min<int64_t>(fg::clip::MAX_GRID, 8 * int64_t(d->sms));
    int64_t partials = 0;
    // pass 0: the sums; pass 1: the scaling (at least one launch, which writes the norm)
    for (int pass = 0; pass < 2; ++pass) {
        bool wrote = false;
        for (int32_t lo = 0; lo < a->count || (pass == 1 && !wrote); lo += fg::clip::MAX_TENSORS) {
            fg::clip::List L;
            L.count = 0;
            int64_t chunks = 0;
            for (int32_t i = lo; i < std::min(a->count, lo + fg::clip::MAX_TENSORS); ++i) {
                const FgGradTensor& t = a->tensors[i];
                if (t.count == 0 || (pass == 1 && t.out == nullptr)) continue;
                const int esz = elem_size(t.dtype);
                fg::clip::Item& it = L.items[L.count++];
                it.in = t.grad; it.out = t.out; it.count = t.count;
                it.dtype = uint8_t(t.dtype); it.out_dtype = uint8_t(t.out_dtype);
                it.first = uint32_t(chunks);
                it.wide_in = reinterpret_cast<uintptr_t>(t.grad) % 16 == 0;
                const int vec = t.out ? std::min(16, 16 / esz * elem_size(t.out_dtype)) : 16;
                it.wide_out = t.out && reinterpret_cast<uintptr_t>(t.out) % vec == 0;
                chunks += (t.count * esz + fg::clip::CHUNK_BYTES - 1) / fg::clip::CHUNK_BYTES;
                if (chunks > (int64_t(1) << 31)) return FG_ENOTSUP;
            }
            L.chunks = uint32_t(chunks);
            if (pass == 0) {
                if (chunks == 0) continue;
                const unsigned grid = unsigned(std::min(cap, chunks));
                const int rc1 = launch_early(fg::clip::norm_kernel, grid, st, L, partial + partials);
                if (rc1 != FG_OK) return rc1;
                partials += grid;
            } else {
                if (chunks == 0 && wrote) continue;
                if (chunks == 0 && lo + fg::clip::MAX_TENSORS < a->count) continue;   // a later launch writes the norm
                const unsigned grid = unsigned(std::max<int64_t>(1, std::min(cap, chunks)));
                const bool one = partials <= cap;
                const int rc1 = launch_early(fg::clip::scale_kernel, grid, st, L, (const double*)(one ? partial : total),
                                             one ? partials : int64_t(1), a->max_norm, a->scale,
                                             wrote ? (float*)nullptr : a->out_norm);
                if (rc1 != FG_OK) return rc1;
                wrote = true;
            }
        }
        if (pass == 0 && partials > cap) {
            const int rc1 = launch_early(fg::clip::total_kernel, 1, st, (const double*)partial, partials, total);
            if (rc1 != FG_OK) return rc1;
        }
    }
    return FG_OK;
}

}  // extern "C"
