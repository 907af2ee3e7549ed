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

// Norm launches of `count` tensors at most: each of the three types may leave one list unfilled.
int64_t launches_for(int64_t count) { return std::min(count, count / fg::clip::MAX_TENSORS + 3); }

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

using ScaleKernel = void (*)(const fg::clip::List, const double*, int64_t, float, float, float*);
ScaleKernel scale_kernel_of(int dt, int odt) {
    using namespace fg::clip;
    static const ScaleKernel table[3][3] = {{scale_kernel<0, 0>, scale_kernel<0, 1>, scale_kernel<0, 2>},
                                            {scale_kernel<1, 0>, scale_kernel<1, 1>, scale_kernel<1, 2>},
                                            {scale_kernel<2, 0>, scale_kernel<2, 1>, scale_kernel<2, 2>}};
    return table[dt][odt];
}

// Calls launch(dtype, result type, list) for the tensors of each type (with `scaling` of
// each pair of types that has results), MAX_TENSORS of them at a time.
template <class F>
int for_lists(const FgClipArgs& a, bool scaling, F launch) {
    for (int dt = 0; dt < 3; ++dt)
        for (int odt = 0; odt < (scaling ? 3 : 1); ++odt) {
            fg::clip::List L;
            L.count = 0;
            int64_t chunks = 0;
            for (int32_t i = 0; i <= a.count; ++i) {
                if (L.count == fg::clip::MAX_TENSORS || (i == a.count && L.count > 0)) {
                    L.chunks = uint32_t(chunks);
                    const int rc = launch(dt, odt, L);
                    if (rc != FG_OK) return rc;
                    L.count = 0;
                    chunks = 0;
                }
                if (i == a.count) break;
                const FgGradTensor& t = a.tensors[i];
                if (t.count == 0 || t.dtype != dt || (scaling && (t.out == nullptr || t.out_dtype != odt))) continue;
                const int esz = elem_size(dt);
                fg::clip::Item& it = L.items[L.count++];
                it.in = t.grad; it.out = t.out; it.count = t.count;
                it.first = uint32_t(chunks);
                it.wide_in = reinterpret_cast<uintptr_t>(t.grad) % 16 == 0;
                // the results of one vector: 16 bytes of the wider type, as many of the other
                it.wide_out = reinterpret_cast<uintptr_t>(t.out) % (16 / std::max(esz, elem_size(odt)) * elem_size(odt)) == 0;
                chunks += (t.count * esz + fg::clip::CHUNK_BYTES - 1) / fg::clip::CHUNK_BYTES;
                if (chunks > (int64_t(1) << 31)) return FG_ENOTSUP;
            }
        }
    return FG_OK;
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
    int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    double* total = reinterpret_cast<double*>(a->workspace);
    double* partial = total + 1;
    const int64_t cap = std::min<int64_t>(fg::clip::MAX_GRID, 6 * int64_t(d->sms));   // what is resident at once
    int64_t partials = 0;
    rc = for_lists(*a, false, [&](int dt, int, const fg::clip::List& L) {
        const unsigned grid = unsigned(std::min<int64_t>(cap, L.chunks));
        double* at = partial + partials;
        partials += grid;
        return launch_early(dt == FG_DTYPE_F32   ? fg::clip::norm_kernel<FG_DTYPE_F32>
                            : dt == FG_DTYPE_F16 ? fg::clip::norm_kernel<FG_DTYPE_F16>
                                                 : fg::clip::norm_kernel<FG_DTYPE_BF16>,
                            grid, st, L, at);
    });
    if (rc != FG_OK) return rc;
    // several launches' sums are added up once, not in every CTA
    const bool one = partials <= cap;
    if (!one && (rc = launch_early(fg::clip::total_kernel, 1, st, (const double*)partial, partials, total)) != FG_OK)
        return rc;
    const double* sums = one ? partial : total;
    const int64_t count = one ? partials : 1;
    float* norm = a->out_norm;   // until a launch writes it
    rc = for_lists(*a, true, [&](int dt, int odt, const fg::clip::List& L) {
        const unsigned grid = unsigned(std::min<int64_t>(cap, L.chunks));
        const int r = launch_early(scale_kernel_of(dt, odt), grid, st, L, sums, count, a->max_norm, a->scale, norm);
        norm = nullptr;
        return r;
    });
    if (rc == FG_OK && norm != nullptr) {   // nothing to scale
        fg::clip::List L;
        L.count = 0;
        L.chunks = 0;
        rc = launch_early(scale_kernel_of(0, 0), 1, st, L, sums, count, a->max_norm, a->scale, norm);
    }
    return rc;
}

}  // extern "C"
