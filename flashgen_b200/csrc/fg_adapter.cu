// fg_adapter.cu — C ABI entry points of the LM head with per-row adapters:
// argument checks, workspace layout and launches.
#include <algorithm>

#include "fg_adapter.cuh"
#include "fg_internal.h"

namespace {

using fg::host::elem_size;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <int DT, int ODT>
int launch(const fg::adapt::Params& P, cudaStream_t st) {
    if (P.slots > 0 || P.out_status) fg::adapt::down_kernel<DT><<<P.batch, fg::adapt::DOWN_THREADS, 0, st>>>(P);
    const dim3 grid((P.vocab + fg::adapt::TILE - 1) / fg::adapt::TILE,
                    (P.batch + fg::adapt::TILE - 1) / fg::adapt::TILE);
    fg::adapt::project_kernel<DT, ODT><<<grid, 256, 0, st>>>(P);
    return cudaGetLastError() == cudaSuccess ? FG_OK : FG_ELAUNCH;
}

constexpr int32_t kMaxRows = 1 << 20;

}  // namespace

extern "C" {

size_t fg_adapter_workspace_size(int32_t batch, int32_t dim, int32_t rank, int32_t slots) {
    if (batch < 0 || batch > kMaxRows || dim < 1 || slots < 0) return 0;
    if (slots > 0 && (rank < 16 || rank > FG_ADAPTER_MAX_RANK || rank % 16 != 0)) return 0;
    return std::max<size_t>(256, slots > 0 ? sizeof(float) * size_t(batch) * rank : 0);
}

int fg_adapter_logits(const FgAdapterArgs* a, void* stream) {
    if (a == nullptr || a->reserved != 0) return FG_EINVAL;
    if (a->dtype != FG_DTYPE_F16 && a->dtype != FG_DTYPE_BF16) return FG_EINVAL;
    if (a->out_dtype != a->dtype && a->out_dtype != FG_DTYPE_F32) return FG_EINVAL;
    if (a->batch < 0 || a->dim < 1 || a->vocab < 1 || a->slots < 0) return FG_EINVAL;
    if (a->hidden == nullptr || a->weight == nullptr || a->out == nullptr) return FG_EINVAL;
    if (a->hidden_stride < a->dim || a->weight_stride < a->dim || a->out_stride < a->vocab) return FG_EINVAL;
    if (!aligned(a->hidden, 2) || !aligned(a->out, elem_size(a->out_dtype))) return FG_EINVAL;
    if (!aligned(a->weight, 16) || a->weight_stride % 8 != 0) return FG_EINVAL;
    if (a->slots > 0) {
        if (a->down == nullptr || a->up == nullptr || a->scales == nullptr) return FG_EINVAL;
        if (a->rank < 16 || a->rank > FG_ADAPTER_MAX_RANK || a->rank % 16 != 0) return FG_EINVAL;
        if (!aligned(a->down, 16) || !aligned(a->up, 16) || a->down_stride < a->dim || a->down_stride % 8 != 0)
            return FG_EINVAL;
    }
    if (a->batch > kMaxRows || a->vocab > (1 << 28) || a->dim > (1 << 20)) return FG_ENOTSUP;
    const size_t need = fg_adapter_workspace_size(a->batch, a->dim, a->rank, a->slots);
    if (a->workspace == nullptr || !aligned(a->workspace, 256) || a->workspace_bytes < need) return FG_EINVAL;
    if (a->batch == 0) return FG_OK;
    fg::adapt::Params P{};
    P.hidden = a->hidden; P.weight = a->weight; P.down = a->down; P.up = a->up; P.scales = a->scales;
    P.adapters = a->slots > 0 || a->out_status ? a->adapters : nullptr;
    P.out = a->out; P.out_status = a->out_status; P.u = reinterpret_cast<float*>(a->workspace);
    P.batch = a->batch; P.dim = a->dim; P.vocab = a->vocab; P.rank = a->rank; P.slots = a->slots;
    P.hidden_stride = a->hidden_stride; P.weight_stride = a->weight_stride; P.down_stride = a->down_stride;
    P.out_stride = a->out_stride;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool f32 = a->out_dtype == FG_DTYPE_F32;
    if (a->dtype == FG_DTYPE_F16)
        return f32 ? launch<FG_DTYPE_F16, FG_DTYPE_F32>(P, st) : launch<FG_DTYPE_F16, FG_DTYPE_F16>(P, st);
    return f32 ? launch<FG_DTYPE_BF16, FG_DTYPE_F32>(P, st) : launch<FG_DTYPE_BF16, FG_DTYPE_BF16>(P, st);
}

}  // extern "C"
