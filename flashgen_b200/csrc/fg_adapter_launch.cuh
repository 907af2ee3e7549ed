// fg_adapter_launch.cuh — launches of the LM-head kernels; included by the units
// that instantiate them.
#pragma once

#include <algorithm>
#include <atomic>

#include "fg_adapter.cuh"

namespace fg {
namespace adapt {

template <int CG, int DT, int ODT, int RC, bool SMALL>
int launch_project(const Params& P, const CUtensorMap& wmap, const CUtensorMap& xmap, bool chained,
                   host::DevInfo* d, cudaStream_t st) {
    auto kern = project_kernel<CG, DT, ODT, RC, SMALL>;
    static std::atomic<bool> attr_set[host::kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return FG_EDEVICE;
    // what the SM has, less this kernel's static part and down_kernel's CTA beside it
    const int room = std::min(d->smem_optin - int(sizeof(Control)) - 256, d->smem_per_sm - 5 * 1024);
    if (!attr_set[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, room) != cudaSuccess)
            return FG_EDEVICE;
        attr_set[dev].store(true, std::memory_order_release);
    }
    Params Q = P;
    Q.chained = chained;
    const int stage = P.kb * (A_BYTES + P.nt / CG * TILE_K * 2);
    Q.stages = std::min(MAX_STAGES, (room - 1024) / stage);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min(P.nvt * P.ntile, d->sms / CG) * CG);
    cfg.blockDim = dim3(Epilogue<ODT, RC, SMALL>::THREADS);
    cfg.dynamicSmemBytes = size_t(1024 + Q.stages * stage);
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    if (CG == 2) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = 2;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
    cfg.attrs = attr;
    return cudaLaunchKernelEx(&cfg, kern, wmap, xmap, Q) == cudaSuccess ? FG_OK : FG_ELAUNCH;
}

template <int DT, int ODT, int RC>
int launch_rank(const Params& P, const CUtensorMap& wmap, const CUtensorMap& xmap, bool pair,
                host::DevInfo* d, cudaStream_t st) {
    const bool first = P.adapters || P.copy || P.out_status;
    if (first) {
        // the same division of the SM's memory as project_kernel's, so that both fit beside each other
        static std::atomic<bool> attr_set[host::kMaxDevices] = {};
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return FG_EDEVICE;
        if (!attr_set[dev].load(std::memory_order_acquire)) {
            if (cudaFuncSetAttribute(down_kernel<DT, RC ? RC : 1>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     (int)cudaSharedmemCarveoutMaxShared) != cudaSuccess)
                return FG_EDEVICE;
            attr_set[dev].store(true, std::memory_order_release);
        }
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(P.batch);
        cfg.blockDim = dim3(DOWN_THREADS);
        cfg.stream = st;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, down_kernel<DT, RC ? RC : 1>, P) != cudaSuccess) return FG_ELAUNCH;
    }
    if (pair) return launch_project<2, DT, ODT, RC, false>(P, wmap, xmap, first, d, st);
    // (Ranks 17 to 32 do better with more warps around 32 rows: dim 2048, V 50257, rank 32, 32
    // rows 52 us against 58, rank 20 51 against 55; 50 and 64 rows differ by less than their
    // spread, 8 and 16 rows lose one to three: dim 4096, V 32000, 16 rows 60.2 against 58.6)
    if constexpr (ODT == FG_DTYPE_F32 && RC != 2)
        if (P.nt <= SMALL_NT) return launch_project<1, DT, ODT, RC, true>(P, wmap, xmap, first, d, st);
    return launch_project<1, DT, ODT, RC, false>(P, wmap, xmap, first, d, st);
}

template <int DT, int ODT>
int launch(const Params& P, const CUtensorMap& wmap, const CUtensorMap& xmap, bool pair, host::DevInfo* d,
           cudaStream_t st) {
    const int rc = P.adapters && P.slots > 0 ? (P.rank + 15) / 16 : 0;
    if (rc == 0) return launch_rank<DT, ODT, 0>(P, wmap, xmap, pair, d, st);
    if (rc == 1) return launch_rank<DT, ODT, 1>(P, wmap, xmap, pair, d, st);
    if (rc == 2) return launch_rank<DT, ODT, 2>(P, wmap, xmap, pair, d, st);
    if (rc <= 4) return launch_rank<DT, ODT, 4>(P, wmap, xmap, pair, d, st);
    return launch_rank<DT, ODT, 8>(P, wmap, xmap, pair, d, st);
}

}  // namespace adapt
}  // namespace fg
