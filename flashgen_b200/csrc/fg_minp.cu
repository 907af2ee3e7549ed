// fg_minp.cu — C ABI entry points of sampling with min-p: argument checks and launches.
#include <algorithm>
#include <atomic>
#include <mutex>

#include "fg_internal.h"
#include "fg_minp.cuh"

namespace {

using fg::host::DevInfo;
using fg::host::elem_size;

constexpr int32_t kMaxBatch = 1 << 24;
constexpr int kMaxClusters = 64;    // of wide_kernel

int slots_for(int64_t ids) {
    int s = 64;
    while (s < 2 * ids) s <<= 1;
    return s;
}
bool penalties(const FgSampleArgs& a) {
    return a.hist_offsets && (a.repetition_penalty || a.presence_penalty || a.frequency_penalty);
}
size_t marks_bytes(int64_t batch) { return size_t(std::max<int64_t>(batch, 1) + 7) / 8 * 8; }
// Distinct columns of a row's history at most.
int64_t distinct(int32_t hist_max_len, int32_t vocab) { return std::max(1, std::min(hist_max_len, vocab)); }

// CTAs a row: a power of two of which the batch fills no more than three an SM (what fits
// without histories), with half a round of copies for each. Kernels alone: one row of 256000
// fp32 with 1, 2, 4, 8 CTAs 41.6, 30, 25, 22 us; 1024 rows of 128256 bf16 182, 207, 254, 340 us.
int ctas_per_row(int32_t batch, int vocab, int elem, const DevInfo* d) {
    const int64_t chunks = int64_t(vocab) * elem / 16;
    int G = 1;
    while (2 * G <= fg::minp::MAX_G && int64_t(batch) * 2 * G <= 3 * int64_t(d->sms) &&
           chunks / (2 * G) >= fg::minp::NT * fg::minp::UNROLL / 2)
        G *= 2;
    return G;
}

// Raises a kernel's limit of dynamic shared memory to `bytes`. Under a lock: of two threads the
// one that needs less must not take back what the other has just set.
std::mutex limits;

template <class K>
bool set_smem(K kern, std::atomic<int>* done, int bytes) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    if (done[dev].load(std::memory_order_acquire) >= bytes) return true;
    std::lock_guard<std::mutex> lock(limits);
    if (done[dev].load(std::memory_order_acquire) >= bytes) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done[dev].store(bytes, std::memory_order_release);
    return true;
}

// Whether a cluster of sixteen CTAs with `smem` bytes each finds room (asked once a size and device).
template <class K>
bool sixteen_fit(K kern, std::atomic<int>* largest, int smem) {
    int dev = 0, active = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    if (largest[dev].load(std::memory_order_acquire) >= smem) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(fg::minp::NT);
    cfg.dynamicSmemBytes = size_t(smem);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 16;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&active, kern, &cfg) != cudaSuccess || active < 1) return false;
    largest[dev].store(smem, std::memory_order_release);
    return true;
}

int launch_early(void (*kern)(fg::minp::Params, int), unsigned grid, unsigned threads, size_t smem, int cluster,
                 cudaStream_t st, const fg::minp::Params& P) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, P, cluster) == cudaSuccess ? FG_OK : FG_ELAUNCH;
}

template <int DT>
int launch(fg::minp::Params P, DevInfo* d, cudaStream_t st) {
    using namespace fg::minp;
    static std::atomic<int> rows_smem[fg::host::kMaxDevices] = {}, wide_smem[fg::host::kMaxDevices] = {};
    static std::atomic<int> uncached_smem[fg::host::kMaxDevices] = {};
    const int esz = fg::Elem<DT>::SIZE;
    int G = ctas_per_row(P.batch, P.vocab, esz, d);
    const int smem = RING_BYTES + CAP * int(sizeof(Candidate)) + (P.penalties ? P.slots * 8 + ROW_FILTER * 4 : 0);
    static std::atomic<int> sixteen[fg::host::kMaxDevices] = {};
    if (!set_smem(rows_kernel<DT>, rows_smem, smem)) return FG_EDEVICE;
    if (G > 8 && !sixteen_fit(rows_kernel<DT>, sixteen, smem)) G = 8;
    int rc = launch_early(rows_kernel<DT>, unsigned(P.batch) * G, NT, smem, G, st, P);
    if (rc != FG_OK) return rc;
    // wide_kernel: the slice's keys in shared memory where they fit
    auto fixed = [&](int g) { return 16 * MEMBERS + bins_bytes(g); };
    auto keys = [&](int g) {
        const int64_t chunks = int64_t(P.vocab) * esz / 16 + 1;
        return (chunks + g - 1) / g * (16 / esz) + 2 * (16 / esz) + KEY_PAD;
    };
    const int room = d->smem_optin - int(sizeof(WideShared) + sizeof(ExpTable)) - 1024;
    // Four CTAs a row where the batch can have work for every SM; how many rows are wide is not known
    // here. wide_kernel with four and with eight CTAs a row: 512 x 128256 bf16, mixed, with
    // histories 142 and 200 us; but where few rows are wide, eight are faster: 1024 x 128256 bf16
    // 55 and 41, 256 x 32000 bf16 38 and 36, 37 x 50257 f16 with histories 51 and 44.
    const int W = P.batch > d->sms / 8 && fixed(4) + 4 * keys(4) <= room ? 4 : WIDE_G;
    const bool cached = fixed(W) + 4 * keys(W) <= room;
    const int wsmem = fixed(W) + 4 * (cached ? int(keys(W)) : P.penalties ? FILTER_WORDS : 0);
    if (!set_smem(cached ? wide_kernel<DT, true> : wide_kernel<DT, false>, cached ? wide_smem : uncached_smem, wsmem))
        return FG_EDEVICE;
    const int clusters = std::min({int(P.batch), kMaxClusters, d->sms / W});
    return launch_early(cached ? wide_kernel<DT, true> : wide_kernel<DT, false>, unsigned(clusters * W), WNT, wsmem, W,
                        st, P);
}

// fg_sample_min_p; with `only` the rows that have min-p.
int sample(const FgMinPArgs* m, bool only, void* stream);

}  // namespace

extern "C" {

size_t fg_sample_min_p_workspace_size(int32_t batch, int32_t vocab, int32_t hist_max_len) {
    if (batch < 0 || vocab < 1 || hist_max_len < 0) return 0;
    return marks_bytes(batch) + (hist_max_len > 0 ? size_t(kMaxClusters) * slots_for(distinct(hist_max_len, vocab)) * 8 : 0);
}

int fg_sample_min_p(const FgMinPArgs* m, void* stream) { return sample(m, false, stream); }

int fg_sample_min_p_rows(const FgMinPArgs* m, void* stream) { return sample(m, true, stream); }

}  // extern "C"

namespace {

int sample(const FgMinPArgs* m, bool only, void* stream) {
    if (m == nullptr || (only && m->min_p == nullptr)) return FG_EINVAL;
    const FgSampleArgs* a = &m->sample;
    const int esz = elem_size(a->dtype);
    if (esz == 0 || a->logits == nullptr || a->batch < 0 || a->vocab < 1 || a->row_stride < a->vocab) return FG_EINVAL;
    if (reinterpret_cast<uintptr_t>(a->logits) % esz != 0) return FG_EINVAL;
    if (a->uniforms == nullptr || a->out_ids == nullptr) return FG_EINVAL;
    if ((a->hist_ids == nullptr) != (a->hist_offsets == nullptr) || a->vocab_offset < 0) return FG_EINVAL;
    const int64_t total = a->vocab_total > 0 ? a->vocab_total : a->vocab;
    // min-p and top-p need the whole row: a shard's maximum is not its
    if (a->vocab_offset != 0 || total != a->vocab) return FG_EINVAL;
    if (a->vocab > (1 << 28) || a->batch > kMaxBatch) return FG_ENOTSUP;
    fg::minp::Params P{};
    if (a->hist_offsets != nullptr && a->hist_max_len < 0) return FG_EINVAL;
    P.penalties = penalties(*a);
    if (P.penalties) {
        // (a bound of 0 leaves room for a few ids, as in fg_sample: rows with more are marked)
        P.hist_max_len = std::max(1, a->hist_max_len);
        P.wide_slots = slots_for(distinct(a->hist_max_len, a->vocab));
        P.slots = std::min(P.wide_slots, slots_for(fg::minp::HIST_CAP));
        P.tables = reinterpret_cast<uint2*>(reinterpret_cast<char*>(a->workspace) + marks_bytes(a->batch));
    }
    const size_t need = fg_sample_min_p_workspace_size(a->batch, a->vocab, P.hist_max_len);
    if (a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 8 != 0 || a->workspace_bytes < need)
        return FG_EINVAL;
    P.marks = reinterpret_cast<uint8_t*>(a->workspace);
    if (a->batch == 0) return FG_OK;
    P.logits = a->logits; P.row_stride = a->row_stride; P.batch = a->batch; P.vocab = a->vocab;
    P.vocab_offset = 0; P.vocab_total = total;
    P.hist_ids = a->hist_ids; P.hist_offsets = a->hist_offsets;
    P.temperature = a->temperature; P.top_p = a->top_p; P.top_k = a->top_k; P.min_p = m->min_p;
    P.rep = a->repetition_penalty; P.pres = a->presence_penalty; P.freq = a->frequency_penalty;
    P.greedy = a->greedy; P.uniforms = a->uniforms;
    P.out_ids = a->out_ids; P.out_status = a->out_status; P.out_probs = a->out_probs;
    P.out_logprobs = m->out_logprobs; P.out_kept = m->out_kept;
    P.only = only;
    P.mass_shift = 62 - fg::host::bits_for(a->vocab);
    DevInfo* d = nullptr;
    const int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (a->dtype) {
        case FG_DTYPE_F32: return launch<FG_DTYPE_F32>(P, d, st);
        case FG_DTYPE_F16: return launch<FG_DTYPE_F16>(P, d, st);
        default: return launch<FG_DTYPE_BF16>(P, d, st);
    }
}

}  // namespace
