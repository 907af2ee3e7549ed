// fg_logprobs.cu — C ABI entry points of the token log probabilities and their
// gradient: argument checks and launches.
#include <algorithm>
#include <atomic>

#include "fg_internal.h"
#include "fg_logprobs.cuh"

namespace {

using fg::host::DevInfo;
using fg::host::elem_size;

bool rows_ok(const void* p, int dtype, int64_t stride, int32_t vocab) {
    return p != nullptr && stride >= vocab && reinterpret_cast<uintptr_t>(p) % elem_size(dtype) == 0;
}

constexpr int32_t kMaxRows = 1 << 30;

// CTAs per row for a batch too small to fill the machine with one each: as many as
// find room at once (three an SM), with at least two chunks for each of their threads.
// Clusters of eight find room less easily. With four an SM instead: 256 rows of 32000
// f16 logits 12.0 us, not 10.9; eight CTAs a row for 50 rows of 128256 bf16 logits: 13.7 us,
// four 11.7; one CTA for a row of 256000 f32 logits: 32 us, eight 9.6.
int ctas_per_row(int32_t batch, int vocab, int elem, const DevInfo* d) {
    const int64_t chunks = int64_t(vocab) * elem / 16;
    int G = 1;
    while (2 * G <= fg::lp::MAX_G && int64_t(batch) * 2 * G <= (2 * G == 8 ? 2 : 3) * d->sms &&
           chunks / (2 * G) >= 2 * fg::lp::THREADS)
        G *= 2;
    return G;
}

template <class K>
bool set_once(K kern, std::atomic<bool>* done, cudaFuncAttribute attr, int value) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    if (done[dev].load(std::memory_order_acquire)) return true;
    if (cudaFuncSetAttribute(kern, attr, value) != cudaSuccess) return false;
    done[dev].store(true, std::memory_order_release);
    return true;
}

// A launch that may begin while the stream's previous kernel ends: the kernel itself
// waits for that one before it touches memory.
template <class... Params, class... Args>
int launch_early(void (*kern)(Params...), unsigned grid, unsigned threads, size_t smem, unsigned cluster,
                 cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? FG_OK : FG_ELAUNCH;
}

template <int DT, bool TOP>
int launch_forward(const fg::lp::Params& P, int32_t batch, cudaStream_t st) {
    DevInfo* d = nullptr;
    const int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;
    const int G = ctas_per_row(batch, P.vocab, fg::Elem<DT>::SIZE, d);
    if (G == 1) {
        auto kern = fg::lp::rows_kernel<DT, TOP>;
        constexpr int smem = fg::lp::RING_BYTES;
        static std::atomic<bool> sized[fg::host::kMaxDevices] = {}, carved[fg::host::kMaxDevices] = {};
        if (!set_once(kern, sized, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ||
            !set_once(kern, carved, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared))
            return FG_EDEVICE;
        const int grid = std::min<int64_t>(batch, fg::lp::CTAS_PER_SM * d->sms);
        return launch_early(kern, grid, fg::lp::THREADS, smem, 1, st, P, int64_t(batch));
    }
    return launch_early(fg::lp::row_kernel<DT, TOP>, unsigned(batch) * G, fg::lp::THREADS, 0, G, st, P, G);
}

template <int DT>
int launch_forward(const fg::lp::Params& P, int32_t batch, cudaStream_t st) {
    return P.top ? launch_forward<DT, true>(P, batch, st) : launch_forward<DT, false>(P, batch, st);
}

template <int DT>
int launch_grad(const fg::lp::GradParams& P, int32_t batch, cudaStream_t st) {
    DevInfo* d = nullptr;
    const int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;
    // steps of GRAD_THREADS * GRAD_UNROLL chunks: one a CTA while there are fewer than eight
    // for an SM, up to four a CTA when there are many (five CTAs are resident with 16-bit
    // logits, six with fp32; cut for five instead, 100, 333 and 500 rows of 32001 and 64 and
    // 1024 of 128256 logits take the same time)
    const int64_t esz = fg::Elem<DT>::SIZE;
    const int64_t step = int64_t(fg::lp::GRAD_THREADS) * fg::lp::GRAD_UNROLL * 16 / esz;
    const int64_t steps = (P.vocab + step - 1) / step;
    const int64_t each = std::max<int64_t>(1, std::min<int64_t>(4, steps * batch / (8 * d->sms)));
    const int per_row = int((steps + each - 1) / each);
    const int32_t rows = std::max(1, (1 << 30) / per_row);   // rows a launch
    for (int32_t lo = 0; lo < batch; lo += rows) {
        fg::lp::GradParams Q = P;
        const int32_t n = std::min(rows, batch - lo);
        Q.logits = reinterpret_cast<const char*>(P.logits) + lo * P.row_stride * esz;
        Q.out_grad = reinterpret_cast<char*>(P.out_grad) + lo * P.grad_stride * esz;
        if (P.tokens) Q.tokens = P.tokens + lo;
        if (P.temperature) Q.temperature = P.temperature + lo;
        Q.max = P.max + lo;
        Q.logsum = P.logsum + lo;
        if (P.entropy) Q.entropy = P.entropy + lo;
        if (P.grad_logprobs) Q.grad_logprobs = P.grad_logprobs + lo;
        if (P.grad_entropy) Q.grad_entropy = P.grad_entropy + lo;
        const int rc = launch_early(fg::lp::logprob_grad_kernel<DT>, unsigned(n) * unsigned(per_row),
                                    fg::lp::GRAD_THREADS, 0, 1, st, Q, per_row);
        if (rc != FG_OK) return rc;
    }
    return FG_OK;
}

}  // namespace

extern "C" {

int fg_token_logprobs(const FgLogprobArgs* a, void* stream) {
    if (a == nullptr || elem_size(a->dtype) == 0 || a->batch < 0 || a->vocab < 1) return FG_EINVAL;
    if (!rows_ok(a->logits, a->dtype, a->row_stride, a->vocab)) return FG_EINVAL;
    if (a->top < 0 || a->top > FG_LOGPROB_MAX_TOP) return FG_EINVAL;
    if (a->batch > kMaxRows || a->vocab > (1 << 28)) return FG_ENOTSUP;
    if (a->batch == 0) return FG_OK;
    fg::lp::Params P{};
    P.logits = a->logits; P.row_stride = a->row_stride; P.vocab = a->vocab;
    P.top = (a->out_top_ids || a->out_top_logprobs) ? a->top : 0;
    P.tokens = a->tokens; P.temperature = a->temperature;
    P.out_logprobs = a->out_logprobs; P.out_entropy = a->out_entropy; P.out_max = a->out_max;
    P.out_logsum = a->out_logsum; P.out_rank = a->out_rank; P.out_top_ids = a->out_top_ids;
    P.out_top_logprobs = a->out_top_logprobs; P.out_status = a->out_status;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (a->dtype) {
        case FG_DTYPE_F32: return launch_forward<FG_DTYPE_F32>(P, a->batch, st);
        case FG_DTYPE_F16: return launch_forward<FG_DTYPE_F16>(P, a->batch, st);
        default: return launch_forward<FG_DTYPE_BF16>(P, a->batch, st);
    }
}

int fg_token_logprobs_grad(const FgLogprobGradArgs* a, void* stream) {
    if (a == nullptr || elem_size(a->dtype) == 0 || a->batch < 0 || a->vocab < 1 || a->reserved != 0)
        return FG_EINVAL;
    if (!rows_ok(a->logits, a->dtype, a->row_stride, a->vocab) ||
        !rows_ok(a->out_grad, a->dtype, a->grad_stride, a->vocab))
        return FG_EINVAL;
    if (a->out_grad == a->logits && a->grad_stride != a->row_stride) return FG_EINVAL;
    if (a->max == nullptr || a->logsum == nullptr) return FG_EINVAL;
    if (a->grad_entropy != nullptr && a->entropy == nullptr) return FG_EINVAL;
    if (a->batch > kMaxRows || a->vocab > (1 << 28)) return FG_ENOTSUP;
    if (a->batch == 0) return FG_OK;
    fg::lp::GradParams P{};
    P.logits = a->logits; P.row_stride = a->row_stride; P.vocab = a->vocab;
    P.tokens = a->tokens; P.temperature = a->temperature; P.max = a->max; P.logsum = a->logsum;
    P.entropy = a->entropy; P.grad_logprobs = a->grad_logprobs; P.grad_entropy = a->grad_entropy;
    P.out_grad = a->out_grad; P.grad_stride = a->grad_stride;
    // the logits themselves may become the gradient (each thread reads what it writes), a
    // part of them may not
    const int64_t esz = elem_size(a->dtype), wide = a->vocab * esz;
    if (a->out_grad != a->logits && fg::host::rows_meet({a->logits, a->batch, a->row_stride * esz, wide},
                                                        {a->out_grad, a->batch, a->grad_stride * esz, wide}))
        return FG_EINVAL;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (a->dtype) {
        case FG_DTYPE_F32: return launch_grad<FG_DTYPE_F32>(P, a->batch, st);
        case FG_DTYPE_F16: return launch_grad<FG_DTYPE_F16>(P, a->batch, st);
        default: return launch_grad<FG_DTYPE_BF16>(P, a->batch, st);
    }
}

}  // extern "C"
