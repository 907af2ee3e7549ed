// fg_linear.cu — C ABI entry points of the fused linear block and its gradients:
// argument checks, workspace layout, the choice of tiles, launches.
#include <algorithm>
#include <atomic>

#include "fg_internal.h"
#include "fg_linear.cuh"
#include "fg_tma.h"

namespace {

using fg::host::DevInfo;
using fg::host::Rows;
using fg::host::rows_meet;
using fg::lin::MAX_STAGES;
using fg::lin::Params;
using fg::lin::TILE_K;
using fg::lin::TILE_L;

constexpr int32_t kMaxTokens = 1 << 20, kMaxInner = 1 << 20, kMaxOuter = 1 << 28;

// fg_linear_set_wait
std::atomic<int64_t> g_wait_ns{fg::lin::DEFAULT_WAIT_NS};
std::atomic<int32_t> g_withhold{-1};

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// A 16-bit matrix as TMA can read it: rows on 16-byte boundaries.
bool tma_ready(const void* p, int64_t rows, int64_t stride) {
    return aligned(p, 16) && (rows <= 1 || stride % 8 == 0);
}
size_t copy_bytes(const void* p, int64_t rows, int64_t dim, int64_t stride) {
    return tma_ready(p, rows, stride) ? 0 : round256(2 * size_t(rows) * size_t(round8(dim)));
}

template <class... Params_, class... Args>
int launch_early(void (*kern)(Params_...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t st,
                 const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
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

// A matrix of an operand: where it is for TMA (the caller's or an aligned copy).
struct Matrix {
    const void* p;
    int64_t rows, dim, stride;
};
// Copies `m` to `room` where TMA cannot read it as it lies.
int make_ready(Matrix& m, void* room, DevInfo* d, cudaStream_t st) {
    if (tma_ready(m.p, m.rows, m.stride)) {
        if (m.rows <= 1) m.stride = round8(m.dim);
        return FG_OK;
    }
    const int64_t stride = round8(m.dim), vecs = m.rows * (stride / 8);
    const unsigned grid = unsigned(std::min<int64_t>((vecs + 255) / 256, 16 * int64_t(d->sms)));
    const int rc = launch_early(fg::lin::align_kernel, dim3(grid), 256, 0, 1, st, (const uint16_t*)m.p, m.stride,
                                (uint16_t*)room, stride, m.rows, int(m.dim));
    m.p = room;
    m.stride = stride;
    return rc;
}

// How a product is cut: CTAs that share a tile's lanes (cg) or its sum (splits), columns.
struct Cut {
    int cg, nt, splits;
};

// The cut with the least estimated time, in SM clocks. A step of K takes a CTA 2 nt clocks
// of tensor pipe, or its operands' bytes at what L2 gave an SM while all of them read (64 bytes
// a clock, 46 each of a pair); a wave ends with its last tile's epilogue, a split sum with the
// parts' way through the cluster. Microseconds measured, bf16, bias, SiLU and residual, for
// columns a tile x splits (pairs: p): 1 token of 4096 x 4096 16 x 4 11.1, 16 x 2 14.3, 16 x 1 20.1;
// 64 tokens 64 x 4 13.7, 64 x 2 17.4, 16 x 1 20.8; 256 tokens 256 x 4 22.1, 128 x 2 22.3, 64 x 1
// 23.2, p64 25.3; 512 tokens 128 x 1 25.6, p128 28.3, p256 30.2; 1024 tokens p256 32.5, 256 x 1 33.2,
// 128 x 1 44.7; 2048 tokens p256 55.8, 256 x 1 57.6; 1024 tokens of 1024 x 1024 64 x 1 9.4, p64 10.5,
// 128 x 1 10.8; 1 token of 2048 x 2048 16 x 4 6.9, 16 x 8 11.2.
Cut choose(int64_t L, int64_t C, int64_t K, bool b_mn, int sms) {
    const int64_t steps = (K + TILE_K - 1) / TILE_K;
    Cut best{1, 64, 1};
    double least = 1e300;
    for (int cg = 1; cg <= 2; ++cg) {
        const int unit = b_mn ? 64 * cg : 16 * cg;
        int last = 0;
        for (int want : {16, 32, 64, 96, 128, 192, 256}) {
            // tiles of equal width, no wider than `want`
            const int64_t n = (C + want - 1) / want;
            const int nt = int(((C + n - 1) / n + unit - 1) / unit * unit);
            if (nt > 256 || nt == last) continue;
            last = nt;
            const int64_t tiles = (L + TILE_L * cg - 1) / (TILE_L * cg) * ((C + nt - 1) / nt);
            for (int s = 1; s <= (cg == 1 ? fg::lin::MAX_SPLITS : 1) && s <= steps; s *= 2) {
                // (clusters of eight find less room than their CTAs: 16 of them take two turns)
                if (s > 1 && tiles * s > (s == 8 ? sms * 3 / 4 : s == 4 ? sms * 15 / 16 : sms)) break;
                const double waves = double((tiles * cg * s + sms - 1) / sms);
                const double bytes = 16384.0 + nt / cg * 128.0;
                const double step = std::max(2.0 * nt, bytes / (cg == 1 ? 64.0 : 46.0));
                const double time = waves * (double((steps + s - 1) / s) * step) + 12.0 * nt + (s > 1 ? 2500.0 + 16.0 * nt : 0.0);
                if (time < least) {
                    least = time;
                    best = {cg, nt, s};
                }
            }
        }
    }
    return best;
}

template <int CG, int DT, bool A_MN, bool B_MN>
int launch_product(Params P, const CUtensorMap& amap, const CUtensorMap& bmap, DevInfo* d, cudaStream_t st) {
    auto kern = fg::lin::product_kernel<CG, DT, A_MN, B_MN>;
    static std::atomic<bool> attr_set[fg::host::kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return FG_EDEVICE;
    const int room = d->smem_optin - int(sizeof(fg::lin::Control)) - 256;
    if (!attr_set[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, room) != cudaSuccess)
            return FG_EDEVICE;
        attr_set[dev].store(true, std::memory_order_release);
    }
    // as many stages as fit: more than half of the SM's memory, so that it never holds two
    // CTAs of these kernels, whose tensor memory one might wait for while its cluster waits
    const int stage = fg::lin::A_BYTES + P.nt / CG * TILE_K * 2;
    P.stages = std::min(MAX_STAGES, (room - 1024) / stage);
    const int64_t tiles = int64_t(P.nl) * P.nc;
    const int share = CG * P.splits;
    const int64_t places = P.splits > 1 ? tiles : std::max<int64_t>(1, std::min<int64_t>(tiles, d->sms / CG));
    return launch_early(kern, dim3(unsigned(places * share)), fg::lin::THREADS, size_t(1024 + P.stages * stage),
                        unsigned(share), st, amap, bmap, P);
}

// out = A B^T as fg_linear.cuh has it: a and b are the operands' matrices, [L, K] and
// [C, K], or [K, L] and [K, C] where the contiguous dimension is not the sum's.
int product(Params P, int dtype, const Matrix& a, bool a_mn, const Matrix& b, bool b_mn, DevInfo* d, cudaStream_t st) {
    const Cut cut = choose(P.L, P.C, P.K, b_mn, d->sms);
    P.nt = cut.nt;
    P.splits = cut.splits;
    P.nl = (P.L + TILE_L * cut.cg - 1) / (TILE_L * cut.cg);
    P.nc = (P.C + P.nt - 1) / P.nt;
    if (int64_t(P.nl) * P.nc > (1 << 30)) return FG_ENOTSUP;
    P.accs = std::min(fg::lin::MAX_ACC, 512 / P.nt);
    P.tmem_cols = 32;
    while (P.tmem_cols < P.accs * P.nt) P.tmem_cols *= 2;
    P.wait_ns = uint64_t(g_wait_ns.load(std::memory_order_relaxed));
    P.withhold = g_withhold.load(std::memory_order_relaxed);
    CUtensorMap amap, bmap;
    if (!fg::host::encode_rows(&amap, dtype, a.p, a.rows, a.dim, a.stride, a_mn ? 64 : TILE_L) ||
        !fg::host::encode_rows(&bmap, dtype, b.p, b.rows, b.dim, b.stride, b_mn ? 64 : cut.nt / cut.cg))
        return FG_EDEVICE;
    const int which = (dtype == FG_DTYPE_BF16 ? 1 : 0) + 2 * (cut.cg - 1) + 4 * (a_mn ? b_mn ? 2 : 1 : 0);
    switch (which) {
        case 0: return launch_product<1, FG_DTYPE_F16, false, false>(P, amap, bmap, d, st);
        case 1: return launch_product<1, FG_DTYPE_BF16, false, false>(P, amap, bmap, d, st);
        case 2: return launch_product<2, FG_DTYPE_F16, false, false>(P, amap, bmap, d, st);
        case 3: return launch_product<2, FG_DTYPE_BF16, false, false>(P, amap, bmap, d, st);
        case 4: return launch_product<1, FG_DTYPE_F16, true, false>(P, amap, bmap, d, st);
        case 5: return launch_product<1, FG_DTYPE_BF16, true, false>(P, amap, bmap, d, st);
        case 6: return launch_product<2, FG_DTYPE_F16, true, false>(P, amap, bmap, d, st);
        case 7: return launch_product<2, FG_DTYPE_BF16, true, false>(P, amap, bmap, d, st);
        case 8: return launch_product<1, FG_DTYPE_F16, true, true>(P, amap, bmap, d, st);
        case 9: return launch_product<1, FG_DTYPE_BF16, true, true>(P, amap, bmap, d, st);
        case 10: return launch_product<2, FG_DTYPE_F16, true, true>(P, amap, bmap, d, st);
        default: return launch_product<2, FG_DTYPE_BF16, true, true>(P, amap, bmap, d, st);
    }
}

bool shape_ok(int dtype, int32_t tokens, int32_t inner, int32_t outer, int32_t act) {
    return (dtype == FG_DTYPE_F16 || dtype == FG_DTYPE_BF16) && tokens >= 0 && inner >= 1 && outer >= 1 &&
           act >= FG_ACT_NONE && act <= FG_ACT_SILU;
}
bool matrix_ok(const void* p, int64_t stride, int64_t dim, size_t align = 2) {
    return p != nullptr && stride >= dim && aligned(p, align);
}
bool room_ok(const void* ws, size_t bytes, size_t need) {
    return need == 0 || (ws != nullptr && aligned(ws, 256) && bytes >= need);
}

// Whether dz needs memory of its own.
bool dz_written(const FgLinearGradArgs& a) {
    const bool wanted = a.grad_x != nullptr || a.grad_weight != nullptr;
    return wanted && (a.activation != FG_ACT_NONE || !tma_ready(a.grad_out, a.tokens, a.grad_out_stride));
}
struct GradLayout {
    size_t dz, sums, x, weight, total;
};
GradLayout grad_layout(const FgLinearGradArgs& a) {
    GradLayout L{};
    const size_t blocks = (size_t(a.tokens) + fg::lin::SLOPE_ROWS - 1) / fg::lin::SLOPE_ROWS;
    L.sums = dz_written(a) ? round256(2 * size_t(a.tokens) * size_t(round8(a.outer))) : 0;
    L.x = L.sums + (a.grad_bias ? round256(4 * blocks * size_t(a.outer)) : 0);
    L.weight = L.x + (a.grad_weight ? copy_bytes(a.x, a.tokens, a.inner, a.x_stride) : 0);
    L.total = L.weight + (a.grad_x ? copy_bytes(a.weight, a.outer, a.inner, a.weight_stride) : 0);
    return L;
}

template <int DT>
int launch_slope(const fg::lin::SlopeParams& S, int act, void* grad_bias, cudaStream_t st) {
    using namespace fg::lin;
    const unsigned blocks = unsigned((S.tokens + SLOPE_ROWS - 1) / SLOPE_ROWS);
    auto kern = act == FG_ACT_RELU        ? slope_kernel<DT, FG_ACT_RELU>
                : act == FG_ACT_GELU      ? slope_kernel<DT, FG_ACT_GELU>
                : act == FG_ACT_GELU_TANH ? slope_kernel<DT, FG_ACT_GELU_TANH>
                : act == FG_ACT_SILU      ? slope_kernel<DT, FG_ACT_SILU>
                                          : slope_kernel<DT, FG_ACT_NONE>;
    int rc = launch_early(kern, dim3(unsigned((S.outer + SLOPE_COLS - 1) / SLOPE_COLS), blocks), SLOPE_THREADS, 0, 1,
                          st, S);
    if (rc == FG_OK && grad_bias)
        rc = launch_early(fg::lin::bias_kernel<DT>, dim3(unsigned((S.outer + 31) / 32)), 256, 0, 1, st,
                          (const float*)S.sums, int(blocks), int(S.outer), (uint16_t*)grad_bias);
    return rc;
}

}  // namespace

extern "C" {

int fg_linear_set_wait(int64_t limit_ns, int32_t withhold) {
    if (limit_ns < 0 || limit_ns > fg::lin::DEFAULT_WAIT_NS || withhold < -1 || withhold >= fg::lin::MAX_ACC)
        return FG_EINVAL;
    g_wait_ns.store(limit_ns > 0 ? limit_ns : fg::lin::DEFAULT_WAIT_NS, std::memory_order_relaxed);
    g_withhold.store(withhold, std::memory_order_relaxed);
    return FG_OK;
}

size_t fg_linear_workspace_size(const FgLinearArgs* a) {
    if (a == nullptr || !shape_ok(a->dtype, a->tokens, a->inner, a->outer, a->activation)) return 0;
    return copy_bytes(a->x, a->tokens, a->inner, a->x_stride) +
           copy_bytes(a->weight, a->outer, a->inner, a->weight_stride);
}

int fg_linear(const FgLinearArgs* a, void* stream) {
    if (a == nullptr || a->reserved != 0) return FG_EINVAL;
    if (!shape_ok(a->dtype, a->tokens, a->inner, a->outer, a->activation)) return FG_EINVAL;
    if (!matrix_ok(a->x, a->x_stride, a->inner) || !matrix_ok(a->weight, a->weight_stride, a->inner) ||
        !matrix_ok(a->out, a->out_stride, a->outer) || !aligned(a->bias, 2) ||
        (a->residual && !matrix_ok(a->residual, a->residual_stride, a->outer)) ||
        (a->preact && !matrix_ok(a->preact, a->preact_stride, a->outer, 4)))
        return FG_EINVAL;
    if (a->tokens > kMaxTokens || a->inner > kMaxInner || a->outer > kMaxOuter) return FG_ENOTSUP;
    if (!room_ok(a->workspace, a->workspace_bytes, fg_linear_workspace_size(a))) return FG_EINVAL;
    if (a->tokens == 0) return FG_OK;
    const Rows x{a->x, a->tokens, a->x_stride * 2, int64_t(a->inner) * 2};
    const Rows w{a->weight, a->outer, a->weight_stride * 2, int64_t(a->inner) * 2};
    const Rows b{a->bias, a->bias ? 1 : 0, 0, int64_t(a->outer) * 2};
    const Rows r{a->residual, a->residual ? a->tokens : 0, a->residual_stride * 2, int64_t(a->outer) * 2};
    const Rows out{a->out, a->tokens, a->out_stride * 2, int64_t(a->outer) * 2};
    const Rows z{a->preact, a->preact ? a->tokens : 0, a->preact_stride * 4, int64_t(a->outer) * 4};
    for (const Rows& o : {out, z})
        if (rows_meet(o, x) || rows_meet(o, w) || rows_meet(o, b)) return FG_EINVAL;
    if (rows_meet(out, z) || rows_meet(z, r)) return FG_EINVAL;
    // the result may take the residual's place: a thread reads what it writes
    if (!(a->residual == a->out && a->residual_stride == a->out_stride) && rows_meet(out, r)) return FG_EINVAL;
    DevInfo* d = nullptr;
    int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    char* room = reinterpret_cast<char*>(a->workspace);
    Matrix xm{a->x, a->tokens, a->inner, a->x_stride}, wm{a->weight, a->outer, a->inner, a->weight_stride};
    const size_t x_room = copy_bytes(a->x, a->tokens, a->inner, a->x_stride);
    if ((rc = make_ready(xm, room, d, st)) != FG_OK || (rc = make_ready(wm, room + x_room, d, st)) != FG_OK) return rc;
    Params P{};
    P.out = a->out; P.out_stride = a->out_stride;
    P.bias = a->bias;
    P.residual = a->residual; P.residual_stride = a->residual_stride;
    P.preact = a->preact; P.preact_stride = a->preact_stride;
    P.L = a->outer; P.C = a->tokens; P.K = a->inner;
    P.act = a->activation;
    return product(P, a->dtype, wm, false, xm, false, d, st);
}

size_t fg_linear_grad_workspace_size(const FgLinearGradArgs* a) {
    if (a == nullptr || !shape_ok(a->dtype, a->tokens, a->inner, a->outer, a->activation)) return 0;
    return grad_layout(*a).total;
}

int fg_linear_grad(const FgLinearGradArgs* a, void* stream) {
    if (a == nullptr || a->reserved != 0) return FG_EINVAL;
    if (!shape_ok(a->dtype, a->tokens, a->inner, a->outer, a->activation)) return FG_EINVAL;
    if (!matrix_ok(a->grad_out, a->grad_out_stride, a->outer)) return FG_EINVAL;
    if (a->activation != FG_ACT_NONE && !matrix_ok(a->preact, a->preact_stride, a->outer, 4)) return FG_EINVAL;
    if (a->grad_x && (!matrix_ok(a->weight, a->weight_stride, a->inner) ||
                      !matrix_ok(a->grad_x, a->grad_x_stride, a->inner)))
        return FG_EINVAL;
    if (a->grad_weight && (!matrix_ok(a->x, a->x_stride, a->inner) ||
                           !matrix_ok(a->grad_weight, a->grad_weight_stride, a->inner)))
        return FG_EINVAL;
    if (!aligned(a->grad_bias, 2)) return FG_EINVAL;
    if (a->tokens > kMaxTokens || a->inner > kMaxInner || a->outer > kMaxOuter) return FG_ENOTSUP;
    if (!room_ok(a->workspace, a->workspace_bytes, fg_linear_grad_workspace_size(a))) return FG_EINVAL;
    const int64_t in2 = int64_t(a->inner) * 2, out2 = int64_t(a->outer) * 2;
    const Rows reads[4] = {{a->grad_out, a->tokens, a->grad_out_stride * 2, out2},
                           {a->preact, a->activation != FG_ACT_NONE ? a->tokens : 0, a->preact_stride * 4, 2 * out2},
                           {a->weight, a->grad_x ? a->outer : 0, a->weight_stride * 2, in2},
                           {a->x, a->grad_weight ? a->tokens : 0, a->x_stride * 2, in2}};
    const Rows writes[3] = {{a->grad_x, a->grad_x ? a->tokens : 0, a->grad_x_stride * 2, in2},
                            {a->grad_weight, a->grad_weight ? a->outer : 0, a->grad_weight_stride * 2, in2},
                            {a->grad_bias, a->grad_bias ? 1 : 0, 0, out2}};
    for (int i = 0; i < 3; ++i) {
        for (const Rows& r : reads)
            if (rows_meet(writes[i], r)) return FG_EINVAL;
        for (int j = 0; j < i; ++j)
            if (rows_meet(writes[i], writes[j])) return FG_EINVAL;
    }
    DevInfo* d = nullptr;
    int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->tokens == 0) {   // sums over nothing
        if (a->grad_weight && cudaMemset2DAsync(a->grad_weight, size_t(a->grad_weight_stride) * 2, 0, size_t(in2),
                                                size_t(a->outer), st) != cudaSuccess)
            return FG_ELAUNCH;
        if (a->grad_bias && cudaMemsetAsync(a->grad_bias, 0, size_t(out2), st) != cudaSuccess) return FG_ELAUNCH;
        return FG_OK;
    }
    const GradLayout W = grad_layout(*a);
    char* room = reinterpret_cast<char*>(a->workspace);
    Matrix dz{a->grad_out, a->tokens, a->outer, a->grad_out_stride};
    const bool written = dz_written(*a);
    if (written || a->grad_bias) {
        fg::lin::SlopeParams S{};
        S.grad = reinterpret_cast<const uint16_t*>(a->grad_out); S.grad_stride = a->grad_out_stride;
        S.preact = a->activation != FG_ACT_NONE ? a->preact : nullptr; S.preact_stride = a->preact_stride;
        S.dz = written ? reinterpret_cast<uint16_t*>(room) : nullptr; S.dz_stride = round8(a->outer);
        S.sums = a->grad_bias ? reinterpret_cast<float*>(room + W.sums) : nullptr;
        S.tokens = a->tokens; S.outer = a->outer;
        S.wide = tma_ready(a->grad_out, a->tokens, a->grad_out_stride) &&
                 (S.preact == nullptr || (aligned(S.preact, 16) && (a->tokens == 1 || a->preact_stride % 4 == 0)));
        rc = a->dtype == FG_DTYPE_F16 ? launch_slope<FG_DTYPE_F16>(S, a->activation, a->grad_bias, st)
                                      : launch_slope<FG_DTYPE_BF16>(S, a->activation, a->grad_bias, st);
        if (rc != FG_OK) return rc;
        if (written) dz = {S.dz, a->tokens, a->outer, S.dz_stride};
    }
    if (dz.rows <= 1) dz.stride = round8(dz.dim);
    if (a->grad_x) {
        Matrix wm{a->weight, a->outer, a->inner, a->weight_stride};
        if ((rc = make_ready(wm, room + W.weight, d, st)) != FG_OK) return rc;
        Params P{};
        P.out = a->grad_x; P.out_stride = a->grad_x_stride;
        P.L = a->inner; P.C = a->tokens; P.K = a->outer;
        if ((rc = product(P, a->dtype, wm, true, dz, false, d, st)) != FG_OK) return rc;
    }
    if (a->grad_weight) {
        Matrix xm{a->x, a->tokens, a->inner, a->x_stride};
        if ((rc = make_ready(xm, room + W.x, d, st)) != FG_OK) return rc;
        Params P{};
        P.out = a->grad_weight; P.out_stride = a->grad_weight_stride;
        P.L = a->inner; P.C = a->outer; P.K = a->tokens;
        if ((rc = product(P, a->dtype, xm, true, dz, true, d, st)) != FG_OK) return rc;
    }
    return FG_OK;
}

}  // extern "C"
