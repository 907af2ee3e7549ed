// fg_adapter.cu — C ABI entry points of the LM head with per-row adapters:
// argument checks, workspace layout and launches.
#include <algorithm>
#include <atomic>

#include "fg_adapter.h"
#include "fg_internal.h"

namespace {

using fg::host::DevInfo;
using fg::host::elem_size;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

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

// A [rows, dim] matrix read in boxes of box_rows x 64 elements; columns past dim
// and rows past `rows` read as zero.
bool encode(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t dim, int64_t stride, int box_rows) {
    EncodeTiledFn f = encoder();
    if (f == nullptr) return false;
    const cuuint64_t extent[2] = {cuuint64_t(dim), cuuint64_t(rows)};
    const cuuint64_t pitch[1] = {cuuint64_t(stride) * 2};
    const cuuint32_t box[2] = {cuuint32_t(fg::adapt::TILE_K), cuuint32_t(box_rows)};
    const cuuint32_t step[2] = {1, 1};
    return f(map, dtype == FG_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(base), extent, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Workspace: U in parts, its units, the order of the rows, their copy.
struct Layout {
    size_t u, unit, order, copy, total;
    int64_t copy_stride;
};
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
Layout layout(int64_t batch, int64_t dim, int64_t rank, int64_t slots) {
    Layout L{};
    const int64_t width = rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128;
    L.copy_stride = (dim + 7) / 8 * 8;
    L.u = 0;
    L.unit = round256(slots > 0 ? 6 * size_t(batch * width) : 0);
    L.order = L.unit + round256(sizeof(float) * size_t(batch));
    L.copy = L.order + round256(sizeof(int32_t) * size_t(batch));
    L.total = std::max<size_t>(256, L.copy + round256(2 * size_t(batch * L.copy_stride)));
    return L;
}

constexpr int32_t kMaxRows = 1 << 20;

// fg_adapter_set_wait
std::atomic<int64_t> g_wait_ns{fg::adapt::DEFAULT_WAIT_NS};
std::atomic<int32_t> g_withhold{-1};

}  // namespace

extern "C" {

size_t fg_adapter_workspace_size(int32_t batch, int32_t dim, int32_t rank, int32_t slots) {
    if (batch < 0 || batch > kMaxRows || dim < 1 || slots < 0) return 0;
    if (slots > 0 && (rank < 8 || rank > FG_ADAPTER_MAX_RANK || rank % 8 != 0)) return 0;
    return layout(batch, dim, rank, slots).total;
}

int fg_adapter_set_wait(int64_t limit_ns, int32_t withhold) {
    if (limit_ns < 0 || limit_ns > fg::adapt::DEFAULT_WAIT_NS || withhold < -1 || withhold >= fg::adapt::MAX_ACC)
        return FG_EINVAL;
    g_wait_ns.store(limit_ns > 0 ? limit_ns : fg::adapt::DEFAULT_WAIT_NS, std::memory_order_relaxed);
    g_withhold.store(withhold, std::memory_order_relaxed);
    return FG_OK;
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
        if (a->rank < 8 || a->rank > FG_ADAPTER_MAX_RANK || a->rank % 8 != 0) return FG_EINVAL;
        if (!aligned(a->down, 16) || !aligned(a->up, 16) || a->down_stride < a->dim || a->down_stride % 8 != 0)
            return FG_EINVAL;
    }
    if (a->batch > kMaxRows || a->vocab > (1 << 28) || a->dim > (1 << 20) || a->slots > (1 << 20)) return FG_ENOTSUP;
    const size_t need = fg_adapter_workspace_size(a->batch, a->dim, a->rank, a->slots);
    if (a->workspace == nullptr || !aligned(a->workspace, 256) || a->workspace_bytes < need) return FG_EINVAL;
    if (a->batch == 0) return FG_OK;
    const int64_t osz = elem_size(a->out_dtype);
    const fg::host::Rows out{a->out, a->batch, a->out_stride * osz, a->vocab * osz};
    if (fg::host::rows_meet(out, {a->hidden, a->batch, a->hidden_stride * 2, int64_t(a->dim) * 2}) ||
        fg::host::rows_meet(out, {a->weight, a->vocab, a->weight_stride * 2, int64_t(a->dim) * 2}))
        return FG_EINVAL;
    DevInfo* d = nullptr;
    const int rc = fg::host::device_info(&d);
    if (rc != FG_OK) return rc;

    const Layout L = layout(a->batch, a->dim, a->rank, a->slots);
    char* ws = reinterpret_cast<char*>(a->workspace);
    fg::adapt::Params P{};
    P.raw_hidden = a->hidden; P.raw_stride = a->hidden_stride;
    P.down = a->down; P.up = a->up; P.scales = a->scales;
    P.adapters = a->slots > 0 || a->out_status ? a->adapters : nullptr;
    P.out = a->out; P.out_status = a->out_status;
    P.u = ws + L.u;
    P.unit = reinterpret_cast<float*>(ws + L.unit);
    P.order = reinterpret_cast<int32_t*>(ws + L.order);
    P.batch = a->batch; P.dim = a->dim; P.vocab = a->vocab; P.rank = a->rank; P.slots = a->slots;
    P.down_stride = a->down_stride; P.out_stride = a->out_stride; P.copy_stride = L.copy_stride;
    // Sorting costs a copy of the hidden rows that the products wait for; it saves fetches of
    // adapters and products with them. Microseconds sorted and not, rank 16, 16-bit results,
    // with 1, 4 and 32 adapters: dim 2048, V 32000, 32 rows 34.9 29.3, 35.4 29.2, 36.9 35.3; 48
    // rows 35.1 33.7, 35.4 34.0, 37.8 37.3; 64 rows 35.1 33.9, 35.6 34.2, 38.7 40.9; 96 rows 38.0
    // 37.8, 38.3 39.2, 43.0 46.8; V 50257, 128 rows 55.6 55.3, 55.9 58.6, 65.4 82.7; dim 4096, V
    // 32768, 256 rows 86.9 84.2, 86.9 90.8, 91.5 119; V 128256, 64 rows 185 184, 187 185, 200 197.
    // How many adapters a batch names is known on the device only: up to 64 rows of few
    // adapters lose 1.5 us by the rule. TMA reads rows that start on 16-byte boundaries:
    // others are copied first too.
    P.sorted = a->slots > 0 && a->adapters != nullptr && a->batch > 48;
    const bool copy = P.sorted || !aligned(a->hidden, 16) || (a->batch > 1 && a->hidden_stride % 8 != 0);
    P.wide_out = aligned(a->out, 16) && (a->batch == 1 || a->out_stride * elem_size(a->out_dtype) % 16 == 0);
    P.f32_out = a->out_dtype == FG_DTYPE_F32;
    P.copy = copy ? ws + L.copy : nullptr;
    P.hidden = copy ? P.copy : a->hidden;
    P.hidden_stride = copy || a->batch == 1 ? L.copy_stride : a->hidden_stride;
    // batch tiles of equal width, at most 256 columns
    P.ntile = (a->batch + fg::adapt::MAX_NT - 1) / fg::adapt::MAX_NT;
    // Two SMs share a product above 128 columns: dim 4096, 32768 words, 1024 rows 255 us against
    // 258 with one SM each. Small batches go either way: dim 2048, 32000 words, 96 rows 41.4
    // against 42.2, 160 rows 51 to 57 against 48; dim 4096, 128256 words, 128 rows 215 against 220.
    const int columns = (a->batch + P.ntile - 1) / P.ntile;
    const bool pair = columns > 128;
    // a pair's product takes its columns in steps of 32, a single CTA's in steps of 16
    P.nt = pair ? (columns + 31) / 32 * 32 : (columns + 15) / 16 * 16;
    P.ntile = (a->batch + P.nt - 1) / P.nt;
    const int tile_v = fg::adapt::TILE_V * (pair ? 2 : 1);
    P.nvt = (a->vocab + tile_v - 1) / tile_v;
    // Steps of K a stage: loads of one row of the weight close to each other in time while
    // the weight's bytes bound the call (dim 4096, 128256 words, one row: four steps 165 us,
    // two 168, one 178; 128 rows: two 219, one 226), more stages when the products do
    // (1024 rows, 32768 words: one 255, two 264). A divisor of PIECE_K.
    P.kb = P.nt <= 64 ? 4 : P.nt <= 128 ? 2 : 1;
    P.tmem_cols = 32;
    P.accs = std::min(fg::adapt::MAX_ACC, 512 / P.nt);
    P.wait_ns = uint64_t(g_wait_ns.load(std::memory_order_relaxed));
    P.withhold = g_withhold.load(std::memory_order_relaxed);
    while (P.tmem_cols < P.accs * P.nt) P.tmem_cols *= 2;
    if (int64_t(P.nvt) * P.ntile > (1 << 30)) return FG_ENOTSUP;
    CUtensorMap wmap, xmap;
    if (!encode(&wmap, a->dtype, a->weight, a->vocab, a->dim, a->weight_stride, fg::adapt::TILE_V) ||
        !encode(&xmap, a->dtype, P.hidden, a->batch, a->dim, P.hidden_stride, pair ? P.nt / 2 : P.nt))
        return FG_EDEVICE;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool f32 = a->out_dtype == FG_DTYPE_F32;
    if (a->dtype == FG_DTYPE_F16)
        return f32 ? fg::adapt::launch<FG_DTYPE_F16, FG_DTYPE_F32>(P, wmap, xmap, pair, d, st)
                   : fg::adapt::launch<FG_DTYPE_F16, FG_DTYPE_F16>(P, wmap, xmap, pair, d, st);
    return f32 ? fg::adapt::launch<FG_DTYPE_BF16, FG_DTYPE_F32>(P, wmap, xmap, pair, d, st)
               : fg::adapt::launch<FG_DTYPE_BF16, FG_DTYPE_BF16>(P, wmap, xmap, pair, d, st);
}

}  // extern "C"
