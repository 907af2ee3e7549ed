// fg_adapter.cuh — logits of a batch that shares an LM head, every row with its
// own low-rank adapter beside it (fg_adapter_logits):
//   out[b, v] = X[b, :] . W[v, :] + U[b, :] . up[a_b, v, :],
//   U[b, i]   = scales[a_b] * (X[b, :] . down[a_b, i, :])
//
// Two launches. down_kernel computes U and sorts the rows of each batch tile by
// adapter (it copies the hidden rows in that order, which also aligns them).
// project_kernel does the rest: the shared product on the tensor cores with the
// vocabulary on the accumulator's 128 lanes and the batch on its columns, so that a
// small batch wastes no tensor-core rows. Its epilogue warps add the adapters'
// product, eight columns at a time, with warp-level products whose fragments match
// the layout in which they read the accumulator.
//
// A row must not see another row's adapter, not even as 0 * NaN. So a product of
// one adapter with eight columns goes to registers of its own and each column takes
// or leaves it; sorting keeps that to about one product per eight columns plus one
// per adapter.
//
// U enters the tensor cores in its fp32 precision: a row of U is scaled by a power of
// two and split into 16-bit parts, whose products are summed in fp32; the power of two
// multiplies the sum. Three parts hold the 24 bits of a component. bf16 has the
// exponents for them; rows of f16 are scaled to the top of its range, and lower parts
// are scaled up once more (part_scale), their sums down: components down to 2^-41 of the
// row's largest keep 23 bits. 16-bit results take two parts: 16 bits of bf16 for results
// of 8 bits; f16, whose results have 11, 16 or more down to 2^-23 of the largest, and a
// third part for rows with smaller components (16 bits down to 2^-36). Three for all: 1024
// rows, dim 4096, V 32768, rank 64, bf16 423 us against 391.
#pragma once

#include "fg_adapter.h"
#include "fg_tcgen05.cuh"

namespace fg {
namespace adapt {

// The slot a row names, or -1 without an adapter: none wanted, or an id out of range.
__device__ __forceinline__ int row_slot(const Params& P, int b) {
    const int a = P.adapters ? P.adapters[b] : -1;
    return (a >= 0 && a < P.slots) ? a : -1;
}

constexpr int DOWN_THREADS = 256;

constexpr int U_PARTS = 3;   // 16-bit parts of a component of U
// What part i (1, 2) is scaled up by against part i - 1.
template <int DT>
__device__ __forceinline__ constexpr float part_scale(bool f32_out, int i) {
    return DT != FG_DTYPE_F16 ? 1.0f : f32_out ? 0x1p12f : i == 1 ? 1.0f : 0x1p24f;
}

template <int DT>
__device__ __forceinline__ float from_bits(uint16_t b) {
    if constexpr (DT == FG_DTYPE_F16) return __half2float(__ushort_as_half(b));
    else return __uint_as_float(uint32_t(b) << 16);
}
template <int DT>
__device__ __forceinline__ uint16_t to_bits(float x) {
    if constexpr (DT == FG_DTYPE_F16) return __half_as_ushort(__float2half_rn(x));
    else return __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// Eight 16-bit elements from any element-aligned address.
template <bool WIDE>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
    if constexpr (WIDE) {
        return *reinterpret_cast<const uint4*>(p);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = uint32_t(p[2 * i]) | (uint32_t(p[2 * i + 1]) << 16);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// This thread's part of the row's products with the warp's rank indices.
template <int DT, int RC, bool WIDE>
__device__ __forceinline__ void down_dots(const Params& P, const uint16_t* src, const uint16_t* dn, int warp, int lane,
                                          float (&acc)[2 * RC]) {
    const int vec = P.dim / 8;
#pragma unroll(RC == 1 ? 4 : RC == 2 ? 2 : 1)
    for (int i = lane; i < vec; i += 32) {
        uint4 q[2 * RC];
#pragma unroll
        for (int j = 0; j < 2 * RC; ++j)
            if (warp + 8 * j < P.rank)
                q[j] = __ldg(reinterpret_cast<const uint4*>(dn + (warp + 8 * j) * P.down_stride) + i);
        float x[8];
        Elem<DT>::unpack(load8<WIDE>(src + 8 * i), x);
#pragma unroll
        for (int j = 0; j < 2 * RC; ++j) {
            if (warp + 8 * j >= P.rank) break;
            float y[8];
            Elem<DT>::unpack(q[j], y);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[j] = fmaf(x[e], y[e], acc[j]);
        }
    }
    const int k = vec * 8 + lane;
    if (k < P.dim) {
        const float x = from_bits<DT>(src[k]);
#pragma unroll
        for (int j = 0; j < 2 * RC; ++j)
            if (warp + 8 * j < P.rank)
                acc[j] = fmaf(x, from_bits<DT>(dn[(warp + 8 * j) * P.down_stride + k]), acc[j]);
    }
}

// One row per CTA: its position in the sorted order of its batch tile (rows with
// the same adapter next to each other, ties in row order), its copy there, and U, a
// warp per rank index (2 * RC of them each, their 16-byte loads in flight together).
// Bound: latency, then L2 (each row reads its own adapter): one row of dim 4096 and
// rank 16 takes 17 us, 1024 rows 29 us (cold caches, alone), beside project_kernel's first
// loads. Half the threads, so that this kernel fits beside project_kernel on an SM: the
// call was 2 to 3 us slower at 64 rows, 15 us at rank 128, 6 us faster at 1024 rows.
// It stages nothing in shared memory: project_kernel's CTAs take nearly all of it
// and start beside this kernel's.
template <int DT, int RC>
__global__ void __launch_bounds__(DOWN_THREADS) down_kernel(const Params P) {
    __shared__ float us[16 * RC];
    // project_kernel may begin once this kernel has: by then what came before both is done
    tc::wait_prerequisites();
    tc::launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b = blockIdx.x;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(P.raw_hidden) + int64_t(b) * P.raw_stride;
    const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0;
    const int b0 = b / P.nt * P.nt, n = min(P.nt, P.batch - b0);
    // the row's slot is the only step on the way to its loads: the scale (0: no
    // adapter), the order and the copy are worked out while those are under way
    const int slot = row_slot(P, b);
    const float scale = slot >= 0 ? P.scales[slot] : 0.0f;
    float acc[2 * RC] = {};
    if (slot >= 0) {
        const uint16_t* dn = reinterpret_cast<const uint16_t*>(P.down) + int64_t(slot) * P.rank * P.down_stride;
        if (wide) down_dots<DT, RC, true>(P, src, dn, warp, lane, acc);
        else down_dots<DT, RC, false>(P, src, dn, warp, lane, acc);
    }
    int pos = b;
    if (P.sorted) {
        const int key = slot * MAX_NT + (b - b0);
        const bool ahead = tid < n && row_slot(P, b0 + tid) * MAX_NT + tid < key;
        pos = b0 + __syncthreads_count(ahead);
    }
    if (tid == 0) {
        P.order[pos] = ((scale != 0.0f ? slot + 1 : 0) << 9) | (b - b0);
        if (P.out_status) P.out_status[b] = (P.adapters && P.adapters[b] >= P.slots) ? FG_ROW_BAD_PARAM : 0;
    }
    if (P.copy) {
        uint16_t* dst = reinterpret_cast<uint16_t*>(P.copy) + int64_t(pos) * P.copy_stride;
        const int vec = P.dim / 8;
        if (wide) {
#pragma unroll 2
            for (int i = tid; i < vec; i += DOWN_THREADS)
                reinterpret_cast<uint4*>(dst)[i] = load8<true>(src + 8 * i);
        } else {
#pragma unroll 2
            for (int i = tid; i < vec; i += DOWN_THREADS)
                reinterpret_cast<uint4*>(dst)[i] = load8<false>(src + 8 * i);
        }
        for (int k = vec * 8 + tid; k < P.dim; k += DOWN_THREADS) dst[k] = src[k];
    }
    if (scale == 0.0f) return;
#pragma unroll
    for (int j = 0; j < 2 * RC; ++j) {
        float v = acc[j];
        for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == 0) us[warp + 8 * j] = v * scale;   // 0 past the rank
    }
    __syncthreads();
    if (warp == 0) {
        float top = 0.0f;   // the largest finite one
        for (int i = lane; i < 16 * RC; i += 32) {
            const float v = fabsf(us[i]);
            top = fmaxf(top, v < INFINITY ? v : 0.0f);
        }
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // |U| 2^-e < 2^HIGH (2 for the largest of bf16); both powers finite
        constexpr int HIGH = DT == FG_DTYPE_F16 ? 15 : 0;
        const int e = top > 0.0f ? max(HIGH - 126, min(HIGH + 127, ilogbf(top) + 1)) - HIGH : 0;
        const float down = ldexpf(1.0f, -e);
        bool small = false;   // components that 16-bit results need the third part for: the unit's sign
        for (int i = lane; i < 16 * RC; i += 32) {
            const float v = fabsf(us[i]) * down;
            small |= DT == FG_DTYPE_F16 && v > 0.0f && v < 0x1p-8f;
        }
        small = __any_sync(0xffffffffu, small);
        if (lane == 0) P.unit[pos] = ldexpf(small ? -1.0f : 1.0f, e);
        uint16_t* dst = reinterpret_cast<uint16_t*>(P.u) + int64_t(pos) * (U_PARTS * 16 * RC);
        for (int i = lane; i < 16 * RC; i += 32) {
            float v = us[i] * down;
#pragma unroll
            for (int part = 0; part < U_PARTS; ++part) {
                if (part > 0) v *= part_scale<DT>(P.f32_out, part);
                // a subnormal operand costs the sum the bits between it and the type's least
                // exponent: to fp32 results it is worth leaving to the next part
                const bool later = DT == FG_DTYPE_F16 && P.f32_out && part == 0 && fabsf(v) < 0x1p-14f;
                const uint16_t h = later ? uint16_t(0) : to_bits<DT>(v);
                dst[part * 16 * RC + i] = h;
                const float left = v - from_bits<DT>(h);
                v = (left - left == 0.0f) ? left : 0.0f;   // inf and NaN live in the first part
            }
        }
    }
}

// ---------------------------------------------------------------------------
// project_kernel: persistent, one CTA per SM (CG = 1) or one pair of CTAs per two
// SMs (CG = 2). Warp 0 loads (TMA), warp 1 issues the products, the others are the
// epilogue (two or four per quarter of the accumulator's lanes). Two to eight
// accumulators in tensor memory: one tile's epilogue runs beside the next products.
//
// Every wait is bounded (P.wait_ns). Where one runs out, the CTA (and its pair) stops
// waiting: the loader and the issuing thread leave off, the epilogue warps write NaN for
// all that they have not stored, so that nothing unwritten can be taken for logits, one
// of them marks every row FG_ROW_TIMEOUT, and the CTA waits for its products and copies
// in flight before it frees the tensor memory and leaves.
//
// Bound: HBM up to about 128 rows (the weight, once), the tensor pipe above. Measured
// (bf16, dim 4096, rank 16): 128256 words, one row 160 to 165 us (6.4 to 6.5 TB/s of weight),
// 64 rows of 32 adapters 198 us (5.3 TB/s); 32768 words, 1024 rows 255 us (1.08 PFLOP/s; SM
// clock held to 1.6 GHz by the power limit, tensor pipe active 58 %), 210 without adapters (the
// epilogue's loads and products are the difference). Few rows of a short weight: 64 rows, dim
// 2048, 32000 words 29 us without adapters, 37 us with 16 of rank 8, 39 us with 32 of rank 16
// (down_kernel's launch and the adapters' bytes; their rows fetched ahead of the epilogue,
// to L2 or to shared memory by a warp of its own, gained nothing).
//
// The tensor core truncates when it adds products to the accumulator: over n elements
// of one sign the sum loses about 0.05 n units of 2^-23. So the sum over K is taken in
// pieces, one accumulator each, that the epilogue warps add with rounding. fp32 results
// take pieces of PIECE_K steps and keep the sum in registers. For 16-bit results pieces of
// LONG_K lose an eighth of half a unit of f16 at most (of one sign; a few 10^-6 of the
// results' norm otherwise, by which one in 400 rounds to the other neighbour); the epilogue
// adds a long dim's pieces in tensor memory, each to the next.
// ---------------------------------------------------------------------------
constexpr int A_BYTES = TILE_V * TILE_K * 2;
constexpr int MAX_STAGES = 12;
// Epilogue warps, and how many windows of its tile each works out before the
// products arrive (the others' adapters are added as they are read). With fp32
// results registers go to the sums, of fewer columns for a SMALL batch tile: next to
// the ring there is no L1 left, and a spilled register would wait for L2.
// Measured (dim 2048, 32000 words, rank 16): 12 warps against 8, 64 rows not sorted, 16-bit
// results: 41 us, 45; 16 against 8, 256 rows, fp32: 66, 81; no early windows at those 64 rows:
// 46; SMALL, 8 rows, 50257 words, fp32: 42, without it 45.
template <int ODT, int RC, bool SMALL>
struct Epilogue {
    static constexpr bool PIECES = ODT == FG_DTYPE_F32;
    static constexpr int WARPS = RC > 2 ? 8 : PIECES && !SMALL ? 16 : 12;
    static constexpr int EARLY = RC == 0 || (PIECES && !SMALL) ? 0
                                 : PIECES ? (RC == 1 ? 2 : RC == 4 ? 1 : 0) : (RC == 1 ? 3 : RC <= 4 ? 2 : 1);
    static constexpr int THREADS = 64 + 32 * WARPS;            // of the CTA
    static constexpr int COLUMNS = SMALL ? SMALL_NT : MAX_NT;
    static constexpr int SUMS = (COLUMNS / 8 + WARPS / 4 - 1) / (WARPS / 4) * 8;   // a warp's share, in eights
};
constexpr int PIECE_K = 8, LONG_K = 64;            // 64-wide steps of K per piece: of fp32 results, of 16-bit ones

// Barrier over `threads` threads that also tells all of them whether any had `p`.
__device__ __forceinline__ bool named_any(int id, int threads, bool p) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %3, 0;\n\tbar.red.or.pred b, %1, %2, a;\n\t"
                 "selp.u32 %0, 1, 0, b;\n\t}"
                 : "=r"(r) : "r"(id), "r"(threads), "r"(uint32_t(p)) : "memory");
    return r != 0;
}

struct Control {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES];
    uint64_t acc_full[MAX_ACC], acc_empty[MAX_ACC], drain;
    uint32_t tmem;
    int abort;      // someone's wait ran out: everyone stops waiting
    int reported;   // the rows' status words say so
};

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8) of 16-bit operands, on one warp.
template <int DT>
__device__ __forceinline__ void warp_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    if constexpr (DT == FG_DTYPE_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                     "{%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}

// The A fragments of one adapter for the warp's 32 vocabulary rows: two tiles of 16
// rows, RC steps of 16 ranks. A thread (g = lane / 4, t = lane % 4) holds ranks
// 4t .. 4t + 3 of a step in rows g and g + 8 of a tile: eight bytes at a time, where
// the instruction's own order would be two pairs (B is laid out alike, so the sum
// does not change).
template <int RC>
struct UpTile {
    uint2 q[RC][4];   // rows g, g + 8, g + 16, g + 24
    __device__ __forceinline__ void load(const Params& P, int slot, int v0, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const uint16_t* up = reinterpret_cast<const uint16_t*>(P.up) + int64_t(slot) * P.vocab * P.rank + 4 * t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t* row = up + int64_t(min(v0 + g + 8 * i, P.vocab - 1)) * P.rank;
#pragma unroll
            for (int c = 0; c < RC; ++c)
                q[c][i] = 16 * c + 4 * t < P.rank ? __ldg(reinterpret_cast<const uint2*>(row + 16 * c))
                                                  : make_uint2(0, 0);
        }
    }
};

// What one epilogue warp keeps while it goes over windows of eight columns: the
// fragments of the adapter used last. A window's other adapters come BATCH at a
// time, their loads in flight together.
template <int DT, int ODT, int RC>
struct Windows {
    static constexpr int PARTS = ODT == FG_DTYPE_F32 ? U_PARTS : 2;   // held in registers
    static constexpr bool LAST = PARTS < U_PARTS && DT == FG_DTYPE_F16;   // the third where a row needs it
    static constexpr int BATCH = RC == 1 && ODT != FG_DTYPE_F32 ? 3 : 1;
    static constexpr uint32_t ALL = 0xffffffffu;
    UpTile<RC> up;
    int cur = -1;

    // This lane's column (lane % 8) of window w: (slot + 1) << 9 | row of the tile,
    // or -1 past the rows.
    __device__ __forceinline__ static int entry(const Params& P, int b0, int rows, int w, int lane) {
        const int p = 8 * w + (lane & 7);
        return p < rows ? P.order[b0 + p] : -1;
    }

    __device__ __forceinline__ static void product(float (&d)[2][4], const UpTile<RC>& tile, int c, const uint2& u) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            warp_mma<DT>(d[h], tile.q[c][2 * h].x, tile.q[c][2 * h + 1].x, tile.q[c][2 * h].y, tile.q[c][2 * h + 1].y, u);
    }
    __device__ __forceinline__ static void scale_down(float (&d)[2][4], int part) {
        constexpr bool F32 = ODT == FG_DTYPE_F32;
        if (part_scale<DT>(F32, part) == 1.0f) return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) d[h][j] *= 1.0f / part_scale<DT>(F32, part);
    }

    // One adapter's product with the window; the columns in `match` take it, no other does.
    __device__ __forceinline__ static void apply(float (&x)[2][4], const UpTile<RC>& tile, const uint2 (&u)[RC][PARTS],
                                                 float unit0, float unit1, uint32_t match, int t) {
        float d[2][4] = {};
#pragma unroll
        for (int i = PARTS - 1; i >= 0; --i) {
#pragma unroll
            for (int c = 0; c < RC; ++c) product(d, tile, c, u[c][i]);
            if (i > 0) scale_down(d, i);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (match >> (2 * t) & (i & 1 ? 2 : 1)) x[h][i] = d[h][i] * fabsf(i & 1 ? unit1 : unit0);
    }

    // Whether any of the columns in `match` needs the part of U that is not held in registers.
    __device__ __forceinline__ static bool needs_last(float unit0, float unit1, uint32_t match, int t) {
        if (!LAST) return false;
        const uint32_t mine = match >> (2 * t);
        return __any_sync(ALL, (unit0 < 0.0f && (mine & 1)) || (unit1 < 0.0f && (mine & 2)));
    }
    // That part's products with every adapter of the window (seldom run: apart from the
    // others, whose instructions interleave).
    __device__ __forceinline__ static void add_last(float (&x)[2][4], UpTile<RC>& tile, const Params& P, const uint2* src,
                                                    int slots, int v0, float unit0, float unit1, int lane) {
        asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane));   // (anew: nothing is kept for this path)
        const int t = lane & 3;
        uint32_t left = __ballot_sync(ALL, slots >= 0) & 0xffu;
        while (left) {
            const int slot = __shfl_sync(ALL, slots, __ffs(left) - 1);
            const uint32_t match = __ballot_sync(ALL, slots == slot) & 0xffu;
            left &= ~match;
            tile.load(P, slot, v0, lane);
            float d[2][4] = {};
#pragma unroll
            for (int c = 0; c < RC; ++c) product(d, tile, c, src[PARTS * 4 * RC + c * 4]);
            scale_down(d, PARTS);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (match >> (2 * t) & (i & 1 ? 2 : 1)) x[h][i] += d[h][i] * fabsf(i & 1 ? unit1 : unit0);
        }
    }

    // The adapters' share of window w, eight columns by 32 vocabulary rows from v0 on:
    // columns 2t, 2t + 1 of rows g + 8 i.
    __device__ __forceinline__ void adapters(float (&x)[2][4], const Params& P, int b0, int rows, int w, int v0,
                                             int ent, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const int slots = ent < 0 ? -1 : (ent >> 9) - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[0][i] = x[1][i] = 0.0f;
        uint32_t left = __ballot_sync(ALL, slots >= 0) & 0xffu;   // columns still without their adapter
        if (left == 0) return;
        const uint32_t all = left;
        // B fragments: parts of U for column g
        uint2 u[RC][PARTS];
        const uint2* src = reinterpret_cast<const uint2*>(P.u) + int64_t(b0 + min(8 * w + g, rows - 1)) * (U_PARTS * 4 * RC) + t;
#pragma unroll
        for (int c = 0; c < RC; ++c)
#pragma unroll
            for (int i = 0; i < PARTS; ++i) u[c][i] = src[i * 4 * RC + c * 4];
        const int p = 8 * w + 2 * t;
        const float unit0 = p < rows ? P.unit[b0 + p] : 0.0f, unit1 = p + 1 < rows ? P.unit[b0 + p + 1] : 0.0f;
        const uint32_t held = __ballot_sync(ALL, slots == cur) & left;
        if (held) {
            left &= ~held;
            apply(x, up, u, unit0, unit1, held, t);
        }
        while (left) {
            // all but the last go through registers of their own; the last stays
            UpTile<RC> tile[BATCH > 1 ? BATCH - 1 : 1];
            uint32_t match[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                match[i] = 0;
                const bool last = i == BATCH - 1;
                if (last ? left != 0 : (left & (left - 1)) != 0) {
                    const int slot = __shfl_sync(ALL, slots, __ffs(left) - 1);
                    match[i] = __ballot_sync(ALL, slots == slot) & 0xffu;
                    left &= ~match[i];
                    if (last) up.load(P, cur = slot, v0, lane);
                    else tile[i].load(P, slot, v0, lane);
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH - 1; ++i)
                if (match[i]) apply(x, tile[i], u, unit0, unit1, match[i], t);
            if (match[BATCH - 1]) apply(x, up, u, unit0, unit1, match[BATCH - 1], t);
        }
        if (needs_last(unit0, unit1, all, t)) {
            add_last(x, up, P, src, slots, v0, unit0, unit1, lane);
            cur = -1;
        }
    }
};

// The adapters' share of the E windows from w0 on, as Windows::adapters, but slot by
// slot over all of them: a slot's rows of up are loaded once, BATCH slots at a time.
template <int DT, int ODT, int RC, int E>
__device__ __forceinline__ void early_windows(float (&x)[E][2][4], const int (&ents)[E], const Params& P, int b0,
                                              int rows, int w0, int w1, int v0, int lane) {
    using W = Windows<DT, ODT, RC>;
    constexpr uint32_t ALL = 0xffffffffu;
    constexpr int BATCH = RC == 1 && ODT != FG_DTYPE_F32 ? 3 : RC <= 2 ? 2 : 1;
    const int g = lane >> 2, t = lane & 3;
    int slots[E];
    uint32_t left = 0;   // columns still without their adapter, eight bits a window
    uint2 u[E][RC][W::PARTS];
    float unit[E][2];
    auto src = [&](int i) {   // this thread's parts of U of window w0 + i
        return reinterpret_cast<const uint2*>(P.u) +
               int64_t(b0 + min(8 * min(w0 + i, w1 - 1) + g, rows - 1)) * (U_PARTS * 4 * RC) + t;
    };
#pragma unroll
    for (int i = 0; i < E; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][0][j] = x[i][1][j] = 0.0f;
        slots[i] = w0 + i < w1 && ents[i] >= 0 ? (ents[i] >> 9) - 1 : -1;
        left |= (__ballot_sync(ALL, slots[i] >= 0) & 0xffu) << (8 * i);
        const int p = 8 * min(w0 + i, w1 - 1) + 2 * t;
#pragma unroll
        for (int c = 0; c < RC; ++c)
#pragma unroll
            for (int j = 0; j < W::PARTS; ++j) u[i][c][j] = src(i)[j * 4 * RC + c * 4];
        unit[i][0] = p < rows ? P.unit[b0 + p] : 0.0f;
        unit[i][1] = p + 1 < rows ? P.unit[b0 + p + 1] : 0.0f;
    }
    while (left) {
        UpTile<RC> tile[BATCH];
        uint32_t match[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            match[k] = 0;
            if (left) {
                const int at = __ffs(left) - 1;
                int mine = slots[0];
#pragma unroll
                for (int i = 1; i < E; ++i)
                    if (at >= 8 * i) mine = slots[i];
                const int slot = __shfl_sync(ALL, mine, at & 7);
#pragma unroll
                for (int i = 0; i < E; ++i) match[k] |= (__ballot_sync(ALL, slots[i] == slot) & 0xffu) << (8 * i);
                left &= ~match[k];
                tile[k].load(P, slot, v0, lane);
            }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (match[k] >> (8 * i) & 0xffu)
                    W::apply(x[i], tile[k], u[i], unit[i][0], unit[i][1], match[k] >> (8 * i), t);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (W::needs_last(unit[i][0], unit[i][1], __ballot_sync(ALL, slots[i] >= 0) & 0xffu, t)) {
            UpTile<RC> tile;
            W::add_last(x[i], tile, P, src(i), slots[i], v0, unit[i][0], unit[i][1], lane);
        }
    }
}

// An infinite element of up meets every part of a component, of which the lower ones may
// be 0 or of the other sign: NaN where the product is infinite. So what came out NaN of an
// adapter is summed again, in fp32 and from whole components (NaN stays NaN).
template <int DT, int ODT, int RC>
__device__ __forceinline__ void settle_nan(float (&x)[2][4], const Params& P, int b0, int w, int v0, int ent, int lane) {
    constexpr uint32_t ALL = 0xffffffffu;
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) all += x[0][i] + x[1][i];
    if (!__any_sync(ALL, isnan(all))) return;
    // (the lane anew, so that nothing worked out from it is kept for this path)
    asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane));
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int e = __shfl_sync(ALL, ent, 2 * t + j);
        const int pos = b0 + 8 * w + 2 * t + j;
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // one at a time: seldom run, and registers are short
            float& y = x[i >> 1][2 * (i & 1) + j];
            if (!isnan(y)) continue;    // (a column without an adapter has 0)
            const uint16_t* u = reinterpret_cast<const uint16_t*>(P.u) + int64_t(pos) * (U_PARTS * 16 * RC);
            const uint16_t* up = reinterpret_cast<const uint16_t*>(P.up) +
                                 (int64_t((e >> 9) - 1) * P.vocab + min(v0 + g + 8 * i, P.vocab - 1)) * P.rank;
            float sum = 0.0f;
#pragma unroll 1
            for (int r = 0; r < P.rank; ++r) {
                float c = 0.0f;
#pragma unroll
                for (int part = U_PARTS - 1; part >= 0; --part) {
                    c += from_bits<DT>(u[part * 16 * RC + r]);
                    if (part > 0) c *= 1.0f / part_scale<DT>(ODT == FG_DTYPE_F32, part);
                }
                sum = fmaf(c, from_bits<DT>(up[r]), sum);
            }
            y = sum * fabsf(P.unit[pos]);
        }
    }
}

// Read window w of the accumulator, add the adapters' share and store it.
template <int DT, int ODT, int RC>
__device__ __forceinline__ void store_window(const Params& P, uint32_t base, int b0, int w, int v0, int ent,
                                             float (&add)[2][4], int lane) {
    if constexpr (RC > 0) settle_nan<DT, ODT, RC>(add, P, b0, w, v0, ent, lane);
    constexpr uint32_t ALL = 0xffffffffu;
    const int g = lane >> 2, t = lane & 3;
    float x[2][4];
    tc::tmem_ld_window(x[0], base + 8 * w);
    tc::tmem_ld_window(x[1], base + 8 * w + (16u << 16));
    tc::tmem_wait_ld(x[0]);
    tc::tmem_wait_ld(x[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[0][i] += add[0][i];
        x[1][i] += add[1][i];
    }
    if (ODT != FG_DTYPE_F32 && P.wide_out && v0 + 32 <= P.vocab) {
        // 16-bit results: transpose 8 x 8 blocks so that a thread holds pairs of
        // neighbouring rows of column g, then exchange among its four threads: eight
        // neighbouring rows, one 16-byte store
        uint32_t r[4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t pack = uint32_t(to_bits<ODT>(x[h][2 * i])) |
                                      (uint32_t(to_bits<ODT>(x[h][2 * i + 1])) << 16);
                asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r[2 * h + i]) : "r"(pack));
            }
        const bool odd = t & 1, high = t & 2;
        uint32_t s0 = __shfl_xor_sync(ALL, odd ? r[0] : r[1], 1), s1 = __shfl_xor_sync(ALL, odd ? r[2] : r[3], 1);
        const uint32_t a0 = odd ? s0 : r[0], a1 = odd ? r[1] : s0;   // block `odd` of threads t & ~1, t | 1
        const uint32_t a2 = odd ? s1 : r[2], a3 = odd ? r[3] : s1;   // block 2 + odd
        s0 = __shfl_xor_sync(ALL, high ? a0 : a2, 2);
        s1 = __shfl_xor_sync(ALL, high ? a1 : a3, 2);
        const uint4 q = high ? make_uint4(s0, s1, a2, a3) : make_uint4(a0, a1, s0, s1);
        const int eg = __shfl_sync(ALL, ent, g);
        if (eg >= 0)
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(P.out) +
                                      int64_t(b0 + (eg & 511)) * P.out_stride + v0 + 8 * t) = q;
    } else {
        const int e0 = __shfl_sync(ALL, ent, 2 * t), e1 = __shfl_sync(ALL, ent, 2 * t + 1);
        const int64_t o0 = int64_t(b0 + (e0 & 511)) * P.out_stride, o1 = int64_t(b0 + (e1 & 511)) * P.out_stride;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int v = v0 + g + 16 * h + 8 * i;
                if (v < P.vocab) {
                    if (e0 >= 0) Elem<ODT>::store(P.out, o0 + v, x[h][2 * i]);
                    if (e1 >= 0) Elem<ODT>::store(P.out, o1 + v, x[h][2 * i + 1]);
                }
            }
    }
}

// NaN in the place of window w, whose products did not come.
template <int ODT, int RC>
__device__ __forceinline__ void store_nan(const Params& P, int b0, int rows, int w, int v0) {
    int lane;
    asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane));   // (anew: nothing is kept for this path)
    if (v0 + lane >= P.vocab) return;
#pragma unroll 1
    for (int p = 8 * w; p < min(rows, 8 * w + 8); ++p) {
        const int row = RC > 0 ? P.order[b0 + p] & 511 : p;
        Elem<ODT>::store(P.out, int64_t(b0 + row) * P.out_stride + v0 + lane, __int_as_float(0x7fc00000));
    }
}

// RC: rank / 16 held in registers (rounded up to 1, 2, 4 or 8), 0: no adapters.
// SMALL: fp32 results and a batch tile of at most SMALL_NT columns.
template <int CG, int DT, int ODT, int RC, bool SMALL>
__global__ void __launch_bounds__(Epilogue<ODT, RC, SMALL>::THREADS, 1)
project_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Params P) {
    extern __shared__ uint8_t dyn[];
    __shared__ Control C;
    constexpr bool PIECES = ODT == FG_DTYPE_F32;
    constexpr int EPI_WARPS = Epilogue<ODT, RC, SMALL>::WARPS;
    uint8_t* ring = dyn + ((1024 - (smem_u32(dyn) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? tc::cta_rank() : 0;
    const int S = P.stages;
    const int box_bytes = A_BYTES + P.nt / CG * TILE_K * 2;   // one 64-wide step of K, this CTA's part
    const int stage_bytes = P.kb * box_bytes;
    const int nk = (P.dim + TILE_K - 1) / TILE_K;
    const int piece = PIECES ? PIECE_K : LONG_K;
    const int tiles = P.nvt * P.ntile;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.empty[s], 1);
        }
        for (int i = 0; i < P.accs; ++i) {
            mbar_init(&C.acc_full[i], i == P.withhold ? 2 : 1);
            mbar_init(&C.acc_empty[i], CG * EPI_WARPS);
        }
        mbar_init(&C.drain, 1);
        C.abort = C.reported = 0;
        fence_mbar_init();
        tc::prefetch_map(&wmap);
        tc::prefetch_map(&xmap);
    }
    if (warp == 1) {
        tc::tmem_alloc<CG>(&C.tmem, P.tmem_cols);
        tc::fence_before();
    }
    __syncthreads();
    if (CG == 2) tc::cluster_sync();   // both CTAs' barriers stand
    tc::fence_after();
    const uint32_t tmem = C.tmem;
    // down_kernel began after everything before it had ended; without it, wait for that here
    if (!P.chained) tc::wait_prerequisites();

    auto give_up = [&]() {   // (the pair's other CTA cannot go on alone)
        *reinterpret_cast<volatile int*>(&C.abort) = 1;
        if (CG == 2) tc::store_cluster(tc::mapa(&C.abort, rank ^ 1), 1);
    };
    int filled = 0;   // stages that the loader has filled
    if (warp == 0) {
        if (lane == 0) {
            const uint32_t ring_a = smem_u32(ring);
            const uint32_t full0 = CG == 2 ? tc::mapa(&C.full[0], 0) : smem_u32(&C.full[0]);
            int stage = 0, used = 0;      // used: stages handed out so far, up to S
            uint32_t parity = 1;          // of the ring's previous round
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                const int v0 = ((t / P.ntile) * CG + rank) * TILE_V;
                const int b0 = (t % P.ntile) * P.nt + rank * (P.nt / CG);
                for (int kc = 0; kc < nk; kc += P.kb) {
                    if (used == S && !mbar_wait(&C.empty[stage], parity, &C.abort, P.wait_ns)) { ok = false; break; }
                    const int boxes = min(P.kb, nk - kc);
                    uint32_t a = ring_a + stage * stage_bytes;
                    if (used < S) {
                        if (++used == 1) {
                            // the first round's weights do not wait for down_kernel
                            int s1 = 0;
                            for (int t1 = first; t1 < tiles && s1 < S; t1 += step)
                                for (int k1 = 0; k1 < nk && s1 < S; k1 += P.kb, ++s1) {
                                    const int n1 = min(P.kb, nk - k1);
                                    if (rank == 0) mbar_arrive_expect_tx(&C.full[s1], CG * n1 * box_bytes);
                                    for (int q = 0; q < n1; ++q)
                                        tc::tma_load_2d<CG>(ring_a + s1 * stage_bytes + q * box_bytes, &wmap,
                                                            (k1 + q) * TILE_K, ((t1 / P.ntile) * CG + rank) * TILE_V,
                                                            full0 + 8 * s1);
                                }
                            if (P.copy) {
                                tc::wait_prerequisites();   // the sorted rows come from down_kernel
                                asm volatile("fence.proxy.async.global;" ::: "memory");
                            }
                        }
                    } else {
                        if (rank == 0) mbar_arrive_expect_tx(&C.full[stage], CG * boxes * box_bytes);
                        for (int q = 0; q < boxes; ++q)
                            tc::tma_load_2d<CG>(a + q * box_bytes, &wmap, (kc + q) * TILE_K, v0, full0 + 8 * stage);
                    }
                    for (int q = 0; q < boxes; ++q)
                        tc::tma_load_2d<CG>(a + q * box_bytes + A_BYTES, &xmap, (kc + q) * TILE_K, b0,
                                            full0 + 8 * stage);
                    ++filled;
                    if (++stage == S) {
                        stage = 0;
                        parity ^= 1;
                    }
                }
            }
            if (!ok) give_up();
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = tc::instr_desc(DT, TILE_V * CG, P.nt);
            const uint64_t desc0 = tc::operand_desc(smem_u32(ring));
            int stage = 0, acc = 0;
            uint32_t parity = 0, acc_parity = 1;   // a fresh barrier counts as passed with parity 1
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                for (int k0 = 0; k0 < nk && ok; k0 += piece) {
                    const int k1 = min(nk, k0 + piece);
                    if (!mbar_wait(&C.acc_empty[acc], acc_parity, &C.abort, P.wait_ns)) { ok = false; break; }
                    tc::fence_after();
                    const uint32_t d = tmem + acc * P.nt;
                    for (int kc = k0; kc < k1; kc += P.kb) {
                        if (!mbar_wait(&C.full[stage], parity, &C.abort, P.wait_ns)) { ok = false; break; }
                        tc::fence_after();
                        const int boxes = min(P.kb, k1 - kc);
                        uint64_t ad = desc0 + uint32_t(stage * stage_bytes) / 16;
                        for (int q = 0; q < boxes; ++q, ad += box_bytes / 16) {
                            const uint64_t bd = ad + A_BYTES / 16;
#pragma unroll
                            for (int k = 0; k < TILE_K / 16; ++k)
                                tc::mma<CG>(d, ad + 2 * k, bd + 2 * k, idesc, kc + q > k0 || k > 0);
                        }
                        tc::commit<CG>(&C.empty[stage]);
                        if (++stage == S) {
                            stage = 0;
                            parity ^= 1;
                        }
                    }
                    if (ok) tc::commit<CG>(&C.acc_full[acc]);
                    if (++acc == P.accs) {
                        acc = 0;
                        acc_parity ^= 1;
                    }
                }
            }
            if (!ok) give_up();
            // no product is in flight when this thread is done, whatever the others made of them
            tc::commit_here<CG>(&C.drain);
            mbar_wait_for(&C.drain, 0, WAIT_LIMIT_NS);
        }
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;   // of PARTS
        constexpr int PARTS = EPI_WARPS / 4;
        const uint32_t empty_bar = CG == 2 ? tc::mapa(&C.acc_empty[0], 0) : smem_u32(&C.acc_empty[0]);
        int acc = 0;
        uint32_t acc_parity = 0;
        auto free_acc = [&](int which) {   // an accumulator is read
            tc::fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) tc::arrive_cluster(empty_bar + 8 * which);
                else mbar_arrive_a(empty_bar + 8 * which);
            }
        };
        auto next_acc = [&]() {
            if (++acc == P.accs) {
                acc = 0;
                acc_parity ^= 1;
            }
        };
        auto release = [&]() {   // the accumulator at hand is read; on to the next
            free_acc(acc);
            next_acc();
        };
        tc::wait_prerequisites();   // U, the order and the status words come from down_kernel
        // a wait of the whole warp: all lanes go on or none
        auto products_done = [&]() {
            return __all_sync(0xffffffffu, mbar_wait(&C.acc_full[acc], acc_parity, &C.abort, P.wait_ns)) != 0;
        };
        bool gone = false;   // gave up
        for (int t = first; t < tiles; t += step) {
            const int v = ((t / P.ntile) * CG + rank) * TILE_V + quarter * 32 + lane, b0 = (t % P.ntile) * P.nt;
            const int rows = min(P.nt, P.batch - b0);
            const int windows = (rows + 7) / 8, w0 = windows * part / PARTS, w1 = windows * (part + 1) / PARTS;
            const int vw = v - lane;   // the warp's first vocabulary row
            const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
            // the adapters' share of the first windows, while the products run
            constexpr int EARLY = Epilogue<ODT, RC, SMALL>::EARLY;
            constexpr int R = RC > 0 ? RC : 1;
            using W = Windows<DT, ODT, R>;
            W win;
            float add[EARLY > 0 ? EARLY : 1][2][4];
            int ents[EARLY > 0 ? EARLY : 1];
            if (gone) {
                if (vw < P.vocab)
                    for (int w = w0; w < w1; ++w) store_nan<ODT, RC>(P, b0, rows, w, vw);
                continue;
            }
            bool ok = true;
            if constexpr (EARLY > 0) {
                if (vw < P.vocab) {
#pragma unroll
                    for (int i = 0; i < EARLY; ++i) ents[i] = W::entry(P, b0, rows, w0 + i, lane);
                    if (w0 < w1) early_windows<DT, ODT, R, EARLY>(add, ents, P, b0, rows, w0, w1, vw, lane);
                }
            }
            if (PIECES && nk > piece) {
                // this warp's columns: every PARTS-th block of eight
                constexpr int SUMS = Epilogue<ODT, RC, SMALL>::SUMS;
                float sum[SUMS];
#pragma unroll
                for (int i = 0; i < SUMS; ++i) sum[i] = 0.0f;
                uint32_t at = 0;
                for (int k0 = 0; k0 < nk; k0 += piece) {
                    ok = products_done();
                    if (!ok) break;
                    tc::fence_after();
                    at = lanes + acc * P.nt + part * 8;
#pragma unroll
                    for (int i = 0; i < SUMS; i += 8) {
                        if (part * 8 + i * PARTS < P.nt) {
                            float x[8];
                            tc::tmem_ld8(x, at + i * PARTS);
                            tc::tmem_wait_ld(x);
#pragma unroll
                            for (int j = 0; j < 8; ++j) sum[i + j] += x[j];
                        }
                    }
                    if (k0 + piece < nk) release();
                }
                if (ok) {
                    // the whole sums go back to where the last piece was
#pragma unroll
                    for (int i = 0; i < SUMS; i += 8)
                        if (part * 8 + i * PARTS < P.nt) tc::tmem_st8(sum + i, at + i * PARTS);
                    tc::tmem_wait_st();
                }
                tc::fence_before();
                // the warps of this quarter of the lanes, which go on or give up together
                ok = !named_any(1 + quarter, 32 * PARTS, !ok);
                tc::fence_after();
            } else if (!PIECES && nk > piece) {
                // this warp's columns of each piece take what the one before it holds
                int before = -1;
                for (int k0 = 0; k0 < nk; k0 += piece) {
                    ok = products_done();
                    if (!ok) break;
                    tc::fence_after();
                    if (before >= 0) {
#pragma unroll 1
                        for (int i = part * 8; i < P.nt; i += 8 * PARTS) {
                            float x[8], y[8];
                            tc::tmem_ld8(x, lanes + acc * P.nt + i);
                            tc::tmem_ld8(y, lanes + before * P.nt + i);
                            tc::tmem_wait_ld(x);
                            tc::tmem_wait_ld(y);
#pragma unroll
                            for (int j = 0; j < 8; ++j) x[j] += y[j];
                            tc::tmem_st8(x, lanes + acc * P.nt + i);
                        }
                        tc::tmem_wait_st();
                        free_acc(before);
                    }
                    before = acc;
                    if (k0 + piece < nk) next_acc();
                }
                tc::fence_before();
                ok = !named_any(1 + quarter, 32 * PARTS, !ok);
                tc::fence_after();
            } else {
                ok = products_done();
                tc::fence_after();
            }
            if (!ok) {
                gone = true;
                if (lane == 0) {
                    give_up();
                    if (P.out_status && atomicExch(&C.reported, 1) == 0)
                        for (int i = 0; i < P.batch; ++i) atomicOr(&P.out_status[i], FG_ROW_TIMEOUT);
                }
                __syncwarp();
                t -= step;   // this tile again, as what was not stored
                continue;
            }
            const uint32_t base = lanes + acc * P.nt;
            if (vw < P.vocab) {
                if constexpr (EARLY > 0) {
#pragma unroll
                    for (int i = 0; i < EARLY; ++i)
                        if (w0 + i < w1) store_window<DT, ODT, RC>(P, base, b0, w0 + i, vw, ents[i], add[i], lane);
                }
                win = W{};
                for (int w = w0 + EARLY; w < w1; ++w) {
                    float more[2][4] = {};
                    int ent = 8 * w + (lane & 7);
                    if constexpr (RC > 0) {
                        ent = W::entry(P, b0, rows, w, lane);
                        win.adapters(more, P, b0, rows, w, vw, ent, lane);
                    } else if (ent >= rows) {
                        ent = -1;
                    }
                    store_window<DT, ODT, RC>(P, base, b0, w, vw, ent, more, lane);
                }
            }
            release();
        }
    }
    tc::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *reinterpret_cast<volatile int*>(&C.abort)) {
        // the copies in flight land before the CTA leaves. A pair's loads are counted on the
        // first CTA's barriers, to which both may not have brought all: a wait by time
        if (CG == 1)
            for (int s = 0; s < min(S, filled); ++s)
                mbar_wait_for(&C.full[s], ((filled - 1 - s) / S) & 1, WAIT_LIMIT_NS);
        else
            for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 10000000;) {}
    }
    __syncwarp();
    if (CG == 2) tc::cluster_sync();   // no CTA leaves while its pair may still signal it
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_free<CG>(tmem, P.tmem_cols);
    }
}

}  // namespace adapt
}  // namespace fg
