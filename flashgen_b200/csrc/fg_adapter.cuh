// fg_adapter.cuh — logits of a batch that shares an LM head, every row with its
// own low-rank adapter beside it (fg_adapter_logits):
//   out[b, v] = X[b, :] . W[v, :] + U[b, :] . up[a_b, v, :],
//   U[b, i]   = scales[a_b] * (X[b, :] . down[a_b, i, :])
//
// Two launches. down_kernel computes U (fp32, a CTA per row), sorts the rows of
// each batch tile by adapter and, where the hidden rows are not 16-byte aligned,
// copies them to aligned ones. project_kernel does the rest: the shared product
// on the tensor cores with the vocabulary on the accumulator's 128 lanes and the
// batch on its columns, so that a small batch wastes no tensor-core rows and a
// warp's stores of one column are 32 neighbouring logits. The adapters' product
// is added by the epilogue warps on the CUDA cores, in fp32, column by column in
// the sorted order: a row touches no adapter but its own (a masked product would
// let NaN from one request's adapter into the others), U needs no rounding to 16
// bits, and each adapter's rows of `up` are read once per tile and kept in
// registers.
#pragma once

#include "fg_adapter.h"
#include "fg_tcgen05.cuh"

namespace fg {
namespace adapt {

// The row's slot, or -1 without an adapter: none wanted, an id out of range, or
// a slot with scale 0.
__device__ __forceinline__ int row_slot(const Params& P, int b) {
    const int a = P.adapters ? P.adapters[b] : -1;
    return (a >= 0 && a < P.slots && P.scales[a] != 0.0f) ? a : -1;
}

constexpr int DOWN_THREADS = 256;
constexpr int DOWN_K = 4096;   // hidden elements staged at a time

// One row per CTA: its position in the sorted order of its batch tile (rows with
// the same adapter next to each other, ties in row order), and U, a warp per rank
// index (2 * RC of them each, their 16-byte loads in flight together).
template <int DT>
__device__ __forceinline__ float from_bits(uint16_t b) {
    if constexpr (DT == FG_DTYPE_F16) return __half2float(__ushort_as_half(b));
    else return __uint_as_float(uint32_t(b) << 16);
}

template <int DT, int RC>
__global__ void __launch_bounds__(DOWN_THREADS) down_kernel(const Params P) {
    __shared__ __align__(16) uint16_t xs[DOWN_K];
    tc::launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b = blockIdx.x;
    const int b0 = b / P.nt * P.nt, n = min(P.nt, P.batch - b0);
    const int slot = row_slot(P, b);
    const int key = ((slot + 1) << 9) | (b - b0);
    int ahead = 0;
    if (tid < n) ahead = (((row_slot(P, b0 + tid) + 1) << 9) | tid) < key;
    const int pos = b0 + __syncthreads_count(ahead);
    if (tid == 0) {
        P.order[pos] = key;
        if (P.out_status) P.out_status[b] = (P.adapters && P.adapters[b] >= P.slots) ? FG_ROW_BAD_PARAM : 0;
    }
    if (slot < 0 && P.copy == nullptr) return;

    const uint16_t* src = reinterpret_cast<const uint16_t*>(P.raw_hidden) + int64_t(b) * P.raw_stride;
    const uint16_t* dn = reinterpret_cast<const uint16_t*>(P.down) + int64_t(max(slot, 0)) * P.rank * P.down_stride;
    const bool wide = reinterpret_cast<uintptr_t>(src) % 16 == 0;
    float acc[2 * RC] = {};
    for (int k0 = 0; k0 < P.dim; k0 += DOWN_K) {
        const int len = min(DOWN_K, P.dim - k0), vec = len / 8;
        __syncthreads();
        if (wide) {
            for (int i = tid; i < vec; i += DOWN_THREADS)
                reinterpret_cast<uint4*>(xs)[i] = reinterpret_cast<const uint4*>(src + k0)[i];
            for (int k = vec * 8 + tid; k < len; k += DOWN_THREADS) xs[k] = src[k0 + k];
        } else {
#pragma unroll 4
            for (int k = tid; k < len; k += DOWN_THREADS) xs[k] = src[k0 + k];
        }
        __syncthreads();
        if (P.copy) {
            uint16_t* dst = reinterpret_cast<uint16_t*>(P.copy) + int64_t(b) * P.copy_stride + k0;
            for (int i = tid; i < vec; i += DOWN_THREADS)
                reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<uint4*>(xs)[i];
            for (int k = vec * 8 + tid; k < len; k += DOWN_THREADS) dst[k] = xs[k];
        }
        if (slot < 0) continue;
#pragma unroll 2
        for (int i = lane; i < vec; i += 32) {
            float x[8];
            Elem<DT>::unpack(reinterpret_cast<const uint4*>(xs)[i], x);
            uint4 q[2 * RC];
#pragma unroll
            for (int j = 0; j < 2 * RC; ++j)
                if (warp + 8 * j < P.rank)
                    q[j] = __ldg(reinterpret_cast<const uint4*>(dn + (warp + 8 * j) * P.down_stride + k0) + i);
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
        if (k < len) {
            const float x = from_bits<DT>(xs[k]);
#pragma unroll
            for (int j = 0; j < 2 * RC; ++j)
                if (warp + 8 * j < P.rank)
                    acc[j] = fmaf(x, Elem<DT>::load(dn + (warp + 8 * j) * P.down_stride + k0, k), acc[j]);
        }
    }
    if (slot < 0) return;
    const float scale = P.scales[slot];
#pragma unroll
    for (int j = 0; j < 2 * RC; ++j) {
        float s = acc[j];
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0 && warp + 8 * j < P.rank) P.u[int64_t(pos) * P.rank + warp + 8 * j] = s * scale;
    }
}

// ---------------------------------------------------------------------------
// project_kernel: persistent, one CTA per SM (CG = 1) or one pair of CTAs per two
// SMs (CG = 2). Warp 0 loads (TMA), warp 1 issues the products, warps 2..9 are the
// epilogue (two per quarter of the accumulator's lanes). Two accumulators in
// tensor memory: one tile's epilogue runs beside the next tile's products.
//
// fp32 results: the tensor core truncates when it adds a product to the
// accumulator, and over hundreds of steps that bias shows in 32 bits. So the sum
// over K is taken in pieces of PIECE_K, alternating between the two accumulators,
// and the epilogue warps add the pieces in registers with rounding. A 16-bit
// result does not see the difference and takes the whole sum in one piece.
// ---------------------------------------------------------------------------
constexpr int A_BYTES = TILE_V * TILE_K * 2;
constexpr int MAX_STAGES = 12;
constexpr int EPI_WARPS = 8;
constexpr int PROJ_THREADS = 64 + 32 * EPI_WARPS;
constexpr int U_FLOATS = 512;                      // U of a group of columns, per epilogue warp
constexpr int U_BYTES = EPI_WARPS * U_FLOATS * 4;
constexpr int PIECE_K = 8;                         // 64-wide steps of K per piece of an fp32 sum

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
    uint64_t acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
          "l"(*reinterpret_cast<uint64_t*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}

// One vocabulary row of an adapter's `up`: 16 * RC elements (zero past the rank).
template <int DT, int RC>
struct UpRow {
    uint4 q[2 * RC];
    __device__ __forceinline__ void load(const Params& P, int slot, int v) {
        const uint4* src = reinterpret_cast<const uint4*>(
            reinterpret_cast<const uint16_t*>(P.up) + (int64_t(slot) * P.vocab + v) * P.rank);
#pragma unroll
        for (int i = 0; i < 2 * RC; ++i) q[i] = (i * 8 < P.rank) ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void unpack(float2 (&w)[8 * RC]) const {
#pragma unroll
        for (int i = 0; i < 2 * RC; ++i) {
            float x[8];
            Elem<DT>::unpack(q[i], x);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * i + j] = make_float2(x[2 * j], x[2 * j + 1]);
        }
    }
};

// x + U[row] . up[v]; `u` in shared memory, the same for the whole warp.
template <int RC>
__device__ __forceinline__ float add_adapter(float x, const float* u, const float2 (&w)[8 * RC], int rank) {
    float2 s0 = make_float2(x, 0.0f), s1 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < RC; ++c) {
        if (c > 0 && c * 16 >= rank) break;
#pragma unroll
        for (int q = 4 * c; q < 4 * c + 4; ++q) {
            const float4 f = reinterpret_cast<const float4*>(u)[q];
            s0 = fma2(make_float2(f.x, f.y), w[2 * q], s0);
            s1 = fma2(make_float2(f.z, f.w), w[2 * q + 1], s1);
        }
    }
    return (s0.x + s0.y) + (s1.x + s1.y);
}

// The epilogue of one warp over positions [p, p1) of the tile's sorted order.
// `base`: the warp's lanes of the accumulator; v: this lane's vocabulary id (in:
// below vocab). Columns go eight at a time where they share an adapter and one at
// a time around the changes; the next adapter's row is on its way meanwhile.
template <int DT, int ODT, int RC>
__device__ __forceinline__ void finish_columns(const Params& P, uint32_t base, int b0, int p, int p1, int v, bool in,
                                               float* ubuf, int lane) {
    constexpr int R = RC > 0 ? RC : 1;
    if constexpr (RC == 0) {
        for (; p < p1; p += 8) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) tc::tmem_ld1(x[i], base + min(p + i, p1 - 1));
            tc::tmem_wait_ld(x);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (p + i < p1 && in) Elem<ODT>::store(P.out, int64_t(b0 + p + i) * P.out_stride + v, x[i]);
        }
    } else {
        constexpr int GROUP = R == 1 ? 32 : U_FLOATS / (16 * R);
        constexpr int STEP = GROUP < 8 ? GROUP : 8;
        constexpr bool AHEAD = R <= 4;   // registers for a second row
        const int rank = P.rank;
        const int vrow = in ? v : P.vocab - 1;
        float2 w[8 * R];
        UpRow<DT, R> next;
        int cur = -1, next_slot = -1;
        int entry = (lane < GROUP && p + lane < p1) ? P.order[b0 + p + lane] : 0;
        float4 un[4];
        auto fetch_u = [&](int at) {
            const int total = min(GROUP, p1 - at) * rank / 4;
            const float4* src = reinterpret_cast<const float4*>(P.u + int64_t(b0 + at) * rank);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 32 * i < total) un[i] = src[lane + 32 * i];
        };
        if (p < p1) fetch_u(p);
        while (p < p1) {
            const int cnt = min(GROUP, p1 - p);
            const int ent = entry;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 32 * i < cnt * rank / 4) reinterpret_cast<float4*>(ubuf)[lane + 32 * i] = un[i];
            __syncwarp();
            const int pn = p + cnt;
            entry = (lane < GROUP && pn + lane < p1) ? P.order[b0 + pn + lane] : 0;
            if (pn < p1) fetch_u(pn);
            const int slots = (ent >> 9) - 1;   // this lane's column's
            for (int j = 0; j < cnt;) {
                const int slot = __shfl_sync(0xffffffffu, slots, j);
                if (slot != cur) {
                    cur = slot;
                    if (slot >= 0) {
                        if (!AHEAD || slot != next_slot) next.load(P, slot, vrow);
                        next.unpack(w);
                    }
                    if (AHEAD) {
                        uint32_t m = __ballot_sync(0xffffffffu, lane > j && lane < cnt && slots != slot);
                        next_slot = -1;
                        if (m) {
                            next_slot = __shfl_sync(0xffffffffu, slots, __ffs(m) - 1);
                        } else {
                            m = __ballot_sync(0xffffffffu, lane < GROUP && pn + lane < p1 && (entry >> 9) - 1 != slot);
                            if (m) next_slot = (__shfl_sync(0xffffffffu, entry, __ffs(m) - 1) >> 9) - 1;
                        }
                        if (next_slot >= 0) next.load(P, next_slot, vrow);
                    }
                }
                const uint32_t same = __ballot_sync(0xffffffffu, lane < cnt && slots == slot) >> j;
                constexpr uint32_t FULL = STEP == 32 ? 0xffffffffu : (1u << STEP) - 1;
                if ((same & FULL) == FULL) {
                    float x[STEP];
                    int col[STEP];
#pragma unroll
                    for (int i = 0; i < STEP; ++i) {
                        col[i] = __shfl_sync(0xffffffffu, ent, j + i) & 511;
                        tc::tmem_ld1(x[i], base + col[i]);
                    }
                    tc::tmem_wait_ld(x);
                    if (slot >= 0) {
#pragma unroll
                        for (int i = 0; i < STEP; ++i) x[i] = add_adapter<R>(x[i], ubuf + (j + i) * rank, w, rank);
                    }
#pragma unroll
                    for (int i = 0; i < STEP; ++i)
                        if (in) Elem<ODT>::store(P.out, int64_t(b0 + col[i]) * P.out_stride + v, x[i]);
                    j += STEP;
                } else {
                    float x[1];
                    const int col = __shfl_sync(0xffffffffu, ent, j) & 511;
                    tc::tmem_ld1(x[0], base + col);
                    tc::tmem_wait_ld(x);
                    if (slot >= 0) x[0] = add_adapter<R>(x[0], ubuf + j * rank, w, rank);
                    if (in) Elem<ODT>::store(P.out, int64_t(b0 + col) * P.out_stride + v, x[0]);
                    ++j;
                }
            }
            __syncwarp();
            p = pn;
        }
    }
}

// RC: rank / 16 held in registers (rounded up to 1, 2, 4 or 8), 0: no adapters.
template <int CG, int DT, int ODT, int RC>
__global__ void __launch_bounds__(PROJ_THREADS, 1)
project_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Params P) {
    extern __shared__ uint8_t dyn[];
    __shared__ Control C;
    constexpr bool PIECES = ODT == FG_DTYPE_F32;
    uint8_t* ring = dyn + ((1024 - (smem_u32(dyn) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? tc::cta_rank() : 0;
    const int S = P.stages;
    const int box_bytes = A_BYTES + P.nt / CG * TILE_K * 2;   // one 64-wide step of K, this CTA's part
    const int stage_bytes = P.kb * box_bytes;
    const int nk = (P.dim + TILE_K - 1) / TILE_K;
    const int piece = PIECES ? PIECE_K : nk;
    const int tiles = P.nvt * P.ntile;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&C.acc_full[i], 1);
            mbar_init(&C.acc_empty[i], CG * EPI_WARPS);
        }
        mbar_init(&C.drain, 1);
        C.abort = 0;
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

    if (warp == 0) {
        if (lane == 0) {
            if (P.copy) tc::wait_prerequisites();   // the aligned rows come from down_kernel
            int it = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                const int v0 = ((t / P.ntile) * CG + rank) * TILE_V;
                const int b0 = (t % P.ntile) * P.nt + rank * (P.nt / CG);
                for (int kc = 0; kc < nk; kc += P.kb, ++it) {
                    const int s = it % S;
                    if (it >= S && !mbar_wait(&C.empty[s], ((it / S) - 1) & 1, &C.abort)) { ok = false; break; }
                    const int boxes = min(P.kb, nk - kc);
                    const uint32_t bar = CG == 2 ? tc::mapa(&C.full[s], 0) : smem_u32(&C.full[s]);
                    if (rank == 0) mbar_arrive_expect_tx(&C.full[s], CG * boxes * box_bytes);
                    uint32_t a = smem_u32(ring + s * stage_bytes);
                    for (int q = 0; q < boxes; ++q, a += box_bytes) {
                        tc::tma_load_2d<CG>(a, &wmap, (kc + q) * TILE_K, v0, bar);
                        tc::tma_load_2d<CG>(a + A_BYTES, &xmap, (kc + q) * TILE_K, b0, bar);
                    }
                }
            }
            if (!ok) {
                // gave up: let the copies in flight land before the block leaves
                *reinterpret_cast<volatile int*>(&C.abort) = 1;
                if (rank == 0)
                    for (int j = max(0, it - S); j < it; ++j)
                        mbar_wait_for(&C.full[j % S], (j / S) & 1, WAIT_LIMIT_NS / 16);
                for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 1000000;) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = tc::instr_desc(DT, TILE_V * CG, P.nt);
            int it = 0, n = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                for (int k0 = 0; k0 < nk && ok; k0 += piece, ++n) {
                    const int acc = n & 1, k1 = min(nk, k0 + piece);
                    if (n >= 2 && !mbar_wait(&C.acc_empty[acc], ((n >> 1) - 1) & 1, &C.abort)) { ok = false; break; }
                    tc::fence_after();
                    const uint32_t d = tmem + acc * P.nt;
                    for (int kc = k0; kc < k1; kc += P.kb, ++it) {
                        const int s = it % S;
                        if (!mbar_wait(&C.full[s], (it / S) & 1, &C.abort)) { ok = false; break; }
                        tc::fence_after();
                        const int boxes = min(P.kb, k1 - kc);
                        for (int q = 0; q < boxes; ++q) {
                            const uint32_t a = smem_u32(ring + s * stage_bytes + q * box_bytes);
                            const uint64_t ad = tc::operand_desc(a), bd = tc::operand_desc(a + A_BYTES);
#pragma unroll
                            for (int k = 0; k < TILE_K / 16; ++k)
                                tc::mma<CG>(d, ad + 2 * k, bd + 2 * k, idesc, kc + q > k0 || k > 0);
                        }
                        tc::commit<CG>(&C.empty[s]);
                    }
                    if (ok) tc::commit<CG>(&C.acc_full[acc]);
                }
            }
            if (!ok) {
                *reinterpret_cast<volatile int*>(&C.abort) = 1;
                tc::commit<CG>(&C.drain);
                mbar_wait_for(&C.drain, 0, WAIT_LIMIT_NS);
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        float* ubuf = reinterpret_cast<float*>(ring + S * stage_bytes) + (warp - 2) * U_FLOATS;
        const uint32_t empty_bar[2] = {CG == 2 ? tc::mapa(&C.acc_empty[0], 0) : smem_u32(&C.acc_empty[0]),
                                       CG == 2 ? tc::mapa(&C.acc_empty[1], 0) : smem_u32(&C.acc_empty[1])};
        auto release = [&](int acc) {
            tc::fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) tc::arrive_cluster(empty_bar[acc]);
                else mbar_arrive_a(empty_bar[acc]);
            }
        };
        tc::wait_prerequisites();   // U, the order and the status words come from down_kernel
        int n = 0;
        bool ok = true;
        for (int t = first; t < tiles && ok; t += step) {
            const int v = ((t / P.ntile) * CG + rank) * TILE_V + quarter * 32 + lane, b0 = (t % P.ntile) * P.nt;
            const int rows = min(P.nt, P.batch - b0);
            const int mid = (rows + 1) / 2;
            const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
            if (PIECES && nk > piece) {
                const int cols = P.nt / 2;   // this warp's share of the columns, a multiple of 8
                float sum[MAX_NT / 2];
#pragma unroll
                for (int i = 0; i < MAX_NT / 2; ++i) sum[i] = 0.0f;
                uint32_t at = 0;
                for (int k0 = 0; k0 < nk; k0 += piece) {
                    ok = mbar_wait(&C.acc_full[n & 1], (n >> 1) & 1, &C.abort);
                    if (!ok) break;
                    tc::fence_after();
                    at = lanes + (n & 1) * P.nt + half * cols;
#pragma unroll
                    for (int i = 0; i < MAX_NT / 2; i += 8) {
                        if (i < cols) {
                            float x[8];
                            tc::tmem_ld8(x, at + i);
                            tc::tmem_wait_ld(x);
#pragma unroll
                            for (int j = 0; j < 8; ++j) sum[i + j] += x[j];
                        }
                    }
                    if (k0 + piece < nk) {
                        release(n & 1);
                        ++n;
                    }
                }
                if (ok) {
                    // the whole sums go back to where the last piece was
#pragma unroll
                    for (int i = 0; i < MAX_NT / 2; i += 8)
                        if (i < cols) tc::tmem_st8(sum + i, at + i);
                    tc::tmem_wait_st();
                }
                tc::fence_before();
                // the two warps of this quarter of the lanes, which go on or give up together
                ok = !named_any(1 + quarter, 64, !ok);
                tc::fence_after();
            } else {
                ok = mbar_wait(&C.acc_full[n & 1], (n >> 1) & 1, &C.abort);
                tc::fence_after();
            }
            if (!ok) {
                *reinterpret_cast<volatile int*>(&C.abort) = 1;
                if (P.out_status && threadIdx.x == 64)
                    for (int i = 0; i < rows; ++i) atomicOr(&P.out_status[b0 + i], FG_ROW_TIMEOUT);
                break;
            }
            finish_columns<DT, ODT, RC>(P, lanes + (n & 1) * P.nt, b0, half ? mid : 0, half ? rows : mid, v,
                                        v < P.vocab, ubuf, lane);
            release(n & 1);
            ++n;
        }
    }
    tc::fence_before();
    __syncthreads();
    if (CG == 2) tc::cluster_sync();   // no CTA leaves while its pair may still signal it
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_free<CG>(tmem, P.tmem_cols);
    }
}

}  // namespace adapt
}  // namespace fg
