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

#include "fg_tcgen05.cuh"

namespace fg {
namespace adapt {

struct Params {
    const void* hidden;       // rows for the products: the caller's, or the aligned copy
    const void* raw_hidden;   // the caller's rows
    int64_t hidden_stride, raw_stride;
    const void* down;
    const void* up;
    const float* scales;
    const int32_t* adapters;
    void* out;
    int32_t* out_status;
    float* u;                 // [B, rank] (workspace)
    int32_t* order;           // [B] per batch tile: (slot + 1) << 9 | column, sorted (workspace)
    void* copy;               // [B, copy_stride] aligned hidden rows, or null (workspace)
    int32_t batch, dim, vocab, rank, slots;
    int64_t down_stride, out_stride, copy_stride;
    // project_kernel
    int32_t ntile;            // batch tiles
    int32_t nt;               // columns of a batch tile, a multiple of 16 up to 256
    int32_t nvt;              // vocabulary tiles of 128
    int32_t stages;
    int32_t tmem_cols;
};

// The row's slot, or -1 without an adapter: none wanted, an id out of range, or
// a slot with scale 0.
__device__ __forceinline__ int row_slot(const Params& P, int b) {
    const int a = P.adapters ? P.adapters[b] : -1;
    return (a >= 0 && a < P.slots && P.scales[a] != 0.0f) ? a : -1;
}

constexpr int DOWN_THREADS = 256;
constexpr int MAX_NT = 256;

// CTAs [0, batch): U of one row, a warp per rank index. CTAs [batch, batch +
// ntile): the sorted order of one batch tile (each thread counts the rows ahead
// of its own).
template <int DT>
__global__ void __launch_bounds__(DOWN_THREADS) down_kernel(const Params P) {
    __shared__ int keys[MAX_NT];
    tc::launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x >= P.batch) {
        const int b0 = (blockIdx.x - P.batch) * P.nt;
        const int n = min(P.nt, P.batch - b0);
        const int i = threadIdx.x;
        int key = 0;
        if (i < n) {
            key = ((row_slot(P, b0 + i) + 1) << 9) | i;
            keys[i] = key;
        }
        __syncthreads();
        if (i < n) {
            int pos = 0;
            for (int j = 0; j < n; ++j) pos += keys[j] < key;
            P.order[b0 + pos] = key;
        }
        return;
    }
    const int b = blockIdx.x;
    if (threadIdx.x == 0 && P.out_status)
        P.out_status[b] = (P.adapters && P.adapters[b] >= P.slots) ? FG_ROW_BAD_PARAM : 0;
    if (P.copy) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(P.raw_hidden) + int64_t(b) * P.raw_stride;
        uint16_t* dst = reinterpret_cast<uint16_t*>(P.copy) + int64_t(b) * P.copy_stride;
        for (int k = threadIdx.x; k < P.dim; k += DOWN_THREADS) dst[k] = src[k];
    }
    const int slot = row_slot(P, b);
    if (slot < 0) return;
    for (int i = warp; i < P.rank; i += DOWN_THREADS / 32) {
        const int64_t at = (int64_t(slot) * P.rank + i) * P.down_stride;
        float s = 0.0f;
        for (int k = lane; k < P.dim; k += 32)
            s = fmaf(Elem<DT>::load(P.raw_hidden, int64_t(b) * P.raw_stride + k), Elem<DT>::load(P.down, at + k), s);
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) P.u[int64_t(b) * P.rank + i] = s * P.scales[slot];
    }
}

// ---------------------------------------------------------------------------
// project_kernel: persistent, one CTA per SM. Warp 0 loads (TMA), warp 1 issues
// the products, warps 2..9 are the epilogue (two per quarter of the accumulator's
// lanes). Two accumulators in tensor memory: one tile's epilogue runs beside the
// next tile's products.
// ---------------------------------------------------------------------------
constexpr int TILE_V = 128, TILE_K = 64;
constexpr int A_BYTES = TILE_V * TILE_K * 2;
constexpr int MAX_STAGES = 12;
constexpr int EPI_WARPS = 8;
constexpr int PROJ_THREADS = 64 + 32 * EPI_WARPS;

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

// `rank` consecutive elements of up for one vocabulary row, 16 per chunk.
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

// RC: rank / 16 held in registers (rounded up to 1, 2, 4 or 8), 0: no adapters.
template <int DT, int ODT, int RC>
__global__ void __launch_bounds__(PROJ_THREADS, 1)
project_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Params P) {
    extern __shared__ uint8_t dyn[];
    __shared__ Control C;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = P.stages;
    const int stage_bytes = A_BYTES + P.nt * TILE_K * 2;
    const int nk = (P.dim + TILE_K - 1) / TILE_K;
    const int tiles = P.nvt * P.ntile;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&C.acc_full[i], 1);
            mbar_init(&C.acc_empty[i], EPI_WARPS);
        }
        mbar_init(&C.drain, 1);
        C.abort = 0;
        fence_mbar_init();
        tc::prefetch_map(&wmap);
        tc::prefetch_map(&xmap);
    }
    if (warp == 1) {
        tc::tmem_alloc(&C.tmem, P.tmem_cols);
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = C.tmem;

    if (warp == 0) {
        if (lane == 0) {
            if (P.copy) tc::wait_prerequisites();   // the aligned rows come from down_kernel
            int it = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                const int v0 = (t / P.ntile) * TILE_V, b0 = (t % P.ntile) * P.nt;
                for (int kc = 0; kc < nk; ++kc, ++it) {
                    const int s = it % S;
                    if (it >= S && !mbar_wait(&C.empty[s], ((it / S) - 1) & 1, &C.abort)) { ok = false; break; }
                    uint8_t* a = ring + s * stage_bytes;
                    mbar_arrive_expect_tx(&C.full[s], stage_bytes);
                    tc::tma_load_2d(a, &wmap, kc * TILE_K, v0, &C.full[s]);
                    tc::tma_load_2d(a + A_BYTES, &xmap, kc * TILE_K, b0, &C.full[s]);
                }
            }
            if (!ok) {
                // gave up: let the copies in flight land before the block leaves
                *reinterpret_cast<volatile int*>(&C.abort) = 1;
                for (int j = max(0, it - S); j < it; ++j) mbar_wait_for(&C.full[j % S], (j / S) & 1, WAIT_LIMIT_NS);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = tc::instr_desc(DT, TILE_V, P.nt);
            int it = 0, n = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++n) {
                const int acc = n & 1;
                if (n >= 2 && !mbar_wait(&C.acc_empty[acc], ((n >> 1) - 1) & 1, &C.abort)) { ok = false; break; }
                tc::fence_after();
                const uint32_t d = tmem + acc * P.nt;
                for (int kc = 0; kc < nk; ++kc, ++it) {
                    const int s = it % S;
                    if (!mbar_wait(&C.full[s], (it / S) & 1, &C.abort)) { ok = false; break; }
                    tc::fence_after();
                    const uint32_t a = smem_u32(ring + s * stage_bytes);
                    const uint64_t ad = tc::operand_desc(a), bd = tc::operand_desc(a + A_BYTES);
#pragma unroll
                    for (int k = 0; k < TILE_K / 16; ++k)
                        tc::mma(d, ad + 2 * k, bd + 2 * k, idesc, (kc | k) != 0);
                    tc::commit(&C.empty[s]);
                }
                if (ok) tc::commit(&C.acc_full[acc]);
            }
            if (!ok) {
                *reinterpret_cast<volatile int*>(&C.abort) = 1;
                tc::commit(&C.drain);
                mbar_wait_for(&C.drain, 0, WAIT_LIMIT_NS);
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        tc::wait_prerequisites();   // U, the order and the status words come from down_kernel
        int n = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
            const int acc = n & 1;
            const int v = (t / P.ntile) * TILE_V + quarter * 32 + lane, b0 = (t % P.ntile) * P.nt;
            const int rows = min(P.nt, P.batch - b0);
            const bool in = v < P.vocab;
            const int p1 = half ? rows : (rows + 1) / 2;
            int p = half ? (rows + 1) / 2 : 0;
            const uint32_t base = tmem + acc * P.nt + lanes;
            bool ok = mbar_wait(&C.acc_full[acc], (n >> 1) & 1, &C.abort);
            if (!ok) {
                *reinterpret_cast<volatile int*>(&C.abort) = 1;
                if (P.out_status && threadIdx.x == 64)
                    for (int i = 0; i < rows; ++i) atomicOr(&P.out_status[b0 + i], FG_ROW_TIMEOUT);
                break;
            }
            tc::fence_after();
            if constexpr (RC == 0) {
                for (; p < p1; p += 8) {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = tc::tmem_column(base + min(p + i, p1 - 1));
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (p + i < p1 && in) Elem<ODT>::store(P.out, int64_t(b0 + p + i) * P.out_stride + v, x[i]);
                }
            } else {
                float2 w[8 * RC];
                while (p < p1) {
                    // the run of rows that share the adapter of position p (at most 32 at a time)
                    const int mine = p + lane < p1 ? P.order[b0 + p + lane] : 0x7fffffff;
                    const int slot = (__shfl_sync(0xffffffffu, mine, 0) >> 9) - 1;
                    const uint32_t other = __ballot_sync(0xffffffffu, (mine >> 9) - 1 != slot);
                    const int run = other ? __ffs(other) - 1 : 32;
                    if (slot >= 0) {
                        UpRow<DT, RC> up;
                        up.load(P, slot, in ? v : P.vocab - 1);
                        up.unpack(w);
                    }
                    for (int j = 0; j < run; j += 4) {
                        float x[4];
                        int col[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            col[i] = __shfl_sync(0xffffffffu, mine, min(j + i, run - 1)) & 511;
                            x[i] = tc::tmem_column(base + col[i]);
                        }
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (j + i >= run) break;
                            if (slot >= 0) {
                                const float4* u = reinterpret_cast<const float4*>(
                                    P.u + int64_t(b0 + col[i]) * P.rank);
                                float2 s0 = make_float2(x[i], 0.0f), s1 = make_float2(0.0f, 0.0f);
#pragma unroll
                                for (int q = 0; q < 4 * RC; ++q) {
                                    if (q * 4 < P.rank) {
                                        const float4 f = u[q];
                                        s0 = fma2(make_float2(f.x, f.y), w[2 * q], s0);
                                        s1 = fma2(make_float2(f.z, f.w), w[2 * q + 1], s1);
                                    }
                                }
                                x[i] = (s0.x + s0.y) + (s1.x + s1.y);
                            }
                            if (in) Elem<ODT>::store(P.out, int64_t(b0 + col[i]) * P.out_stride + v, x[i]);
                        }
                    }
                    p += run;
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&C.acc_empty[acc]);
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_free(tmem, P.tmem_cols);
    }
}

}  // namespace adapt
}  // namespace fg
