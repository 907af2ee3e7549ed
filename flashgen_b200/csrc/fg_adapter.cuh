// fg_adapter.cuh — logits of a batch that shares an LM head, every row with its
// own low-rank adapter beside it (fg_adapter_logits):
//   out[b, v] = X[b, :] . W[v, :] + U[b, :] . up[a_b, v, :],
//   U[b, i]   = scales[a_b] * (X[b, :] . down[a_b, i, :])
// U is held in fp32 in the workspace; the second term is added in fp32 to the
// first one's accumulator, row by row, so a row touches no adapter but its own.
#pragma once

#include "fg_common.cuh"

namespace fg {
namespace adapt {

struct Params {
    const void* hidden;
    const void* weight;
    const void* down;
    const void* up;
    const float* scales;
    const int32_t* adapters;
    void* out;
    int32_t* out_status;
    float* u;                 // [B, rank] (workspace)
    int32_t batch, dim, vocab, rank, slots;
    int64_t hidden_stride, weight_stride, down_stride, out_stride;
};

// The row's slot, or -1 without an adapter: none wanted, an id out of range, or
// a slot with scale 0.
__device__ __forceinline__ int row_slot(const Params& P, int b) {
    const int a = P.adapters ? P.adapters[b] : -1;
    return (a >= 0 && a < P.slots && P.scales[a] != 0.0f) ? a : -1;
}

constexpr int DOWN_THREADS = 256;

// U of one row per CTA, a warp per rank index.
template <int DT>
__global__ void __launch_bounds__(DOWN_THREADS) down_kernel(const Params P) {
    const int b = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0 && P.out_status)
        P.out_status[b] = (P.adapters && P.adapters[b] >= P.slots) ? FG_ROW_BAD_PARAM : 0;
    const int slot = row_slot(P, b);
    if (slot < 0) return;
    for (int i = warp; i < P.rank; i += DOWN_THREADS / 32) {
        const int64_t at = (int64_t(slot) * P.rank + i) * P.down_stride;
        float s = 0.0f;
        for (int k = lane; k < P.dim; k += 32)
            s = fmaf(Elem<DT>::load(P.hidden, int64_t(b) * P.hidden_stride + k), Elem<DT>::load(P.down, at + k), s);
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) P.u[int64_t(b) * P.rank + i] = s * P.scales[slot];
    }
}

constexpr int TILE = 64, KSTEP = 16;

// One 64 x 64 output tile per CTA of 256 threads, 4 x 4 outputs a thread.
template <int DT, int ODT>
__global__ void __launch_bounds__(256) project_kernel(const Params P) {
    __shared__ float xs[KSTEP][TILE + 1], ws[KSTEP][TILE + 1];
    const int v0 = blockIdx.x * TILE, b0 = blockIdx.y * TILE;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < P.dim; k0 += KSTEP) {
        for (int e = threadIdx.x; e < TILE * KSTEP; e += 256) {
            const int row = e / KSTEP, k = e % KSTEP;
            const bool in = k0 + k < P.dim;
            xs[k][row] = (in && b0 + row < P.batch)
                             ? Elem<DT>::load(P.hidden, int64_t(b0 + row) * P.hidden_stride + k0 + k) : 0.0f;
            ws[k][row] = (in && v0 + row < P.vocab)
                             ? Elem<DT>::load(P.weight, int64_t(v0 + row) * P.weight_stride + k0 + k) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KSTEP; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty + 16 * i], ws[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const int b = b0 + ty + 16 * i;
        if (b >= P.batch) continue;
        const int slot = row_slot(P, b);
        for (int j = 0; j < 4; ++j) {
            const int v = v0 + tx + 16 * j;
            if (v >= P.vocab) continue;
            float d = acc[i][j];
            if (slot >= 0)
                for (int q = 0; q < P.rank; ++q)
                    d = fmaf(P.u[int64_t(b) * P.rank + q],
                             Elem<DT>::load(P.up, (int64_t(slot) * P.vocab + v) * P.rank + q), d);
            Elem<ODT>::store(P.out, int64_t(b) * P.out_stride + v, d);
        }
    }
}

}  // namespace adapt
}  // namespace fg
