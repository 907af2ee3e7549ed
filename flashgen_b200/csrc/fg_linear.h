// fg_linear.h — what the entry points of the fused linear block (fg_linear.cu) and its
// kernels (fg_linear.cuh) share.
#pragma once

#include <cuda.h>

#include "fg_internal.h"

namespace fg {
namespace lin {

constexpr int TILE_L = 128, TILE_K = 64;   // accumulator lanes of a CTA; elements of a K step
constexpr int MAX_NT = 256;                // columns of a tile
constexpr int MAX_STAGES = 12;
constexpr int MAX_SPLITS = 8;
constexpr int MAX_ACC = 4;                 // accumulators that take turns
constexpr int64_t DEFAULT_WAIT_NS = 1000000000;   // limit of a wait: 1 s, far above any legitimate one

// One product: out[c, l] = act(sum_k A[l, k] B[c, k] + bias[l]) + residual[c, l], l being the
// contiguous dimension of out.
struct Params {
    void* out;
    const void* bias;         // [L] or null
    const void* residual;     // [C, L] or null
    float* preact;            // [C, L]: the sum with the bias, or null
    int64_t out_stride, residual_stride, preact_stride;
    int32_t L, C, K;
    int32_t act;              // FG_ACT_*
    int32_t nt;               // columns of a tile
    int32_t nl, nc;           // tiles along l (of 128; 256 for a pair) and along c
    int32_t stages, accs, tmem_cols;
    int32_t splits;           // CTAs (a cluster) that share a tile's sum over K
    uint64_t wait_ns;         // limit of each wait
    int32_t withhold;         // accumulator whose products are never reported (for tests); -1: none
};

}  // namespace lin
}  // namespace fg
