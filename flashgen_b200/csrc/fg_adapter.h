// fg_adapter.h — what the entry points (fg_adapter.cu) and the launches
// (fg_adapter_*.cu, one unit per operand and result type) share.
#pragma once

#include <cuda.h>

#include "fg_internal.h"

namespace fg {
namespace adapt {

constexpr int TILE_V = 128, TILE_K = 64;   // accumulator lanes; elements of a K step (128 bytes)
constexpr int MAX_NT = 256;                // batch columns of a tile
constexpr int SMALL_NT = 64;
constexpr int MAX_ACC = 8;                 // accumulators in tensor memory
constexpr int64_t DEFAULT_WAIT_NS = 1000000000;   // limit of a wait: 1 s, far above any legitimate one

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
    void* u;                  // [B, 3, 16 RC] in the sorted order: 16-bit parts of U times powers of two (workspace)
    float* unit;              // [B] in the sorted order: the first power's inverse, negative where 16-bit results need all parts (workspace)
    int32_t* order;           // [B] per batch tile: (slot + 1) << 9 | column, sorted (workspace)
    void* copy;               // [B, copy_stride] hidden rows, sorted and aligned, or null (workspace)
    int32_t batch, dim, vocab, rank, slots;
    int64_t down_stride, out_stride, copy_stride;
    int32_t ntile;            // batch tiles
    int32_t sorted;           // rows of a tile in the order of their adapters (else as they come)
    int32_t wide_out;         // rows of out 16-byte aligned
    int32_t f32_out;
    int32_t nt;               // columns of a batch tile, a multiple of 16 up to 256
    // project_kernel
    int32_t nvt;              // vocabulary tiles of 128 (256 for a pair)
    int32_t stages;           // of the operand ring
    int32_t kb;               // 64-wide boxes of K in a stage
    int32_t accs;             // accumulators of nt columns in tensor memory
    int32_t tmem_cols;
    int32_t chained;          // down_kernel goes before
    int32_t withhold;         // accumulator whose products are never reported (tests), or -1
    uint64_t wait_ns;         // limit of each wait
};

// Both launches of a call: operands of type DT, result of type ODT. `pair`: two
// CTAs share each product (tiles of 256 vocabulary rows).
template <int DT, int ODT>
int launch(const Params& P, const CUtensorMap& wmap, const CUtensorMap& xmap, bool pair, host::DevInfo* d,
           cudaStream_t st);

}  // namespace adapt
}  // namespace fg
