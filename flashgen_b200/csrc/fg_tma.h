// fg_tma.h — host side of tiled TMA loads: tensor maps of row-major matrices (fg_host.cu).
#pragma once

#include <cuda.h>

#include <cstdint>

namespace fg {
namespace host {

// A [rows, dim] matrix of 16-bit elements read in boxes of box_rows x 64 elements with the
// 128-byte swizzle; columns past dim and rows past `rows` read as zero. False where the
// driver refuses it.
bool encode_rows(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t dim, int64_t stride,
                 int box_rows);

}  // namespace host
}  // namespace fg
