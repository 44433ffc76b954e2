// tmap.cuh -- host-side creation of TMA tensor maps (CUtensorMap) without linking libcuda:
// the driver's cuTensorMapEncodeTiled is fetched once through the runtime's entry-point
// query.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace k3 {

// 2-D row-major tensor [outer][inner] of `elem_bytes` elements with `row_bytes` between
// rows; box [box_outer][box_inner]; 128-byte swizzle when box_inner * elem_bytes == 128.
// Returns K3CUDA_OK or an error code with the message set.
int make_tmap_2d(CUtensorMap *map, const void *base, CUtensorMapDataType dtype,
                 uint32_t elem_bytes, uint64_t inner, uint64_t outer, uint64_t row_bytes,
                 uint32_t box_inner, uint32_t box_outer);

// 3-D tensor [d2][d1][d0] with byte strides s1 (between d1 rows) and s2 (between d2 planes);
// box [b2][b1][b0], 128-byte swizzle.
int make_tmap_3d(CUtensorMap *map, const void *base, CUtensorMapDataType dtype,
                 uint32_t elem_bytes, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1,
                 uint64_t s2, uint32_t b0, uint32_t b1, uint32_t b2);

// bf16 tensor [rows][inner] (packed, inner a multiple of 64, rows of 8), cut so that one load of
// box_rows rows (a multiple of 8, at most 2048) x box_blocks 64-value blocks lands as
// [box_rows / 8][box_blocks][8 rows][128 B] with the 128-byte swizzle: eight-row groups
// box_blocks * 1024 bytes apart for any number of rows, so that loads of short runs of rows put
// together one matrix operand. Coordinates: (0, 0, first block, first row / 8).
int make_tmap_rows8(CUtensorMap *map, const void *base, uint64_t inner, uint64_t rows,
                    uint32_t box_blocks, uint32_t box_rows);

}  // namespace k3
