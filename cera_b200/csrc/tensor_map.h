// TMA tensor maps of row-major matrices.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace cera {

// [rows][ld] elements of elem_bytes (ld * elem_bytes a multiple of 16), boxes of box_cols x box_rows elements; elements outside
// read as zero.
int32_t tensor_map_2d(CUtensorMap *map, CUtensorMapDataType type, uint32_t elem_bytes, const void *base, uint64_t rows, uint64_t ld, uint32_t box_cols,
                      uint32_t box_rows, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion);

// Four dimensions, the innermost contiguous, strides in bytes (multiples of 16), boxes of 128 bytes of it laid down with the 128-byte swizzle.
int32_t tensor_map_4d(CUtensorMap *map, CUtensorMapDataType type, const void *base, const uint64_t (&dims)[4], const uint64_t (&strides)[3],
                      const uint32_t (&box)[4]);

// bf16, boxes laid down with the 128-byte swizzle (box_cols = 64).
inline int32_t tensor_map_bf16(CUtensorMap *map, const void *base, uint64_t rows, uint64_t ld, uint32_t box_cols, uint32_t box_rows) {
    return tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, rows, ld, box_cols, box_rows, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

}  // namespace cera
