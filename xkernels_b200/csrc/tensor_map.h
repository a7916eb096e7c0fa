// Encoded 2-D tensor maps, kept per (base, shape, box, type, swizzle) (moe_tc.cu).
#pragma once
#include <cuda.h>
#include "common.cuh"

namespace xkb {

// 2-D row-major tensor [rows, cols] of `elem_bits` elements, box [box_rows, box_cols].
int make_map_2d(CUtensorMap* map, CUtensorMapDataType dt, int elem_bits, const void* base, uint64_t rows,
                uint64_t cols, uint32_t box_rows, uint32_t box_cols, CUtensorMapSwizzle swz, const char* what);

// The same with rows `pitch_bytes` apart (a multiple of 16).
int make_map_2d_pitched(CUtensorMap* map, CUtensorMapDataType dt, const void* base, uint64_t rows, uint64_t cols,
                        uint64_t pitch_bytes, uint32_t box_rows, uint32_t box_cols, CUtensorMapSwizzle swz, const char* what);
// And planes of such rows, `plane_bytes` apart.
int make_map_3d_pitched(CUtensorMap* map, CUtensorMapDataType dt, const void* base, uint64_t planes, uint64_t rows, uint64_t cols,
                        uint64_t plane_bytes, uint64_t pitch_bytes, uint32_t box_planes, uint32_t box_rows, uint32_t box_cols,
                        CUtensorMapSwizzle swz, const char* what);

}  // namespace xkb
