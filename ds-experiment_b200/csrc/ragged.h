// What the products grouped by expert share between their CUDA-core and
// tensor-core parts.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace dsb {

constexpr int kSmallTile = 64;    // rows of a small group's tile
constexpr int kTensorTile = 256;  // rows of a tile of the tensor-core product
// Groups of at least this many rows take the tensor-core product.
constexpr int64_t kTensorRows = 128;

// Rows [row, row + rows) of a group.
struct RaggedTile {
  int32_t group, row, rows, pad;
};

// Made by prep_kernel in the workspace.
struct RaggedPlan {
  int32_t* row;           // [G + 1] first row of each group, then the end of the last
  int32_t* small_start;   // [G + 1] first tile of each small group
  int32_t* tensor_start;  // [G + 1] first tile of each large one
  RaggedTile* small;      // null: not wanted
  RaggedTile* tensor;
  int64_t small_cap, tensor_cap;
  int32_t* counter;       // cleared
  int64_t counters;
  int64_t tensor_rows;    // a group of as many rows is large
};

#ifdef __CUDACC__
__device__ __forceinline__ double result_value(const DotResult& c, int64_t i) {
  return c.f64 ? c.f64[i]
               : __dadd_rn(static_cast<double>(c.hi[i]), static_cast<double>(c.lo[i]));
}
#endif

}  // namespace dsb
