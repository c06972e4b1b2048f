// What the products grouped by expert share between their CUDA-core
// (ragged.cu) and tensor-core (ragged_ozaki.cu) parts.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels.h"

namespace dsb {

constexpr int kSmallTile = 64;    // rows of a small group's tile
constexpr int kTensorTile = 256;  // rows of a tile of the tensor-core product
// Groups of at least this many rows are large: the tensor-core product takes
// them.  Its fixed costs are a matrix's split (products) or rebuilding (contraction):
// 32 groups of 96 rows, 2048 x 2048 matrices, take 1.18 ms with it and 1.11 without
// as products, of 128 rows 1.20 and 1.43; as a contraction 32 of 192 rows 1.96 and
// 1.96, of 256 2.06 and 2.53 (1024 x 1024 matrices: of 192 0.58 and 0.50, of 256 0.64
// and 0.65).
constexpr int64_t tensor_rows(bool contract) { return contract ? 256 : 128; }
// Longest contraction over rows that is taken at once.
constexpr int64_t kRaggedWindow = 1 << 15;
// Most workspace that the tensor-core product may ask for.
constexpr size_t kRaggedTensorBytes = static_cast<size_t>(48) << 30;

// Large groups among G with M rows, and their tiles, at most.
inline int64_t ragged_slots(int64_t M, int64_t G, bool contract) {
  const int64_t most = M / tensor_rows(contract);
  return G < most ? G : most;
}
inline int64_t ragged_tensor_tiles(int64_t M, int64_t G, bool contract) {
  return M / kTensorTile + ragged_slots(M, G, contract);
}

// Rows [row, row + rows) of a group; slot: its number among the large ones.
struct RaggedTile {
  int32_t group, row, rows, slot;
};

// Bits that an operand keeps (of the tensor-core product): 50 - i up to
// limit[i] terms.
constexpr int kBitsLimits = 6;

// Made by prep_kernel in the workspace.
struct RaggedPlan {
  int64_t groups;
  int32_t* row;           // [G + 1] first row of each group, then the end of the last
  int32_t* small_start;   // [G + 2] full tiles of the small groups before each, then their
                          // number, then that of all small tiles
  int32_t* tensor_start;  // [G + 1] the same of the large ones
  int32_t* slot;          // [G + 1] large groups before each, then their number
  int32_t* order;         // [G] contraction: the groups by falling number of rows; products:
                          // prep_kernel's own
  RaggedTile* small;      // [small_cap] products; null: contraction
  RaggedTile* tensor;
  int32_t* slot_group;    // of each large group: its number among all,
  int32_t* slot_bits;     // and the bits its rows allow as a contraction
  int64_t small_cap, tensor_cap;
  int64_t tensor_rows;    // a group of as many rows is large
  int32_t bits_limit[kBitsLimits];
};

// The large groups' part (ragged_ozaki.cu), after prep_kernel on the stream.
// `clusters`: CTA pairs of the GEMM on this device (0: not available).
int ragged_bits(int64_t K);
int ragged_tensor_clusters(int* clusters);
bool ragged_tensor_fits(int64_t M, int64_t K, int64_t N, int64_t G, bool contract);
size_t ragged_tensor_bytes(int64_t M, int64_t K, int64_t N, int64_t G, bool contract);
int ragged_tensor_dot(const RaggedProblem& q, const RaggedPlan& p, void* workspace, int clusters,
                      cudaStream_t s);
// add: onto the result rather than over it.
int ragged_tensor_contract(const RaggedProblem& q, const RaggedPlan& p, bool add, void* workspace,
                           int clusters, cudaStream_t s);

#ifdef __CUDACC__
__device__ __forceinline__ double result_value(const DotResult& c, int64_t i) {
  return c.f64 ? c.f64[i]
               : __dadd_rn(static_cast<double>(c.hi[i]), static_cast<double>(c.lo[i]));
}
#endif

}  // namespace dsb
