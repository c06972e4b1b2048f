// Products grouped by expert: rows of consecutive groups times their group's
// matrix, and the contraction over each group's rows.
#include <string>

#include "common.cuh"
#include "ds_arith.cuh"
#include "kernels.h"
#include "profile.h"

namespace dsb {
namespace {

__device__ __forceinline__ double value_at(const DotOperand& o, int64_t i) {
  return o.f64 ? o.f64[i] : to_f64(ds2{o.hi[i], o.lo[i]});
}

__device__ __forceinline__ void put(const DotResult& c, int64_t i, double v) {
  if (c.f64) {
    c.f64[i] = v;
  } else {
    const ds2 d = from_f64(v);
    c.hi[i] = d.hi;
    c.lo[i] = d.lo;
  }
}

// Exclusive ends of the groups: offsets[g] = first row of group g,
// offsets[G] = first row behind the last one.  A negative size counts as 0
// and no group passes row M.
__global__ void __launch_bounds__(32)
offsets_kernel(const int32_t* __restrict__ sizes, int64_t G, int64_t M,
               int32_t* __restrict__ offsets) {
  wait_previous_grid();
  if (threadIdx.x != 0) return;
  int64_t at = 0;
  for (int64_t g = 0; g < G; ++g) {
    offsets[g] = static_cast<int32_t>(at);
    at += sizes[g] > 0 ? sizes[g] : 0;
    if (at > M) at = M;
  }
  offsets[G] = static_cast<int32_t>(at);
}

// The group of row `row`: the last g with offsets[g] <= row, or G behind them.
__device__ __forceinline__ int64_t group_of(const int32_t* offsets, int64_t G, int64_t row) {
  if (row >= offsets[G]) return G;
  int64_t lo = 0, hi = G;  // offsets[lo] <= row < offsets[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

constexpr int kThreads = 128;

__global__ void __launch_bounds__(kThreads)
ragged_dot_kernel(RaggedProblem p, const int32_t* __restrict__ offsets) {
  wait_previous_grid();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (j >= p.N) return;
  for (int64_t i = blockIdx.y; i < p.M; i += gridDim.y) {
    const int64_t g = group_of(offsets, p.G, i);
    double s = 0.0;
    if (g < p.G)
      for (int64_t k = 0; k < p.K; ++k)
        s = __fma_rn(value_at(p.lhs, i * p.lhs.s_r + k * p.lhs.s_k),
                     value_at(p.rhs, g * p.rhs.s_b + j * p.rhs.s_r + k * p.rhs.s_k), s);
    put(p.out, i * p.N + j, s);
  }
}

__global__ void __launch_bounds__(kThreads)
ragged_contract_kernel(RaggedProblem p, const int32_t* __restrict__ offsets) {
  wait_previous_grid();
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (j >= p.N) return;
  for (int64_t r = blockIdx.y; r < p.G * p.K; r += gridDim.y) {
    const int64_t g = r / p.K, i = r - g * p.K;
    double s = 0.0;
    for (int64_t t = offsets[g]; t < offsets[g + 1]; ++t)
      s = __fma_rn(value_at(p.lhs, i * p.lhs.s_r + t * p.lhs.s_k),
                   value_at(p.rhs, j * p.rhs.s_r + t * p.rhs.s_k), s);
    put(p.out, r * p.N + j, s);
  }
}

size_t offsets_bytes(int64_t G) { return (static_cast<size_t>(G + 1) * 4 + 255) / 256 * 256; }

int launch_offsets(const RaggedProblem& p, int32_t* offsets, cudaStream_t s) {
  DSB_CUDA_TRY(launch_dependent(offsets_kernel, dim3(1), dim3(32), s, p.group_sizes, p.G, p.M,
                                offsets));
  return DS_OK;
}

dim3 row_grid(int64_t N, int64_t rows) {
  return dim3(static_cast<unsigned>((N + kThreads - 1) / kThreads),
              static_cast<unsigned>(rows < 65535 ? rows : 65535));
}

}  // namespace

size_t ragged_dot_workspace_bytes(int64_t, int64_t, int64_t, int64_t G, bool) {
  return offsets_bytes(G);
}

int ragged_dot(const RaggedProblem& p, void* workspace, size_t, cudaStream_t s) {
  if (p.M == 0 || p.N == 0) return ok();
  int32_t* offsets = static_cast<int32_t*>(workspace);
  ProfileScope prof("ragged_dot", s);
  if (int st = launch_offsets(p, offsets, s)) return st;
  DSB_CUDA_TRY(launch_dependent(ragged_dot_kernel, row_grid(p.N, p.M), dim3(kThreads), s, p,
                                offsets));
  return launch_status();
}

size_t ragged_contract_workspace_bytes(int64_t, int64_t, int64_t, int64_t G) {
  return offsets_bytes(G);
}

int ragged_contract(const RaggedProblem& p, void* workspace, size_t, cudaStream_t s) {
  if (p.G == 0 || p.K == 0 || p.N == 0) return ok();
  int32_t* offsets = static_cast<int32_t*>(workspace);
  ProfileScope prof("ragged_dot_contract", s);
  if (int st = launch_offsets(p, offsets, s)) return st;
  DSB_CUDA_TRY(launch_dependent(ragged_contract_kernel, row_grid(p.N, p.G * p.K), dim3(kThreads),
                                s, p, offsets));
  return launch_status();
}

}  // namespace dsb
