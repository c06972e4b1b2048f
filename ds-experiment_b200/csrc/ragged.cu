// Products grouped by expert: rows of consecutive groups times their group's
// matrix, and the contraction over each group's rows.
//
// Groups are sorted by their number of rows, on the device (prep_kernel): a
// group of at least kTensorRows rows goes to the tensor-core product
// (ragged_ozaki.cu), the others are multiplied here with FP64 matrix
// instructions.  One launch serves all of a call's small groups.
//
// Bound: HBM while a group has few rows (each matrix is read once, 8 bytes a
// value, for 2 rows operations), the FP64 pipe (64 FMA per clock and SM) above
// about 20 rows.
#include <climits>
#include <mutex>
#include <string>
#include <vector>

#include "common.cuh"
#include "ds_arith.cuh"
#include "kernels.h"
#include "profile.h"
#include "ragged.h"

namespace dsb {
namespace {

__device__ __forceinline__ void put(const DotResult& c, int64_t i, double v) {
  if (c.f64) {
    c.f64[i] = v;
  } else {
    const ds2 d = from_f64(v);
    c.hi[i] = d.hi;
    c.lo[i] = d.lo;
  }
}

// ---- the groups' rows and tiles ------------------------------------------------

constexpr int kPrepThreads = 1024;

// Exclusive sum over the block, and the block's total.
__device__ int64_t block_scan(int64_t v, int64_t& total) {
  __shared__ int64_t s_warp[kPrepThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t w = s_warp[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const int64_t before = (warp > 0 ? s_warp[warp - 1] : 0) + x - v;
  total = s_warp[kPrepThreads / 32 - 1];
  __syncthreads();
  return before;
}

// start[g] <= t < start[g + 1] for t in [0, start[G]).
__device__ __forceinline__ int64_t owner_of(const int32_t* start, int64_t G, int32_t t) {
  int64_t lo = 0, hi = G;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One block: the groups' first rows inside [begin, end) of the call's rows (a
// negative size counts as 0, no group passes row M), and the tiles of the two
// kinds of groups.
__global__ void __launch_bounds__(kPrepThreads)
prep_kernel(const int32_t* __restrict__ sizes, int64_t G, int64_t M, int64_t begin, int64_t end,
            RaggedPlan p) {
  wait_previous_grid();
  const int64_t tid = threadIdx.x;
  for (int64_t i = tid; i < p.counters; i += kPrepThreads) p.counter[i] = 0;
  int64_t rows_before = 0, tiles_before = 0, slots_before = 0;
  for (int64_t g0 = 0; g0 < G; g0 += kPrepThreads) {
    const int64_t g = g0 + tid;
    const int64_t n = g < G && sizes[g] > 0 ? sizes[g] : 0;
    int64_t sum, tsum, ssum;
    int64_t lo = rows_before + block_scan(n, sum), hi = lo + n;
    rows_before += sum;
    // the group's rows inside the call's window
    auto clip = [&](int64_t r) {
      r = r < M ? r : M;
      return r < begin ? begin : r > end ? end : r;
    };
    lo = clip(lo);
    hi = clip(hi);
    const int64_t rows = hi - lo;
    const bool tensor = rows >= p.tensor_rows;
    const int64_t d = tensor ? 0 : (rows + kSmallTile - 1) / kSmallTile;
    const int64_t t = tensor ? (rows + kTensorTile - 1) / kTensorTile : 0;
    // both counts stay below 2^31
    const int64_t both = tiles_before + block_scan(d << 32 | t, tsum);
    tiles_before += tsum;
    const int64_t slot = slots_before + block_scan(tensor, ssum);
    slots_before += ssum;
    if (g < G) {
      p.row[g] = static_cast<int32_t>(lo);
      p.small_start[g] = static_cast<int32_t>(both >> 32);
      p.tensor_start[g] = static_cast<int32_t>(both & 0xffffffff);
      p.slot[g] = static_cast<int32_t>(slot);
      if (tensor) {
        int bits = 50;
        for (int i = 0; i < kBitsLimits && rows > p.bits_limit[i]; ++i) --bits;
        p.slot_group[slot] = static_cast<int32_t>(g);
        p.slot_bits[slot] = bits;
      }
      if (g == G - 1) {
        p.row[G] = static_cast<int32_t>(hi);
        p.small_start[G] = static_cast<int32_t>((both >> 32) + d);
        p.tensor_start[G] = static_cast<int32_t>((both & 0xffffffff) + t);
        p.slot[G] = static_cast<int32_t>(slot + tensor);
      }
    }
  }
  if (G == 0 && tid == 0) p.row[0] = p.small_start[0] = p.tensor_start[0] = p.slot[0] = 0;
  __syncthreads();
  auto fill = [&](const int32_t* start, int tile, RaggedTile* out, int64_t cap) {
    const int64_t n = start[G] < cap ? start[G] : cap;
    for (int64_t t = tid; t < n; t += kPrepThreads) {
      const int64_t g = owner_of(start, G, static_cast<int32_t>(t));
      const int32_t row = p.row[g] + static_cast<int32_t>(t - start[g]) * tile;
      const int32_t left = p.row[g + 1] - row;
      out[t] = RaggedTile{static_cast<int32_t>(g), row, left < tile ? left : tile, p.slot[g]};
    }
  };
  if (p.small) fill(p.small_start, kSmallTile, p.small, p.small_cap);
  if (p.tensor) fill(p.tensor_start, kTensorTile, p.tensor, p.tensor_cap);
}

// ---- small groups: FP64 matrix instructions ---------------------------------------

constexpr int kThreads = 256;
constexpr int kTN = 64;      // columns of a tile
constexpr int kKS = 32;      // contraction per pipeline stage
constexpr int kStages = 3;
// Row pitches of the staged tiles, in values: 4 (mod 16) puts the 4 x 4
// values that half a warp reads for a fragment in 16 different 8-byte banks.
constexpr int kPitchK = kKS + 4;       // [row or column][k]
constexpr int kPitchN = kSmallTile + 4;  // [k][row or column]
constexpr int kOperand = kSmallTile * kPitchK > kKS * kPitchN ? kSmallTile * kPitchK : kKS * kPitchN;
constexpr size_t kSmallBytes = sizeof(double) * 2 * kStages * kOperand;
static_assert(kTN == kSmallTile, "A and B are staged alike");

template <int kBytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool valid) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  const int n = valid ? kBytes : 0;
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(src), "r"(n)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(at), "l"(src), "n"(kBytes),
                 "r"(n)
                 : "memory");
}

// d += a b for an 8 x 4 and a 4 x 8 fragment: lane l holds a[l / 4][l % 4],
// b[l % 4][l / 4] and d[l / 4][2 (l % 4) + {0, 1}].
__device__ __forceinline__ void mma_f64(double (&d)[2], double a, double b) {
  asm volatile(
      "mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
      : "+d"(d[0]), "+d"(d[1])
      : "d"(a), "d"(b));
}

// A staged operand: f64 values, or (kPair) the hi words and behind them the
// lo words.
template <bool kPair>
__device__ __forceinline__ double staged(const double* tile, int at) {
  if constexpr (kPair) {
    const float* f = reinterpret_cast<const float*>(tile);
    return __dadd_rn(static_cast<double>(f[at]), static_cast<double>(f[kOperand + at]));
  } else {
    return tile[at];
  }
}

// One operand's part of a unit: `lines` lines of `len` consecutive values,
// line t at offset origin + t stride of the operand.
struct Block2d {
  int64_t origin, stride;
  int lines, len;
};

// kLines lines of kLen values (powers of two) of the block into a staged tile
// (pitch values per line), zeros outside it; kVec values per copy.
template <bool kPair, int kLen, int kVec>
__device__ __forceinline__ void stage_lines(const DotOperand& o, const Block2d& b, int lines,
                                            double* tile, int pitch) {
  constexpr int kElem = kPair ? 4 : 8;
  constexpr int kPerLine = kLen / kVec, kStep = kThreads / kPerLine;
  const int at = threadIdx.x % kPerLine * kVec;
  const bool in_line = at < b.len;  // kVec divides len
#pragma unroll 4
  for (int line = threadIdx.x / kPerLine; line < lines; line += kStep) {
    const bool in = in_line && line < b.lines;
    const int64_t src = in ? b.origin + line * b.stride + at : 0;
    if constexpr (kPair) {
      float* f = reinterpret_cast<float*>(tile) + line * pitch + at;
      copy_async<kElem * kVec>(f, o.hi + src, in);
      copy_async<kElem * kVec>(f + kOperand, o.lo + src, in);
    } else {
      copy_async<kElem * kVec>(tile + line * pitch + at, o.f64 + src, in);
    }
  }
}

template <bool kPair, int kLen>
__device__ __forceinline__ void stage_block(const DotOperand& o, const Block2d& b, int lines,
                                            double* tile, int pitch, int vec) {
  if (vec > 1) stage_lines<kPair, kLen, kPair ? 4 : 2>(o, b, lines, tile, pitch);
  else stage_lines<kPair, kLen, 1>(o, b, lines, tile, pitch);
}

struct SmallArgs {
  RaggedProblem q;
  RaggedPlan p;
  bool contract;
  bool add;        // contraction: add to the result (a later window of rows)
  int tiles_k;     // contraction: tiles of the result's rows
  int tiles_n;
  int splits;      // of the contraction (products only)
  int64_t split_k;
  double* partial;  // [splits][M][N]
  int vec_a, vec_b;  // values per copy
};

// A unit of work: an output tile over a range of the contraction.
struct SmallUnit {
  int64_t g, row, col;  // group, first output row (in the group's rows or matrix) and column
  int rows, cols;
  int64_t k0, k1;       // contraction range (contraction: rows of the call)
  int split;
  int64_t id;           // of its output tile
};

__device__ __forceinline__ int64_t units_of(const SmallArgs& a) {
  if (a.contract) return a.q.G * a.tiles_k * a.tiles_n;
  return static_cast<int64_t>(a.p.small_start[a.q.G]) * a.tiles_n * a.splits;
}

// False for a unit that belongs to the tensor-core product, or that adds
// nothing.
__device__ __forceinline__ bool unit_at(const SmallArgs& a, int64_t u, SmallUnit& x) {
  if (a.contract) {
    const int64_t per = static_cast<int64_t>(a.tiles_k) * a.tiles_n;
    x.g = u / per;
    const int64_t r = u - x.g * per;
    x.row = r / a.tiles_n * kSmallTile;
    x.col = r % a.tiles_n * kTN;
    x.k0 = a.p.row[x.g];
    x.k1 = a.p.row[x.g + 1];
    x.rows = a.q.K - x.row < kSmallTile ? static_cast<int>(a.q.K - x.row) : kSmallTile;
    x.split = 0;
    x.id = u;
    if (x.k1 - x.k0 >= a.p.tensor_rows || (a.add && x.k1 == x.k0)) return false;
  } else {
    const int64_t n = a.p.small_start[a.q.G];
    const int64_t rest = u / n;
    const RaggedTile t = a.p.small[u - rest * n];
    x.g = t.group;
    x.row = t.row;
    x.rows = t.rows;
    x.split = static_cast<int>(rest % a.splits);
    const int64_t tn = rest / a.splits;
    x.col = tn * kTN;
    x.k0 = x.split * a.split_k;
    x.k1 = x.k0 + a.split_k < a.q.K ? x.k0 + a.split_k : a.q.K;
    x.id = tn * n + (u - rest * n);
  }
  x.cols = a.q.N - x.col < kTN ? static_cast<int>(a.q.N - x.col) : kTN;
  return true;
}

// kA: A is staged as [k][row] (its rows are contiguous) rather than [row][k];
// kB: B as [k][column] rather than [column][k].
template <bool kPair, bool kA, bool kB>
__device__ __forceinline__ void stage_unit(const SmallArgs& a, const SmallUnit& x, int64_t k,
                                           double* sa, double* sb) {
  const int kn = x.k1 - k < kKS ? static_cast<int>(x.k1 - k) : kKS;
  const RaggedProblem& q = a.q;
  [[maybe_unused]] const int rows_pad = x.rows <= 16 ? 16 : kSmallTile;
  Block2d A, B;
  if constexpr (kA) {
    A = Block2d{x.row + k * q.lhs.s_k, q.lhs.s_k, kn, x.rows};
    stage_block<kPair, kSmallTile>(q.lhs, A, kKS, sa, kPitchN, a.vec_a);
  } else {
    A = Block2d{x.row * q.lhs.s_r + k, q.lhs.s_r, x.rows, kn};
    stage_block<kPair, kKS>(q.lhs, A, rows_pad, sa, kPitchK, a.vec_a);
  }
  const int64_t base = a.contract ? 0 : x.g * q.rhs.s_b;
  if constexpr (kB) {
    B = Block2d{base + k * q.rhs.s_k + x.col, q.rhs.s_k, kn, x.cols};
    stage_block<kPair, kTN>(q.rhs, B, kKS, sb, kPitchN, a.vec_b);
  } else {
    B = Block2d{base + x.col * q.rhs.s_r + k, q.rhs.s_r, x.cols, kn};
    stage_block<kPair, kKS>(q.rhs, B, kTN, sb, kPitchK, a.vec_b);
  }
}

// The products of one stage: warps stand kWM x (8 / kWM), each with MF x NF
// fragments.
template <bool kPair, bool kA, bool kB, int MF, int NF, int kWM>
__device__ __forceinline__ void multiply_stage(const double* sa, const double* sb, int kn,
                                               double (&acc)[4][2][2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % kWM * MF * 8, wn = warp / kWM * NF * 8;
  const int r = lane >> 2, kk = lane & 3;
#pragma unroll 4
  for (int k = 0; k < kn; k += 4) {
    double fa[MF], fb[NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
      fa[i] = staged<kPair>(sa, kA ? (k + kk) * kPitchN + wm + i * 8 + r
                                   : (wm + i * 8 + r) * kPitchK + k + kk);
#pragma unroll
    for (int j = 0; j < NF; ++j)
      fb[j] = staged<kPair>(sb, kB ? (k + kk) * kPitchN + wn + j * 8 + r
                                   : (wn + j * 8 + r) * kPitchK + k + kk);
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) mma_f64(acc[i][j], fa[i], fb[j]);
  }
}

template <int MF, int NF, int kWM>
__device__ __forceinline__ void store_unit(const SmallArgs& a, const SmallUnit& x,
                                           const double (&acc)[4][2][2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % kWM * MF * 8, wn = warp / kWM * NF * 8;
  const int64_t first = (a.contract ? x.g * a.q.K : 0) + x.row;
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int r = wm + i * 8 + (lane >> 2);
    if (r >= x.rows) continue;
    const int64_t row = (first + r) * a.q.N + x.col;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = wn + j * 8 + 2 * (lane & 3) + h;
        if (c >= x.cols) continue;
        double v = acc[i][j][h];
        if (a.splits > 1) {
          a.partial[static_cast<int64_t>(x.split) * a.q.M * a.q.N + row + c] = v;
          continue;
        }
        if (a.add) v = __dadd_rn(result_value(a.q.out, row + c), v);
        put(a.q.out, row + c, v);
      }
    }
  }
}

// Blocks stay and take every gridDim.x-th unit; the pipeline of stages runs on
// across units.
template <bool kPair, bool kA, bool kB>
__global__ void __launch_bounds__(kThreads, 2)
small_kernel(const __grid_constant__ SmallArgs a) {
  extern __shared__ __align__(16) double stage[];
  __shared__ int s_last;
  wait_previous_grid();
  // rows behind the last group
  if (!a.contract) {
    const int64_t end = a.q.M * a.q.N;
    for (int64_t i = a.p.row[a.q.G] * a.q.N + static_cast<int64_t>(blockIdx.x) * kThreads +
                     threadIdx.x;
         i < end; i += static_cast<int64_t>(gridDim.x) * kThreads)
      put(a.q.out, i, 0.0);
  }
  const int64_t units = units_of(a);
  auto next_unit = [&](int64_t u, SmallUnit& x) {
    while (u < units && !unit_at(a, u, x)) u += gridDim.x;
    return u;
  };
  // loading runs kStages - 1 stages ahead of multiplying
  SmallUnit lx, x;
  int64_t lu = next_unit(blockIdx.x, lx);
  int64_t lk = lu < units ? lx.k0 : 0;
  int ls = 0;
  auto load_one = [&] {
    if (lu < units) {
      double* sa = stage + ls * 2 * kOperand;
      if (lk < lx.k1) stage_unit<kPair, kA, kB>(a, lx, lk, sa, sa + kOperand);
      lk += kKS;
      if (lk >= lx.k1) {
        lu = next_unit(lu + gridDim.x, lx);
        if (lu < units) lk = lx.k0;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ls = ls + 1 == kStages ? 0 : ls + 1;
  };
#pragma unroll 1
  for (int i = 0; i < kStages - 1; ++i) load_one();
  int cs = 0;
#pragma unroll 1
  for (int64_t u = next_unit(blockIdx.x, x); u < units; u = next_unit(u + gridDim.x, x)) {
    double acc[4][2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j][0] = acc[i][j][1] = 0.0;
    int64_t k = x.k0;
    do {  // a unit without contraction takes one (empty) stage
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncthreads();
      const double* sa = stage + cs * 2 * kOperand;
      const int kn = x.k1 - k < kKS ? static_cast<int>(x.k1 - k) : kKS;
      load_one();
      if (x.rows <= 16) multiply_stage<kPair, kA, kB, 2, 1, 1>(sa, sa + kOperand, kn, acc);
      else multiply_stage<kPair, kA, kB, 4, 2, 2>(sa, sa + kOperand, kn, acc);
      cs = cs + 1 == kStages ? 0 : cs + 1;
      k += kKS;
    } while (k < x.k1);
    if (x.rows <= 16) store_unit<2, 1, 1>(a, x, acc);
    else store_unit<4, 2, 2>(a, x, acc);
    if (a.splits > 1) {
      // the last of a tile's splits adds them up in order
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) s_last = atomicAdd(a.p.counter + x.id, 1) == a.splits - 1;
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int e = threadIdx.x; e < x.rows * x.cols; e += kThreads) {
          const int64_t at = (x.row + e / x.cols) * a.q.N + x.col + e % x.cols;
          double v = 0.0;
          for (int s = 0; s < a.splits; ++s)
            v = __dadd_rn(v, __ldcg(a.partial + static_cast<int64_t>(s) * a.q.M * a.q.N + at));
          put(a.q.out, at, v);
        }
      }
      __syncthreads();
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- host ------------------------------------------------------------------------

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Contraction splits of the products: enough units for about four per
// resident block when the rows are few, each of at least kSplitMin.  From the
// call's sizes alone, so a row's rounding does not depend on other groups.
constexpr int64_t kSplitMin = 128;
constexpr int kMaxSplits = 16;

int splits_of(int64_t M, int64_t K, int64_t N, int64_t G) {
  const int64_t tiles = (M / kSmallTile + (G < M ? G : M)) * ceil_div(N, kTN);
  int64_t s = tiles > 0 ? ceil_div(1184, tiles) : 1;
  const int64_t most = K / kSplitMin;
  s = s > most ? most : s;
  s = s > kMaxSplits ? kMaxSplits : s;
  return s < 1 ? 1 : static_cast<int>(s);
}

// Whether the tensor-core product takes groups of many rows: its tiles are
// padded to 256 columns and 128 of the contraction.
bool tensor_allowed(int64_t M, int64_t K, int64_t N, int64_t G, bool contract) {
  return M >= kTensorRows && (contract ? K >= 128 : K >= 64) && N >= 128 &&
         ragged_tensor_fits(M, K, N, G, contract);
}

struct Layout {
  size_t row, small_start, tensor_start, slot, small, tensor, slot_group, slot_bits, counter,
      partial, tensor_ws, total;
  int64_t small_cap, tensor_cap, slots, counters;
  int splits;
  bool tensor_ok;
};

Layout layout_of(int64_t M, int64_t K, int64_t N, int64_t G, bool contract) {
  Layout l{};
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at = (at + bytes + 1023) / 1024 * 1024;
    return here;
  };
  const int64_t groups = G < M ? G : M;  // with rows
  l.tensor_ok = tensor_allowed(M, K, N, G, contract);
  l.small_cap = contract ? 0 : M / kSmallTile + groups;
  if (l.tensor_ok) {
    const int64_t rows = contract && M > kRaggedWindow ? kRaggedWindow : M;
    l.slots = ragged_slots(rows, G);
    l.tensor_cap = ragged_tensor_tiles(rows, G);
  }
  l.splits = contract ? 1 : splits_of(M, K, N, G);
  l.counters = l.splits > 1 ? l.small_cap * ceil_div(N, kTN) : 0;
  l.row = take((G + 1) * 4);
  l.small_start = take((G + 1) * 4);
  l.tensor_start = take((G + 1) * 4);
  l.slot = take((G + 1) * 4);
  l.small = take(l.small_cap * sizeof(RaggedTile));
  l.tensor = take(l.tensor_cap * sizeof(RaggedTile));
  l.slot_group = take(l.slots * 4);
  l.slot_bits = take(l.slots * 4);
  l.counter = take(l.counters * 4);
  l.partial = take(l.splits > 1 ? static_cast<size_t>(l.splits) * M * N * 8 : 0);
  l.tensor_ws = take(l.tensor_ok ? ragged_tensor_bytes(M, K, N, G, contract) : 0);
  // the tensor-core part is aligned to 1024 whatever the workspace's start
  l.total = at + 1024;
  return l;
}

const int32_t* bits_limits() {
  static int32_t limit[kBitsLimits];
  static std::once_flag once;
  std::call_once(once, [] {
    for (int i = 0; i < kBitsLimits; ++i) {
      int64_t lo = 1, hi = kRaggedWindow + 1;  // ragged_bits(lo) >= 50 - i, not so at hi
      if (ragged_bits(kRaggedWindow) >= 50 - i) lo = kRaggedWindow;
      while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        (ragged_bits(mid) >= 50 - i ? lo : hi) = mid;
      }
      limit[i] = static_cast<int32_t>(lo);
    }
  });
  return limit;
}

uint8_t* align_ws(void* workspace) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 1023) &
                                    ~static_cast<uintptr_t>(1023));
}

RaggedPlan plan_at(const Layout& l, int64_t G, uint8_t* ws, bool tensor) {
  auto ints = [&](size_t off) { return reinterpret_cast<int32_t*>(ws + off); };
  RaggedPlan p{};
  p.groups = G;
  p.row = ints(l.row);
  p.small_start = ints(l.small_start);
  p.tensor_start = ints(l.tensor_start);
  p.slot = ints(l.slot);
  p.small = l.small_cap ? reinterpret_cast<RaggedTile*>(ws + l.small) : nullptr;
  p.tensor = l.tensor_cap ? reinterpret_cast<RaggedTile*>(ws + l.tensor) : nullptr;
  p.slot_group = ints(l.slot_group);
  p.slot_bits = ints(l.slot_bits);
  p.small_cap = l.small_cap;
  p.tensor_cap = l.tensor_cap;
  p.counter = ints(l.counter);
  p.counters = l.counters;
  p.tensor_rows = tensor ? kTensorRows : INT32_MAX;
  if (tensor)
    for (int i = 0; i < kBitsLimits; ++i) p.bits_limit[i] = bits_limits()[i];
  return p;
}

// Values per copy of an operand whose lines are `len` values long at a stride
// of `stride` values, from `origin` on.
int copy_width(const DotOperand& o, int64_t len, int64_t stride, int64_t batch) {
  const int wide = o.f64 ? 2 : 4;
  const bool at = o.f64 ? aligned(o.f64, 16) : aligned(o.hi, 16) && aligned(o.lo, 16);
  return at && len % wide == 0 && stride % wide == 0 && batch % wide == 0 ? wide : 1;
}

template <bool kPair, bool kA, bool kB>
int launch_small(const SmallArgs& a, int64_t most_units, cudaStream_t s) {
  static std::mutex mu;
  static std::vector<bool> done;
  int dev = 0;
  DSB_CUDA_TRY(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= static_cast<int>(done.size())) done.resize(dev + 1, false);
    if (!done[dev]) {
      DSB_CUDA_TRY(cudaFuncSetAttribute(small_kernel<kPair, kA, kB>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(kSmallBytes)));
      done[dev] = true;
    }
  }
  const int64_t resident = 2 * static_cast<int64_t>(sm_count());
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(most_units < resident ? (most_units < 1 ? 1 : most_units)
                                                                 : resident));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmallBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DSB_CUDA_TRY(cudaLaunchKernelEx(&cfg, small_kernel<kPair, kA, kB>, a));
  return launch_status();
}

int launch_prep(const RaggedProblem& q, int64_t begin, int64_t end, const RaggedPlan& p,
                cudaStream_t s) {
  DSB_CUDA_TRY(launch_dependent(prep_kernel, dim3(1), dim3(kPrepThreads), s, q.group_sizes, q.G,
                                q.M, begin, end, p));
  return launch_status();
}

}  // namespace

size_t ragged_dot_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t G, bool) {
  return layout_of(M, K, N, G, false).total;
}

int ragged_dot(const RaggedProblem& q, void* workspace, size_t, cudaStream_t s) {
  if (q.M == 0 || q.N == 0) return ok();
  const Layout l = layout_of(q.M, q.K, q.N, q.G, false);
  int clusters = 0;
  if (l.tensor_ok)
    if (int st = ragged_tensor_clusters(&clusters)) return st;
  uint8_t* ws = align_ws(workspace);
  SmallArgs a{};
  a.q = q;
  a.p = plan_at(l, q.G, ws, clusters > 0);
  a.tiles_n = static_cast<int>(ceil_div(q.N, kTN));
  a.splits = l.splits;
  a.split_k = ceil_div(ceil_div(q.K, a.splits), kKS) * kKS;
  a.partial = reinterpret_cast<double*>(ws + l.partial);
  a.vec_a = copy_width(q.lhs, q.K, q.lhs.s_r, 0);
  a.vec_b = copy_width(q.rhs, q.rhs_t ? q.K : q.N, q.rhs_t ? q.rhs.s_r : q.rhs.s_k, q.rhs.s_b);
  if (int st = launch_prep(q, 0, q.M, a.p, s)) return st;
  if (clusters > 0)
    if (int st = ragged_tensor_dot(q, a.p, ws + l.tensor_ws, clusters, s)) return st;
  ProfileScope prof("ragged_small", s);
  const int64_t units = l.small_cap * a.tiles_n * a.splits;
  const bool pair = q.lhs.f64 == nullptr;
  if (q.rhs_t)
    return pair ? launch_small<true, false, false>(a, units, s)
                : launch_small<false, false, false>(a, units, s);
  return pair ? launch_small<true, false, true>(a, units, s)
              : launch_small<false, false, true>(a, units, s);
}

size_t ragged_contract_workspace_bytes(int64_t M, int64_t K, int64_t N, int64_t G) {
  return layout_of(M, K, N, G, true).total;
}

int ragged_contract(const RaggedProblem& q, void* workspace, size_t, cudaStream_t s) {
  if (q.G == 0 || q.K == 0 || q.N == 0) return ok();
  const Layout l = layout_of(q.M, q.K, q.N, q.G, true);
  int clusters = 0;
  if (l.tensor_ok)
    if (int st = ragged_tensor_clusters(&clusters)) return st;
  uint8_t* ws = align_ws(workspace);
  SmallArgs a{};
  a.q = q;
  a.p = plan_at(l, q.G, ws, clusters > 0);
  a.contract = true;
  a.tiles_k = static_cast<int>(ceil_div(q.K, kSmallTile));
  a.tiles_n = static_cast<int>(ceil_div(q.N, kTN));
  a.splits = 1;
  a.vec_a = copy_width(q.lhs, q.K, q.lhs.s_k, 0);
  a.vec_b = copy_width(q.rhs, q.N, q.rhs.s_k, 0);
  const int64_t units = q.G * a.tiles_k * a.tiles_n;
  // without the tensor-core product one window takes all rows
  const int64_t window = clusters > 0 ? kRaggedWindow : q.M + 1;
  for (int64_t begin = 0; begin == 0 || begin < q.M; begin += window) {
    a.add = begin > 0;
    if (int st = launch_prep(q, begin, begin + window, a.p, s)) return st;
    if (clusters > 0)
      if (int st = ragged_tensor_contract(q, a.p, a.add, ws + l.tensor_ws, clusters, s)) return st;
    ProfileScope prof("ragged_small", s);
    const int st = q.lhs.f64 == nullptr ? launch_small<true, true, true>(a, units, s)
                                        : launch_small<false, true, true>(a, units, s);
    if (st) return st;
  }
  return ok();
}

}  // namespace dsb
