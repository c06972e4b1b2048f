// Products grouped by expert: rows of consecutive groups times their group's
// matrix, and the contraction over each group's rows.
//
// Groups are sorted by their number of rows, on the device (prep_kernel): a
// group of many rows goes to the tensor-core product
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
// Most groups that are put in order of their rows (each compares itself with all).
constexpr int64_t kOrderedGroups = 2048;

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

// A group's rows inside [begin, end) of the call's rows, given its first row and
// number (a negative one counts as 0; no group passes row M), and its tiles.
struct GroupShape {
  int32_t row, end;
  int32_t full, tail;  // small: tiles of kSmallTile rows, and rows of one more (or 0)
  int32_t tensor;      // large: tiles
  bool large;
};

__device__ __forceinline__ GroupShape shape_of(int64_t first, int64_t n, int64_t M, int64_t begin,
                                               int64_t end, const RaggedPlan& p) {
  auto clip = [&](int64_t r) {
    r = r < M ? r : M;
    return r < begin ? begin : r > end ? end : r;
  };
  const int64_t lo = clip(first), hi = clip(first + n), rows = hi - lo;
  GroupShape g;
  g.row = static_cast<int32_t>(lo);
  g.end = static_cast<int32_t>(hi);
  g.large = rows >= p.tensor_rows;
  g.full = g.large ? 0 : static_cast<int32_t>(rows / kSmallTile);
  g.tail = g.large ? 0 : static_cast<int32_t>(rows % kSmallTile);
  g.tensor = g.large ? static_cast<int32_t>((rows + kTensorTile - 1) / kTensorTile) : 0;
  return g;
}

// Small tiles stand in falling order of the work they take (full ones, then
// tails by the accumulators that small_kernel gives them), so that the last units
// of a call are its short ones: 0 .. 3, or 4 for no tail.
constexpr int kTailKinds = 4;
__device__ __forceinline__ int tail_kind(int tail) {
  return tail == 0 ? kTailKinds : tail <= 8 ? 3 : tail <= 16 ? 2 : tail <= 32 ? 1 : 0;
}

__device__ __forceinline__ void put_tail(const RaggedPlan& p, int64_t g, int32_t end, int32_t tail,
                                         int64_t at) {
  p.small[at] = RaggedTile{static_cast<int32_t>(g), end - tail, tail, 0};
}

// Writes group g's places, given the full small tiles, large tiles and large
// groups before it.
__device__ __forceinline__ void put_group(const RaggedPlan& p, int64_t g, const GroupShape& x,
                                          int64_t full, int64_t tensor, int64_t slot) {
  p.row[g] = x.row;
  p.small_start[g] = static_cast<int32_t>(full);
  p.tensor_start[g] = static_cast<int32_t>(tensor);
  p.slot[g] = static_cast<int32_t>(slot);
  if (x.large) {
    int bits = 50;
    for (int i = 0; i < kBitsLimits && x.end - x.row > p.bits_limit[i]; ++i) --bits;
    p.slot_group[slot] = static_cast<int32_t>(g);
    p.slot_bits[slot] = bits;
  }
  if (g == p.groups - 1) {
    p.row[g + 1] = x.end;
    p.small_start[g + 1] = static_cast<int32_t>(full + x.full);
    p.tensor_start[g + 1] = static_cast<int32_t>(tensor + x.tensor);
    p.slot[g + 1] = static_cast<int32_t>(slot + x.large);
  }
}

// The tables of whole tiles and the groups' order, from what put_group wrote.
__device__ void put_tables(const RaggedPlan& p, int64_t G, int64_t tid, int64_t threads) {
  // a contraction's groups by falling number of rows
  if (!p.small) {
    for (int64_t g = tid; g < G; g += threads) {
      const int32_t n = p.row[g + 1] - p.row[g];
      int32_t rank = static_cast<int32_t>(g);
      if (G <= kOrderedGroups) {
        rank = 0;
        for (int64_t h = 0; h < G; ++h) {
          const int32_t m = p.row[h + 1] - p.row[h];
          rank += m > n || (m == n && h < g);
        }
      }
      p.order[rank] = static_cast<int32_t>(g);
    }
  }
  auto fill = [&](const int32_t* start, int tile, RaggedTile* out, int64_t cap) {
    const int64_t n = start[G] < cap ? start[G] : cap;
    for (int64_t t = tid; t < n; t += threads) {
      const int64_t g = owner_of(start, G, static_cast<int32_t>(t));
      const int32_t row = p.row[g] + static_cast<int32_t>(t - start[g]) * tile;
      const int32_t left = p.row[g + 1] - row;
      out[t] = RaggedTile{static_cast<int32_t>(g), row, left < tile ? left : tile, p.slot[g]};
    }
  };
  if (p.small) fill(p.small_start, kSmallTile, p.small, p.small_cap);
  if (p.tensor) fill(p.tensor_start, kTensorTile, p.tensor, p.tensor_cap);
}

// One block for any number of groups.
__global__ void __launch_bounds__(kPrepThreads)
prep_kernel(const int32_t* __restrict__ sizes, int64_t G, int64_t M, int64_t begin, int64_t end,
            RaggedPlan p) {
  wait_previous_grid();
  const int64_t tid = threadIdx.x;
  int64_t rows_before = 0, tiles_before = 0, slots_before = 0;
  int64_t tails_before = 0;  // 16 bits for each kind
  for (int64_t g0 = 0; g0 < G; g0 += kPrepThreads) {
    const int64_t g = g0 + tid;
    const int64_t n = g < G && sizes[g] > 0 ? sizes[g] : 0;
    int64_t rows, tiles, slots;
    const GroupShape x = shape_of(rows_before + block_scan(n, rows), n, M, begin, end, p);
    // both counts stay below 2^31
    const int64_t both =
        tiles_before + block_scan(static_cast<int64_t>(x.full) << 32 | x.tensor, tiles);
    const int64_t slot = slots_before + block_scan(x.large, slots);
    rows_before += rows;
    tiles_before += tiles;
    slots_before += slots;
    if (g < G) put_group(p, g, x, both >> 32, both & 0xffffffff, slot);
    if (p.small) {
      int64_t tails;
      const int kind = tail_kind(x.tail);
      const int64_t one = kind < kTailKinds ? 1ll << (16 * kind) : 0;
      const int64_t before = tails_before + block_scan(one, tails);
      tails_before += tails;
      // the tail's number among its kind
      if (one) p.order[g] = static_cast<int32_t>(before >> (16 * kind) & 0xffff);
    }
  }
  if (G == 0 && tid == 0) p.row[0] = p.small_start[0] = p.tensor_start[0] = p.slot[0] = 0;
  __syncthreads();
  put_tables(p, G, tid, kPrepThreads);
  if (!p.small) return;
  int64_t kinds[kTailKinds + 1] = {tiles_before >> 32};
#pragma unroll
  for (int k = 0; k < kTailKinds; ++k) kinds[k + 1] = kinds[k] + (tails_before >> (16 * k) & 0xffff);
  for (int64_t g = tid; g < G; g += kPrepThreads) {
    const int32_t end = p.row[g + 1], rows = end - p.row[g];
    const int kind = tail_kind(rows >= p.tensor_rows ? 0 : rows % kSmallTile);
#pragma unroll
    for (int k = 0; k < kTailKinds; ++k)
      if (kind == k) put_tail(p, g, end, rows % kSmallTile, kinds[k] + p.order[g]);
  }
  if (tid == 0) p.small_start[G + 1] = static_cast<int32_t>(kinds[kTailKinds]);
}

// The same for at most kFewGroups, by one warp's shuffles (3.6 us instead of 5.3).
constexpr int kFewGroups = 32;
constexpr int kPrepFewThreads = 128;

__device__ __forceinline__ void prep_few(const int32_t* __restrict__ sizes, int64_t G, int64_t M,
                                         int64_t begin, int64_t end, const RaggedPlan& p) {
  const int lane = threadIdx.x;
  if (lane < 32) {
    const int64_t n = lane < G && sizes[lane] > 0 ? sizes[lane] : 0;
    auto before = [&](int64_t v) {
      int64_t x = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      return x - v;
    };
    const GroupShape x = shape_of(before(n), n, M, begin, end, p);
    const int64_t both = before(static_cast<int64_t>(x.full) << 32 | x.tensor);
    const uint32_t earlier = (1u << lane) - 1u;
    const int slot = __popc(__ballot_sync(0xffffffffu, x.large) & earlier);
    if (lane < G) put_group(p, lane, x, both >> 32, both & 0xffffffff, slot);
    if (p.small) {
      int at = __shfl_sync(0xffffffffu, static_cast<int>(both >> 32) + x.full, 31);
      const int kind = tail_kind(x.tail);
#pragma unroll
      for (int k = 0; k < kTailKinds; ++k) {
        const uint32_t same = __ballot_sync(0xffffffffu, kind == k);
        if (kind == k) put_tail(p, lane, x.end, x.tail, at + __popc(same & earlier));
        at += __popc(same);
      }
      if (lane == 0) p.small_start[G + 1] = at;
    }
    if (G == 0 && lane == 0) p.row[0] = p.small_start[0] = p.tensor_start[0] = p.slot[0] = 0;
  }
  __syncthreads();
  put_tables(p, G, threadIdx.x, blockDim.x);
}

__global__ void __launch_bounds__(kPrepFewThreads)
prep_few_kernel(const int32_t* __restrict__ sizes, int64_t G, int64_t M, int64_t begin,
                int64_t end, RaggedPlan p) {
  wait_previous_grid();
  prep_few(sizes, G, M, begin, end, p);
}

// ---- small groups: FP64 matrix instructions ---------------------------------------

constexpr int kThreads = 256;
constexpr int kTN = 64;      // columns of a tile
constexpr int kKS = 32;      // contraction per pipeline stage
// Row pitches of the staged tiles, in values: 4 (mod 16) puts the 4 x 4
// values that half a warp reads for a fragment in 16 different 8-byte banks.
constexpr int kPitchK = kKS + 4;         // [row or column][k]
constexpr int kPitchN = kSmallTile + 4;  // [k][row or column]

// Values of a staged operand of up to `rows` rows or columns.
__host__ __device__ constexpr int operand_values(int rows) {
  return rows * kPitchK > kKS * kPitchN && rows == kSmallTile ? rows * kPitchK
         : rows == kSmallTile                                  ? kKS * kPitchN
                                                               : rows * kPitchK;
}
constexpr int kOperandB = operand_values(kTN);

// Stages in flight: two blocks per SM share 227 KB.  With A tiles of at most 16
// rows a fourth one fits.
template <int kRows>
struct Stages {
  static constexpr int kCount = kRows == kSmallTile ? 3 : 4;
  static constexpr int kOperandA = operand_values(kRows);
  static constexpr int kStride = kOperandA + kOperandB;
  static constexpr size_t kBytes = sizeof(double) * kCount * kStride;
};

// The first n bytes from src, zeros for the rest of kBytes.
template <int kBytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src, int n) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
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

// The same of a 16 x 8 and an 8 x 8 fragment: a[8 (i % 2) + l / 4][4 (i / 2) +
// l % 4], b[4 i + l % 4][l / 4], d[8 (i / 2) + l / 4][2 (l % 4) + i % 2].
__device__ __forceinline__ void mma_f64_wide(double (&d0)[2], double (&d1)[2],
                                             const double (&a)[4], const double (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f64.f64.f64.f64 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+d"(d0[0]), "+d"(d0[1]), "+d"(d1[0]), "+d"(d1[1])
      : "d"(a[0]), "d"(a[1]), "d"(a[2]), "d"(a[3]), "d"(b[0]), "d"(b[1]));
}

// A staged operand: f64 values, or (kPair) the hi words and, kOperand of them
// further on, the lo words.
template <bool kPair, int kOperand>
__device__ __forceinline__ double staged(const double* tile, int at) {
  if constexpr (kPair) {
    const float* f = reinterpret_cast<const float*>(tile);
    return __dadd_rn(static_cast<double>(f[at]), static_cast<double>(f[kOperand + at]));
  } else {
    return tile[at];
  }
}

// One operand's part of a stage: `lines` lines of `len` consecutive values,
// line t at offset origin + t stride of the operand.
struct Block2d {
  int64_t origin, stride;
  int lines, len;
};

// f64 lines move in 16-byte words wherever they start: a line whose first value
// lies off the 16-byte boundary is staged one place later (odd_start), its first
// and last value moved alone.
__device__ __forceinline__ int odd_start(const DotOperand& o, int64_t origin, int64_t stride,
                                         int line) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(o.f64) >> 3) + origin + line * stride) & 1;
}

// `lines_pad` lines of kLen values of the block into a staged tile (kPitch values
// per line), zeros outside it.
template <int kLen, int kPitch>
__device__ __forceinline__ void stage_f64(const DotOperand& o, const Block2d& b, int lines_pad,
                                          double* tile) {
  constexpr int kWords = kLen / 2, kStep = kThreads / kWords;  // lines at once (even)
  const int c = threadIdx.x % kWords, l0 = threadIdx.x / kWords;
  const int odd = odd_start(o, b.origin, b.stride, l0);
  const int first = 2 * c - odd, left = b.len - first;
  const double* src = o.f64 + b.origin + l0 * b.stride + first;
  double* dst = tile + l0 * kPitch + 2 * c;
  if (first < 0) {  // the first value, and the last one
    const bool last = kLen - 1 < b.len;
#pragma unroll 4
    for (int line = l0; line < lines_pad; line += kStep) {
      const bool in = line < b.lines && b.len > 0;
      copy_async<8>(dst + 1, in ? src + 1 : o.f64, in ? 8 : 0);
      copy_async<8>(dst + kLen, in && last ? src + kLen : o.f64, in && last ? 8 : 0);
      src += kStep * b.stride;
      dst += kStep * kPitch;
    }
    return;
  }
  const int bytes = left >= 2 ? 16 : left == 1 ? 8 : 0;
#pragma unroll 4
  for (int line = l0; line < lines_pad; line += kStep) {
    const int n = line < b.lines ? bytes : 0;
    copy_async<16>(dst, n ? src : o.f64 - odd_start(o, 0, 0, 0), n);
    src += kStep * b.stride;
    dst += kStep * kPitch;
  }
}

// The same of DS pairs, kVec of them per copy.
template <int kLen, int kPitch, int kVec, int kOperand>
__device__ __forceinline__ void stage_pairs(const DotOperand& o, const Block2d& b, int lines_pad,
                                            double* tile) {
  constexpr int kWords = kLen / kVec, kStep = kThreads / kWords;
  const int at = threadIdx.x % kWords * kVec;
  float* f = reinterpret_cast<float*>(tile);
#pragma unroll 4
  for (int line = threadIdx.x / kWords; line < lines_pad; line += kStep) {
    const bool in = line < b.lines && at < b.len;  // kVec divides len
    const int64_t src = in ? b.origin + line * b.stride + at : 0;
    const int n = in ? 4 * kVec : 0;
    copy_async<4 * kVec>(f + line * kPitch + at, o.hi + src, n);
    copy_async<4 * kVec>(f + kOperand + line * kPitch + at, o.lo + src, n);
  }
}

template <bool kPair, int kLen, int kPitch, int kOperand>
__device__ __forceinline__ void stage_block(const DotOperand& o, const Block2d& b, int lines_pad,
                                            double* tile, int vec) {
  if constexpr (!kPair) {
    stage_f64<kLen, kPitch>(o, b, lines_pad, tile);
  } else {
    if (vec > 1) stage_pairs<kLen, kPitch, 4, kOperand>(o, b, lines_pad, tile);
    else stage_pairs<kLen, kPitch, 1, kOperand>(o, b, lines_pad, tile);
  }
}

// A thread's word of each line of an f64 operand through a unit: where it is, and
// how it moves in a stage with all its contraction.  Lines are positions of the
// contraction (kLinesK: [k][row]) or rows ([row][k]); values past the operand's
// rows or columns are not staged, since their products are not stored.
template <int kLen, int kPitch, bool kLinesK>
struct Words {
  static constexpr int kWords = kLen / 2, kStep = kThreads / kWords;
  const double* src;  // of this stage
  int bytes;          // 16; 8: half a word; 0: none; -1: the first and last value

  // From `origin` on; len: rows or columns when they run along the lines.
  __device__ __forceinline__ void start(const DotOperand& o, int64_t origin, int64_t stride,
                                        int len) {
    const int c = threadIdx.x % kWords, l0 = threadIdx.x / kWords;
    const int odd = odd_start(o, origin, stride, l0), first = 2 * c - odd;
    const int left = (kLinesK ? len : kLen) - first;
    src = o.f64 + origin + l0 * stride + first;
    bytes = first < 0 ? -1 : left >= 2 ? 16 : left == 1 ? 8 : 0;
  }

  // One stage of `lines` lines.  kLinesK: zeros in the lines up to kKS; else the
  // stage has all its contraction.
  __device__ __forceinline__ void stage(const DotOperand& o, double* tile, int64_t stride,
                                        int lines, int len) const {
    if (bytes == 0) return;
    const int l0 = threadIdx.x / kWords;
    double* dst = tile + l0 * kPitch + threadIdx.x % kWords * 2;
    const double* p = src;
    const int64_t step = kStep * stride;
    constexpr int kPasses = (kLinesK ? kKS : kSmallTile) / kStep;
    if (kLinesK && lines < kKS) {
      const double* none = o.f64 - odd_start(o, 0, 0, 0);  // nothing is read from it
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const bool in = l0 + i * kStep < lines;
        if (bytes > 0) {
          copy_async<16>(dst, in ? p : none, in ? bytes : 0);
        } else {
          copy_async<8>(dst + 1, in ? p + 1 : none, in ? 8 : 0);
          if (kLen - 1 < len) copy_async<8>(dst + kLen, in ? p + kLen : none, in ? 8 : 0);
        }
        p += step;
        dst += kStep * kPitch;
      }
      return;
    }
    if (bytes == 16) {
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        if (!kLinesK && l0 + i * kStep >= lines) break;
        copy_async<16>(dst + i * kStep * kPitch, p, 16);
        p += step;
      }
      return;
    }
    const bool last = !kLinesK || kLen - 1 < len;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if (!kLinesK && l0 + i * kStep >= lines) break;
      if (bytes == 8) {
        copy_async<16>(dst + i * kStep * kPitch, p, 8);
      } else {
        copy_async<8>(dst + i * kStep * kPitch + 1, p + 1, 8);
        if (last) copy_async<8>(dst + i * kStep * kPitch + kLen, p + kLen, 8);
      }
      p += step;
    }
  }
};

struct SmallArgs {
  RaggedProblem q;
  RaggedPlan p;
  bool contract;
  bool add;          // contraction: add to the result (a later window of rows)
  uint32_t tiles_k;  // contraction: tiles of the result's rows
  uint32_t tiles_n;
  uint32_t splits;   // of the contraction (products only)
  int64_t split_k;
  double* partial;   // [splits][M][N]
  int vec_a, vec_b;  // DS pairs per copy
  bool own_plan;     // each block makes the plan (of at most kFewGroups) for itself
};

// A block's own plan: of calls without large groups and with few tiles, which are
// short enough for the launch before them to count ([16] x [16, 1024, 2048]: 35 us
// with prep_few_kernel, 32.5 without).
constexpr int kOwnTiles = 96;

struct OwnPlan {
  int32_t row[kFewGroups + 1], small_start[kFewGroups + 2], tensor_start[kFewGroups + 1];
  int32_t slot[kFewGroups + 1], order[kFewGroups];
  RaggedTile small[kOwnTiles];
};

__device__ __forceinline__ void make_own_plan(const SmallArgs& a, OwnPlan& own) {
  RaggedPlan p = a.p;
  p.row = own.row;
  p.small_start = own.small_start;
  p.tensor_start = own.tensor_start;
  p.slot = own.slot;
  p.order = own.order;
  p.small = a.contract ? nullptr : own.small;
  prep_few(a.q.group_sizes, a.q.G, a.q.M, 0, a.q.M, p);
  __syncthreads();
  // small_sum_kernel asks for the last group's end
  if (blockIdx.x == 0 && threadIdx.x == 0) a.p.row[a.q.G] = own.row[a.q.G];
}

// A unit of work: an output tile over a range of the contraction.
struct SmallUnit {
  int g, rows, cols;
  int64_t row, col;  // first output row (of the call, or of the group's matrix) and column
  int64_t k0, k1;    // contraction range (contraction: rows of the call)
  int split;
};

__device__ __forceinline__ uint32_t units_of(const SmallArgs& a, const OwnPlan& own) {
  if (a.contract) return static_cast<uint32_t>(a.q.G) * a.tiles_k * a.tiles_n;
  const int tiles = (a.own_plan ? own.small_start : a.p.small_start)[a.q.G + 1];
  return static_cast<uint32_t>(tiles) * a.tiles_n * a.splits;
}

// False for a unit that belongs to the tensor-core product, or that adds
// nothing.
__device__ __forceinline__ bool unit_at(const SmallArgs& a, const OwnPlan& own, uint32_t u,
                                        SmallUnit& x) {
  if (a.contract) {
    const uint32_t per = a.tiles_k * a.tiles_n, at = u / per, r = u - at * per;
    const uint32_t tk = r / a.tiles_n, g = (a.own_plan ? own.order : a.p.order)[at];
    const int32_t* rows = (a.own_plan ? own.row : a.p.row) + g;
    x.g = static_cast<int>(g);
    x.row = static_cast<int64_t>(tk) * kSmallTile;
    x.col = static_cast<int64_t>(r - tk * a.tiles_n) * kTN;
    x.k0 = rows[0];
    x.k1 = rows[1];
    x.rows = a.q.K - x.row < kSmallTile ? static_cast<int>(a.q.K - x.row) : kSmallTile;
    x.split = 0;
    if (x.k1 - x.k0 >= a.p.tensor_rows || (a.add && x.k1 == x.k0)) return false;
  } else {
    const uint32_t per = a.tiles_n * a.splits, at = u / per, r = u - at * per, tn = r / a.splits;
    const RaggedTile t = (a.own_plan ? own.small : a.p.small)[at];
    x.g = t.group;
    x.row = t.row;
    x.rows = t.rows;
    x.split = static_cast<int>(r - tn * a.splits);
    x.col = static_cast<int64_t>(tn) * kTN;
    x.k0 = x.split * a.split_k;
    x.k1 = x.k0 + a.split_k < a.q.K ? x.k0 + a.split_k : a.q.K;
  }
  x.cols = a.q.N - x.col < kTN ? static_cast<int>(a.q.N - x.col) : kTN;
  return true;
}

// First value of each operand at contraction position k.
__device__ __forceinline__ int64_t origin_a(const SmallArgs& a, const SmallUnit& x, int64_t k) {
  return x.row * a.q.lhs.s_r + k * a.q.lhs.s_k;
}
__device__ __forceinline__ int64_t origin_b(const SmallArgs& a, const SmallUnit& x, int64_t k) {
  return (a.contract ? 0 : x.g * a.q.rhs.s_b) + x.col * a.q.rhs.s_r + k * a.q.rhs.s_k;
}

// kA: A is staged as [k][row] (its rows are contiguous) rather than [row][k];
// kB: B as [k][column] rather than [column][k].
template <bool kPair, bool kA, bool kB, int kRows>
__device__ __forceinline__ void stage_unit(const SmallArgs& a, const SmallUnit& x, int64_t k,
                                           double* sa, double* sb) {
  const int kn = x.k1 - k < kKS ? static_cast<int>(x.k1 - k) : kKS;
  const DotOperand &A = a.q.lhs, &B = a.q.rhs;
  const int64_t oa = origin_a(a, x, k), ob = origin_b(a, x, k);
  constexpr int kOperandA = Stages<kRows>::kOperandA;
  if constexpr (kA) {
    stage_block<kPair, kSmallTile, kPitchN, kOperandA>(A, Block2d{oa, A.s_k, kn, x.rows}, kKS, sa,
                                                       a.vec_a);
  } else {
    const int pad = x.rows <= 16 ? 16 : x.rows <= 32 ? 32 : kSmallTile;
    stage_block<kPair, kKS, kPitchK, kOperandA>(A, Block2d{oa, A.s_r, x.rows, kn}, pad, sa,
                                                a.vec_a);
  }
  if constexpr (kB)
    stage_block<kPair, kTN, kPitchN, kOperandB>(B, Block2d{ob, B.s_k, kn, x.cols}, kKS, sb,
                                                a.vec_b);
  else
    stage_block<kPair, kKS, kPitchK, kOperandB>(B, Block2d{ob, B.s_r, x.cols, kn}, kTN, sb,
                                                a.vec_b);
}

// The products of one stage: warps stand kWM x (8 / kWM), each with MF x NF
// 8 x 8 accumulators.  odd_a, odd_b: where this lane's lines of A and B start
// (odd_start; the same for all its lines, which are an even number apart).
template <bool kFull, bool kPair, bool kA, bool kB, int kRows, int MF, int NF, int kWM>
__device__ __forceinline__ void multiply_part(const double* sa, const double* sb, int kn, int odd_a,
                                              int odd_b, double (&acc)[4][2][2]) {
  constexpr int kOperandA = Stages<kRows>::kOperandA;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % kWM * MF * 8, wn = warp / kWM * NF * 8;
  const int r = lane >> 2, kk = lane & 3;
  const int ia = odd_a + (kA ? kk * kPitchN + wm + r : (wm + r) * kPitchK + kk);
  const int ib = odd_b + (kB ? kk * kPitchN + wn + r : (wn + r) * kPitchK + kk);
  auto value_a = [&](int i, int k) {
    return staged<kPair, kOperandA>(sa, ia + (kA ? k * kPitchN + i * 8 : i * 8 * kPitchK + k));
  };
  auto value_b = [&](int j, int k) {
    return staged<kPair, kOperandB>(sb, ib + (kB ? k * kPitchN + j * 8 : j * 8 * kPitchK + k));
  };
  if constexpr (MF == 1) {
    // one accumulator would chain the instructions: four take turns, added up
    // at the end (finish_few)
#pragma unroll
    for (int k = 0; k < kKS; k += 4) {
      if (!kFull && k >= kn) break;
      mma_f64(acc[k / 4 % 4][0], value_a(0, k), value_b(0, k));
    }
  } else {
#pragma unroll
    for (int k = 0; k < kKS; k += 8) {
      if (!kFull && k >= kn) break;
      double fa[MF / 2][4], fb[NF][2];
#pragma unroll
      for (int i = 0; i < MF / 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) fa[i][e] = value_a(2 * i + e % 2, k + 4 * (e / 2));
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) fb[j][e] = value_b(j, k + 4 * e);
      if constexpr (MF == 2 && NF == 1) {
        constexpr int kTurn = 8;
        mma_f64_wide(acc[2 * (k / kTurn % 2)][0], acc[2 * (k / kTurn % 2) + 1][0], fa[0], fb[0]);
      } else {
#pragma unroll
        for (int i = 0; i < MF / 2; ++i)
#pragma unroll
          for (int j = 0; j < NF; ++j)
            mma_f64_wide(acc[2 * i][j], acc[2 * i + 1][j], fa[i], fb[j]);
      }
    }
  }
}

template <bool kPair, bool kA, bool kB, int kRows, int MF, int NF, int kWM>
__device__ __forceinline__ void multiply_stage(const double* sa, const double* sb, int kn,
                                               int odd_a, int odd_b, double (&acc)[4][2][2]) {
  if (kn == kKS)
    multiply_part<true, kPair, kA, kB, kRows, MF, NF, kWM>(sa, sb, kn, odd_a, odd_b, acc);
  else
    multiply_part<false, kPair, kA, kB, kRows, MF, NF, kWM>(sa, sb, kn, odd_a, odd_b, acc);
}

// The accumulators that took turns, added up in order.
template <int MF>
__device__ __forceinline__ void finish_few(double (&acc)[4][2][2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (MF == 1) {
      acc[0][0][h] = __dadd_rn(__dadd_rn(acc[0][0][h], acc[1][0][h]),
                               __dadd_rn(acc[2][0][h], acc[3][0][h]));
    } else {
      acc[0][0][h] = __dadd_rn(acc[0][0][h], acc[2][0][h]);
      acc[1][0][h] = __dadd_rn(acc[1][0][h], acc[3][0][h]);
    }
  }
}

template <int MF, int NF, int kWM>
__device__ __forceinline__ void store_unit(const SmallArgs& a, const SmallUnit& x,
                                           const double (&acc)[4][2][2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = warp % kWM * MF * 8 + (lane >> 2), c0 = warp / kWM * NF * 8 + 2 * (lane & 3);
  const int64_t N = a.q.N, first = (a.contract ? x.g * a.q.K : 0) + x.row;
  DotResult out = a.q.out;
  if (a.splits > 1) out = DotResult{a.partial + x.split * a.q.M * N, nullptr, nullptr};
  int64_t at = (first + r0) * N + x.col + c0;
  if (out.f64 && !a.add) {
    const bool words = (N & 1) == 0 && (reinterpret_cast<uintptr_t>(out.f64) & 15) == 0;
    double* p = out.f64 + at;
#pragma unroll
    for (int i = 0; i < MF; ++i, p += 8 * N) {
      if (r0 + i * 8 >= x.rows) break;
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const int left = x.cols - c0 - j * 8;
        if (words && left >= 2) {
          *reinterpret_cast<double2*>(p + j * 8) = make_double2(acc[i][j][0], acc[i][j][1]);
        } else {
          if (left > 0) p[j * 8] = acc[i][j][0];
          if (left > 1) p[j * 8 + 1] = acc[i][j][1];
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < MF; ++i, at += 8 * N) {
    if (r0 + i * 8 >= x.rows) break;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (c0 + j * 8 + h >= x.cols) continue;
        double v = acc[i][j][h];
        if (a.add) v = __dadd_rn(result_value(out, at + j * 8 + h), v);
        put(out, at + j * 8 + h, v);
      }
    }
  }
}

constexpr uint32_t kNoUnit = 0xffffffffu;

// Blocks stay and share the units out; the pipeline of stages runs on across
// units.  kRows: most rows of a tile.
template <bool kPair, bool kA, bool kB, int kRows>
__global__ void __launch_bounds__(kThreads, 2)
small_kernel(const __grid_constant__ SmallArgs a) {
  using St = Stages<kRows>;
  extern __shared__ __align__(16) double stage[];
  __shared__ OwnPlan own;
  wait_previous_grid();
  if (a.own_plan) make_own_plan(a, own);
  // rows behind the last group
  if (!a.contract) {
    const int64_t end = a.q.M * a.q.N;
    for (int64_t i = (a.own_plan ? own.row : a.p.row)[a.q.G] * a.q.N + static_cast<int64_t>(blockIdx.x) * kThreads +
                     threadIdx.x;
         i < end; i += static_cast<int64_t>(gridDim.x) * kThreads)
      put(a.q.out, i, 0.0);
  }
  const uint32_t units = units_of(a, own);
  // the block's units: every gridDim.x-th.  They fall in size and are taken there
  // and back, so that every block gets about as much
  auto unit_number = [&](uint32_t step) {
    return step * gridDim.x + (step & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  };
  auto next_unit = [&](uint32_t step, SmallUnit& x) {
    while (step * gridDim.x < units) {
      const uint32_t u = unit_number(step);
      if (u < units && unit_at(a, own, u, x)) return step;
      ++step;
    }
    return kNoUnit;
  };
  // loading runs kCount - 1 stages ahead of multiplying
  const DotOperand &A = a.q.lhs, &B = a.q.rhs;
  const int64_t line_a = kA ? A.s_k : A.s_r, line_b = kB ? B.s_k : B.s_r;
  Words<kA ? kSmallTile : kKS, kA ? kPitchN : kPitchK, kA> wa;
  Words<kB ? kTN : kKS, kB ? kPitchN : kPitchK, kB> wb;
  SmallUnit lx, x;
  uint32_t lu = 0;
  int64_t lk = 0;
  auto start_unit = [&](uint32_t step) {
    lu = next_unit(step, lx);
    if (lu == kNoUnit) return;
    lk = lx.k0;
    if constexpr (!kPair) {
      wa.start(A, origin_a(a, lx, lk), line_a, lx.rows);
      wb.start(B, origin_b(a, lx, lk), line_b, lx.cols);
    }
  };
  start_unit(0);
  int ls = 0;
  auto load_one = [&] {
    if (lu != kNoUnit) {
      double* sa = stage + ls * St::kStride;
      double* sb = sa + St::kOperandA;
      const int64_t left = lx.k1 - lk;
      if (!kPair && (left >= kKS || (kA && kB && left > 0))) {
        const int kn = left < kKS ? static_cast<int>(left) : kKS;
        wa.stage(A, sa, line_a, kA ? kn : lx.rows, lx.rows);
        wb.stage(B, sb, line_b, kB ? kn : lx.cols, lx.cols);
      } else if (left > 0) {
        stage_unit<kPair, kA, kB, kRows>(a, lx, lk, sa, sb);
      }
      lk += kKS;
      if (lk >= lx.k1) {
        start_unit(lu + 1);
      } else if constexpr (!kPair) {
        wa.src += kKS * A.s_k;
        wb.src += kKS * B.s_k;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ls = ls + 1 == St::kCount ? 0 : ls + 1;
  };
#pragma unroll 1
  for (int i = 0; i < St::kCount - 1; ++i) load_one();
  int cs = 0;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (uint32_t u = next_unit(0, x); u != kNoUnit; u = next_unit(u + 1, x)) {
    double acc[4][2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j][0] = acc[i][j][1] = 0.0;
    int odd_a = 0, odd_b = 0;
    if constexpr (!kPair) {
      odd_a = kA ? odd_start(a.q.lhs, origin_a(a, x, x.k0), a.q.lhs.s_k, lane & 3)
                 : odd_start(a.q.lhs, origin_a(a, x, x.k0), a.q.lhs.s_r, lane >> 2);
      odd_b = kB ? odd_start(a.q.rhs, origin_b(a, x, x.k0), a.q.rhs.s_k, lane & 3)
                 : odd_start(a.q.rhs, origin_b(a, x, x.k0), a.q.rhs.s_r, lane >> 2);
    }
    int64_t k = x.k0;
    do {  // a unit without contraction takes one (empty) stage
      asm volatile("cp.async.wait_group %0;" ::"n"(St::kCount - 2) : "memory");
      __syncthreads();
      const double* sa = stage + cs * St::kStride;
      const double* sb = sa + St::kOperandA;
      const int kn = x.k1 - k < kKS ? static_cast<int>(x.k1 - k) : kKS;
      load_one();
      if (x.rows <= 8)
        multiply_stage<kPair, kA, kB, kRows, 1, 1, 1>(sa, sb, kn, odd_a, odd_b, acc);
      else if (kRows == 16 || x.rows <= 16)
        multiply_stage<kPair, kA, kB, kRows, 2, 1, 1>(sa, sb, kn, odd_a, odd_b, acc);
      else if (x.rows <= 32)
        multiply_stage<kPair, kA, kB, kRows, 2, 2, 2>(sa, sb, kn, odd_a, odd_b, acc);
      else
        multiply_stage<kPair, kA, kB, kRows, 4, 2, 2>(sa, sb, kn, odd_a, odd_b, acc);
      cs = cs + 1 == St::kCount ? 0 : cs + 1;
      k += kKS;
    } while (k < x.k1);
    if (x.rows <= 8) {
      finish_few<1>(acc);
      store_unit<1, 1, 1>(a, x, acc);
    } else if (kRows == 16 || x.rows <= 16) {
      finish_few<2>(acc);
      store_unit<2, 1, 1>(a, x, acc);
    } else if (x.rows <= 32) store_unit<2, 2, 2>(a, x, acc);
    else store_unit<4, 2, 2>(a, x, acc);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The splits of every small tile (blockIdx.y) added up in order; where the blocks
// made the plan themselves all rows are small groups' and blockIdx.y stands for
// kSmallTile of them.
__global__ void __launch_bounds__(kThreads)
small_sum_kernel(const __grid_constant__ SmallArgs a) {
  wait_previous_grid();
  RaggedTile t;
  if (a.own_plan) {
    t.row = static_cast<int>(blockIdx.y) * kSmallTile;
    t.rows = a.p.row[a.q.G] - t.row;
    t.rows = t.rows < kSmallTile ? t.rows : kSmallTile;
  } else {
    if (static_cast<int>(blockIdx.y) >= a.p.small_start[a.q.G + 1]) return;
    t = a.p.small[blockIdx.y];
  }
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= a.q.N) return;
  const int64_t plane = a.q.M * a.q.N;
  for (int r = blockIdx.z; r < t.rows; r += gridDim.z) {
    const int64_t at = (t.row + r) * a.q.N + c;
    double v = 0.0;
#pragma unroll 4
    for (uint32_t s = 0; s < a.splits; ++s) v = __dadd_rn(v, __ldcg(a.partial + s * plane + at));
    put(a.q.out, at, v);
  }
}

// ---- host ------------------------------------------------------------------------

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Contraction splits of the products: where the tiles are few, units of at least
// kSplitMin of the contraction, enough of them to share out evenly among the
// resident blocks (more when no tile has over 16 rows: those only stream the
// matrices).  From the call's sizes alone, so a row's rounding does not depend
// on other groups.
constexpr int64_t kSplitMin = 256;
constexpr int kMaxSplits = 16;

int splits_of(int64_t M, int64_t K, int64_t N, int64_t G) {
  const int64_t units = M <= 16 ? 2400 : 600;
  const int64_t tiles = (M / kSmallTile + (G < M ? G : M)) * ceil_div(N, kTN);
  if (tiles == 0 || tiles >= units) return 1;
  int64_t s = ceil_div(units, tiles);
  const int64_t most = K / kSplitMin;
  s = s > most ? most : s;
  s = s > kMaxSplits ? kMaxSplits : s;
  return s < 1 ? 1 : static_cast<int>(s);
}

// Whether the tensor-core product takes the large groups: where its estimated
// time is below the FP64 path's.  In microseconds, from measurements on one B200:
// the FP64 path takes 9 us and does 26 TFLOP/s; the tensor-core product has
// launches of 60 us (50 with K-contiguous matrices) for each 32768 of K, as a
// contraction 80, splits a value in 5 to 7.2 ps, multiplies at 3 POPS of its 28
// operations per product but takes at least 0.76 us per 256 x 256 outputs (short
// contractions), and rebuilds an output in 5.5 ps; a matrix counts with whole tiles
// of 256 columns.  Measured with / without: 2048 x 1024 x 1024 in 4 groups 132 /
// 190 us (contraction 173 / 169), 4096 x 1024 x 1024 in 8 groups 208 / 333 (232 / 318),
// 2048 x 2048 x 2048 in 4 groups 286 / 646 (368 / 624), 8192 x 512 x 512 in 8 groups
// 175 / 177 (159 / 183), 1024 x 1024 x 1024 in one 90 / 106 (128 / 97), 4096 x 256 x
// 2048 in 4 groups 208 / 173 (177 / 183), 494 x 1910 x 1292 in one 109 / 104
// (K-contiguous 91 / 105), 700 x 33041 x 300 in 3 groups 966 / 630, 33041 rows of 300
// x 400 contracted in 2 groups 608 / 788, in 5 545 / 550.
bool tensor_allowed(int64_t M, int64_t K, int64_t N, int64_t G, bool contract, bool rhs_t) {
  if (G < 1 || M < tensor_rows(contract) || K < 64 || N < 64) return false;
  const double m = M, k = K, n = N, slots = static_cast<double>(ragged_slots(M, G, contract));
  const double macs = m * k * n, matrices = slots * k * n, outputs = contract ? matrices : m * n;
  const double padded = static_cast<double>(ceil_div(N, 256) * 256) / n;
  const double plain = 9 + 7.7e-8 * macs;
  const double chunks = static_cast<double>(ceil_div(K, kRaggedWindow));
  const double launches = contract ? 80 : (rhs_t ? 50 : 60) * chunks;
  const double split =
      contract ? 6.5e-6 * m * (k + n)
               : 5.5e-6 * m * k + (rhs_t ? 5e-6 : 7.2e-6) * matrices * padded;
  const double gemm = 9.3e-9 * macs * padded, least = 1.15e-5 * outputs;
  const double tensor = launches + split + (gemm > least ? gemm : least) + 5.5e-6 * outputs;
  return tensor < plain && ragged_tensor_fits(M, K, N, G, contract);
}

struct Layout {
  size_t row, small_start, tensor_start, slot, order, small, tensor, slot_group, slot_bits, partial, tensor_ws, total;
  int64_t small_cap, tensor_cap, slots;
  int splits;
  bool tensor_ok;
};

Layout layout_of(const RaggedProblem& q, bool contract) {
  const int64_t M = q.M, K = q.K, N = q.N, G = q.G;
  Layout l{};
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at = (at + bytes + 1023) / 1024 * 1024;
    return here;
  };
  const int64_t groups = G < M ? G : M;  // with rows
  l.tensor_ok = q.tensor && tensor_allowed(M, K, N, G, contract, q.rhs_t);
  l.small_cap = contract ? 0 : M / kSmallTile + groups;
  if (l.tensor_ok) {
    const int64_t rows = contract && M > kRaggedWindow ? kRaggedWindow : M;
    l.slots = ragged_slots(rows, G, contract);
    l.tensor_cap = ragged_tensor_tiles(rows, G, contract);
  }
  l.splits = contract ? 1 : splits_of(M, K, N, G);
  l.row = take((G + 1) * 4);
  l.small_start = take((G + 2) * 4);
  l.tensor_start = take((G + 1) * 4);
  l.slot = take((G + 1) * 4);
  l.order = take(G * 4);
  l.small = take(l.small_cap * sizeof(RaggedTile));
  l.tensor = take(l.tensor_cap * sizeof(RaggedTile));
  l.slot_group = take(l.slots * 4);
  l.slot_bits = take(l.slots * 4);
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

RaggedPlan plan_at(const Layout& l, int64_t G, bool contract, uint8_t* ws, bool tensor) {
  auto ints = [&](size_t off) { return reinterpret_cast<int32_t*>(ws + off); };
  RaggedPlan p{};
  p.groups = G;
  p.row = ints(l.row);
  p.small_start = ints(l.small_start);
  p.tensor_start = ints(l.tensor_start);
  p.slot = ints(l.slot);
  p.order = ints(l.order);
  p.small = contract ? nullptr : reinterpret_cast<RaggedTile*>(ws + l.small);
  p.tensor = l.tensor_cap ? reinterpret_cast<RaggedTile*>(ws + l.tensor) : nullptr;
  p.slot_group = ints(l.slot_group);
  p.slot_bits = ints(l.slot_bits);
  p.small_cap = l.small_cap;
  p.tensor_cap = l.tensor_cap;
  p.tensor_rows = tensor ? tensor_rows(contract) : INT32_MAX;
  if (tensor)
    for (int i = 0; i < kBitsLimits; ++i) p.bits_limit[i] = bits_limits()[i];
  return p;
}

// DS pairs per copy of an operand whose lines are `len` values long at a stride
// of `stride` values.
int copy_width(const DotOperand& o, int64_t len, int64_t stride, int64_t batch) {
  const bool at = aligned(o.hi, 16) && aligned(o.lo, 16);
  return at && len % 4 == 0 && stride % 4 == 0 && batch % 4 == 0 ? 4 : 1;
}

template <bool kPair, bool kA, bool kB, int kRows>
int launch_small(const SmallArgs& a, int64_t most_units, cudaStream_t s) {
  constexpr size_t kBytes = Stages<kRows>::kBytes;
  static std::mutex mu;
  static std::vector<bool> done;
  int dev = 0;
  DSB_CUDA_TRY(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= static_cast<int>(done.size())) done.resize(dev + 1, false);
    if (!done[dev]) {
      DSB_CUDA_TRY(cudaFuncSetAttribute(small_kernel<kPair, kA, kB, kRows>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(kBytes)));
      done[dev] = true;
    }
  }
  if (most_units > 0x7fffffff)
    return set_error(DS_INVALID_ARGUMENT, "ds_ragged_dot: too many output tiles");
  const int64_t resident = 2 * static_cast<int64_t>(sm_count());
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(most_units < resident ? (most_units < 1 ? 1 : most_units)
                                                                 : resident));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DSB_CUDA_TRY(cudaLaunchKernelEx(&cfg, small_kernel<kPair, kA, kB, kRows>, a));
  if (a.splits > 1) {
    const int64_t most = a.own_plan ? kSmallTile : 8, rows = a.q.M < most ? a.q.M : most;
    DSB_CUDA_TRY(launch_dependent(small_sum_kernel,
                                  dim3(static_cast<unsigned>(ceil_div(a.q.N, kThreads)),
                                       static_cast<unsigned>(
                                           a.own_plan ? ceil_div(a.q.M, kSmallTile) : a.p.small_cap),
                                       static_cast<unsigned>(rows)),
                                  dim3(kThreads), s, a));
  }
  return launch_status();
}

template <bool kB>
int launch_products(const SmallArgs& a, int64_t units, cudaStream_t s) {
  // no group has more rows than the call
  const bool few = a.q.M <= 16;
  if (a.q.lhs.f64)
    return few ? launch_small<false, false, kB, 16>(a, units, s)
               : launch_small<false, false, kB, kSmallTile>(a, units, s);
  return few ? launch_small<true, false, kB, 16>(a, units, s)
             : launch_small<true, false, kB, kSmallTile>(a, units, s);
}

int launch_prep(const RaggedProblem& q, int64_t begin, int64_t end, const RaggedPlan& p,
                cudaStream_t s) {
  if (q.G <= kFewGroups)
    DSB_CUDA_TRY(launch_dependent(prep_few_kernel, dim3(1), dim3(kPrepFewThreads), s,
                                  q.group_sizes, q.G, q.M, begin, end, p));
  else
    DSB_CUDA_TRY(launch_dependent(prep_kernel, dim3(1), dim3(kPrepThreads), s, q.group_sizes, q.G,
                                  q.M, begin, end, p));
  return launch_status();
}

}  // namespace

size_t ragged_dot_workspace_bytes(const RaggedProblem& q) { return layout_of(q, false).total; }

int ragged_dot(const RaggedProblem& q, void* workspace, size_t, cudaStream_t s) {
  if (q.M == 0 || q.N == 0) return ok();
  const Layout l = layout_of(q, false);
  int clusters = 0;
  if (l.tensor_ok)
    if (int st = ragged_tensor_clusters(&clusters)) return st;
  uint8_t* ws = align_ws(workspace);
  SmallArgs a{};
  a.q = q;
  a.p = plan_at(l, q.G, false, ws, clusters > 0);
  a.tiles_n = static_cast<uint32_t>(ceil_div(q.N, kTN));
  a.splits = static_cast<uint32_t>(l.splits);
  a.split_k = ceil_div(ceil_div(q.K, l.splits), kKS) * kKS;
  a.partial = reinterpret_cast<double*>(ws + l.partial);
  a.vec_a = copy_width(q.lhs, q.K, q.lhs.s_r, 0);
  a.vec_b = copy_width(q.rhs, q.rhs_t ? q.K : q.N, q.rhs_t ? q.rhs.s_r : q.rhs.s_k, q.rhs.s_b);
  a.own_plan = clusters == 0 && q.G <= kFewGroups && l.small_cap <= kOwnTiles;
  if (!a.own_plan)
    if (int st = launch_prep(q, 0, q.M, a.p, s)) return st;
  if (clusters > 0)
    if (int st = ragged_tensor_dot(q, a.p, ws + l.tensor_ws, clusters, s)) return st;
  ProfileScope prof("ragged_small", s);
  const int64_t units = l.small_cap * a.tiles_n * a.splits;
  return q.rhs_t ? launch_products<false>(a, units, s) : launch_products<true>(a, units, s);
}

size_t ragged_contract_workspace_bytes(const RaggedProblem& q) { return layout_of(q, true).total; }

int ragged_contract(const RaggedProblem& q, void* workspace, size_t, cudaStream_t s) {
  if (q.G == 0 || q.K == 0 || q.N == 0) return ok();
  const Layout l = layout_of(q, true);
  int clusters = 0;
  if (l.tensor_ok)
    if (int st = ragged_tensor_clusters(&clusters)) return st;
  uint8_t* ws = align_ws(workspace);
  SmallArgs a{};
  a.q = q;
  a.p = plan_at(l, q.G, true, ws, clusters > 0);
  a.contract = true;
  a.tiles_k = static_cast<uint32_t>(ceil_div(q.K, kSmallTile));
  a.tiles_n = static_cast<uint32_t>(ceil_div(q.N, kTN));
  a.splits = 1;
  a.vec_a = copy_width(q.lhs, q.K, q.lhs.s_k, 0);
  a.vec_b = copy_width(q.rhs, q.N, q.rhs.s_k, 0);
  a.own_plan = clusters == 0 && q.G <= kFewGroups;
  const int64_t units = q.G * a.tiles_k * a.tiles_n;
  // without the tensor-core product one window takes all rows
  const int64_t window = clusters > 0 ? kRaggedWindow : q.M + 1;
  for (int64_t begin = 0; begin == 0 || begin < q.M; begin += window) {
    a.add = begin > 0;
    if (!a.own_plan)
      if (int st = launch_prep(q, begin, begin + window, a.p, s)) return st;
    if (clusters > 0)
      if (int st = ragged_tensor_contract(q, a.p, a.add, ws + l.tensor_ws, clusters, s)) return st;
    ProfileScope prof("ragged_small", s);
    const int st = q.lhs.f64 == nullptr ? launch_small<true, true, true, kSmallTile>(a, units, s)
                                        : launch_small<false, true, true, kSmallTile>(a, units, s);
    if (st) return st;
  }
  return ok();
}

}  // namespace dsb
