// The large groups of the products grouped by expert on the int8 tcgen05
// tensor cores: the integer-residue product of dot_ozaki.cu (split, GEMM,
// reconstruction, certificate and recomputation, with their error bounds) with
// the groups' sizes read on the device.
//
// Products (rows of a group times its matrix): the rows keep their places in
// the planes of A, [14][M][K]; a tile of the GEMM starts at any row of its
// group and stores only the group's rows.  The matrices of the large groups
// take slots, [14][slots][K][N] (or [N][K]): the others' are not read.
//
// Contraction (rows of a group contracted): both operands are split into
// planes [14][positions][features] whose positions are the groups' rows, each
// group padded with zeros to whole tiles of 256, and read as MN-major operands;
// a unit of the GEMM runs over its group's tiles.  Every (group, feature) has
// its own scale, and every group the bits its own length allows.
//
// A contraction longer than 32768 runs in chunks whose results are added.
#include <mutex>
#include <string>
#include <vector>

#include "common.cuh"
#include "ds_arith.cuh"
#include "kernels.h"
#include "ozaki.cuh"
#include "profile.h"
#include "ragged.h"

namespace dsb {
namespace {

// The operand with its values moved by `off`.
__device__ __forceinline__ DotOperand moved(DotOperand o, int64_t off) {
  if (o.f64) {
    o.f64 += off;
  } else {
    o.hi += off;
    o.lo += off;
  }
  return o;
}

__device__ __forceinline__ int slots_of(const RaggedPlan& p) { return p.slot[p.groups]; }

// ---- split ---------------------------------------------------------------------

// Values k .. k + 7 of the row that starts at `base` (contiguous in k), zeros
// from K on.
__device__ __forceinline__ void load_8(const DotOperand& o, int64_t base, bool words, int64_t k,
                                       int64_t K, double (&v)[8]) {
  if (words && k + 8 <= K) {
    const double2* p = reinterpret_cast<const double2*>(o.f64 + base + k);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double2 d = __ldg(p + j);
      v[2 * j] = d.x;
      v[2 * j + 1] = d.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? op_value(o, base + k + j) : 0.0;
  }
}

// A row's largest magnitude (as high and, where that is 0, low word: its exponent
// is all that counts) and 1-norm.
struct RowStats {
  int high = 0;
  uint32_t low = 0;
  double sum = 0.0;
  __device__ __forceinline__ void add(const double (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int h = __double2hiint(v[j]) & 0x7fffffff;
      high = h > high ? h : high;
      low |= static_cast<uint32_t>(__double2loint(v[j]));
      sum += fabs(v[j]);
    }
  }
};

// One row into its planes by one block, eight values per thread, modulus and
// 8-byte store.  The first 2048 values stay in registers, later ones are read
// twice.
//
// Bound by the instructions of 14 residues per value (119 in all): 16.8 million
// values in rows of 2048 take 88 us (22 bytes per value, 4.2 TB/s).  With four
// values per thread and store, the maximum taken in f64 and all values read twice
// it was 109 us.  Blocks of eight rows that load the next one early keep the
// residues' constants in registers and spill: within 1% of this either way.
constexpr int kSplitThreads = 256;

__device__ __forceinline__ void split_row(const DotOperand& o, int64_t base, int64_t K, int64_t Kp,
                                          int P, uint8_t* __restrict__ out, size_t plane_stride,
                                          int* shift_to, float* part_to) {
  __shared__ int s_high[kSplitThreads / 32];
  __shared__ uint32_t s_low[kSplitThreads / 32];
  __shared__ double s_sum[kSplitThreads / 32];
  const bool words = o.f64 && (reinterpret_cast<uintptr_t>(o.f64 + base) & 15) == 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int64_t kStep = 8 * kSplitThreads;
  const int64_t first = 8 * static_cast<int64_t>(threadIdx.x);
  double v[8];
  load_8(o, base, words, first, K, v);
  RowStats stats;
  stats.add(v);
  for (int64_t k = first + kStep; k < K; k += kStep) {
    double w[8];
    load_8(o, base, words, k, K, w);
    stats.add(w);
  }
  int high = __reduce_max_sync(0xffffffffu, stats.high);
  uint32_t low = __reduce_or_sync(0xffffffffu, stats.low);
  double sum = stats.sum;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) {
    s_high[warp] = high;
    s_low[warp] = low;
    s_sum[warp] = sum;
  }
  __syncthreads();
  constexpr int kWarps = kSplitThreads / 32;
  high = __reduce_max_sync(0xffffffffu, s_high[lane % kWarps]);
  low = __reduce_or_sync(0xffffffffu, s_low[lane % kWarps]);
  const int shift = shift_for(__hiloint2double(high, high == 0 ? static_cast<int>(low) : 0),
                              high >= 0x7ff00000, P);
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < kWarps; ++w) sum += s_sum[w];
    *shift_to = shift;
    *part_to = certify_part(sum, shift, K);
  }
  const bool zero = !shift_ordinary(shift);
  const int sh = zero ? 0 : shift;
#pragma unroll 1
  for (int64_t k = first; k < Kp; k += kStep) {
    if (k != first) load_8(o, base, words, k, K, v);
    Limbs x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = limbs_of(quantise(zero ? 0.0 : v[j], sh));
    store_planes_n<8, true>(x, out + k, plane_stride);
  }
}

struct RowSplit {
  DotOperand o;
  int64_t K, Mp, Kp;
  int P;
  uint8_t* planes;
  int* shifts;
  int* row_slot;
  float* part;
};

// Rows of the large groups, one block each: blockIdx.y is the row in tile
// blockIdx.x.  (In one launch with the column maxima of the matrices, their
// blocks interleaved, it took as long as both.)
__global__ void __launch_bounds__(kSplitThreads, 4)
ragged_split_rows_kernel(RowSplit r, RaggedPlan p) {
  wait_previous_grid();
  if (static_cast<int>(blockIdx.x) >= p.tensor_start[p.groups]) return;
  const RaggedTile t = p.tensor[blockIdx.x];
  if (static_cast<int>(blockIdx.y) >= t.rows) return;
  const int64_t at = t.row + static_cast<int64_t>(blockIdx.y);
  if (threadIdx.x == 0) r.row_slot[at] = t.slot + 1;
  split_row(r.o, at * r.o.s_r, r.K, r.Kp, r.P, r.planes + at * r.Kp,
            static_cast<size_t>(r.Mp) * r.Kp, r.shifts + at, r.part + at);
}

// Matrices with K contiguous ([G, N, K]): column blockIdx.x of slot blockIdx.y.
__global__ void __launch_bounds__(kSplitThreads, 4)
ragged_split_matrix_rows_kernel(DotOperand o, int64_t K, int64_t Np, int64_t Kp, int64_t slots,
                                int P, RaggedPlan p, uint8_t* __restrict__ planes,
                                int* __restrict__ shifts, float* __restrict__ part) {
  wait_previous_grid();
  const int slot = blockIdx.y;
  if (slot >= slots_of(p)) return;
  const int64_t at = slot * Np + blockIdx.x;
  split_row(o, p.slot_group[slot] * o.s_b + blockIdx.x * o.s_r, K, Kp, P, planes + at * Kp,
            static_cast<size_t>(slots) * Np * Kp, shifts + at, part + at);
}

struct ColumnMax {
  DotOperand o;
  int64_t N, K, Np;
  int* codes;
  int* norms;
};

// Column maxima of the matrices ([G, K, N]): slot blockIdx.z.
__global__ void __launch_bounds__(256, 6)
ragged_colmax_kernel(ColumnMax c, RaggedPlan p) {
  wait_previous_grid();
  const int slot = blockIdx.z;
  if (slot >= slots_of(p)) return;
  DotOperand x = moved(c.o, p.slot_group[slot] * c.o.s_b);
  x.s_b = 0;
  colmax_body<true>(x, c.N, c.K, c.Np, c.codes, blockIdx.x, blockIdx.y, slot, c.norms);
}

// The same per group and feature of a contraction's operand: half blockIdx.y
// % 2 of tile blockIdx.y / 2.
__global__ void __launch_bounds__(256, 6)
ragged_tile_colmax_kernel(DotOperand o, int64_t F, int64_t Fp, RaggedPlan p,
                          int* __restrict__ codes, int* __restrict__ norms) {
  wait_previous_grid();
  const int tile = blockIdx.y >> 1;
  if (tile >= p.tensor_start[p.groups]) return;
  const RaggedTile t = p.tensor[tile];
  if (static_cast<int>(blockIdx.y & 1) * kColmaxSlab >= t.rows) return;
  const int64_t at = static_cast<int64_t>(t.slot) * Fp;
  colmax_body<true>(moved(o, t.row * o.s_k), F, t.rows, Fp, codes + at, blockIdx.x,
                    blockIdx.y & 1, 0, norms + at);
}

// DS pairs into row-contiguous planes, as split_mn_async_body does for f64:
// each thread takes kMnCols rows at k = blockIdx.y, + gridDim.y, ...
__device__ __forceinline__ void split_mn_pairs_body(const DotOperand& o, int64_t rows, int64_t K,
                                                    int64_t rows_pad, int64_t Kp, int P,
                                                    const int* __restrict__ codes,
                                                    uint8_t* __restrict__ planes,
                                                    size_t plane_stride, int* __restrict__ shifts) {
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kMnRows + threadIdx.x * kMnCols;
  if (r0 >= rows_pad) return;
  int sh[kMnCols];
  bool z[kMnCols];
#pragma unroll
  for (int j = 0; j < kMnCols; ++j) {
    const int64_t r = r0 + j;
    const int sv = r < rows ? shift_from_code(codes[r], P) : 0;
    if (blockIdx.y == 0) shifts[r] = sv;
    z[j] = r >= rows || !shift_ordinary(sv);
    sh[j] = z[j] ? 0 : sv;
  }
#pragma unroll 1
  for (int64_t k = blockIdx.y; k < Kp; k += gridDim.y) {
    Limbs x[kMnCols];
#pragma unroll
    for (int j = 0; j < kMnCols; ++j)
      x[j] = limbs_of(quantise(z[j] || k >= K ? 0.0 : op_value(o, (r0 + j) * o.s_r + k * o.s_k),
                               sh[j]));
    store_planes_n<kMnCols, true>(x, planes + static_cast<size_t>(k) * rows_pad + r0,
                                  plane_stride);
  }
}

template <bool kPair>
__device__ __forceinline__ void split_mn_body(const DotOperand& o, int64_t rows, int64_t K,
                                              int64_t rows_pad, int64_t Kp, int P,
                                              const int* codes, uint8_t* planes,
                                              size_t plane_stride, int* shifts) {
  if constexpr (kPair)
    split_mn_pairs_body(o, rows, K, rows_pad, Kp, P, codes, planes, plane_stride, shifts);
  else
    split_mn_async_body(o, 0, true, rows, K, rows_pad, Kp, P, codes, planes, plane_stride, shifts);
}

// Certificate parts of this thread's columns, from the column maxima's codes, by
// the blocks that start at k = 0.
__device__ __forceinline__ void column_parts(int64_t rows, int64_t rows_pad, int64_t K, int P,
                                             const int* __restrict__ codes,
                                             const int* __restrict__ norms,
                                             float* __restrict__ part) {
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kMnRows + threadIdx.x * kMnCols;
  if (blockIdx.y != 0 || r0 >= rows_pad) return;
  const double slabs = static_cast<double>((K + kColmaxSlab - 1) / kColmaxSlab);
#pragma unroll
  for (int j = 0; j < kMnCols; ++j) {
    const int64_t r = r0 + j;
    part[r] = r < rows ? certify_part(slabs * norm_of(norms[r]), shift_from_code(codes[r], P), K)
                       : 0.0f;
  }
}

// Matrices [G, K, N] into planes [14][slots][Kp][Np]: slot blockIdx.z.
template <bool kPair>
__global__ void __launch_bounds__(256, 2)
ragged_split_matrix_kernel(DotOperand o, int64_t N, int64_t K, int64_t Np, int64_t Kp,
                           int64_t slots, int P, RaggedPlan p, const int* __restrict__ codes,
                           const int* __restrict__ norms, uint8_t* __restrict__ planes,
                           int* __restrict__ shifts, float* __restrict__ part) {
  wait_previous_grid();
  const int64_t slot = blockIdx.z;
  if (slot >= slots_of(p)) return;
  column_parts(N, Np, K, P, codes + slot * Np, norms + slot * Np, part + slot * Np);
  split_mn_body<kPair>(moved(o, p.slot_group[slot] * o.s_b), N, K, Np, Kp, P, codes + slot * Np,
                       planes + static_cast<size_t>(slot) * Kp * Np,
                       static_cast<size_t>(slots) * Kp * Np, shifts + slot * Np);
}

// A contraction's operand into planes [14][positions][Fp]: tile blockIdx.z.
template <bool kPair>
__global__ void __launch_bounds__(256, 2)
ragged_split_tiles_kernel(DotOperand o, int64_t F, int64_t Fp, int64_t positions, RaggedPlan p,
                          const int* __restrict__ codes, const int* __restrict__ norms,
                          uint8_t* __restrict__ planes, int* __restrict__ shifts,
                          float* __restrict__ part) {
  wait_previous_grid();
  const int tile = blockIdx.z;
  if (tile >= p.tensor_start[p.groups]) return;
  const RaggedTile t = p.tensor[tile];
  const int64_t at = static_cast<int64_t>(t.slot) * Fp;
  if (tile == p.tensor_start[t.group])
    column_parts(F, Fp, p.row[t.group + 1] - p.row[t.group], p.slot_bits[t.slot], codes + at,
                 norms + at, part + at);
  split_mn_body<kPair>(moved(o, t.row * o.s_k), F, t.rows, Fp, kTensorTile, p.slot_bits[t.slot],
                       codes + t.slot * Fp,
                       planes + static_cast<size_t>(tile) * kTensorTile * Fp,
                       static_cast<size_t>(positions) * Fp, shifts + t.slot * Fp);
}

// ---- GEMM ----------------------------------------------------------------------

struct RaggedGemm {
  RaggedPlan p;
  int slots;                // of the planes
  int tiles_m, tiles_n;     // tiles_m: contraction only
  int stages;               // products only
  int64_t Mp, Np;           // rows of a plane of A, columns
  uint8_t* cres;
};

// Units (modulus, tile of rows, tile of columns), modulus outermost, so that
// one modulus's planes stay in L2.
template <bool kBMnPlanes>
struct ProductWork {
  static constexpr bool kAMn = false, kBMn = kBMnPlanes, kMasked = true;
  const RaggedGemm& g;
  int64_t tiles;
  __device__ __forceinline__ int64_t units() const { return kL * tiles * g.tiles_n; }
  __device__ __forceinline__ GemmTile at(int64_t u, uint32_t rank) const {
    const int64_t per = tiles * g.tiles_n;
    GemmTile t;
    t.l = static_cast<int>(u / per);
    const int64_t r = u - t.l * per;
    const RaggedTile x = g.p.tensor[r / g.tiles_n];
    const int tn = static_cast<int>(r % g.tiles_n), half = static_cast<int>(rank) * 128;
    t.stages = g.stages;
    t.k0 = 0;
    t.za = 0;
    t.a = static_cast<int>(t.l * g.Mp) + x.row + half;
    t.zb = t.l * g.slots + x.slot;
    t.b = (kBMn ? 0 : static_cast<int>(t.zb * g.Np)) + tn * 256 + half;
    t.out = g.cres + (t.l * g.Mp + x.row + half) * g.Np + tn * 256;
    t.rows = x.rows - half;
    return t;
  }
};

// Units (modulus, slot, tile of rows, tile of columns).
struct ContractWork {
  static constexpr bool kAMn = true, kBMn = true, kMasked = false;
  const RaggedGemm& g;
  int64_t slots;
  __device__ __forceinline__ int64_t units() const {
    return kL * slots * g.tiles_m * g.tiles_n;
  }
  __device__ __forceinline__ GemmTile at(int64_t u, uint32_t rank) const {
    const int per = g.tiles_m * g.tiles_n;
    const int64_t s = u / per;
    const int r = static_cast<int>(u - s * per);
    GemmTile t;
    t.l = static_cast<int>(s / slots);
    const int slot = static_cast<int>(s - t.l * slots);
    const int group = g.p.slot_group[slot];
    const int first = g.p.tensor_start[group];
    const int half = static_cast<int>(rank) * 128;
    t.stages = g.p.tensor_start[group + 1] - first;
    t.k0 = first * kTensorTile;
    t.za = t.zb = t.l;
    t.a = r / g.tiles_n * 256 + half;
    t.b = r % g.tiles_n * 256 + half;
    t.out = g.cres + (static_cast<int64_t>(t.l * g.slots + slot) * g.Mp + t.a) * g.Np +
            r % g.tiles_n * 256;
    t.rows = 128;
    return t;
  }
};
static_assert(kTensorTile == kSub2 * kTileK, "a stage is a tile of positions");
static_assert(kRaggedWindow == kMaxK, "a window of rows is one exact product");

template <bool kBMn>
__global__ void __launch_bounds__(kGemm2Threads, 1)
ragged_product_gemm_kernel(const __grid_constant__ CUtensorMap ta,
                           const __grid_constant__ CUtensorMap tb, RaggedGemm g, int* err) {
  gemm2_body(ta, tb, ProductWork<kBMn>{g, g.p.tensor_start[g.p.groups]}, g.Np, err);
}

__global__ void __launch_bounds__(kGemm2Threads, 1)
ragged_contract_gemm_kernel(const __grid_constant__ CUtensorMap ta,
                            const __grid_constant__ CUtensorMap tb, RaggedGemm g, int* err) {
  gemm2_body(ta, tb, ContractWork{g, slots_of(g.p)}, g.Np, err);
}

// ---- reconstruction ----------------------------------------------------------------

// The modular sum of an output's 14 residues. A residue byte r becomes the f64
// 4096 + r by one byte permutation (byte 1 of the high word of 2^12), and the
// weights W_l, each less the modulus product M where that keeps the running sums
// of the weights within M / 2, sum to 1: the 4096s leave 4096 times 1, which
// the sums start below zero. In limbs of 70 bits (hi rounded to nearest) the high
// sum stays below 2^51.5 in magnitude and is exact; the low one's partial sums
// stay below 2^86, so its 15 roundings lose at most 2^37 together.
struct CrtSum {
  double w[kL][2];
  double start[2];
  double mlimb[2];
  double inv_m;  // 2^70 / M
};

CrtSum crt_sum() {
  CrtSum c{};
  using i128 = __int128;
  i128 M = 1, sum = 0, sum_hi = 0;
  for (int l = 0; l < kL; ++l) M *= mod_of(l);
  const i128 unit = static_cast<i128>(1) << kCrtSplit;
  for (int l = 0; l < kL; ++l) {
    const i128 Ml = M / mod_of(l);
    int inv = 1;
    while (static_cast<int>(Ml % mod_of(l)) * inv % mod_of(l) != 1) ++inv;
    i128 w = Ml * inv;
    if (sum + w > M / 2) w -= M;
    sum += w;
    // floor(w / 2^70 + 1/2)
    const i128 hi = (w + unit / 2) >> kCrtSplit;
    sum_hi += hi;
    c.w[l][0] = static_cast<double>(static_cast<int64_t>(hi));
    c.w[l][1] = static_cast<double>(w - hi * unit);
  }
  c.start[0] = -4096.0 * static_cast<double>(static_cast<int64_t>(sum_hi));
  c.start[1] = -4096.0 * static_cast<double>(sum - sum_hi * unit);
  c.mlimb[0] = crt_consts().mlimb[0];
  c.mlimb[1] = crt_consts().mlimb[1];
  c.inv_m = crt_consts().inv_m * 0x1p70;
  return c;
}

struct RaggedCrt {
  CrtSum sum;
  RaggedPlan p;
  DotOperand a, b;
  DotResult c;
  int64_t M, K, N;       // rows; products: contraction; contraction: rows of a matrix
  int64_t Mp, Np, slots;
  int P;                 // products
  uint32_t blocks_n;     // of columns, and (contraction) of a slot's rows, of
  uint32_t blocks_m;     // ragged_crt_kernel
  const uint8_t* cres;
  const int* sa;
  const int* sb;
  const float* pa;       // certificate parts of the rows and columns
  const float* pb;
  const int* row_slot;   // products: slot + 1 of each row
  const int* err;
  int* fix_count;
  uint64_t* fix_list;
  int64_t fix_cap;
};

// A row of the result: where its residues, scales and operands are.
struct RowView {
  bool live;
  int slot, sa, P;
  int64_t residues;      // row of the residue planes
  int64_t out;           // row of the result
  int64_t a, b, K;       // first elements and length of the contraction
};

// The certificate's K / 4 and the low limb's rounding.
__device__ __forceinline__ float certify_rest(int64_t K) {
  return __double2float_ru((0.25 * static_cast<double>(K) + 0x1p37) * pow2_normal(kCertifyBits));
}

template <bool kContract>
__device__ __forceinline__ int64_t rows_of(const RaggedCrt& p) {
  return kContract ? slots_of(p.p) * p.K : p.M;
}

template <bool kContract>
__device__ __forceinline__ RowView view(const RaggedCrt& p, int64_t row) {
  RowView v;
  if constexpr (kContract) {
    v.live = true;
    v.slot = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(p.K));
    const int64_t i = row - v.slot * p.K;
    const int g = p.p.slot_group[v.slot];
    const int64_t first = p.p.row[g];
    v.residues = v.slot * p.Mp + i;
    v.out = g * p.K + i;
    v.a = first * p.a.s_k + i;
    v.b = first * p.b.s_k;
    v.K = p.p.row[g + 1] - first;
    v.P = p.p.slot_bits[v.slot];
    v.sa = p.sa[v.residues];
  } else {
    v.slot = p.row_slot[row] - 1;
    v.live = v.slot >= 0;
    if (!v.live) return v;
    v.residues = v.out = row;
    v.a = row * p.a.s_r;
    v.b = p.p.slot_group[v.slot] * p.b.s_b;
    v.K = p.K;
    v.P = p.P;
    v.sa = p.sa[row];
  }
  return v;
}

// C from an output's residues: the modular sum, less the multiple of M that
// brings it within M / 4 (so near that the high sum alone tells which).
__device__ __forceinline__ double crt_value(const CrtSum& k, double s_hi, double s_lo) {
  const double qt = rint(s_hi * k.inv_m);
  const double t_hi = __fma_rn(-qt, k.mlimb[0], s_hi);
  const double t_lo = __fma_rn(-qt, k.mlimb[1], s_lo);
  return __fma_rn(t_hi, 0x1p70, t_lo);
}

// bytes of the high word: 0, byte q of `word`, 0xb0, 0x40
__device__ __forceinline__ double biased_byte(uint32_t word, int q) {
  return __hiloint2double(static_cast<int>(__byte_perm(word, 0x40b00000u, 0x7604u | (q << 4))), 0);
}

__device__ __forceinline__ bool scales_ordinary(int sa, int sb) {
  return shift_ordinary(sa) && shift_ordinary(sb);
}
__device__ __forceinline__ bool in_range(int s) { return s <= 1022 && s >= -1023; }

// Outputs of one row at four columns that ragged_crt_kernel leaves out of its
// loop: scales whose sum leaves the f64 range, and (the IEEE sum of the products)
// non-finite operands.
struct SpecialRow {
  const uint8_t* residues;
  int64_t a, b, K;  // first elements of the row and of the column, and length
  int64_t out;
  int columns, sa;
};

__device__ __noinline__ void special_outputs(const RaggedCrt& p, const SpecialRow& r,
                                             const int* sb_of, size_t plane) {
  for (int q = 0; q < r.columns; ++q) {
    const int sa = r.sa, sb = sb_of[q];
    double out = 0.0;
    if (scales_ordinary(sa, sb)) {
      if (in_range(sa + sb)) continue;
      double s_hi = p.sum.start[0], s_lo = p.sum.start[1];
      for (int l = 0; l < kL; ++l) {
        const double x = biased_byte(r.residues[l * plane + q], 0);
        s_hi = __fma_rn(x, p.sum.w[l][0], s_hi);
        s_lo = __fma_rn(x, p.sum.w[l][1], s_lo);
      }
      out = scale2(crt_value(p.sum, s_hi, s_lo), -(sa + sb));
    } else {
      if (sa != kShiftNonFinite && sb != kShiftNonFinite) continue;
      for (int64_t k = 0; k < r.K; ++k)
        out += op_value(p.a, r.a + k * p.a.s_k) *
               op_value(p.b, r.b + q * p.b.s_r + k * p.b.s_k);
    }
    put_result(p.c, r.out + q, out);
  }
}

// A block takes kCrtRows rows of one group x 512 columns, each thread kCols
// consecutive columns, whose scales and certificate parts it keeps.  14 bytes in
// and 8 out per output: bound by HBM once enough rows are on their way, which
// the loop's own loads (64 to 126 registers, 20 to 32 warps) did not reach.  Each
// warp copies its rows to shared memory three ahead: 16.8 million outputs of
// 2048 x 2048 matrices take 68 us (5.4 TB/s), with loads in the loop and a
// residue's bias subtracted 117; 33.5 million of a contraction 114 and 226.
// 8 or 32 rows, or 4 or 6 blocks per SM, are within 1%, and so is five rows ahead.
constexpr int kRaggedCrtThreads = 128, kCols = 4;
constexpr int kCrtRows = 16, kCrtAhead = 3, kWarpCols = 32 * kCols;
static_assert(kCrtRows <= 32, "a lane per row");

template <bool kContract>
__global__ void __launch_bounds__(kRaggedCrtThreads, 5)
ragged_crt_kernel(const __grid_constant__ RaggedCrt p) {
  wait_previous_grid();
  const uint32_t bm = blockIdx.x / p.blocks_n, bn = blockIdx.x - bm * p.blocks_n;
  int64_t row0;
  int rows;
  if constexpr (kContract) {
    const uint32_t slot = bm / p.blocks_m;
    if (slot >= static_cast<uint32_t>(slots_of(p.p))) return;
    const int64_t i = static_cast<int64_t>(bm - slot * p.blocks_m) * kCrtRows;
    row0 = slot * p.K + i;
    rows = p.K - i < kCrtRows ? static_cast<int>(p.K - i) : kCrtRows;
  } else {
    constexpr uint32_t kParts = kTensorTile / kCrtRows;
    if (bm / kParts >= static_cast<uint32_t>(p.p.tensor_start[p.p.groups])) return;
    const RaggedTile x = p.p.tensor[bm / kParts];
    const int i = static_cast<int>(bm % kParts) * kCrtRows, left = x.rows - i;
    row0 = x.row + i;
    rows = left < kCrtRows ? left : kCrtRows;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t w0 = (static_cast<int64_t>(bn) * (kRaggedCrtThreads / 32) + warp) * kWarpCols;
  const int64_t j0 = w0 + lane * kCols;
  if (rows <= 0 || w0 >= p.N) return;  // the whole warp
  const RowView v = view<kContract>(p, row0);
  const size_t plane = static_cast<size_t>(kContract ? p.slots : 1) * p.Mp * p.Np;
  // the warp's columns of the 14 planes of a row, kCrtAhead rows ahead
  __shared__ __align__(16) uint8_t s_rows[kRaggedCrtThreads / 32][kCrtAhead + 1][kL * kWarpCols];
  const uint8_t* from = p.cres + v.residues * p.Np + w0 + lane / 8 * plane + lane % 8 * 16;
  auto copy_row = [&](int r) {
    if (r < rows) {
      const uint32_t to = smem_u32(&s_rows[warp][r % (kCrtAhead + 1)][lane * 16]);
#pragma unroll
      for (int i = 0; i < (kL + 3) / 4; ++i)
        if (4 * i + lane / 8 < kL)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 512),
                       "l"(from + 4 * i * plane)
                       : "memory");
      from += p.Np;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int r = 0; r < kCrtAhead; ++r) copy_row(r);
  // row r's scale and certificate part in lane r
  const int sa_of = lane < rows ? p.sa[v.residues + lane] : 0;
  const float pa_of = lane < rows ? p.pa[v.residues + lane] : 0.0f;
  const bool failed = *p.err != 0;
  const int4 sbv = *reinterpret_cast<const int4*>(p.sb + v.slot * p.Np + j0);
  const int sb[kCols] = {sbv.x, sbv.y, sbv.z, sbv.w};
  const float4 pbv = *reinterpret_cast<const float4*>(p.pb + v.slot * p.Np + j0);
  const float pb[kCols] = {pbv.x, pbv.y, pbv.z, pbv.w};
  int sb_min = sb[0], sb_max = sb[0];
  bool plain = !failed && j0 + kCols <= p.N;
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
    plain &= shift_ordinary(sb[q]);
    sb_min = sb[q] < sb_min ? sb[q] : sb_min;
    sb_max = sb[q] > sb_max ? sb[q] : sb_max;
  }
  const float rest = certify_rest(v.K);
  const bool words =
      p.c.f64 && (p.N & 1) == 0 && (reinterpret_cast<uintptr_t>(p.c.f64) & 15) == 0;
  int64_t at = v.out * p.N + j0;
  uint32_t special = 0;  // rows with outputs for special_outputs
#pragma unroll 1
  for (int r = 0; r < rows; ++r, at += p.N) {
    const int sa = __shfl_sync(0xffffffffu, sa_of, r);
    const float part = __fadd_ru(rest, __shfl_sync(0xffffffffu, pa_of, r));
    asm volatile("cp.async.wait_group %0;" ::"n"(kCrtAhead - 1) : "memory");
    __syncwarp();
    copy_row(r + kCrtAhead);
    const uint32_t* row = reinterpret_cast<const uint32_t*>(s_rows[warp][r % (kCrtAhead + 1)]);
    uint32_t cur[kL];
#pragma unroll
    for (int l = 0; l < kL; ++l) cur[l] = row[l * (kWarpCols / 4) + lane];
    double s_hi[kCols], s_lo[kCols];
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      s_hi[q] = p.sum.start[0];
      s_lo[q] = p.sum.start[1];
    }
#pragma unroll
    for (int l = 0; l < kL; ++l) {
      const double w_hi = p.sum.w[l][0], w_lo = p.sum.w[l][1];
#pragma unroll
      for (int q = 0; q < kCols; ++q) {
        const double x = biased_byte(cur[l], q);
        s_hi[q] = __fma_rn(x, w_hi, s_hi[q]);  // exact
        s_lo[q] = __fma_rn(x, w_lo, s_lo[q]);
      }
    }
    double c[kCols];
    bool sure[kCols];
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      c[q] = crt_value(p.sum, s_hi[q], s_lo[q]);
      // the high word of the bound as an f64, rounded down, against c's
      const int bound = (__float_as_int(__fadd_ru(part, pb[q])) >> 3) + (896 << 20);
      sure[q] = (__double2hiint(c[q]) & 0x7fffffff) > bound;
      const uint32_t e = 1023u - static_cast<uint32_t>(sa) - static_cast<uint32_t>(sb[q]);
      c[q] = __dmul_rn(c[q], __hiloint2double(static_cast<int>(e << 20), 0));
    }
    if (words && plain && shift_ordinary(sa) && in_range(sa + sb_max) && in_range(sa + sb_min) &&
        sure[0] && sure[1] && sure[2] && sure[3]) {
      double2* dst = reinterpret_cast<double2*>(p.c.f64 + at);
      dst[0] = make_double2(c[0], c[1]);
      dst[1] = make_double2(c[2], c[3]);
      continue;
    }
#pragma unroll
    for (int q = 0; q < kCols; ++q) {
      if (j0 + q >= p.N) continue;
      if (failed) {
        c[q] = __longlong_as_double(0x7ff8000000000000LL);
      } else if (!scales_ordinary(sa, sb[q])) {
        c[q] = 0.0;  // a row or column of zeros
        if (sa == kShiftNonFinite || sb[q] == kShiftNonFinite) special |= 1u << r;
      } else if (!sure[q]) {
        // uncertified: listed for ragged_fix_kernel, which writes this output
        const int64_t n = list_place(p.fix_count, p.fix_cap);
        if (n < p.fix_cap) p.fix_list[n] = static_cast<uint64_t>((row0 + r) * p.N + j0 + q);
        continue;
      } else if (!in_range(sa + sb[q])) {
        special |= 1u << r;
      }
      put_result(p.c, at + q, c[q]);
    }
  }
  while (special != 0) {
    const int r = __ffs(special) - 1;
    special &= special - 1;
    const int left = p.N - j0 < kCols ? static_cast<int>(p.N - j0) : kCols;
    const SpecialRow x{p.cres + (v.residues + r) * p.Np + j0,
                       v.a + r * (kContract ? 1 : p.a.s_r), v.b + j0 * p.b.s_r, v.K,
                       (v.out + r) * p.N + j0, left, p.sa[v.residues + r]};
    special_outputs(p, x, p.sb + v.slot * p.Np + j0, plane);
  }
}

// ---- recomputation of uncertified outputs -----------------------------------------

constexpr int kRaggedFixThreads = 256, kFixTile = 64;

// One output by one block (as dot2_block in dot_ozaki.cu): thread t sums k =
// t, t + 256, ... in eight chains, merged in a fixed tree.
__device__ double ragged_dot2(const RaggedCrt& p, const RowView& v, int64_t j, int da, int db) {
  constexpr int kChains = 8;
  __shared__ Dot2 s_warp[kRaggedFixThreads / 32];
  const int64_t b0 = v.b + j * p.b.s_r;
  Dot2 ch[kChains];
  int64_t k = threadIdx.x;
  auto add = [&](Dot2& d, int64_t at) {
    dot2_add(d, scale2(op_value(p.a, v.a + at * p.a.s_k), da),
             scale2(op_value(p.b, b0 + at * p.b.s_k), db));
  };
  for (; k + (kChains - 1) * kRaggedFixThreads < v.K; k += kChains * kRaggedFixThreads) {
#pragma unroll
    for (int u = 0; u < kChains; ++u) add(ch[u], k + u * kRaggedFixThreads);
  }
  for (; k < v.K; k += kRaggedFixThreads) add(ch[0], k);
#pragma unroll
  for (int w = 1; w < kChains; w <<= 1)
#pragma unroll
    for (int u = 0; u + w < kChains; u += 2 * w) dot2_merge(ch[u], ch[u + w]);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    Dot2 o;
    o.p = __shfl_down_sync(0xffffffffu, ch[0].p, off);
    o.s = __shfl_down_sync(0xffffffffu, ch[0].s, off);
    if (lane + off < 32) dot2_merge(ch[0], o);
  }
  if (lane == 0) s_warp[threadIdx.x >> 5] = ch[0];
  __syncthreads();
  double r = 0.0;
  if (threadIdx.x == 0) {
    Dot2 d = s_warp[0];
    for (int w = 1; w < kRaggedFixThreads / 32; ++w) dot2_merge(d, s_warp[w]);
    r = scale2(__dadd_rn(d.p, d.s), -(da + db));  // at once: in two steps it may underflow
  }
  __syncthreads();  // s_warp is reused
  return r;
}

// Up to 64 rows from row0 on (of one group, `rows` of them) x 64 columns by
// one block, as dot2_tile in dot_ozaki.cu.
template <bool kContract>
__device__ void ragged_dot2_tile(const RaggedCrt& p, int64_t row0, int rows, int64_t j0) {
  __shared__ double sA[kFixTile][17];
  __shared__ double sB[16][kFixTile + 1];
  __shared__ int sShA[kFixTile], sShB[kFixTile];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const RowView v = view<kContract>(p, row0);
  const int64_t a_row = kContract ? 1 : p.a.s_r;  // from a row to the next
  if (tid < kFixTile) {
    sShA[tid] = tid < rows ? p.sa[v.residues + tid] : kShiftZero;
    sShB[tid] = j0 + tid < p.N ? p.sb[v.slot * p.Np + j0 + tid] : kShiftZero;
  }
  __syncthreads();
  Dot2 acc[4][4];
  for (int64_t k0 = 0; k0 < v.K; k0 += 16) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int e = tid + t * kRaggedFixThreads;
      {
        const int r = e >> 4, kk = e & 15;
        const bool in = k0 + kk < v.K && shift_ordinary(sShA[r]);
        sA[r][kk] = in ? scale2(op_value(p.a, v.a + r * a_row + (k0 + kk) * p.a.s_k),
                                sShA[r] - v.P)
                       : 0.0;
      }
      {
        const int kk = e >> 6, c = e & 63;
        const bool in = k0 + kk < v.K && shift_ordinary(sShB[c]);
        sB[kk][c] = in ? scale2(op_value(p.b, v.b + (j0 + c) * p.b.s_r + (k0 + kk) * p.b.s_k),
                                sShB[c] - v.P)
                       : 0.0;
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int kk = 0; kk < 16; ++kk) {
      double x[4], y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = sA[ty + 16 * u][kk];
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = sB[kk][tx + 16 * u];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) dot2_add(acc[u][w], x[u], y[w]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = ty + 16 * u;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int c = tx + 16 * w;
      if (shift_ordinary(sShA[r]) && shift_ordinary(sShB[c]))
        put_result(p.c, (v.out + r) * p.N + j0 + c,
                   scale2(__dadd_rn(acc[u][w].p, acc[u][w].s), 2 * v.P - sShA[r] - sShB[c]));
    }
  }
  __syncthreads();
}

// Every uncertified output: one block per listed output, or with more than
// the list holds every output of the large groups.
template <bool kContract>
__global__ void __launch_bounds__(kRaggedFixThreads, 2)
ragged_fix_kernel(const __grid_constant__ RaggedCrt p) {
  wait_previous_grid();
  const int count = *p.fix_count;
  if (count == 0 || *p.err != 0) return;
  if (count <= p.fix_cap) {
    for (int e = blockIdx.x; e < count; e += gridDim.x) {
      const int64_t flat = static_cast<int64_t>(p.fix_list[e]);
      const int64_t row = flat / p.N, j = flat - row * p.N;
      const RowView v = view<kContract>(p, row);
      const double r = ragged_dot2(p, v, j, v.sa - v.P, p.sb[v.slot * p.Np + j] - v.P);
      if (threadIdx.x == 0) put_result(p.c, v.out * p.N + j, r);
    }
    return;
  }
  const int64_t tn = (p.N + kFixTile - 1) / kFixTile;
  if constexpr (kContract) {
    const int64_t tk = (p.K + kFixTile - 1) / kFixTile, tiles = slots_of(p.p) * tk * tn;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int64_t i = t / tn % tk * kFixTile;
      ragged_dot2_tile<true>(p, t / (tn * tk) * p.K + i,
                             p.K - i < kFixTile ? static_cast<int>(p.K - i) : kFixTile,
                             t % tn * kFixTile);
    }
  } else {
    constexpr int kParts = kTensorTile / kFixTile;
    const int64_t tiles = p.p.tensor_start[p.p.groups] * kParts * tn;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      const RaggedTile x = p.p.tensor[t / (tn * kParts)];
      const int i = static_cast<int>(t / tn % kParts) * kFixTile, left = x.rows - i;
      if (left > 0)
        ragged_dot2_tile<false>(p, x.row + i, left < kFixTile ? left : kFixTile,
                                t % tn * kFixTile);
    }
  }
}

// A later chunk of the contraction: the large groups' part added to the result.
template <bool kContract>
__global__ void __launch_bounds__(256)
ragged_add_kernel(const __grid_constant__ RaggedCrt p, DotResult out) {
  wait_previous_grid();
  const int64_t rows = rows_of<kContract>(p);
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const RowView v = view<kContract>(p, row);
    if (!v.live) continue;
    for (int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; j < p.N;
         j += static_cast<int64_t>(gridDim.x) * 256) {
      const int64_t at = v.out * p.N + j;
      put_result(out, at, __dadd_rn(result_value(out, at), p.c.f64[at]));
    }
  }
}

// ---- host ------------------------------------------------------------------------

struct TensorLayout {
  int64_t chunk;            // longest contraction of a chunk
  int64_t Mp, Np, Kp;       // contraction: Kp positions, Mp rows of a matrix
  int64_t slots;
  size_t a, b, c, sa, sb, pa, pb, clear, ca, cb, na, nb, err, row_slot, clear_end, list, part, total;
  int64_t fix_cap;
};

int64_t pad(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

TensorLayout tensor_layout(int64_t M, int64_t K, int64_t N, int64_t G, bool contract) {
  TensorLayout g{};
  const int64_t length = contract ? M : K;
  g.chunk = length < kMaxK ? length : kMaxK;
  g.slots = ragged_slots(contract ? g.chunk : M, G, contract);
  g.Np = pad(N, 256);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at = (at + bytes + 1023) / 1024 * 1024;
    return here;
  };
  const size_t l = kL;
  int64_t a_scales;
  if (contract) {
    g.Mp = pad(K, 256);
    g.Kp = ragged_tensor_tiles(g.chunk, G, true) * kTensorTile;
    g.a = take(l * g.Kp * g.Mp);
    g.b = take(l * g.Kp * g.Np);
    g.c = take(l * g.slots * g.Mp * g.Np);
    a_scales = g.slots * g.Mp;
  } else {
    g.Mp = pad(M, 128);
    g.Kp = pad(g.chunk, kTileK);
    g.a = take(l * g.Mp * g.Kp);
    g.b = take(l * g.slots * g.Np * g.Kp);
    g.c = take(l * g.Mp * g.Np);
    a_scales = g.Mp;
  }
  g.sa = take(4 * a_scales);
  g.sb = take(4 * g.slots * g.Np);
  g.pa = take(4 * a_scales);
  g.pb = take(4 * g.slots * g.Np);
  // cleared together: column codes and norms, error word and count, slots of the
  // rows
  g.clear = at;
  g.ca = take(contract ? 4 * a_scales : 0);
  g.cb = take(4 * g.slots * g.Np);
  g.na = take(contract ? 4 * a_scales : 0);
  g.nb = take(4 * g.slots * g.Np);
  g.err = take(16);
  g.row_slot = take(contract ? 0 : 4 * M);
  g.clear_end = at;
  const int64_t outputs = contract ? g.slots * K * N : M * N;
  g.fix_cap = outputs < (1 << 20) ? outputs : 1 << 20;
  g.list = take(8 * g.fix_cap);
  g.part = take(length > g.chunk ? 8 * static_cast<size_t>(contract ? G * K * N : M * N) : 0);
  g.total = at;
  return g;
}

// The kernels' shared memory limit, once per device.
int prepare_device(int* clusters) {
  static std::mutex mu;
  static std::vector<int> by_device;
  int dev = 0;
  DSB_CUDA_TRY(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= static_cast<int>(by_device.size())) by_device.resize(dev + 1, -1);
  if (by_device[dev] < 0) {
    int pairs = 0, query = 0;
    if (int st = dot_ozaki_kernel_info(&pairs, &query)) return st;
    const int bytes = static_cast<int>(gemm2_smem_bytes());
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    DSB_CUDA_TRY(cudaFuncSetAttribute(ragged_product_gemm_kernel<false>, attr, bytes));
    DSB_CUDA_TRY(cudaFuncSetAttribute(ragged_product_gemm_kernel<true>, attr, bytes));
    DSB_CUDA_TRY(cudaFuncSetAttribute(ragged_contract_gemm_kernel, attr, bytes));
    by_device[dev] = pairs;
  }
  *clusters = by_device[dev];
  return DS_OK;
}

template <class Kernel>
int launch_gemm(Kernel kernel, int clusters, const CUtensorMap& ta, const CUtensorMap& tb,
                const RaggedGemm& g, int* err, cudaStream_t s) {
  ProfileScope prof("ozaki_gemm", s);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * clusters));
  cfg.blockDim = dim3(kGemm2Threads);
  cfg.dynamicSmemBytes = gemm2_smem_bytes();
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DSB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ta, tb, g, err));
  return DS_OK;
}

unsigned grid_y(int64_t n) { return static_cast<unsigned>(n < 1 ? 1 : n > 65535 ? 65535 : n); }

template <bool kContract>
int launch_rebuild(const RaggedCrt& c, int64_t rows, const DotResult* add_to, cudaStream_t s) {
  {
    ProfileScope prof("ozaki_crt", s);
    const int64_t parts =
        kContract ? c.slots * c.blocks_m : c.p.tensor_cap * (kTensorTile / kCrtRows);
    DSB_CUDA_TRY(launch_dependent(ragged_crt_kernel<kContract>,
                                  dim3(static_cast<unsigned>(parts * c.blocks_n)),
                                  dim3(kRaggedCrtThreads), s, c));
  }
  ProfileScope prof("ozaki_fix", s);
  DSB_CUDA_TRY(launch_dependent(ragged_fix_kernel<kContract>,
                                dim3(static_cast<unsigned>(2 * sm_count())),
                                dim3(kRaggedFixThreads), s, c));
  if (add_to)
    DSB_CUDA_TRY(launch_dependent(ragged_add_kernel<kContract>,
                                  dim3(static_cast<unsigned>((c.N + 255) / 256), grid_y(rows)),
                                  dim3(256), s, c, *add_to));
  return launch_status();
}

DotOperand at_k(DotOperand o, int64_t k) {
  if (o.f64) o.f64 += k * o.s_k;
  if (o.hi) o.hi += k * o.s_k;
  if (o.lo) o.lo += k * o.s_k;
  return o;
}

// Everything after the splits' shapes: fills what products and contraction
// share.
struct TensorRun {
  uint8_t* ws;
  TensorLayout g;
  uint8_t *planes_a, *planes_b;
  int *sa, *sb, *ca, *cb, *na, *nb, *err, *row_slot;
  float *pa, *pb;
  RaggedCrt crt;
  RaggedGemm gemm;
};

TensorRun tensor_run(const RaggedProblem& q, const RaggedPlan& p, const TensorLayout& g, void* at) {
  TensorRun r{};
  r.ws = static_cast<uint8_t*>(at);
  r.g = g;
  auto ints = [&](size_t off) { return reinterpret_cast<int*>(r.ws + off); };
  r.planes_a = r.ws + g.a;
  r.planes_b = r.ws + g.b;
  r.sa = ints(g.sa);
  r.sb = ints(g.sb);
  r.ca = ints(g.ca);
  r.cb = ints(g.cb);
  r.na = ints(g.na);
  r.nb = ints(g.nb);
  r.pa = reinterpret_cast<float*>(r.ws + g.pa);
  r.pb = reinterpret_cast<float*>(r.ws + g.pb);
  r.err = ints(g.err);
  r.row_slot = ints(g.row_slot);
  static const CrtSum sum = crt_sum();
  r.crt.sum = sum;
  constexpr int64_t kBlockN = kRaggedCrtThreads * kCols;
  r.crt.blocks_n = static_cast<uint32_t>((q.N + kBlockN - 1) / kBlockN);
  r.crt.blocks_m = static_cast<uint32_t>((q.K + kCrtRows - 1) / kCrtRows);
  r.crt.p = p;
  r.crt.a = q.lhs;
  r.crt.b = q.rhs;
  r.crt.c = q.out;
  r.crt.M = q.M;
  r.crt.K = q.K;
  r.crt.N = q.N;
  r.crt.Mp = g.Mp;
  r.crt.Np = g.Np;
  r.crt.slots = g.slots;
  r.crt.cres = r.ws + g.c;
  r.crt.sa = r.sa;
  r.crt.sb = r.sb;
  r.crt.pa = r.pa;
  r.crt.pb = r.pb;
  r.crt.row_slot = r.row_slot;
  r.crt.err = r.err;
  r.crt.fix_count = r.err + 1;
  r.crt.fix_list = reinterpret_cast<uint64_t*>(r.ws + g.list);
  r.crt.fix_cap = g.fix_cap;
  r.gemm.p = p;
  r.gemm.slots = static_cast<int>(g.slots);
  r.gemm.tiles_n = static_cast<int>(g.Np / 256);
  r.gemm.Mp = g.Mp;
  r.gemm.Np = g.Np;
  r.gemm.cres = r.ws + g.c;
  return r;
}

}  // namespace

int ragged_bits(int64_t K) { return bits_for_k(K); }

int ragged_tensor_clusters(int* clusters) { return prepare_device(clusters); }

bool ragged_tensor_fits(int64_t M, int64_t K, int64_t N, int64_t G, bool contract) {
  const TensorLayout g = tensor_layout(M, K, N, G, contract);
  const int64_t most = (1LL << 31) - 1;  // TMA coordinates and tile numbers are int32
  if (g.total > kRaggedTensorBytes) return false;
  // blocks of ragged_crt_kernel
  const int64_t rows = contract ? g.slots * pad(K, kCrtRows)
                                : ragged_tensor_tiles(M, G, false) * kTensorTile;
  if (rows / kCrtRows * (N / (kRaggedCrtThreads * kCols) + 1) > most) return false;
  if (contract) return g.slots * g.Mp <= most && g.Np <= most;
  return kL * g.Mp <= most && kL * g.slots * g.Np <= most && g.slots <= 65535;
}

size_t ragged_tensor_bytes(int64_t M, int64_t K, int64_t N, int64_t G, bool contract) {
  return tensor_layout(M, K, N, G, contract).total;
}

int ragged_tensor_dot(const RaggedProblem& q, const RaggedPlan& p, void* workspace, int clusters,
                      cudaStream_t s) {
  const TensorLayout g = tensor_layout(q.M, q.K, q.N, q.G, false);
  TensorRun r = tensor_run(q, p, g, workspace);
  const unsigned tiles = static_cast<unsigned>(p.tensor_cap);
  for (int64_t k0 = 0; k0 < q.K; k0 += g.chunk) {
    const int64_t K = q.K - k0 < g.chunk ? q.K - k0 : g.chunk;
    const int64_t Kp = pad(K, kTileK);  // of this chunk's planes
    const int P = bits_for_k(K);
    CUtensorMap ta, tb;
    if (int st = make_tmap(&ta, r.planes_a, Kp, kL * g.Mp, kTileM)) return st;
    if (q.rhs_t) {
      if (int st = make_tmap(&tb, r.planes_b, Kp, kL * g.slots * g.Np, 128)) return st;
    } else {
      if (int st = make_tmap_mn(&tb, r.planes_b, g.Np, Kp, kL * g.slots)) return st;
    }
    const DotOperand a = at_k(q.lhs, k0), b = at_k(q.rhs, k0);
    {
      ProfileScope prof("ozaki_split", s);
      DSB_CUDA_TRY(cudaMemsetAsync(r.ws + g.clear, 0, g.clear_end - g.clear, s));
      const RowSplit rows{a, K, g.Mp, Kp, P, r.planes_a, r.sa, r.row_slot, r.pa};
      const ColumnMax cols{b, q.N, K, g.Np, r.cb, r.nb};
      const unsigned slots = static_cast<unsigned>(g.slots);
      const unsigned cgx = static_cast<unsigned>(g.Np / kColTileR);
      const unsigned cgy = static_cast<unsigned>((K + kColmaxSlab - 1) / kColmaxSlab);
      DSB_CUDA_TRY(launch_dependent(ragged_split_rows_kernel, dim3(tiles, kTensorTile),
                                    dim3(kSplitThreads), s, rows, p));
      if (q.rhs_t) {
        DSB_CUDA_TRY(launch_dependent(ragged_split_matrix_rows_kernel,
                                      dim3(static_cast<unsigned>(q.N), slots),
                                      dim3(kSplitThreads), s, b, K, g.Np, Kp, g.slots, P, p,
                                      r.planes_b, r.sb, r.pb));
      } else {
        DSB_CUDA_TRY(launch_dependent(ragged_colmax_kernel, dim3(cgx, cgy, slots), dim3(256), s,
                                      cols, p));
        const int64_t cx = (g.Np + kMnRows - 1) / kMnRows;
        int64_t ky = (2 * static_cast<int64_t>(sm_count()) + cx - 1) / cx;
        ky = ky > Kp / 16 ? Kp / 16 : ky;
        const dim3 grid(static_cast<unsigned>(cx), grid_y(ky), slots);
        if (q.rhs.f64)
          DSB_CUDA_TRY(launch_dependent(ragged_split_matrix_kernel<false>, grid, dim3(256), s, b,
                                        q.N, K, g.Np, Kp, g.slots, P, p, r.cb, r.nb, r.planes_b,
                                        r.sb, r.pb));
        else
          DSB_CUDA_TRY(launch_dependent(ragged_split_matrix_kernel<true>, grid, dim3(256), s, b,
                                        q.N, K, g.Np, Kp, g.slots, P, p, r.cb, r.nb, r.planes_b,
                                        r.sb, r.pb));
      }
    }
    r.gemm.stages = static_cast<int>((Kp / kTileK + kSub2 - 1) / kSub2);
    if (int st = q.rhs_t ? launch_gemm(ragged_product_gemm_kernel<false>, clusters, ta, tb, r.gemm,
                                       r.err, s)
                         : launch_gemm(ragged_product_gemm_kernel<true>, clusters, ta, tb, r.gemm,
                                       r.err, s))
      return st;
    r.crt.a = a;
    r.crt.b = b;
    r.crt.K = K;
    r.crt.P = P;
    if (k0 > 0) r.crt.c = DotResult{reinterpret_cast<double*>(r.ws + g.part), nullptr, nullptr};
    if (int st = launch_rebuild<false>(r.crt, q.M, k0 > 0 ? &q.out : nullptr, s)) return st;
  }
  return DS_OK;
}

int ragged_tensor_contract(const RaggedProblem& q, const RaggedPlan& p, bool add, void* workspace,
                           int clusters, cudaStream_t s) {
  const TensorLayout g = tensor_layout(q.M, q.K, q.N, q.G, true);
  TensorRun r = tensor_run(q, p, g, workspace);
  const unsigned tiles = static_cast<unsigned>(p.tensor_cap);
  CUtensorMap ta, tb;
  if (int st = make_tmap_mn(&ta, r.planes_a, g.Mp, g.Kp, kL)) return st;
  if (int st = make_tmap_mn(&tb, r.planes_b, g.Np, g.Kp, kL)) return st;
  {
    ProfileScope prof("ozaki_split", s);
    DSB_CUDA_TRY(cudaMemsetAsync(r.ws + g.clear, 0, g.clear_end - g.clear, s));
    auto split = [&](const DotOperand& o, int64_t F, int64_t Fp, int* codes, int* norms,
                     uint8_t* planes, int* shifts, float* part) -> int {
      DSB_CUDA_TRY(launch_dependent(ragged_tile_colmax_kernel,
                                    dim3(static_cast<unsigned>(Fp / kColTileR), 2 * tiles),
                                    dim3(256), s, o, F, Fp, p, codes, norms));
      const dim3 grid(static_cast<unsigned>((Fp + kMnRows - 1) / kMnRows), 8, tiles);
      if (o.f64)
        DSB_CUDA_TRY(launch_dependent(ragged_split_tiles_kernel<false>, grid, dim3(256), s, o, F,
                                      Fp, g.Kp, p, codes, norms, planes, shifts, part));
      else
        DSB_CUDA_TRY(launch_dependent(ragged_split_tiles_kernel<true>, grid, dim3(256), s, o, F,
                                      Fp, g.Kp, p, codes, norms, planes, shifts, part));
      return DS_OK;
    };
    if (int st = split(q.lhs, q.K, g.Mp, r.ca, r.na, r.planes_a, r.sa, r.pa)) return st;
    if (int st = split(q.rhs, q.N, g.Np, r.cb, r.nb, r.planes_b, r.sb, r.pb)) return st;
  }
  r.gemm.tiles_m = static_cast<int>(g.Mp / 256);
  if (int st = launch_gemm(ragged_contract_gemm_kernel, clusters, ta, tb, r.gemm, r.err, s))
    return st;
  if (add) r.crt.c = DotResult{reinterpret_cast<double*>(r.ws + g.part), nullptr, nullptr};
  return launch_rebuild<true>(r.crt, g.slots * q.K, add ? &q.out : nullptr, s);
}

}  // namespace dsb
