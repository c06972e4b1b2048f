// Device pieces of the tensor-core integer-residue product (Ozaki scheme II)
// shared by dot_general (dot_ozaki.cu) and the products grouped by expert
// (ragged_ozaki.cu): moduli and weights, the split into residues, the int8
// tcgen05 GEMM over CTA pairs, the reconstruction and the compensated dot
// product.  The scheme is described in dot_ozaki.cu.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <climits>
#include <cmath>
#include <mutex>

#include "common.cuh"
#include "ds_arith.cuh"
#include "kernels.h"

namespace dsb {
namespace {

constexpr int kL = 14;
constexpr int kTileM = 128, kTileN = 256, kTileK = 128;  // int8: 128 bytes of K
constexpr int kStages = 4;
constexpr int kStageA = kTileM * kTileK;  // 16 KB
constexpr int kStageB = kTileN * kTileK;  // 32 KB
constexpr int kGemmThreads = 192;
// u8 x u8 products summed in int32: K * 255^2 < 2^31 needs K <= 33025.
constexpr int kMaxK = 1 << 15;
constexpr int kShiftNonFinite = INT_MIN;
// Shift code of a row (column) whose values are all zero: its products are
// exactly zero, so its outputs need no error certificate.
constexpr int kShiftZero = INT_MIN + 1;
constexpr long long kTimeoutCycles = 4000000000LL;  // ~2 s at 1.9 GHz

__host__ __device__ constexpr int mod_of(int l) {
  return l == 0 ? 256 : l == 1 ? 255 : l == 2 ? 253 : l == 3 ? 251 : l == 4 ? 247
       : l == 5 ? 241 : l == 6 ? 239 : l == 7 ? 233 : l == 8 ? 229 : l == 9 ? 227
       : l == 10 ? 223 : l == 11 ? 217 : l == 12 ? 211 : 199;
}

// Moduli whose split residue is taken from the FP64 pipe (one FMA and one
// integer multiply-add) rather than the integer pipes (two byte dot
// products and a multiply-high reduction).  Ten of the thirteen were
// fastest: with all thirteen the row split spills (its group loop keeps
// every 1 / m in a register), with seven both splits are 4 to 6% slower.
__host__ __device__ constexpr bool residue_fp64(int l) { return l >= 1 && l <= 10; }

// ---------------------------------------------------------------------------
// Host-side constants: P from K, and the CRT weights in 40-bit limbs.

// The weights and the modulus product split at bit kCrtSplit: W = W_hi 2^70 +
// W_lo.  W_hi < 2^40.2, so the 14 products r W_hi (r < 2^8) sum exactly in
// f64 (< 2^53); W_lo < 2^70 is rounded to 53 bits.
constexpr int kCrtSplit = 70;

struct CrtConsts {
  double w[kL][2];  // W_l = (Mprod/m_l) * ((Mprod/m_l)^-1 mod m_l): {W_hi, W_lo}
  double mlimb[2];  // Mprod: {hi, lo}
  double inv_m;     // 1 / Mprod
  double log2_m;
};

using u128 = unsigned __int128;

const CrtConsts& crt_consts() {
  static CrtConsts c;
  static std::once_flag once;
  std::call_once(once, [] {
    u128 M = 1;
    for (int l = 0; l < kL; ++l) M *= static_cast<u128>(mod_of(l));
    const u128 lo_mask = (static_cast<u128>(1) << kCrtSplit) - 1;
    auto to_double = [](u128 v) { return static_cast<double>(v); };  // rounded to nearest
    for (int l = 0; l < kL; ++l) {
      const int m = mod_of(l);
      const u128 Ml = M / m;
      const int r = static_cast<int>(Ml % m);
      int inv = 1;
      while ((r * inv) % m != 1) ++inv;  // m <= 256: trivial search
      const u128 W = Ml * static_cast<u128>(inv);  // < M
      c.w[l][0] = static_cast<double>(static_cast<uint64_t>(W >> kCrtSplit));
      c.w[l][1] = to_double(W & lo_mask);
    }
    c.mlimb[0] = static_cast<double>(static_cast<uint64_t>(M >> kCrtSplit));
    c.mlimb[1] = to_double(M & lo_mask);
    const double Md = to_double(M);
    c.inv_m = 1.0 / Md;
    c.log2_m = std::log2(Md);
  });
  return c;
}

int bits_for_k(int64_t K) {
  const double lk = std::log2(static_cast<double>(K < 1 ? 1 : K));
  int P = static_cast<int>(std::floor((crt_consts().log2_m - 2.0 - lk) / 2.0));
  return P > 50 ? 50 : P;
}

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// ---------------------------------------------------------------------------
// Step 1: split.

// The value an operand element contributes: an f64 input as it is (it is at
// least as precise as its DS split), a SoA DS input as hi + lo.
__device__ __forceinline__ double op_value(const DotOperand& o, int64_t idx) {
  return o.f64 ? o.f64[idx]
               : __dadd_rn(static_cast<double>(o.hi[idx]), static_cast<double>(o.lo[idx]));
}

// v * 2^s for any int s (exact unless the result under/overflows).
__device__ __forceinline__ double scale2(double v, int s) {
  if (s >= -1000 && s <= 1000) return v * __longlong_as_double(static_cast<long long>(1023 + s) << 52);
  return ldexp(v, s);
}

constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52

// The biased integer t = rint(v * 2^shift) + 2^51, for |v * 2^shift| <= 2^50:
// adding 1.5 * 2^52 rounds to an integer (to nearest even) and leaves t in
// the low 52 bits of the sum, so no conversion instruction is needed.
__device__ __forceinline__ uint64_t quantise(double v, int shift) {
  const double y = (shift >= -1000 && shift <= 1000)
                       ? __fma_rn(v, __longlong_as_double(static_cast<long long>(1023 + shift) << 52), kMagic)
                       : __dadd_rn(ldexp(v, shift), kMagic);
  return static_cast<uint64_t>(__double_as_longlong(y)) & ((1ull << 52) - 1);
}

// t = hi * 2^32 + lo (hi < 2^20): the seven bytes of t in two words, and
// x - 128 as an f64 for the unbiased integer x = t - 2^51 (exact:
// |x| <= 2^50).
struct Limbs {
  uint32_t lo, hi;
  double xs;
};

__device__ __forceinline__ Limbs limbs_of(uint64_t t) {
  // t is the mantissa of 1.5 * 2^52 + x_int, a double in [2^52, 2^53)
  const double y = __longlong_as_double(static_cast<long long>(0x4330000000000000ull | t));
  return Limbs{static_cast<uint32_t>(t), static_cast<uint32_t>(t >> 32),
               __dsub_rn(y, kMagic + 128.0)};
}

// 2^e mod m, for the byte weights below.
__host__ __device__ constexpr uint32_t pow2_mod(int e, uint32_t m) {
  uint32_t r = 1 % m;
  for (int i = 0; i < e; ++i) r = (r * 2u) % m;
  return r;
}

// Four byte weights packed for __dp4a: byte j of the word is 2^(8 (j + j0)) mod m.
__host__ __device__ constexpr uint32_t byte_weights(int j0, int count, uint32_t m) {
  uint32_t w = 0;
  for (int j = 0; j < count; ++j) w |= pow2_mod(8 * (j0 + j), m) << (8 * j);
  return w;
}

// Residue in [0, m) of the unbiased integer t - 2^51 modulo m = mod_of(l).
// The bytes of t dotted with the weights 2^(8j) mod m (two byte dot
// products), plus the constant that cancels the bias, give s < 2^19 with
// s = t - 2^51 (mod m); then s mod m = s - m * umulhi(s, ceil(2^32 / m)),
// exact because s * (ceil(2^32 / m) * m - 2^32) < 2^19 * 2^8 < 2^32.
// m = 256 is the low byte of t (2^51 = 0 mod 256).
// Per modulus: {byte weights of the low word, of the high word, the bias
// correction, ceil(2^32 / m)}.  In the constant bank, so the instructions
// read them as operands instead of materialising 52 immediates per element.
struct SplitConsts {
  uint32_t w_lo, w_hi, unbias, magic;
};

__host__ __device__ constexpr SplitConsts split_consts(uint32_t m) {
  return SplitConsts{byte_weights(0, 4, m), byte_weights(4, 3, m), (m - pow2_mod(51, m)) % m,
                     m == 256u ? 0u : 0xFFFFFFFFu / m + 1u};
}

__constant__ SplitConsts c_split[kL] = {
    split_consts(mod_of(0)),  split_consts(mod_of(1)),  split_consts(mod_of(2)),
    split_consts(mod_of(3)),  split_consts(mod_of(4)),  split_consts(mod_of(5)),
    split_consts(mod_of(6)),  split_consts(mod_of(7)),  split_consts(mod_of(8)),
    split_consts(mod_of(9)),  split_consts(mod_of(10)), split_consts(mod_of(11)),
    split_consts(mod_of(12)), split_consts(mod_of(13))};

// 1 / m rounded, for the residue from the FP64 pipe: (x - 128) / m to
// 2^-10 for |x| <= 2^50.
__constant__ double c_inv_m[kL] = {
    1.0 / mod_of(0),  1.0 / mod_of(1),  1.0 / mod_of(2),  1.0 / mod_of(3),  1.0 / mod_of(4),
    1.0 / mod_of(5),  1.0 / mod_of(6),  1.0 / mod_of(7),  1.0 / mod_of(8),  1.0 / mod_of(9),
    1.0 / mod_of(10), 1.0 / mod_of(11), 1.0 / mod_of(12), 1.0 / mod_of(13)};

// With kMixed, the moduli of residue_fp64 take the FP64 path and the others
// the integer one; otherwise all take the integer path.  0 (256) is a mask.
template <bool kMixed>
constexpr bool residue_on_fp64(int l) { return kMixed && residue_fp64(l); }

// Residue from the FP64 pipe, two instructions: one FMA gives
// 1.5 * 2^52 + q with q = rint((x - 128) / m) (x.xs = x - 128; the rounded
// 1 / m puts q within one of the nearest integer), so r = x - q m =
// 128 + ((x - 128) - q m) lies in [128 - m / 2 - m 2^-10,
// 128 + m / 2 + m 2^-10], inside [0, 255] for m <= 255.  r is then exact in
// 32-bit integer arithmetic from the low words: x mod 2^32 is x.lo (2^51 is
// 0 mod 2^32) and q mod 2^32 is the low word of the FMA's result, so one
// multiply-add x.lo - q m gives r.  r is a residue of x in [0, 256) but not
// always below m; the GEMM only needs an unsigned byte of the right class.
__device__ __forceinline__ uint32_t residue_fp64_path(const Limbs& x, double inv, uint32_t m) {
  const double qd = __fma_rn(x.xs, inv, kMagic);
  return x.lo - static_cast<uint32_t>(__double2loint(qd)) * m;
}

// Residue in [0, m) on the integer pipes.
__device__ __forceinline__ uint32_t residue_int(const Limbs& x, const SplitConsts& c, uint32_t m) {
  const uint32_t s = __dp4a(x.lo, c.w_lo, __dp4a(x.hi, c.w_hi, c.unbias));
  return s - __umulhi(s, c.magic) * m;
}

template <int l, bool kMixed>
__device__ __forceinline__ uint32_t residue(const Limbs& x) {
  constexpr uint32_t m = mod_of(l);
  if constexpr (m == 256u) {
    return x.lo & 0xFFu;
  } else if constexpr (residue_on_fp64<kMixed>(l)) {
    return residue_fp64_path(x, c_inv_m[l], m);
  } else {
    return residue_int(x, c_split[l], m);
  }
}

// Four residues (each < 256) as the bytes of one word: three byte permutes.
__device__ __forceinline__ uint32_t pack4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  return __byte_perm(__byte_perm(r0, r1, 0x0040), __byte_perm(r2, r3, 0x0040), 0x5410);
}

// Residues of N = 4, 8 or 16 consecutive values -> one 4-, 8- or 16-byte
// store per modulus plane.
template <int N, bool kMixed, int l = 0>
__device__ __forceinline__ void store_planes_n(const Limbs (&x)[N], uint8_t* base,
                                               size_t plane_stride) {
  if constexpr (l < kL) {
    uint32_t w[N / 4];
#pragma unroll
    for (int q = 0; q < N / 4; ++q)
      w[q] = pack4(residue<l, kMixed>(x[q * 4]), residue<l, kMixed>(x[q * 4 + 1]),
                   residue<l, kMixed>(x[q * 4 + 2]), residue<l, kMixed>(x[q * 4 + 3]));
    uint8_t* dst = base + l * plane_stride;
    if constexpr (N == 4) {
      *reinterpret_cast<uint32_t*>(dst) = w[0];
    } else if constexpr (N == 8) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    store_planes_n<N, kMixed, l + 1>(x, base, plane_stride);
  }
}

// The residue with the modulus picked at run time: the same arithmetic as
// residue<l, true>, its constants read from the constant bank by index
// (m = 256 works on the integer path too: its weights select byte 0 and its
// magic is 0).  A loop over the moduli built from it is a fourteenth of the
// unrolled code, which keeps the column split's instruction stream in cache.
__constant__ uint32_t c_mod_rt[kL] = {mod_of(0), mod_of(1), mod_of(2),  mod_of(3),  mod_of(4),
                                      mod_of(5), mod_of(6), mod_of(7),  mod_of(8),  mod_of(9),
                                      mod_of(10), mod_of(11), mod_of(12), mod_of(13)};

__device__ __forceinline__ uint32_t residue_rt(const Limbs& x, int l) {
  if (residue_fp64(l)) return residue_fp64_path(x, c_inv_m[l], c_mod_rt[l]);
  return residue_int(x, c_split[l], c_mod_rt[l]);
}

// Residues of 16 consecutive values -> one 16-byte store per modulus plane,
// the moduli looped at run time.
__device__ __forceinline__ void store_planes_16_rt(const Limbs (&x)[16], uint8_t* base,
                                                   size_t plane_stride) {
#pragma unroll 1
  for (int l = 0; l < kL; ++l) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      w[q] = pack4(residue_rt(x[q * 4], l), residue_rt(x[q * 4 + 1], l),
                   residue_rt(x[q * 4 + 2], l), residue_rt(x[q * 4 + 3], l));
    *reinterpret_cast<uint4*>(base + l * plane_stride) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ int shift_for(double mx, bool nonfinite, int P) {
  if (nonfinite) return kShiftNonFinite;
  if (mx == 0.0) return kShiftZero;
  return P - (ilogb(mx) + 1);  // |v| <= mx < 2^(ilogb+1)
}

// Encoded row exponent for atomicMax across blocks: 0 = all zero,
// kExpNonFinite = a NaN/Inf seen, else ilogb(max) + 1 + kExpBias.
constexpr int kExpBias = 2048;
constexpr int kExpNonFinite = 0x7FFFFFFF;

__device__ __forceinline__ int shift_from_code(int code, int P) {
  if (code == kExpNonFinite) return kShiftNonFinite;
  if (code == 0) return kShiftZero;
  return P - (code - kExpBias);
}

// Place of an uncertified output in the list of those to recompute: at least `cap`
// where that is full.  A count past `cap` says so and is not raised further (a call
// may have more than 2^31 such outputs): it stays within the resident threads of
// cap + 1, as each looks before it adds one.
__device__ __forceinline__ int64_t list_place(int* count, int64_t cap) {
  if (*reinterpret_cast<volatile int*>(count) > cap) return cap;
  return atomicAdd(count, 1);
}

// The certificate by the operands' own 1-norms (the products grouped by expert).
// In units of C_int the quantisation error of an output is at most
// (||a_int||_1 + ||b_int||_1) / 2 + K / 4, and ||a_int||_1 <= sum |a| 2^sa + K / 2.
// A row's (column's) part of 2^kCertifyBits times that, rounded up: the sums and
// the conversion lose less than 2^-20 of it.
constexpr int kCertifyBits = 24;

__device__ __forceinline__ float certify_part(double sum, int shift, int64_t K) {
  if (shift == kShiftNonFinite || shift == kShiftZero) return 0.0f;
  const double units = scale2(sum, shift) + 0.5 * static_cast<double>(K);
  return __double2float_ru(0.5 * units * ((1 << kCertifyBits) * (1.0 + 0x1p-18)));
}

// A slab's sum, rounded up, as an int that keeps the order: the largest one over
// the slabs does not depend on their order, as a sum of them would.
__device__ __forceinline__ int norm_code(double sum) { return __double2hiint(sum) + 1; }
__device__ __forceinline__ double norm_of(int code) { return __hiloint2double(code, 0); }

// Operand rows contiguous in K (s_k == 1): one block per (row, batch), of
// 256 threads, or 512 for rows longer than 4096.  An f64 row of at most 16
// values per thread at a 16-byte aligned address is read into registers
// (four groups of four consecutive k, 4 * blockDim.x apart, so every load
// is coalesced) and reduced to the row maximum; the groups are then read
// again one at a time (L1 hits) and quantised.  Other rows take the same two
// passes with the second mostly from L2.  Four residues per thread per
// modulus make one coalesced 4-byte store.
constexpr int kSplitRowsMaxThreads = 512;

__host__ __device__ constexpr int split_rows_threads(int64_t K) {
  return K > 4096 && K <= 16 * kSplitRowsMaxThreads ? kSplitRowsMaxThreads : 256;
}

__device__ __forceinline__ void split_rows_body(const DotOperand& o, int64_t rows, int64_t K,
                                                int64_t rows_pad, int64_t Kp, int64_t batch,
                                                int P, uint8_t* __restrict__ planes,
                                                int* __restrict__ shifts, int64_t r, int64_t b) {
  __shared__ double s_max[kSplitRowsMaxThreads / 32];
  __shared__ int s_bad[kSplitRowsMaxThreads / 32];
  const bool live = r < rows;
  const int64_t base = b * o.s_b + r * o.s_r;
  const bool vec = o.f64 && o.s_k == 1 && (reinterpret_cast<uintptr_t>(o.f64 + base) & 15) == 0;
  const int64_t group = 4 * static_cast<int64_t>(blockDim.x);  // k covered by one group
  const bool in_regs = vec && K <= 4 * group;
  double v[16];
  double mx = 0.0;
  bool bad = false;
  if (in_regs) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int64_t k0 = g * group + threadIdx.x * 4;
      if (live && k0 + 4 <= K) {
        const double2* p = reinterpret_cast<const double2*>(o.f64 + base + k0);
        const double2 v01 = __ldg(p), v23 = __ldg(p + 1);
        v[g * 4 + 0] = v01.x;
        v[g * 4 + 1] = v01.y;
        v[g * 4 + 2] = v23.x;
        v[g * 4 + 3] = v23.y;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[g * 4 + j] = (live && k0 + j < K) ? o.f64[base + k0 + j] : 0.0;
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      bad |= !isfinite(v[j]);
      mx = fmax(mx, fabs(v[j]));
    }
  } else if (live) {
    for (int64_t k = threadIdx.x; k < K; k += blockDim.x) {
      const double x = op_value(o, base + k * o.s_k);
      bad |= !isfinite(x);
      mx = fmax(mx, fabs(x));
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    bad |= __shfl_xor_sync(0xffffffffu, static_cast<int>(bad), d) != 0;
  }
  if ((threadIdx.x & 31) == 0) {
    s_max[threadIdx.x >> 5] = mx;
    s_bad[threadIdx.x >> 5] = bad;
  }
  __syncthreads();
  mx = 0.0;
  bad = false;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    mx = fmax(mx, s_max[w]);
    bad |= s_bad[w] != 0;
  }
  const int shift = live ? shift_for(mx, bad, P) : 0;
  if (threadIdx.x == 0) shifts[b * rows_pad + r] = shift;
  const bool zero = !live || shift == kShiftNonFinite || shift == kShiftZero;
  const int sh = zero ? 0 : shift;
  const size_t plane_stride = static_cast<size_t>(batch) * rows_pad * Kp;
  uint8_t* row_out = planes + (static_cast<size_t>(b) * rows_pad + r) * Kp;
  if (in_regs) {
    // the groups again, one at a time from L1 (the first pass read them
    // through it): the residue code appears once rather than four times
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
      const int64_t k0 = g * group + threadIdx.x * 4;
      if (k0 < Kp) {
        double w[4];
        if (!zero && k0 + 4 <= K) {
          const double2* p = reinterpret_cast<const double2*>(o.f64 + base + k0);
          const double2 v01 = __ldg(p), v23 = __ldg(p + 1);
          w[0] = v01.x;
          w[1] = v01.y;
          w[2] = v23.x;
          w[3] = v23.y;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = (zero || k0 + j >= K) ? 0.0 : o.f64[base + k0 + j];
        }
        Limbs x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = limbs_of(quantise(w[j], sh));
        store_planes_n<4, true>(x, row_out + k0, plane_stride);
      }
    }
    return;
  }
  for (int64_t k0 = static_cast<int64_t>(threadIdx.x) * 4; k0 < Kp; k0 += 4 * blockDim.x) {
    double w[4];
    if (!zero && vec && k0 + 4 <= K) {
      const double2* p = reinterpret_cast<const double2*>(o.f64 + base + k0);
      const double2 v01 = p[0], v23 = p[1];
      w[0] = v01.x;
      w[1] = v01.y;
      w[2] = v23.x;
      w[3] = v23.y;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t k = k0 + j;
        w[j] = (zero || k >= K) ? 0.0 : op_value(o, base + k * o.s_k);
      }
    }
    Limbs x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = limbs_of(quantise(w[j], sh));
    store_planes_n<4, true>(x, row_out + k0, plane_stride);
  }
}

// Operand rows contiguous across rows (s_r == 1, e.g. B[K, N] row-major):
// blocks of 64 rows x 256 K.  Pairs of adjacent rows load as one 16-byte
// value when the layout allows it (paired_rows).
constexpr int kColTileR = 64;

__device__ __forceinline__ bool paired_rows(const DotOperand& o) {
  return o.f64 && o.s_r == 1 && (reinterpret_cast<uintptr_t>(o.f64) & 15) == 0 &&
         (o.s_k & 1) == 0 && (o.s_b & 1) == 0;
}

// Values of rows (row, row + 1) at k; zero outside the operand.
__device__ __forceinline__ void load_row_pair(const DotOperand& o, bool paired, int64_t b,
                                              int64_t row, int64_t k, int64_t rows, int64_t K,
                                              double& x0, double& x1) {
  x0 = x1 = 0.0;
  if (k >= K) return;
  const int64_t off = b * o.s_b + row * o.s_r + k * o.s_k;
  if (paired && row + 2 <= rows) {
    const double2 d = __ldcs(reinterpret_cast<const double2*>(o.f64 + off));
    x0 = d.x;
    x1 = d.y;
  } else {
    if (row < rows) x0 = op_value(o, off);
    if (row + 1 < rows) x1 = op_value(o, off + o.s_r);
  }
}

// Pass 1: per-row maximum over a kColmaxSlab-deep slab of K per block, merged
// across blocks with atomicMax on an encoded exponent (codes start at 0).
constexpr int kColmaxSlab = 128;

// kNorm: norm_codes also takes the largest slab sum of each row's magnitudes
// (norm_code).
template <bool kNorm = false>
__device__ __forceinline__ void colmax_body(const DotOperand& o, int64_t rows, int64_t K,
                                            int64_t rows_pad, int* __restrict__ codes,
                                            int64_t bx, int64_t by, int64_t b,
                                            int* __restrict__ norm_codes = nullptr) {
  __shared__ double s_max[8][kColTileR];
  __shared__ int s_bad[8][kColTileR];
  __shared__ double s_sum[kNorm ? 8 : 1][kColTileR];
  double n0 = 0.0, n1 = 0.0;
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t r0 = bx * kColTileR;
  const int64_t row = r0 + 2 * lane;
  const int64_t k0 = by * kColmaxSlab;
  double m0 = 0.0, m1 = 0.0;
  bool bad = false, bad1 = false;
  const int64_t k1 = k0 + kColmaxSlab < K ? k0 + kColmaxSlab : K;
  if (paired_rows(o) && row + 2 <= rows) {
    const double* p = o.f64 + b * o.s_b + row;
#pragma unroll 4
    for (int64_t k = k0 + ty; k < k1; k += 8) {
      const double2 d = __ldcs(reinterpret_cast<const double2*>(p + k * o.s_k));
      bad |= !isfinite(d.x);
      bad1 |= !isfinite(d.y);
      m0 = fmax(m0, fabs(d.x));
      m1 = fmax(m1, fabs(d.y));
      if constexpr (kNorm) {
        n0 += fabs(d.x);
        n1 += fabs(d.y);
      }
    }
  } else {
    for (int64_t k = k0 + ty; k < k1; k += 8) {
      double x0, x1;
      load_row_pair(o, false, b, row, k, rows, K, x0, x1);
      bad |= !isfinite(x0);
      bad1 |= !isfinite(x1);
      m0 = fmax(m0, fabs(x0));
      m1 = fmax(m1, fabs(x1));
      if constexpr (kNorm) {
        n0 += fabs(x0);
        n1 += fabs(x1);
      }
    }
  }
  s_max[ty][2 * lane] = m0;
  s_max[ty][2 * lane + 1] = m1;
  s_bad[ty][2 * lane] = bad;
  s_bad[ty][2 * lane + 1] = bad1;
  if constexpr (kNorm) {
    s_sum[ty][2 * lane] = n0;
    s_sum[ty][2 * lane + 1] = n1;
  }
  __syncthreads();
  if (threadIdx.x < kColTileR) {
    const int64_t r = r0 + threadIdx.x;
    double mx = 0.0;
    bool nf = false;
    for (int w = 0; w < 8; ++w) {
      mx = fmax(mx, s_max[w][threadIdx.x]);
      nf |= s_bad[w][threadIdx.x] != 0;
    }
    const int code = nf ? kExpNonFinite : (mx == 0.0 ? 0 : ilogb(mx) + 1 + kExpBias);
    if (r < rows && code != 0) atomicMax(&codes[b * rows_pad + r], code);
    if constexpr (kNorm) {
      double sum = 0.0;
      for (int w = 0; w < 8; ++w) sum += s_sum[w][threadIdx.x];
      if (r < rows && sum > 0.0) atomicMax(&norm_codes[b * rows_pad + r], norm_code(sum));
    }
  }
}

constexpr int kMnCols = 4, kMnRows = 256 * kMnCols, kMnSlab = 2;

constexpr int kMnStages = 4;

__device__ __forceinline__ void cp_async8(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src),
               "r"(valid ? 8 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Split of an f64 operand whose rows are contiguous into row-contiguous
// planes [l][Kp][rows_pad] with its loads made asynchronous:
// block (c, g) of gridDim.x = chunks of kMnRows rows takes chunk c at
// k = g, g + gridDim.y, ...; each thread copies its four values of the next
// kMnStages - 1 k into its own shared-memory slots with cp.async (zero fill
// past K or the rows) while it quantises the current ones, so no register
// holds a load in flight and the column shifts are loaded once per block.
// Two blocks per SM: with four (64 registers) the k loop keeps every 1 / m
// in a register and spills, and runs at half the speed; six stages were no
// faster than four.  (The same pipeline for A's rows, with B's column
// maxima in a kernel of their own, was slower than split_rows_colmax_kernel:
// 0.095 + 0.030 ms against 0.102 ms for both.)
__device__ __forceinline__ void split_mn_async_body(const DotOperand& o, int64_t off, bool even_off,
                                                    int64_t rows, int64_t K, int64_t rows_pad,
                                                    int64_t Kp, int P,
                                                    const int* __restrict__ codes,
                                                    uint8_t* __restrict__ planes,
                                                    size_t plane_stride,
                                                    int* __restrict__ shifts) {
  __shared__ __align__(16) double stage[kMnStages][256][kMnCols];
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kMnRows + threadIdx.x * kMnCols;
  if (r0 >= rows_pad) return;  // rows_pad is a multiple of kMnCols
  int sh[kMnCols];
  bool z[kMnCols];
#pragma unroll
  for (int j = 0; j < kMnCols; ++j) {
    const int64_t r = r0 + j;
    const int sv = r < rows ? shift_from_code(codes[r], P) : 0;
    if (blockIdx.y == 0) shifts[r] = sv;
    z[j] = r >= rows || sv == kShiftNonFinite || sv == kShiftZero;
    sh[j] = z[j] ? 0 : sv;
  }
  const bool vec = r0 + kMnCols <= rows && (o.s_k & 1) == 0 && even_off &&
                   (reinterpret_cast<uintptr_t>(o.f64) & 15) == 0;
  // addresses of copies that read nothing (zero fill) still point inside
  // the operand
  const double* base = o.f64 + off + (r0 < rows ? r0 : 0);
  const int64_t kstep = gridDim.y;
  auto issue = [&](int64_t k, int slot) {
    double* dst = stage[slot][threadIdx.x];
    const bool in = k < K;
    const double* src = base + (in ? k : 0) * o.s_k;
    if (vec) {
      cp_async16(dst, src, in);
      cp_async16(dst + 2, src + 2, in);
    } else {
#pragma unroll
      for (int j = 0; j < kMnCols; ++j) {
        const bool valid = in && r0 + j < rows;
        cp_async8(dst + j, valid ? src + j : base, valid);
      }
    }
  };
  // prologue: the first kMnStages - 1 k of this block (empty groups past Kp)
  int64_t kn = blockIdx.y;
#pragma unroll
  for (int st = 0; st < kMnStages - 1; ++st, kn += kstep) {
    if (kn < Kp) issue(kn, st);
    cp_async_commit();
  }
  int slot = 0;
#pragma unroll 1
  for (int64_t k = blockIdx.y; k < Kp; k += kstep) {
    if (kn < Kp) issue(kn, (slot + kMnStages - 1) % kMnStages);
    cp_async_commit();
    kn += kstep;
    cp_async_wait<kMnStages - 1>();  // this thread's copies of k have landed
    const double* w = stage[slot][threadIdx.x];
    Limbs x[kMnCols];
#pragma unroll
    for (int j = 0; j < kMnCols; ++j) x[j] = limbs_of(quantise(z[j] ? 0.0 : w[j], sh[j]));
    store_planes_n<kMnCols, true>(x, planes + static_cast<size_t>(k) * rows_pad + r0,
                                  plane_stride);
    slot = slot + 1 == kMnStages ? 0 : slot + 1;
  }
  cp_async_wait<0>();
}

// ---- tcgen05 int8 GEMM primitives

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded wait: false (and an error code recorded) after ~2 s, or at once if
// another role of any CTA has already given up.  The first try is inlined
// into the pipeline loops; only a wait that has to spin makes the call (a
// call per K-block cost the GEMM 9% of its time).
__device__ __noinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity, int* err, int code) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*reinterpret_cast<volatile int*>(err) != 0) return false;
    if (clock64() - t0 > kTimeoutCycles) {
      atomicCAS(err, 0, code);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return mbar_try_wait(bar, parity) || mbar_wait_slow(bar, parity, err, code);
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// K-major operand tile with 128-byte swizzle: rows of 128 B, 8-row atoms of
// 1024 B (stride byte offset), descriptor version 1 (sm_100).
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(1) << 16;          // leading byte offset (unused here): 16 B
  d |= static_cast<uint64_t>(1024 >> 4) << 32;  // stride byte offset
  d |= static_cast<uint64_t>(1) << 46;          // version
  d |= static_cast<uint64_t>(2) << 61;          // SWIZZLE_128B
  return d;
}

// MN-major operand tile with 128-byte swizzle, 128 bytes (one swizzle atom)
// of M or N per CTA: rows of 128 B along MN, one per k; 8-k atoms of 1024 B
// (stride byte offset).  The leading byte offset steps between 128-byte MN
// atoms, of which a CTA's tile has one, so it is never applied.
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(1) << 16;          // leading byte offset (unused here): 16 B
  d |= static_cast<uint64_t>(1024 >> 4) << 32;  // stride byte offset: 8 k of 128 B
  d |= static_cast<uint64_t>(1) << 46;          // version
  d |= static_cast<uint64_t>(2) << 61;          // SWIZZLE_128B
  return d;
}

// kind::i8, D = s32, A = B = unsigned 8-bit (residues in [0, m)), both
// K-major, N = 256, M = 128.
constexpr uint32_t kIdesc = (2u << 4) | (0u << 7) | (0u << 10) |
                            (static_cast<uint32_t>(kTileN >> 3) << 17) |
                            (static_cast<uint32_t>(kTileM >> 4) << 24);

__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
        "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
        "=r"(v[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// v mod m for 0 <= v < 2^31 (a u8 x u8 -> s32 accumulator, K <= 32768):
// floor(v / m) = umulhi(v, ceil(2^39 / m)) >> 7 exactly, because
// v * (ceil(2^39 / m) * m - 2^39) < 2^31 * 2^8 = 2^39.  Integer pipes only.
__host__ __device__ constexpr uint32_t epilogue_magic(uint32_t m) {
  return static_cast<uint32_t>(((1ull << 39) + m - 1) / m);
}

__device__ __forceinline__ uint32_t mod_u8(uint32_t v, uint32_t m, uint32_t magic) {
  return v - (__umulhi(v, magic) >> 7) * m;
}

// Four accumulators -> their residues as the bytes of one word.
__device__ __forceinline__ uint32_t mod_pack4(const uint32_t* v, uint32_t m, uint32_t magic) {
  return __byte_perm(__byte_perm(mod_u8(v[0], m, magic), mod_u8(v[1], m, magic), 0x0040),
                     __byte_perm(mod_u8(v[2], m, magic), mod_u8(v[3], m, magic), 0x0040), 0x5410);
}

// Epilogue warps of each CTA (eight, sharing the columns, were 1 to 3% slower).
constexpr int kEpilogueWarps2 = 4;
constexpr int kGemm2Threads = 64 + 32 * kEpilogueWarps2;
constexpr int kStages2 = 3;
constexpr int kSub2 = 2;  // 128-byte K sub-tiles per stage
constexpr int kStage2 = kTileM * kTileK;  // 16 KB: A rows, or half of the B tile
// Residues of a CTA's 128 x 256 outputs on their way to memory: a thread
// holds a row of the accumulator, so a store from its registers would write 16
// bytes of 32 rows at a time; staged here, each warp stores whole lines of its
// rows.
constexpr int kOut2 = kTileM * 256;
constexpr uint32_t kIdesc2 = (2u << 4) | (0u << 7) | (0u << 10) | ((256u >> 3) << 17) |
                             ((256u >> 4) << 24);
constexpr uint32_t kIdescAMajorMN = 1u << 15;  // A MN-major
constexpr uint32_t kIdescBMajorMN = 1u << 16;  // B MN-major

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_id_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t nclusters_x() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%nclusterid.x;" : "=r"(r));
  return r;
}
// Shared::cluster address of the same variable in CTA rank 0 of the cluster.
__device__ __forceinline__ uint32_t in_rank0(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __noinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int* err, int code) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait_cluster(bar, parity)) {
    if (*reinterpret_cast<volatile int*>(err) != 0) return false;
    if (clock64() - t0 > kTimeoutCycles) {
      atomicCAS(err, 0, code);
      return false;
    }
  }
  return true;
}

// Arrival on another CTA's barrier, ordered after this thread's reads of TMEM
// (tcgen05.wait::ld and the fence before it), not after its global stores: with
// .release.cluster it waited for them too, which held the GEMM at 1.9 POPS for
// K = 1024 (2.6 now) and at 3.32 for K = 4096 (3.46 now).
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y,
                                                 uint32_t mbar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(mbar_cluster)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int x, int y,
                                                 int z, uint32_t mbar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(mbar_cluster)
      : "memory");
}

__device__ __forceinline__ void mma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// Arrive (when the prior MMAs complete) on the barrier at this address in
// both CTAs of the pair.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
  const uint16_t mask = 0x3;
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(mask)
      : "memory");
}

__device__ __forceinline__ void mma_commit_pair_self(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

// A unit of the CTA-pair GEMM: a 256 x 256 output tile of one modulus.
struct GemmTile {
  int l;         // modulus
  int stages;    // pipeline stages of kSub2 * kTileK of the contraction
  int k0;        // first position of the contraction
  int a, za;     // this CTA's first row of A (over all planes) or, MN-major, its
                 // first row in plane za
  int b, zb;     // the same of B
  uint8_t* out;  // residue of this CTA's first row and the tile's first column
  int rows;      // rows to store of the CTA's 128 (kMasked)
};

// The persistent GEMM over the units of `work`, shared by dot_general and the
// grouped products: Work gives units(), at(unit, CTA rank) and whether A and
// B are MN-major planes (3-D tensor maps {rows, contraction, planes}).
template <class Work>
__device__ __forceinline__ void gemm2_body(const CUtensorMap& tmap_a, const CUtensorMap& tmap_b,
                                           const Work& work, int64_t Np, int* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kStages2 * kSub2 * kStage2;
  uint8_t* smem_out = smem + 2 * kStages2 * kSub2 * kStage2;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_out + kOut2);
  uint64_t* empty = full + kStages2;
  uint64_t* tfull = empty + kStages2;
  uint64_t* tempty = tfull + 2;
  uint64_t* drained = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages2; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * kEpilogueWarps2);  // the epilogue warps of both CTAs
    }
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t cid = cluster_id_x(), ncl = nclusters_x();
  const int64_t units = work.units();

  if (warp == 0) {
    // ---- TMA producer (both CTAs) ----
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_a)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_b)) : "memory");
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      // each unit's place is looked up while the one before it is under way
      GemmTile next = cid < units ? work.at(cid, rank) : GemmTile{};
      for (int64_t u = cid; u < units && ok; u += ncl) {
        const GemmTile w = next;
        if (u + ncl < units) next = work.at(u + ncl, rank);
        for (int kb = 0; kb < w.stages; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, err, 11)) {
            ok = false;
            break;
          }
          if (leader) mbar_expect_tx(&full[stage], 4 * kSub2 * kStage2);
          const uint32_t full0 = in_rank0(&full[stage]);
#pragma unroll
          for (int sub = 0; sub < kSub2; ++sub) {
            const int x = w.k0 + (kb * kSub2 + sub) * kTileK;
            uint8_t* sa = smem_a + (stage * kSub2 + sub) * kStage2;
            uint8_t* sb = smem_b + (stage * kSub2 + sub) * kStage2;
            if constexpr (Work::kAMn) tma_load_3d_pair(sa, &tmap_a, w.a, x, w.za, full0);
            else tma_load_2d_pair(sa, &tmap_a, x, w.a, full0);
            if constexpr (Work::kBMn) tma_load_3d_pair(sb, &tmap_b, w.b, x, w.zb, full0);
            else tma_load_2d_pair(sb, &tmap_b, x, w.b, full0);
          }
          if (++stage == kStages2) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) {
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer (even CTA only) ----
    if (lane == 0 && leader) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      int next = cid < units ? work.at(cid, rank).stages : 0;
      for (int64_t u = cid; u < units && ok; u += ncl) {
        if (!mbar_wait_cluster(&tempty[acc], acc_phase ^ 1, err, 12)) break;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(acc * 256);
        constexpr uint32_t idesc = kIdesc2 | (Work::kAMn ? kIdescAMajorMN : 0u) |
                                   (Work::kBMn ? kIdescBMajorMN : 0u);
        const int stages = next;
        if (u + ncl < units) next = work.at(u + ncl, rank).stages;
        for (int kb = 0; kb < stages; ++kb) {
          if (!mbar_wait(&full[stage], phase, err, 13)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int sub = 0; sub < kSub2; ++sub) {
            const uint32_t a0 = smem_u32(smem_a + (stage * kSub2 + sub) * kStage2);
            const uint32_t b0 = smem_u32(smem_b + (stage * kSub2 + sub) * kStage2);
#pragma unroll
            for (int k = 0; k < kTileK / 32; ++k) {
              // 32 k per instruction: 32 bytes along a K-major row, or 32
              // rows of 128 bytes of an MN-major tile
              const uint64_t adesc = Work::kAMn ? sdesc_mn(a0 + k * 32 * 128) : sdesc(a0 + k * 32);
              const uint64_t bdesc = Work::kBMn ? sdesc_mn(b0 + k * 32 * 128) : sdesc(b0 + k * 32);
              mma_i8_pair(d, adesc, bdesc, idesc, (kb | sub | k) != 0 ? 1u : 0u);
            }
          }
          mma_commit_pair(&empty[stage]);
          if (++stage == kStages2) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit_pair(&tfull[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      mma_commit_pair_self(drained);
      const long long t0 = clock64();
      while (!mbar_try_wait(drained, 0) && clock64() - t0 < kTimeoutCycles) {
      }
    }
  } else {
    // ---- epilogue (both CTAs; warps 2.., TMEM lanes 32*(warp%4) .., the
    // columns shared out among the warps of the same lanes) ----
    const int quad = warp & 3;
    constexpr int kCols = 256 * 4 / kEpilogueWarps2;
    const int col0 = (warp - 2) / 4 * kCols;
    const uint32_t tempty0[2] = {in_rank0(&tempty[0]), in_rank0(&tempty[1])};
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int64_t u = cid; u < units; u += ncl) {
      const GemmTile w = work.at(u, rank);
      if (!mbar_wait(&tfull[acc], acc_phase, err, 14)) break;
      tc_fence_after();
      const uint32_t m = static_cast<uint32_t>(mod_of(w.l));
      const uint32_t magic = epilogue_magic(m);
      const uint32_t tbase = tmem + (static_cast<uint32_t>(quad * 32) << 16) +
                             static_cast<uint32_t>(acc * 256);
      // the warp's 32 rows x kCols bytes, 16-byte words swizzled by the row
      constexpr int kWords = kCols / 16;
      uint4* own = reinterpret_cast<uint4*>(smem_out) + (warp - 2) * 32 * kWords;
#pragma unroll 1
      for (int c0 = 0; c0 < kCols; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(tbase + col0 + c0, v);
        uint32_t packed[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) packed[q] = mod_pack4(v + q * 4, m, magic);
        const int word = c0 / 16;
        own[lane * kWords + (word ^ lane % kWords)] =
            make_uint4(packed[0], packed[1], packed[2], packed[3]);
        own[lane * kWords + ((word + 1) ^ lane % kWords)] =
            make_uint4(packed[4], packed[5], packed[6], packed[7]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(tempty0[acc]);
      constexpr int kRowsAtOnce = 32 / kWords;
#pragma unroll 4
      for (int r0 = 0; r0 < 32; r0 += kRowsAtOnce) {
        const int r = r0 + lane / kWords, word = lane % kWords;
        if (!Work::kMasked || quad * 32 + r < w.rows)
          *reinterpret_cast<uint4*>(w.out + static_cast<int64_t>(quad * 32 + r) * Np + col0 +
                                    word * 16) = own[r * kWords + (word ^ r % kWords)];
      }
      __syncwarp();
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }

  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

__device__ __forceinline__ void put_result(const DotResult& c, int64_t idx, double v) {
  if (c.f64) {
    c.f64[idx] = v;
  } else {
    const ds2 d = from_f64(v);
    c.hi[idx] = d.hi;
    c.lo[idx] = d.lo;
  }
}

// Byte q of `word` as an f64: the bits of 2^52 + byte, minus 2^52 -- one
// add on the FP64 pipe instead of a quarter-rate integer conversion.
__device__ __forceinline__ double byte_to_f64(uint32_t word, int q) {
  const uint32_t byte = __byte_perm(word, 0u, 0x4440u + static_cast<uint32_t>(q));
  return __dsub_rn(__hiloint2double(0x43300000, static_cast<int>(byte)), 0x1p52);
}

// 2^e as an f64 for a normal exponent.
__device__ __forceinline__ double pow2_normal(int e) {
  return __longlong_as_double(static_cast<long long>(1023 + e) << 52);
}

// Error certificate.  A row of A enters the GEMM as a_int = rint(a 2^sa)
// with |a_int| <= 2^P, so |a 2^sa - a_int| <= 1/2; likewise for B.  In units
// of C_int the quantisation error of an output is at most
//     (||b_int||_1 + ||a_int||_1) / 2 + K / 4 <= K 2^P (+ K / 4),
// and the CRT's low limb adds below 2^34.  An output is certified when
// |C_int| >= 2^24 (K 2^P + 2^35): its error is then at most 2^-24 |C| (in
// practice far less: the quantisation errors are not aligned).  This bound
// is relative to the row maximum of A and the column maximum of B, so it
// fails exactly where those maxima do not take part in the output: a large
// entry facing zeros, values spread over many binades, or cancellation.
// Such outputs are recomputed with a compensated dot product (fix_kernel).

__device__ __forceinline__ bool shift_ordinary(int s) {
  return s != kShiftNonFinite && s != kShiftZero;
}

// ---- recomputation of uncertified outputs ----------------------------------
//
// sum_k a_ik b_kj by Ogita, Rump and Oishi's Dot2: each product split exactly
// by an FMA, the products summed with two_sum and the error terms summed
// aside, which is as accurate as the dot product evaluated in twice the
// working precision and then rounded.  Operands are scaled by 2^(sa - P) and
// 2^(sb - P) (below 1 in magnitude, so no product overflows); the scaling is
// undone at the end.

struct Dot2 {
  double p = 0.0, s = 0.0;
};

__device__ __forceinline__ void two_sum64(double a, double b, double& s, double& e) {
  s = __dadd_rn(a, b);
  const double bb = __dsub_rn(s, a);
  e = __dadd_rn(__dsub_rn(a, __dsub_rn(s, bb)), __dsub_rn(b, bb));
}

__device__ __forceinline__ void dot2_add(Dot2& d, double x, double y) {
  const double h = __dmul_rn(x, y);
  const double r = __fma_rn(x, y, -h);
  double q;
  two_sum64(d.p, h, d.p, q);
  d.s = __dadd_rn(d.s, __dadd_rn(q, r));
}

__device__ __forceinline__ void dot2_merge(Dot2& d, const Dot2& o) {
  double q;
  two_sum64(d.p, o.p, d.p, q);
  d.s = __dadd_rn(__dadd_rn(d.s, o.s), q);
}

// ---------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

int make_tmap(CUtensorMap* map, const void* base, int64_t Kp, int64_t rows, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return set_error(DS_INTERNAL, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(Kp), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(Kp)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(kTileK), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides,
                  box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(DS_INTERNAL, "cuTensorMapEncodeTiled failed");
  return DS_OK;
}

// Row-contiguous planes [planes][Kp][Np] (MN-major B): boxes of 128 rows
// (128 bytes) x 128 k of one plane.  k past Kp reads as zero.
int make_tmap_mn(CUtensorMap* map, const void* base, int64_t Np, int64_t Kp, int64_t planes) {
  auto fn = encode_fn();
  if (!fn) return set_error(DS_INTERNAL, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(Np), static_cast<cuuint64_t>(Kp),
                              static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(Np), static_cast<cuuint64_t>(Np * Kp)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(kTileN / 2), static_cast<cuuint32_t>(kTileK),
                             1};
  const cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides,
                  box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(DS_INTERNAL, "cuTensorMapEncodeTiled failed");
  return DS_OK;
}

size_t gemm_smem_bytes() {
  return 1024 + kStages * (kStageA + kStageB) + (2 * kStages + 5) * sizeof(uint64_t) + 16;
}

size_t gemm2_smem_bytes() {
  return 1024 + 2 * kStages2 * kSub2 * kStage2 + kOut2 + (2 * kStages2 + 5) * sizeof(uint64_t) + 16;
}

}  // namespace
}  // namespace dsb
