// The linear recurrence h_t = a_t h_{t-1} + x_t along a sequence, and its
// gradient.
//
// A step is the map s -> a s + x; a run of steps composes to s -> P s + S with
// P the product of the coefficients and S the run's result from a zero state.
// The gradient is the same recurrence backwards in time: with p = T - 1 - t,
//     g_p = grad_h + a_{t+1} g_{p-1},
// so one kernel does both, reading its coefficients one row later.
//
// Both are bound by HBM: 24 (gradient: 40) bytes of f64 per value for one FMA.
// Every value is therefore read once.  A unit of work is CT channels x a chunk
// of S * R steps, held in registers by 256 threads of R steps each; each
// thread composes its steps, a scan over the S threads of a channel joins
// them, and once the state at the chunk's start is known each thread runs its
// steps again from its own start and stores them.
//
// The state at a chunk's start is the last one's end where a block takes all
// chunks of its channels (many channels).  Otherwise it comes from the chunks
// before it through the workspace: chunks stand in rounds of `round` chunks; a
// chunk publishes (P, S) as soon as it has read its values; it takes those of the
// earlier chunks of its round and the state the last round ended with, and
// applies them in order; the round's last chunk publishes that state.  So the
// chain has one hop per round rather than per chunk, and the order of every
// operation is fixed by the shape.  A published value is its own message: the
// workspace starts as all ones (a NaN no result has), and a reader polls the
// value itself, so there is no flag, fence or barrier between the two.
//
// Blocks stay on their SM; the next unit's values travel to shared memory
// (cp.async, each thread into slots of its own) while the current one is worked
// on.  Chunks of all tiles are taken from a counter, chunk by chunk, one ahead:
// what a unit waits for is an earlier unit, and the earliest unfinished one is
// always some block's current one, so the chain moves; each wait is bounded
// (about 2 s), after which the unit works with NaN.
//
// A composed map is not the steps where a product of coefficients leaves the f64
// range and the states do not.  Such a channel's chunk is stepped through, thread
// after thread, and hands on the state at its end in place of its map (see tiny):
// with every chunk stepped [8, 2048, 1024] of f64 takes 119 us instead of 69,
// [1, 65536, 250], whose chunks then wait for one another, 2.7 ms instead of 110 us.
//
// Measured on one B200 (cold L2, launch included): f64 [8, 2048, 1024] 76 us =
// 5.3 TB/s, its gradient 121 us = 5.5 TB/s, [1, 65536, 250] 113 us, f32 [4, 4096,
// 2048] 90 us.  A plain kernel that reads two arrays of that size and writes a
// third takes 70 us (5.8 TB/s), whatever the width of its rows.
#include <mutex>
#include <vector>

#include "common.cuh"
#include "ds_arith.cuh"
#include "kernels.h"
#include "profile.h"

namespace dsb {
namespace {

// Element types: f64, f32, packed DS pair.  Held as loaded, computed with as
// the exact f64 value, stored with one rounding (a pair: hi = f32(v),
// lo = f32(v - hi)).
template <class T> struct SeqIO;
template <> struct SeqIO<double> {
  static __device__ __forceinline__ double load(const double* p) { return __ldcs(p); }
  static __device__ __forceinline__ double value(double v) { return v; }
  static __device__ __forceinline__ double zero() { return 0.0; }
  static __device__ __forceinline__ double one() { return 1.0; }
  static __device__ __forceinline__ void store(double* p, double v) { __stcs(p, v); }
  template <int V> static __device__ __forceinline__ void put(double* p, const double (&v)[V]) {
    if constexpr (V == 1) store(p, v[0]);
    else __stcs(reinterpret_cast<double2*>(p), make_double2(v[0], v[1]));
  }
};
template <> struct SeqIO<float> {
  static __device__ __forceinline__ float load(const float* p) { return __ldcs(p); }
  static __device__ __forceinline__ double value(float v) { return static_cast<double>(v); }
  static __device__ __forceinline__ float zero() { return 0.0f; }
  static __device__ __forceinline__ float one() { return 1.0f; }
  static __device__ __forceinline__ void store(float* p, double v) {
    __stcs(p, __double2float_rn(v));
  }
  template <int V> static __device__ __forceinline__ void put(float* p, const double (&v)[V]) {
    if constexpr (V == 1) store(p, v[0]);
    else __stcs(reinterpret_cast<float2*>(p),
                make_float2(__double2float_rn(v[0]), __double2float_rn(v[1])));
  }
};
template <> struct SeqIO<float2> {
  static __device__ __forceinline__ float2 load(const float2* p) { return __ldcs(p); }
  static __device__ __forceinline__ double value(float2 v) { return to_f64(ds2{v.x, v.y}); }
  static __device__ __forceinline__ float2 zero() { return make_float2(0.0f, 0.0f); }
  static __device__ __forceinline__ float2 one() { return make_float2(1.0f, 0.0f); }
  static __device__ __forceinline__ void store(float2* p, double v) {
    const ds2 d = from_f64(v);
    __stcs(p, make_float2(d.hi, d.lo));
  }
  template <int V> static __device__ __forceinline__ void put(float2* p, const double (&v)[V]) {
    if constexpr (V == 1) {
      store(p, v[0]);
    } else {
      const ds2 d = from_f64(v[0]), e = from_f64(v[1]);
      __stcs(reinterpret_cast<float4*>(p), make_float4(d.hi, d.lo, e.hi, e.lo));
    }
  }
};

constexpr int kThreads = 256;
constexpr long long kTimeoutCycles = 4000000000LL;  // ~2 s at 1.9 GHz

// Sequences of at most kShort steps run one thread per channel.
constexpr int64_t kShort = 16;

template <class E>
__global__ void __launch_bounds__(kThreads)
scan_short_kernel(const E* __restrict__ a, const E* __restrict__ b, const E* __restrict__ h0,
                  E* __restrict__ h, int64_t C, int64_t T, int64_t D) {
  wait_previous_grid();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= C) return;
  const int64_t seq = c / D;
  int64_t at = seq * T * D + (c - seq * D);
  double s = h0 ? SeqIO<E>::value(SeqIO<E>::load(h0 + c)) : 0.0;
#pragma unroll 4
  for (int64_t t = 0; t < T; ++t, at += D) {
    s = __fma_rn(SeqIO<E>::value(SeqIO<E>::load(a + at)), s,
                 SeqIO<E>::value(SeqIO<E>::load(b + at)));
    SeqIO<E>::store(h + at, s);
  }
}

template <class E>
__global__ void __launch_bounds__(kThreads)
scan_vjp_short_kernel(const E* __restrict__ a, const E* __restrict__ h, const E* __restrict__ gh,
                      const E* __restrict__ h0, E* __restrict__ ga, E* __restrict__ gb,
                      E* __restrict__ gh0, int64_t C, int64_t T, int64_t D) {
  wait_previous_grid();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= C) return;
  const int64_t seq = c / D;
  int64_t at = (seq * T + T - 1) * D + (c - seq * D);
  double carry = 0.0;  // a_{t+1} g_{t+1}
#pragma unroll 4
  for (int64_t t = T - 1; t >= 0; --t, at -= D) {
    const double g = __dadd_rn(SeqIO<E>::value(SeqIO<E>::load(gh + at)), carry);
    const E before = t > 0 ? SeqIO<E>::load(h + at - D)
                           : (h0 ? SeqIO<E>::load(h0 + c) : SeqIO<E>::zero());
    SeqIO<E>::store(gb + at, g);
    SeqIO<E>::store(ga + at, __dmul_rn(g, SeqIO<E>::value(before)));
    carry = __dmul_rn(SeqIO<E>::value(SeqIO<E>::load(a + at)), g);
  }
  SeqIO<E>::store(gh0 + c, carry);
}

struct Map {
  double p, s;  // state -> p state + s
};

__device__ __forceinline__ bool not_finite(double v) {
  return (__double2hiint(v) & 0x7ff00000) == 0x7ff00000;
}

__device__ __forceinline__ double apply(const Map& m, double state) {
  return __fma_rn(m.p, state, m.s);
}

// first, then second.
__device__ __forceinline__ Map compose(const Map& first, const Map& second) {
  return Map{__dmul_rn(second.p, first.p), apply(second, first.s)};
}

// Products of coefficients may leave the f64 range where no state does: one that
// overflows meets a tiny state, or a coefficient of zero (inf 0 is NaN, the state
// is 0); one that underflows meets a large state, or coefficients that make it
// large again.  So a channel's chunk is stepped through one step after another, as
// the loop does, where
//   a map of its threads or of their composition is not finite,
//   a product is below the normal range (tiny) and a coefficient of the chunk is
//   above 1, or
//   a tiny product meets a state above 2^64.
// Elsewhere a tiny product is below 2^-1021 and off by at most 2^-1075 in each of
// up to 1024 roundings, and the state that it is multiplied with is at most 2^71
// (a thread's is at most 2^64): a result is off by at most 2^-994.
__device__ __forceinline__ bool tiny(double p) {
  return (__double2hiint(p) & 0x7ff00000) == 0;
}
__device__ __forceinline__ bool beyond(double state) {
  return (__double2hiint(state) & 0x7fffffff) >= (1023 + 64) << 20;
}
__device__ __forceinline__ bool large(double state) {
  return beyond(state) && !not_finite(state);
}

// Bit 30 is set for |a| >= 1 + 2^-20 (1024 factors below that are 2^0.002), also
// in the bitwise or of several.  A NaN may not set it; it is not finite.
__device__ __forceinline__ uint32_t growth_bits(double a) {
  return static_cast<uint32_t>(__double2hiint(a)) + 0xfffffu;
}
__device__ __forceinline__ bool grows(uint32_t bits) { return (bits & 0x40000000u) != 0; }

template <class E>
struct ChunkArgs {
  const E *a, *x, *h, *h0;
  E *out, *ga, *gh0;
  uint32_t C, D;      // channels of all sequences, of one
  int64_t T;          // steps
  uint32_t tiles;     // of CT channels
  uint32_t chunks, units;
  uint32_t round;     // chunks per round, at most kMaxRound
  uint32_t* counter;  // units taken, minus one (null: a block takes whole tiles)
  uint32_t* err;      // all ones, or 1 when a wait has run out
  ulonglong2* maps;   // [chunks][tiles][CT]
  uint64_t* states;   // [rounds][tiles][CT]
};

constexpr int kMaxRound = 16;
constexpr uint64_t kEmpty = ~0ull;

// The bits of v, a NaN's made the ordinary one (never kEmpty).
__device__ __forceinline__ uint64_t message(double v) {
  return v == v ? static_cast<uint64_t>(__double_as_longlong(v)) : 0x7ff8000000000000ull;
}

__device__ __forceinline__ void put_map(ulonglong2* at, const Map& m) {
  asm volatile(
      "{\n\t.reg .b128 v;\n\tmov.b128 v, {%1, %2};\n\tst.relaxed.gpu.global.b128 [%0], v;\n\t}" ::"l"(
          at),
      "l"(message(m.p)), "l"(message(m.s))
      : "memory");
}
__device__ __forceinline__ ulonglong2 look_at_map(const ulonglong2* at) {
  ulonglong2 v;
  asm volatile(
      "{\n\t.reg .b128 v;\n\tld.relaxed.gpu.global.b128 v, [%2];\n\tmov.b128 {%0, %1}, v;\n\t}"
      : "=l"(v.x), "=l"(v.y)
      : "l"(at)
      : "memory");
  return v;
}
__device__ __forceinline__ void put_state(uint64_t* at, double v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(at), "l"(message(v)) : "memory");
}
__device__ __forceinline__ uint64_t look_at_state(const uint64_t* at) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(at) : "memory");
  return v;
}

// Whether to look again: false about 2 s after t0, or when another wait has
// run out.  Asked every 64th look only: it reads memory itself.
__device__ __noinline__ bool keep_waiting(long long t0, uint32_t* err) {
  if (*reinterpret_cast<volatile uint32_t*>(err) == 1u) return false;
  if (clock64() - t0 <= kTimeoutCycles) return true;
  *reinterpret_cast<volatile uint32_t*>(err) = 1u;
  return false;
}

// Looks until the value is there; false when the wait runs out.
template <class Look>
__device__ __forceinline__ bool poll(Look look, uint32_t* err) {
  const long long t0 = clock64();
  for (uint32_t n = 1; !look(); ++n)
    if (n % 64 == 0 && !keep_waiting(t0, err)) return false;
  return true;
}

__device__ __forceinline__ Map wait_map(const ulonglong2* at, ulonglong2 v, uint32_t* err) {
  if (v.x == kEmpty && !poll([&] { return (v = look_at_map(at)).x != kEmpty; }, err))
    v.x = v.y = 0x7ff8000000000000ull;
  return Map{__longlong_as_double(static_cast<long long>(v.x)),
             __longlong_as_double(static_cast<long long>(v.y))};
}

__device__ __forceinline__ double wait_state(const uint64_t* at, uint32_t* err) {
  uint64_t v = kEmpty;
  if (!poll([&] { return (v = look_at_state(at)) != kEmpty; }, err)) v = 0x7ff8000000000000ull;
  return __longlong_as_double(static_cast<long long>(v));
}

// The state at the end of a chunk that was stepped through, in place of its map: an
// infinite product says so.
constexpr uint64_t kEnd = 0x7ff0000000000000ull;
__device__ __forceinline__ void put_end(ulonglong2* at, double end) {
  put_map(at, Map{__longlong_as_double(static_cast<long long>(kEnd)), end});
}

// The state after the chunk whose message at `at` was m, from the one before it.
// A tiny product and a large state: that chunk gives its end after its map.
__device__ __forceinline__ double pass(const ulonglong2* at, const Map& m, double state,
                                       uint32_t* err) {
  if (not_finite(m.p)) return m.s;
  if (!(tiny(m.p) && large(state))) return apply(m, state);
  ulonglong2 v;
  if (!poll([&] { return (v = look_at_map(at)).x == kEnd; }, err)) v.y = 0x7ff8000000000000ull;
  return __longlong_as_double(static_cast<long long>(v.y));
}

// V neighbouring channels, moved as one word.
template <class E, int V>
struct alignas(sizeof(E) * V) Word {
  E v[V];
};

template <class W>
__device__ __forceinline__ void copy_async(W* dst, const void* src) {
  static_assert(sizeof(W) == 4 || sizeof(W) == 8 || sizeof(W) == 16, "cp.async sizes");
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (sizeof(W) == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(src), "n"(sizeof(W))
                 : "memory");
}

// One thread's part of a unit: R steps of V channels.
template <int V, int CT, int R>
struct Part {
  static constexpr int N = CT / V, S = kThreads / N;
  uint32_t chunk, tile;
  int64_t row;  // element of the first step's row
  int n;        // steps it has
  // first channel, and first step (gradient: counted from the end)
  __device__ __forceinline__ uint32_t c() const { return tile * CT + threadIdx.x % N * V; }
  __device__ __forceinline__ int64_t p0() const {
    return (static_cast<int64_t>(chunk) * S + threadIdx.x / N) * R;
  }
};

template <class E, int V, int CT, int R, bool kGrad>
__device__ __forceinline__ Part<V, CT, R> part_of(const ChunkArgs<E>& p, uint32_t unit) {
  Part<V, CT, R> q;
  q.chunk = unit / p.tiles;
  q.tile = unit - q.chunk * p.tiles;
  const uint32_t c = q.c(), seq = c / p.D;
  const int64_t p0 = q.p0(), left = c < p.C ? p.T - p0 : 0;
  q.n = left < 0 ? 0 : left < R ? static_cast<int>(left) : R;
  q.row = (seq * p.T + (kGrad ? p.T - 1 - p0 : p0)) * p.D + (c - seq * p.D);
  return q;
}

template <class E, int V, int R, bool kGrad>
constexpr size_t stage_bytes() {
  return sizeof(E) * V * (kGrad ? 3 : 2) * R * kThreads;
}

// A thread's slots in shared memory: R words each of the coefficients, the
// added values and (gradient) the states before.
template <class E, int V, int R>
struct Slots {
  Word<E, V> *a, *x, *h;
};

// Values of a part on their way.  kFull: it has all R steps.
template <bool kFull, class E, int V, int CT, int R, bool kGrad>
__device__ __forceinline__ void issue_part(const ChunkArgs<E>& p, const Part<V, CT, R>& q,
                                           const Slots<E, V, R>& s) {
  const int64_t dir = kGrad ? -static_cast<int64_t>(p.D) : static_cast<int64_t>(p.D);
  const E* x = p.x + q.row;
  const E* a = p.a + q.row + (kGrad ? p.D : 0);
  const E* h = kGrad ? p.h + q.row - p.D : nullptr;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (!kFull && i >= q.n) break;
    copy_async(s.x + i * kThreads, x);
    if constexpr (kGrad) {
      // the last step in time has no coefficient after it, the first one the
      // state h0 before it
      if (i > 0 || q.p0() > 0) copy_async(s.a + i * kThreads, a);
      if ((kFull && i < R - 1) || q.p0() + i < p.T - 1) copy_async(s.h + i * kThreads, h);
      else if (p.h0) copy_async(s.h + i * kThreads, p.h0 + q.c());
      h += dir;
    } else {
      copy_async(s.a + i * kThreads, a);
    }
    x += dir;
    a += dir;
  }
}

template <class E, int V, int CT, int R, bool kGrad>
__device__ __forceinline__ void issue(const ChunkArgs<E>& p, const Part<V, CT, R>& q,
                                      const Slots<E, V, R>& s) {
  if (q.n == R) issue_part<true, E, V, CT, R, kGrad>(p, q, s);
  else if (q.n > 0) issue_part<false, E, V, CT, R, kGrad>(p, q, s);
}

// A part's values, those used twice widened once: a conversion costs a quarter of
// the FP64 rate.
template <class E, int V, int R, bool kGrad>
struct Values {
  double a[R][V], x[R][V];
  E h[kGrad ? R : 1][V];
};

// Steps that the part does not have do nothing: s -> 1 s + 0.
template <class E, int V, int CT, int R, bool kGrad>
__device__ __forceinline__ void read(const ChunkArgs<E>& p, const Part<V, CT, R>& q,
                                     const Slots<E, V, R>& s, Values<E, V, R, kGrad>& v) {
  using IO = SeqIO<E>;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const Word<E, V> x = s.x[i * kThreads], a = s.a[i * kThreads];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v.x[i][j] = IO::value(x.v[j]);
      v.a[i][j] = IO::value(a.v[j]);
    }
    if constexpr (kGrad) {
      const Word<E, V> h = s.h[i * kThreads];
#pragma unroll
      for (int j = 0; j < V; ++j) v.h[i][j] = h.v[j];
    }
  }
  if (kGrad && q.p0() == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) v.a[0][j] = 1.0;
  }
  if (q.n == R && !(kGrad && !p.h0 && q.p0() + R == p.T)) return;
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (i >= q.n) {
        v.x[i][j] = 0.0;
        v.a[i][j] = 1.0;
      }
      if constexpr (kGrad) {
        if (!p.h0 && q.p0() + i == p.T - 1) v.h[i][j] = IO::zero();
      }
    }
  }
}

// The steps from `state` on, stored.
template <bool kFull, class E, int V, int CT, int R, bool kGrad>
__device__ __forceinline__ void run_part(const ChunkArgs<E>& p, const Part<V, CT, R>& q,
                                         const Values<E, V, R, kGrad>& v, double (&state)[V]) {
  using IO = SeqIO<E>;
  const int64_t dir = kGrad ? -static_cast<int64_t>(p.D) : static_cast<int64_t>(p.D);
  E* out = p.out + q.row;
  E* ga = kGrad ? p.ga + q.row : nullptr;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (!kFull && i >= q.n) break;
    double g[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      state[j] = __fma_rn(v.a[i][j], state[j], v.x[i][j]);
      if constexpr (kGrad) g[j] = __dmul_rn(state[j], IO::value(v.h[i][j]));
    }
    IO::template put<V>(out, state);
    out += dir;
    if constexpr (kGrad) {
      IO::template put<V>(ga, g);
      ga += dir;
      if ((!kFull || i == R - 1) && q.p0() + i == p.T - 1) {
        const E* a0 = p.a + q.row + i * dir;
#pragma unroll
        for (int j = 0; j < V; ++j)
          IO::store(p.gh0 + q.c() + j, __dmul_rn(IO::value(IO::load(a0 + j)), state[j]));
      }
    }
  }
}

// The state before the first step of channel threadIdx.x of a tile.
template <class E, int CT, bool kGrad>
__device__ __forceinline__ double state_h0(const ChunkArgs<E>& p, uint32_t tile) {
  const uint32_t c = tile * CT + threadIdx.x;
  return !kGrad && p.h0 && c < p.C ? SeqIO<E>::value(SeqIO<E>::load(p.h0 + c)) : 0.0;
}

template <class E, int V, int CT, int R, bool kGrad>
__global__ void __launch_bounds__(kThreads, 2)
scan_chunk_kernel(const __grid_constant__ ChunkArgs<E> p) {
  constexpr int N = CT / V;         // threads across the channels
  constexpr int S = kThreads / N;   // and along the steps
  // Whether a thread's smallest product is kept from step to step, or found by a
  // second pass where a coefficient is above 1.  The pass costs most threads nothing
  // (f32 [4, 4096, 2048] 86 us, kept 87), but spills with the more steps of V = 1
  // (f64 [8, 2048, 1023] 83 us, kept 80).
  constexpr bool kTrack = V == 1;
  extern __shared__ __align__(16) uint8_t smem[];
  Slots<E, V, R> slots;
  slots.a = reinterpret_cast<Word<E, V>*>(smem) + threadIdx.x;
  slots.x = slots.a + R * kThreads;
  slots.h = slots.x + R * kThreads;  // gradient only
  __shared__ Map s_map[2][S][CT];  // channel V c + j at j N + c: no bank twice
  __shared__ Map s_before[kMaxRound][CT];
  __shared__ double s_start[CT];
  __shared__ uint32_t s_unit[2];
  // the last of the block's units in which a channel has a
  // coefficient above 1, has a tiny product, and is stepped through
  __shared__ uint32_t s_grows[CT], s_tiny[CT], s_stepped[CT];
  // the last one with a coefficient above 1 or a state beyond 2^64 in a thread's
  // map, with a channel that is stepped through, and with a map from another block
  // that is not an ordinary one
  __shared__ uint32_t s_careful, s_any_stepped, s_special;
  const int tid = threadIdx.x, cl = tid % N * V, sub = tid / N;

  wait_previous_grid();
  // a block with tiles of its own takes their chunks one after another
  uint32_t unit = blockIdx.x;
  auto after = [&](uint32_t u) {
    if (u + p.tiles < p.units) return u + p.tiles;
    return u % p.tiles + gridDim.x < p.tiles ? u % p.tiles + gridDim.x : p.units;
  };
  if (tid < CT) s_grows[tid] = s_tiny[tid] = s_stepped[tid] = ~0u;
  if (tid == 0) s_careful = s_any_stepped = s_special = ~0u;
  if (p.counter && tid == 0) s_unit[0] = atomicAdd(p.counter, 1u) + 1u;
  __syncthreads();
  if (p.counter) unit = s_unit[0];
  if (unit >= p.units) return;
  Part<V, CT, R> q = part_of<E, V, CT, R, kGrad>(p, unit);
  issue<E, V, CT, R, kGrad>(p, q, slots);
  int turn = 0;
  for (;;) {
    turn ^= 1;
    if (p.counter && tid == 0) s_unit[turn] = atomicAdd(p.counter, 1u) + 1u;
    if (!p.counter && tid < CT && q.chunk == 0)
      s_start[tid] = state_h0<E, CT, kGrad>(p, q.tile);
    asm volatile("cp.async.wait_all;" ::: "memory");
    Values<E, V, R, kGrad> val;
    read<E, V, CT, R, kGrad>(p, q, slots, val);
    // the slots are this thread's own: the next unit's values may come
    const Part<V, CT, R> cur = q;
    uint32_t next = p.units;
    if (!p.counter) {
      next = after(unit);
      if (next < p.units) {
        q = part_of<E, V, CT, R, kGrad>(p, next);
        issue<E, V, CT, R, kGrad>(p, q, slots);
      }
    }
    Map m[V];
    uint32_t growth[V];
    int lowest[V];  // high word of the smallest product
#pragma unroll
    for (int j = 0; j < V; ++j) {
      m[j] = Map{1.0, 0.0};
      growth[j] = 0;
      lowest[j] = 0x7fffffff;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        m[j].s = __fma_rn(val.a[i][j], m[j].s, val.x[i][j]);
        m[j].p = __dmul_rn(m[j].p, val.a[i][j]);
        growth[j] |= growth_bits(val.a[i][j]);
        if constexpr (kTrack) lowest[j] = min(lowest[j], __double2hiint(m[j].p) & 0x7fffffff);
      }
    }
    bool low[V], steps[V];  // a product is tiny; the channel is to be stepped through
    // inclusive scan over the S threads of a channel
    int buf = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      steps[j] = false;
      s_map[0][sub][j * N + tid % N] = m[j];
      low[j] = kTrack ? lowest[j] < 0x00100000 : tiny(m[j].p);
      if (grows(growth[j])) {
        s_grows[cl + j] = s_careful = unit;
        if constexpr (!kTrack) {
          double product = 1.0;
#pragma unroll
          for (int i = 0; i < R; ++i) {
            product = __dmul_rn(product, val.a[i][j]);
            low[j] |= tiny(product);
          }
        }
      }
      if (beyond(m[j].s)) s_careful = unit;
    }
    __syncthreads();
    if (p.counter) {
      next = s_unit[turn];
      if (next < p.units) {
        q = part_of<E, V, CT, R, kGrad>(p, next);
        issue<E, V, CT, R, kGrad>(p, q, slots);
      }
    }
    // Without a coefficient above 1 and a state beyond 2^64 in a thread's map no
    // product or state of a composition passes 2^71, and one that is tiny makes
    // those after it tiny.
    const bool careful = s_careful == unit;
    if (careful) {
      // a product with a coefficient of zero is exact
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!low[j]) continue;
#pragma unroll
        for (int i = 0; i < R; ++i) low[j] &= val.a[i][j] != 0.0;
      }
    }
#pragma unroll
    for (int d = 1; d < S; d <<= 1) {
      buf ^= 1;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (sub >= d) {
          const Map first = s_map[buf ^ 1][sub - d][j * N + tid % N];
          const bool zero = m[j].p == 0.0 || first.p == 0.0;
          if (careful) steps[j] |= tiny(m[j].p) && large(first.s);
          m[j] = compose(first, m[j]);
          if (careful) low[j] |= tiny(m[j].p) && !zero;
        }
        s_map[buf][sub][j * N + tid % N] = m[j];
      }
      if (2 * d < S) __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (careful)
        steps[j] |= not_finite(m[j].p) || not_finite(m[j].s) ||
                    (low[j] && s_grows[cl + j] == unit);
      low[j] |= tiny(m[j].p);
      if (low[j]) {
        steps[j] |= !p.counter && large(s_start[cl + j]);
        s_tiny[cl + j] = unit;
      }
      if (steps[j]) s_stepped[cl + j] = s_any_stepped = unit;
    }
    __syncthreads();
    bool any_stepped = s_any_stepped == unit;
    auto stepped = [&](int c) { return any_stepped && s_stepped[c] == unit; };
    if (p.counter) {
      const int64_t slot = static_cast<int64_t>(cur.chunk) * p.tiles + cur.tile;
      const uint32_t rnd = cur.chunk / p.round;
      const int idx = static_cast<int>(cur.chunk - rnd * p.round);
      const bool last = cur.chunk == p.chunks - 1, ends = idx == static_cast<int>(p.round) - 1;
      // a later chunk of the round reads it
#pragma unroll
      for (int j = 0; j < V; ++j) {
        steps[j] = stepped(cl + j);
        if (!last && !ends && sub == S - 1 && !steps[j]) put_map(p.maps + slot * CT + cl + j, m[j]);
      }
      // the round's earlier maps, spread over all threads
      const ulonglong2* maps = p.maps + (slot - static_cast<int64_t>(idx) * p.tiles) * CT;
      const int64_t step = static_cast<int64_t>(p.tiles) * CT;
      constexpr int Q = kThreads / CT;
      const int cm = tid % CT;
      for (int i = tid / CT; i < idx; i += 4 * Q) {
        ulonglong2 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u * Q < idx) v[u] = look_at_map(maps + (i + u * Q) * step + cm);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u * Q < idx) {
            const Map b = wait_map(maps + (i + u * Q) * step + cm, v[u], p.err);
            s_before[i + u * Q][cm] = b;
            if (not_finite(b.p) || tiny(b.p)) s_special = unit;
          }
      }
      __syncthreads();
      // the state at the chunk's start, by one thread per channel (cs)
      const int cs = tid;
      if (cs < CT) {
        double start;
        if (rnd > 0)
          start = wait_state(
              p.states + (static_cast<int64_t>(rnd - 1) * p.tiles + cur.tile) * CT + cs, p.err);
        else
          start = state_h0<E, CT, kGrad>(p, cur.tile);
        if (s_special != unit)
          for (int i = 0; i < idx; ++i) start = apply(s_before[i][cs], start);
        else
          for (int i = 0; i < idx; ++i)
            start = pass(maps + i * step + cs, s_before[i][cs], start, p.err);
        s_start[cs] = start;
        const bool late = s_tiny[cs] == unit && large(start);
        if (late) s_stepped[cs] = s_any_stepped = unit;
        if (!last && ends && !late && !stepped(cs))
          put_state(p.states + (static_cast<int64_t>(rnd) * p.tiles + cur.tile) * CT + cs,
                    apply(s_map[buf][S - 1][cs % V * N + cs / V], start));
      }
      __syncthreads();
      any_stepped = s_any_stepped == unit;
    }
    double state[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      state[j] = s_start[cl + j];
      if (sub > 0) state[j] = apply(s_map[buf][sub - 1][j * N + tid % N], state[j]);
    }
    if (any_stepped) {
      // thread after thread, the state in s_start
#pragma unroll 1
      for (int k = 0; k < S; ++k) {
        if (sub == k) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (!stepped(cl + j)) continue;
            double s = state[j] = s_start[cl + j];
#pragma unroll
            for (int i = 0; i < R; ++i) s = __fma_rn(val.a[i][j], s, val.x[i][j]);
            s_start[cl + j] = s;
          }
        }
        __syncthreads();
      }
      if (p.counter && cur.chunk != p.chunks - 1 && sub == S - 1) {
        const uint32_t rnd = cur.chunk / p.round;
        const bool ends = cur.chunk - rnd * p.round == p.round - 1;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (!stepped(cl + j)) continue;
          const double end = s_start[cl + j];
          // a map that was given already counts unless its product is tiny
          if (ends)
            put_state(p.states + (static_cast<int64_t>(rnd) * p.tiles + cur.tile) * CT + cl + j, end);
          else if (steps[j] || tiny(s_map[buf][S - 1][j * N + tid % N].p))
            put_end(p.maps + (static_cast<int64_t>(cur.chunk) * p.tiles + cur.tile) * CT + cl + j, end);
        }
      }
    }
    if (cur.n == R) run_part<true, E, V, CT, R, kGrad>(p, cur, val, state);
    else if (cur.n > 0) run_part<false, E, V, CT, R, kGrad>(p, cur, val, state);
    __syncthreads();  // s_map, s_before and s_start are written again
    if (!p.counter && cur.chunk != p.chunks - 1 && sub == S - 1) {
      // where the tile's next chunk starts
#pragma unroll
      for (int j = 0; j < V; ++j) s_start[cl + j] = state[j];
    }
    if (next >= p.units) break;
    unit = next;
  }
}

// Steps of one channel per thread, half as many of two channels (f32; f64 and
// pairs).  Registers hold two (gradient: three) f64 values of each: two blocks per
// SM with 128 registers.  12 of f64 instead of 16 take as long for [8, 2048, 1024]
// and 14% longer for [1, 65536, 250] (76 and 113 us), 8 5% and 40%, 20 of f32 9% for
// [4, 4096, 2048]; 6 or 8 of the f64 gradient's 10 are within 2% for [8, 2048, 1024].
constexpr int steps_of(int type, bool gradient) {
  return type == 1 ? (gradient ? 12 : 16) : (gradient ? 10 : 16);
}

// ScanArgs::type of an element type (packed pairs and f64 are alike here).
template <class E>
constexpr int type_of() {
  return sizeof(E) == 4 ? 1 : 0;
}

struct Plan {
  int ct;
  bool own;  // a block takes whole tiles
  int64_t C, tiles, chunks, rounds;
  int round;
  size_t off_maps, off_states, total;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Blocks that work at a time: two per SM of B200 (the plan goes by it on every
// device, so that results do not depend on the device).
constexpr int64_t kBlocks = 296;

// Channels per unit, and who carries the state.  Where tiles of 64, 32 or 16
// channels keep at least 0.8 of the blocks busy, each block takes whole tiles,
// chunk by chunk, and nothing is waited for: [8, 2048, 1024] of f64 in 256 tiles
// of 32 takes 76 us, through the workspace 83, and f32 [4, 4096, 2048] 92 and 112.
// Otherwise the chunks of all tiles are shared out: 64 channels per unit (512
// contiguous bytes of f64 per step), 16 where the channels are few, so that a
// unit has more steps and the chain fewer hops ([1, 65536, 250]: 113 us, with 64
// channels 144), 4 for a handful of channels.  The workspace holds the counter,
// the error word, maps and states; every call sets it to ones.
Plan plan_of(int64_t B, int64_t T, int64_t D, int steps) {
  Plan g{};
  g.C = B * D;
  if (g.C == 0 || T <= kShort) return g;
  for (int ct = 64; ct >= 16 && !g.own; ct /= 2) {
    const int64_t tiles = ceil_div(g.C, ct);
    if (tiles * 5 >= ceil_div(tiles, kBlocks) * kBlocks * 4 || T <= kThreads / ct * steps) {
      g.own = true;
      g.ct = ct;
    }
  }
  if (!g.own) g.ct = g.C >= 2048 ? 64 : g.C >= 16 ? 16 : 4;
  const int64_t rows = kThreads / g.ct * steps;
  g.tiles = ceil_div(g.C, g.ct);
  g.chunks = ceil_div(T, rows);
  if (g.chunks == 1) g.own = true;
  if (g.own) return g;
  const int64_t want = ceil_div(512, g.tiles);
  g.round = want < 4 ? 4 : want > kMaxRound ? kMaxRound : static_cast<int>(want);
  g.rounds = ceil_div(g.chunks, g.round);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  g.off_maps = 256;
  g.off_states = g.off_maps + up(static_cast<size_t>(g.chunks * g.tiles) * g.ct * 16);
  g.total = g.off_states + up(static_cast<size_t>(g.rounds * g.tiles) * g.ct * 8);
  return g;
}

// Blocks of the kernel resident on the current device (its shared memory
// limit raised first), once per device.
template <class E, int V, int CT, int R, bool kGrad>
int resident_blocks(int* blocks) {
  static std::mutex mu;
  static std::vector<int> by_device;
  int dev = 0;
  DSB_CUDA_TRY(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= static_cast<int>(by_device.size())) by_device.resize(dev + 1, 0);
  if (by_device[dev] == 0) {
    const int bytes = static_cast<int>(stage_bytes<E, V, R, kGrad>());
    DSB_CUDA_TRY(cudaFuncSetAttribute(scan_chunk_kernel<E, V, CT, R, kGrad>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    int n = 0;
    DSB_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(
        &n, scan_chunk_kernel<E, V, CT, R, kGrad>, kThreads, bytes));
    by_device[dev] = (n < 1 ? 1 : n) * sm_count();
  }
  *blocks = by_device[dev];
  return DS_OK;
}

template <class E, int V, int CT, bool kGrad>
int launch_chunks(const ScanArgs& s, const Plan& g, cudaStream_t st) {
  constexpr int R = steps_of(type_of<E>(), kGrad) / V;
  int resident = 0;
  if (int rc = resident_blocks<E, V, CT, R, kGrad>(&resident)) return rc;
  ChunkArgs<E> p{};
  p.a = static_cast<const E*>(s.a);
  p.x = static_cast<const E*>(s.x);
  p.h = static_cast<const E*>(s.h);
  p.h0 = static_cast<const E*>(s.h0);
  p.out = static_cast<E*>(s.out);
  p.ga = static_cast<E*>(s.grad_a);
  p.gh0 = static_cast<E*>(s.grad_h0);
  p.C = static_cast<uint32_t>(g.C);
  p.T = s.T;
  p.D = static_cast<uint32_t>(s.D);
  p.tiles = static_cast<uint32_t>(g.tiles);
  p.chunks = static_cast<uint32_t>(g.chunks);
  p.units = static_cast<uint32_t>(g.chunks * g.tiles);
  p.round = static_cast<uint32_t>(g.round);
  if (!g.own) {
    uint8_t* ws = static_cast<uint8_t*>(s.workspace);
    p.counter = reinterpret_cast<uint32_t*>(ws);
    p.err = p.counter + 1;
    p.maps = reinterpret_cast<ulonglong2*>(ws + g.off_maps);
    p.states = reinterpret_cast<uint64_t*>(ws + g.off_states);
    DSB_CUDA_TRY(cudaMemsetAsync(ws, 0xff, g.total, st));
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  const uint32_t most = g.own ? p.tiles : p.units;
  cfg.gridDim = dim3(most < static_cast<uint32_t>(resident) ? most : resident);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = stage_bytes<E, V, R, kGrad>();
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DSB_CUDA_TRY(cudaLaunchKernelEx(&cfg, scan_chunk_kernel<E, V, CT, R, kGrad>, p));
  return launch_status();
}

// Two channels per thread where every row starts on a word of two.
template <class E>
bool pairs(const ScanArgs& s) {
  const size_t w = 2 * sizeof(E);
  return s.D % 2 == 0 && aligned(s.a, w) && aligned(s.x, w) && aligned(s.h, w) &&
         aligned(s.h0, w) && aligned(s.out, w) && aligned(s.grad_a, w);
}

template <class E, int CT, bool kGrad>
int launch_chunks(const ScanArgs& s, const Plan& g, cudaStream_t st) {
  return pairs<E>(s) ? launch_chunks<E, 2, CT, kGrad>(s, g, st)
                     : launch_chunks<E, 1, CT, kGrad>(s, g, st);
}

template <class E, bool kGrad>
int launch(const ScanArgs& s, cudaStream_t st) {
  const Plan g = plan_of(s.B, s.T, s.D, steps_of(type_of<E>(), kGrad));
  const int64_t units = g.ct ? g.chunks * g.tiles : ceil_div(g.C, kThreads);
  if (units > 0x7fffffff || g.C > 0x7fffffff)
    return set_error(DS_INVALID_ARGUMENT, "ds_linear_recurrence: too many channels");
  if (g.ct == 64) return launch_chunks<E, 64, kGrad>(s, g, st);
  if (g.ct == 32) return launch_chunks<E, 32, kGrad>(s, g, st);
  if (g.ct == 16) return launch_chunks<E, 16, kGrad>(s, g, st);
  if (g.ct == 4) return launch_chunks<E, 4, kGrad>(s, g, st);
  auto in = [](const void* p) { return static_cast<const E*>(p); };
  auto out = [](void* p) { return static_cast<E*>(p); };
  const dim3 grid(static_cast<unsigned>(units)), block(kThreads);
  if constexpr (kGrad) {
    DSB_CUDA_TRY(launch_dependent(scan_vjp_short_kernel<E>, grid, block, st, in(s.a), in(s.h),
                                  in(s.x), in(s.h0), out(s.grad_a), out(s.out), out(s.grad_h0),
                                  g.C, s.T, s.D));
  } else {
    DSB_CUDA_TRY(launch_dependent(scan_short_kernel<E>, grid, block, st, in(s.a), in(s.x),
                                  in(s.h0), out(s.out), g.C, s.T, s.D));
  }
  return launch_status();
}

template <class E>
int launch(const ScanArgs& s, bool gradient, cudaStream_t st) {
  return gradient ? launch<E, true>(s, st) : launch<E, false>(s, st);
}

}  // namespace

size_t scan_workspace_bytes(int type, int64_t B, int64_t T, int64_t D) {
  const size_t f = plan_of(B, T, D, steps_of(type, false)).total;
  const size_t g = plan_of(B, T, D, steps_of(type, true)).total;
  return f > g ? f : g;
}

int scan_launch(const ScanArgs& a, bool gradient, cudaStream_t s) {
  if (a.B * a.D == 0 || (a.T == 0 && !gradient)) return ok();
  ProfileScope prof("linear_recurrence", s);
  if (a.type == 0) return launch<double>(a, gradient, s);
  if (a.type == 1) return launch<float>(a, gradient, s);
  return launch<float2>(a, gradient, s);
}

}  // namespace dsb
