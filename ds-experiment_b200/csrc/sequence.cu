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
// The state at a chunk's start comes from the chunks before it through the
// workspace.  Chunks stand in rounds of `round` chunks: a chunk publishes
// (P, S) as soon as it has read its values; it takes those of the earlier
// chunks of its round and the state the last round ended with, and applies
// them in order; the round's last chunk publishes that state.  So the chain
// has one hop per round rather than per chunk, and the order of every
// operation is fixed by the shape.  A published value is its own message: the
// workspace starts as all ones (a NaN no result has), and a reader polls the
// value itself, so there is no flag, fence or barrier between the two.
//
// Blocks stay on their SM and take units from a counter, chunk by chunk, one
// ahead: the next unit's values travel to shared memory (cp.async, each thread
// into slots of its own) while the current one waits for its state.  What a
// unit waits for is an earlier unit, and the earliest unfinished one is always
// some block's current one, so the chain moves; each wait is bounded (about
// 2 s), after which the unit works with NaN.
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
};
template <> struct SeqIO<float> {
  static __device__ __forceinline__ float load(const float* p) { return __ldcs(p); }
  static __device__ __forceinline__ double value(float v) { return static_cast<double>(v); }
  static __device__ __forceinline__ float zero() { return 0.0f; }
  static __device__ __forceinline__ float one() { return 1.0f; }
  static __device__ __forceinline__ void store(float* p, double v) {
    __stcs(p, __double2float_rn(v));
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

// A zero state stays out of the product, so that coefficients whose product
// has overflowed do not turn it into NaN (a coefficient that is itself NaN or
// infinite has made s NaN already).
__device__ __forceinline__ double apply(const Map& m, double state) {
  return state == 0.0 ? m.s : __fma_rn(m.p, state, m.s);
}

// first, then second.
__device__ __forceinline__ Map compose(const Map& first, const Map& second) {
  return Map{first.p == 0.0 ? 0.0 : __dmul_rn(second.p, first.p), apply(second, first.s)};
}

template <class E>
struct ChunkArgs {
  const E *a, *x, *h, *h0;
  E *out, *ga, *gh0;
  int64_t C, T, D;  // channels of all sequences, steps, channels of one
  int64_t tiles;    // of CT channels
  int64_t chunks, units;
  int round;         // chunks per round, at most kMaxRound
  uint32_t* counter;  // units taken, minus one (null: one chunk, nothing to wait for)
  uint32_t* err;      // all ones, or 1 when a wait has run out
  ulonglong2* maps;   // [chunks][tiles][CT]
  uint64_t* states;   // [rounds][tiles][CT]
};

#ifndef SEQ_MR
#define SEQ_MR 24
#endif
constexpr int kMaxRound = SEQ_MR;
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
// run out.
__device__ __noinline__ bool keep_waiting(long long t0, uint32_t* err) {
  if (*reinterpret_cast<volatile uint32_t*>(err) == 1u) return false;
  if (clock64() - t0 <= kTimeoutCycles) return true;
  *reinterpret_cast<volatile uint32_t*>(err) = 1u;
  return false;
}

__device__ __forceinline__ Map wait_map(const ulonglong2* at, ulonglong2 v, uint32_t* err) {
  if (v.x == kEmpty) {
    const long long t0 = clock64();
    do {
      if (!keep_waiting(t0, err)) {
        v.x = v.y = 0x7ff8000000000000ull;
        break;
      }
      v = look_at_map(at);
    } while (v.x == kEmpty);
  }
  return Map{__longlong_as_double(static_cast<long long>(v.x)),
             __longlong_as_double(static_cast<long long>(v.y))};
}

__device__ __forceinline__ double wait_state(const uint64_t* at, uint32_t* err) {
  uint64_t v = look_at_state(at);
  if (v == kEmpty) {
    const long long t0 = clock64();
    do {
      if (!keep_waiting(t0, err)) {
        v = 0x7ff8000000000000ull;
        break;
      }
      v = look_at_state(at);
    } while (v == kEmpty);
  }
  return __longlong_as_double(static_cast<long long>(v));
}

template <class E>
__device__ __forceinline__ void copy_async(E* dst, const E* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "n"(sizeof(E))
               : "memory");
}

// One thread's part of a unit: R steps of a channel.
struct Part {
  int64_t chunk, tile;
  int64_t c;     // channel
  int64_t p0;    // first step (gradient: counted from the end)
  int64_t base;  // element of the channel's first row
  int64_t row;   // element of the first step's row
  int n;         // steps it has
};

template <class E, int CT, int R, bool kGrad>
__device__ __forceinline__ Part part_of(const ChunkArgs<E>& p, int64_t unit) {
  constexpr int S = kThreads / CT;
  Part q;
  q.chunk = unit / p.tiles;
  q.tile = unit - q.chunk * p.tiles;
  q.c = q.tile * CT + threadIdx.x % CT;
  const int64_t seq = q.c / p.D;
  q.base = seq * p.T * p.D + (q.c - seq * p.D);
  q.p0 = (q.chunk * S + threadIdx.x / CT) * R;
  const int64_t left = q.c < p.C ? p.T - q.p0 : 0;
  q.n = left < 0 ? 0 : left < R ? static_cast<int>(left) : R;
  q.row = q.base + (kGrad ? p.T - 1 - q.p0 : q.p0) * p.D;
  return q;
}

template <class E, int R, bool kGrad>
constexpr size_t stage_bytes() {
  return sizeof(E) * (kGrad ? 3 : 2) * R * kThreads;
}

template <class E, int CT, int R, bool kGrad>
__global__ void __launch_bounds__(kThreads, 2)
scan_chunk_kernel(const __grid_constant__ ChunkArgs<E> p) {
  constexpr int S = kThreads / CT;  // threads of one channel
  using IO = SeqIO<E>;
  extern __shared__ __align__(16) uint8_t smem[];
  E* stage_a = reinterpret_cast<E*>(smem) + threadIdx.x;
  E* stage_x = stage_a + R * kThreads;
  E* stage_h = stage_x + R * kThreads;  // gradient only
  __shared__ Map s_map[2][S][CT];
  __shared__ Map s_before[kMaxRound][CT];
  __shared__ double s_start[CT];
  __shared__ uint32_t s_unit[2];
  const int cl = threadIdx.x % CT, sub = threadIdx.x / CT;

  auto issue = [&](const Part& q) {
    const int64_t dir = kGrad ? -p.D : p.D;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i < q.n) {
        const int64_t at = q.row + i * dir;
        copy_async(stage_x + i * kThreads, p.x + at);
        if constexpr (kGrad) {
          if (q.p0 + i > 0) copy_async(stage_a + i * kThreads, p.a + at + p.D);
          if (q.p0 + i < p.T - 1) copy_async(stage_h + i * kThreads, p.h + at - p.D);
          else if (p.h0) copy_async(stage_h + i * kThreads, p.h0 + q.c);
        } else {
          copy_async(stage_a + i * kThreads, p.a + at);
        }
      }
    }
  };

  wait_previous_grid();
  int64_t unit = blockIdx.x;
  if (p.counter) {
    if (threadIdx.x == 0) s_unit[0] = atomicAdd(p.counter, 1u) + 1u;
    __syncthreads();
    unit = s_unit[0];
  }
  Part q{};
  if (unit < p.units) {
    q = part_of<E, CT, R, kGrad>(p, unit);
    issue(q);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  int turn = 0;
  while (unit < p.units) {
    turn ^= 1;
    if (p.counter && threadIdx.x == 0) s_unit[turn] = atomicAdd(p.counter, 1u) + 1u;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    E av[R], xv[R], hv[kGrad ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool in = i < q.n;
      xv[i] = in ? stage_x[i * kThreads] : IO::zero();
      av[i] = in && (!kGrad || q.p0 + i > 0) ? stage_a[i * kThreads] : IO::one();
      if constexpr (kGrad)
        hv[i] = in && (q.p0 + i < p.T - 1 || p.h0) ? stage_h[i * kThreads] : IO::zero();
    }
    Map m{1.0, 0.0};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const double a = IO::value(av[i]);
      m.s = __fma_rn(a, m.s, IO::value(xv[i]));
      m.p = __dmul_rn(m.p, a);
    }
    // inclusive scan over the S threads of a channel
    int buf = 0;
    s_map[0][sub][cl] = m;
    __syncthreads();
    const int64_t next = p.counter ? static_cast<int64_t>(s_unit[turn]) : unit + gridDim.x;
    const Part cur = q;
    if (next < p.units) {
      q = part_of<E, CT, R, kGrad>(p, next);
      issue(q);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int d = 1; d < S; d <<= 1) {
      if (sub >= d) m = compose(s_map[buf][sub - d][cl], m);
      buf ^= 1;
      s_map[buf][sub][cl] = m;
      __syncthreads();
    }
    double start = 0.0;  // state at the chunk's start (threads of sub 0)
    if (p.counter) {
      const int64_t slot = cur.chunk * p.tiles + cur.tile;
      const int64_t rnd = cur.chunk / p.round;
      const int idx = static_cast<int>(cur.chunk - rnd * p.round);
      const bool last = cur.chunk == p.chunks - 1, ends = idx == p.round - 1;
      // a later chunk of the round reads it
      if (!last && !ends && sub == S - 1) put_map(p.maps + slot * CT + cl, m);
      const ulonglong2* maps = p.maps + (slot - idx * p.tiles) * CT + cl;
      const int64_t step = p.tiles * CT;
      for (int i = sub; i < idx; i += 4 * S) {
        ulonglong2 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u * S < idx) v[u] = look_at_map(maps + (i + u * S) * step);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u * S < idx)
            s_before[i + u * S][cl] = wait_map(maps + (i + u * S) * step, v[u], p.err);
      }
      __syncthreads();
      if (sub == 0) {
        if (rnd > 0)
          start = wait_state(p.states + ((rnd - 1) * p.tiles + cur.tile) * CT + cl, p.err);
        else if (!kGrad && p.h0 && cur.c < p.C)
          start = IO::value(IO::load(p.h0 + cur.c));
        for (int i = 0; i < idx; ++i) start = apply(s_before[i][cl], start);
        s_start[cl] = start;
        if (!last && ends)
          put_state(p.states + (rnd * p.tiles + cur.tile) * CT + cl,
                    apply(s_map[buf][S - 1][cl], start));
      }
    } else if (sub == 0) {
      if (!kGrad && p.h0 && cur.c < p.C) start = IO::value(IO::load(p.h0 + cur.c));
      s_start[cl] = start;
    }
    __syncthreads();
    double state = s_start[cl];
    if (sub > 0) state = apply(s_map[buf][sub - 1][cl], state);
    const int64_t dir = kGrad ? -p.D : p.D;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      state = __fma_rn(IO::value(av[i]), state, IO::value(xv[i]));
      if (i < cur.n) {
        const int64_t at = cur.row + i * dir;
        IO::store(p.out + at, state);
        if constexpr (kGrad) {
          IO::store(p.ga + at, __dmul_rn(state, IO::value(hv[i])));
          if (cur.p0 + i == p.T - 1)
            IO::store(p.gh0 + cur.c, __dmul_rn(IO::value(IO::load(p.a + cur.base)), state));
        }
      }
    }
    __syncthreads();  // s_map, s_before and s_start are written again
    unit = next;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Steps per thread: registers hold two (gradient: three) values of each.
#ifndef SEQ_RF
#define SEQ_RF 16
#endif
#ifndef SEQ_RG
#define SEQ_RG 12
#endif
constexpr int kSteps = SEQ_RF, kStepsGrad = SEQ_RG;

// Channels per unit: 64 where there are as many (512 contiguous bytes of f64
// per step), fewer where a unit would be mostly empty.
int unit_channels(int64_t C, int64_t T, int steps) {
  if (C >= 64 || T <= 4 * steps) return 64;
  return C >= 16 || T <= 16 * steps ? 16 : 4;
}

struct Plan {
  int ct;
  int64_t C, tiles, chunks, rounds;
  int round;
  size_t off_maps, off_states, total;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The workspace: counter, error word, maps, states; every call sets it to
// ones.
Plan plan_of(int64_t B, int64_t T, int64_t D, int steps) {
  Plan g{};
  g.C = B * D;
  if (g.C == 0 || T <= kShort) return g;
  g.ct = unit_channels(g.C, T, steps);
  g.tiles = ceil_div(g.C, g.ct);
  g.chunks = ceil_div(T, kThreads / g.ct * steps);
  if (g.chunks == 1) return g;
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
template <class E, int CT, int R, bool kGrad>
int resident_blocks(int* blocks) {
  static std::mutex mu;
  static std::vector<int> by_device;
  int dev = 0;
  DSB_CUDA_TRY(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= static_cast<int>(by_device.size())) by_device.resize(dev + 1, 0);
  if (by_device[dev] == 0) {
    const int bytes = static_cast<int>(stage_bytes<E, R, kGrad>());
    DSB_CUDA_TRY(cudaFuncSetAttribute(scan_chunk_kernel<E, CT, R, kGrad>,
                                      cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    int n = 0;
    DSB_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(
        &n, scan_chunk_kernel<E, CT, R, kGrad>, kThreads, bytes));
    by_device[dev] = (n < 1 ? 1 : n) * sm_count();
  }
  *blocks = by_device[dev];
  return DS_OK;
}

template <class E, int CT, bool kGrad>
int launch_chunks(const ScanArgs& s, const Plan& g, cudaStream_t st) {
  constexpr int R = kGrad ? kStepsGrad : kSteps;
  int resident = 0;
  if (int rc = resident_blocks<E, CT, R, kGrad>(&resident)) return rc;
  ChunkArgs<E> p{};
  p.a = static_cast<const E*>(s.a);
  p.x = static_cast<const E*>(s.x);
  p.h = static_cast<const E*>(s.h);
  p.h0 = static_cast<const E*>(s.h0);
  p.out = static_cast<E*>(s.out);
  p.ga = static_cast<E*>(s.grad_a);
  p.gh0 = static_cast<E*>(s.grad_h0);
  p.C = g.C;
  p.T = s.T;
  p.D = s.D;
  p.tiles = g.tiles;
  p.chunks = g.chunks;
  p.units = g.chunks * g.tiles;
  p.round = g.round;
  if (g.chunks > 1) {
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
  cfg.gridDim = dim3(static_cast<unsigned>(p.units < resident ? p.units : resident));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = stage_bytes<E, R, kGrad>();
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DSB_CUDA_TRY(cudaLaunchKernelEx(&cfg, scan_chunk_kernel<E, CT, R, kGrad>, p));
  return launch_status();
}

template <class E, bool kGrad>
int launch(const ScanArgs& s, cudaStream_t st) {
  const Plan g = plan_of(s.B, s.T, s.D, kGrad ? kStepsGrad : kSteps);
  const int64_t units = g.ct ? g.chunks * g.tiles : ceil_div(g.C, kThreads);
  if (units > 0x7fffffff)
    return set_error(DS_INVALID_ARGUMENT, "ds_linear_recurrence: too many channels");
  if (g.ct == 64) return launch_chunks<E, 64, kGrad>(s, g, st);
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

size_t scan_workspace_bytes(int64_t B, int64_t T, int64_t D) {
  const size_t f = plan_of(B, T, D, kSteps).total, g = plan_of(B, T, D, kStepsGrad).total;
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
