// The linear recurrence h_t = a_t h_{t-1} + x_t along a sequence, and its
// gradient.
#include "common.cuh"
#include "ds_arith.cuh"
#include "kernels.h"
#include "profile.h"

namespace dsb {
namespace {

// Element types: f64, f32, packed DS pair.  Loaded as the exact f64 value,
// stored with one rounding (a pair: hi = f32(v), lo = f32(v - hi)).
template <class T> struct SeqIO;
template <> struct SeqIO<double> {
  static __device__ __forceinline__ double load(const double* p) { return __ldcs(p); }
  static __device__ __forceinline__ void store(double* p, double v) { __stcs(p, v); }
};
template <> struct SeqIO<float> {
  static __device__ __forceinline__ double load(const float* p) {
    return static_cast<double>(__ldcs(p));
  }
  static __device__ __forceinline__ void store(float* p, double v) {
    __stcs(p, __double2float_rn(v));
  }
};
template <> struct SeqIO<float2> {
  static __device__ __forceinline__ double load(const float2* p) {
    const float2 v = __ldcs(p);
    return to_f64(ds2{v.x, v.y});
  }
  static __device__ __forceinline__ void store(float2* p, double v) {
    const ds2 d = from_f64(v);
    __stcs(p, make_float2(d.hi, d.lo));
  }
};

constexpr int kThreads = 128;

// One thread per channel, step by step.
template <class E>
__global__ void __launch_bounds__(kThreads)
scan_kernel(const E* __restrict__ a, const E* __restrict__ b, const E* __restrict__ h0,
            E* __restrict__ h, int64_t B, int64_t T, int64_t D) {
  wait_previous_grid();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= B * D) return;
  const int64_t seq = c / D;
  int64_t at = seq * T * D + (c - seq * D);
  double s = h0 ? SeqIO<E>::load(h0 + c) : 0.0;
  for (int64_t t = 0; t < T; ++t, at += D) {
    s = __fma_rn(SeqIO<E>::load(a + at), s, SeqIO<E>::load(b + at));
    SeqIO<E>::store(h + at, s);
  }
}

template <class E>
__global__ void __launch_bounds__(kThreads)
scan_vjp_kernel(const E* __restrict__ a, const E* __restrict__ h, const E* __restrict__ gh,
                const E* __restrict__ h0, E* __restrict__ ga, E* __restrict__ gb,
                E* __restrict__ gh0, int64_t B, int64_t T, int64_t D) {
  wait_previous_grid();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= B * D) return;
  const int64_t seq = c / D;
  int64_t at = (seq * T + T - 1) * D + (c - seq * D);
  double carry = 0.0;  // a_{t+1} g_{t+1}
  for (int64_t t = T - 1; t >= 0; --t, at -= D) {
    const double g = __dadd_rn(SeqIO<E>::load(gh + at), carry);
    const double before = t > 0 ? SeqIO<E>::load(h + at - D)
                                : (h0 ? SeqIO<E>::load(h0 + c) : 0.0);
    SeqIO<E>::store(gb + at, g);
    SeqIO<E>::store(ga + at, __dmul_rn(g, before));
    carry = __dmul_rn(SeqIO<E>::load(a + at), g);
  }
  SeqIO<E>::store(gh0 + c, carry);
}

template <class E>
int launch(const ScanArgs& s, bool gradient, cudaStream_t st) {
  const int64_t blocks = (s.B * s.D + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return set_error(DS_INVALID_ARGUMENT, "too many channels");
  auto in = [](const void* p) { return static_cast<const E*>(p); };
  auto out = [](void* p) { return static_cast<E*>(p); };
  if (gradient) {
    DSB_CUDA_TRY(launch_dependent(scan_vjp_kernel<E>, dim3(static_cast<unsigned>(blocks)),
                                  dim3(kThreads), st, in(s.a), in(s.h), in(s.x), in(s.h0),
                                  out(s.grad_a), out(s.out), out(s.grad_h0), s.B, s.T, s.D));
  } else {
    DSB_CUDA_TRY(launch_dependent(scan_kernel<E>, dim3(static_cast<unsigned>(blocks)),
                                  dim3(kThreads), st, in(s.a), in(s.x), in(s.h0), out(s.out), s.B,
                                  s.T, s.D));
  }
  return launch_status();
}

}  // namespace

size_t scan_workspace_bytes(int, int64_t, int64_t, int64_t) { return 0; }

int scan_launch(const ScanArgs& a, bool gradient, cudaStream_t s) {
  if (a.B * a.D == 0 || (a.T == 0 && !gradient)) return ok();
  ProfileScope prof("linear_recurrence", s);
  if (a.type == 0) return launch<double>(a, gradient, s);
  if (a.type == 1) return launch<float>(a, gradient, s);
  return launch<float2>(a, gradient, s);
}

}  // namespace dsb
