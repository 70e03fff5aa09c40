// One AdamW step over many tensors.
//
//   t = step + 1
//   m = b1 * m + (1 - b1) * g
//   v = b2 * v + (1 - b2) * g * g
//   p = p * (1 - lr * decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound: HBM.  Every value is read once (p, g, m, v) and written once (p, m,
// v): 28 bytes in float32.  All tensors of a step go through one launch: the
// table of their addresses travels in the kernel's parameters, so a captured
// graph holds it by value, and a CTA finds its chunk of 16 KB of values by a
// binary search in the table's running chunk count.
//
// The step count lives on the device, so that a recorded step counts its own
// replays: every CTA reads it first, and the last CTA to finish (a ticket)
// advances it, after everybody has read it.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"

namespace lmpb {
namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 64;  // of one launch: 64 x 44 bytes of parameters
template <typename T>
constexpr int chunk_of() { return 16384 / (int)sizeof(T); }

struct Table {
  void* p[kTensors];
  const void* g[kTensors];
  void* m[kTensors];
  void* v[kTensors];
  int64_t n[kTensors];
  unsigned first[kTensors + 1];  // chunks before each tensor
  int count;
};

struct Rates {
  double lr, b1, b2, eps, decay;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Packet {
  T v[VEC];
};

__device__ __forceinline__ float root(float v) { return __fsqrt_rn(v); }
__device__ __forceinline__ double root(double v) { return sqrt(v); }

template <typename T>
struct Coef {
  T b1, c1, b2, c2, keep, rate, iroot, eps;
};

template <typename T>
__device__ __forceinline__ void update(T& p, T g, T& m, T& v, const Coef<T>& k) {
  m = k.b1 * m + k.c1 * g;
  v = k.b2 * v + k.c2 * (g * g);
  p = p * k.keep - k.rate * (m / (root(v) * k.iroot + k.eps));
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    adamw_kernel(const __grid_constant__ Table tab, Rates r, long long* __restrict__ step, int advance) {
  constexpr int VEC = 16 / sizeof(T), CHUNK = chunk_of<T>();
  __shared__ double power[2];
  if (threadIdx.x < 64 && (threadIdx.x & 31) == 0) {
    const double t = (double)(*(volatile long long*)step + 1);
    power[threadIdx.x >> 5] = pow(threadIdx.x ? r.b2 : r.b1, t);
  }
  int lo = 0, hi = tab.count;  // the last tensor whose first chunk is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const int64_t base = (int64_t)(blockIdx.x - tab.first[lo]) * CHUNK;
  const int n = (int)min((int64_t)CHUNK, tab.n[lo] - base);
  T* p = (T*)tab.p[lo] + base;
  const T* g = (const T*)tab.g[lo] + base;
  T* m = (T*)tab.m[lo] + base;
  T* v = (T*)tab.v[lo] + base;
  __syncthreads();
  const Coef<T> k{T(r.b1), T(1.0 - r.b1), T(r.b2), T(1.0 - r.b2), T(1.0 - r.lr * r.decay),
                  T(r.lr / (1.0 - power[0])), T(1.0 / sqrt(1.0 - power[1])), T(r.eps)};
  const bool vec = (((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15u) == 0;
  if (vec) {
    using P = Packet<T, VEC>;
#pragma unroll
    for (int i = 0; i < CHUNK / VEC / kThreads; ++i) {
      const int c = (i * kThreads + threadIdx.x) * VEC;
      if (c + VEC <= n) {
        P pp = *(P*)(p + c), pg = *(const P*)(g + c), pm = *(P*)(m + c), pv = *(P*)(v + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) update(pp.v[j], pg.v[j], pm.v[j], pv.v[j], k);
        *(P*)(p + c) = pp;
        *(P*)(m + c) = pm;
        *(P*)(v + c) = pv;
      } else {
        for (int j = c; j < n; ++j) update(p[j], g[j], m[j], v[j], k);
      }
    }
  } else {
    for (int c = threadIdx.x; c < n; c += kThreads) update(p[c], g[c], m[c], v[c], k);
  }
  if (advance) {
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      if (atomicAdd((unsigned long long*)step + 1, 1ull) == gridDim.x - 1) {
        step[1] = 0;
        step[0] += 1;
      }
    }
  }
}

// A step over no values still counts.
__global__ void advance_kernel(long long* step) { step[0] += 1; }

template <typename T>
lmpb_status run(const lmpb_adamw_tensor* ts, int count, const Rates& r, int64_t* step, cudaStream_t st) {
  int i = 0;
  while (i < count && ts[i].n == 0) ++i;
  if (i == count) {
    advance_kernel<<<1, 1, 0, st>>>((long long*)step);
    return launch_status("adamw");
  }
  while (i < count) {
    Table tab;
    tab.count = 0;
    int64_t chunks = 0;
    for (; i < count && tab.count < kTensors; ++i) {
      if (ts[i].n == 0) continue;
      const int64_t c = (ts[i].n + chunk_of<T>() - 1) / chunk_of<T>();
      if (tab.count && chunks + c > 0x7fffffff) break;
      const int k = tab.count++;
      tab.p[k] = ts[i].param;
      tab.g[k] = ts[i].grad;
      tab.m[k] = ts[i].exp_avg;
      tab.v[k] = ts[i].exp_avg_sq;
      tab.n[k] = ts[i].n;
      tab.first[k] = (unsigned)chunks;
      chunks += c;
    }
    tab.first[tab.count] = (unsigned)chunks;
    while (i < count && ts[i].n == 0) ++i;
    adamw_kernel<T><<<(unsigned)chunks, kThreads, 0, st>>>(tab, r, (long long*)step, i == count);
    const lmpb_status s = launch_status("adamw");
    if (s != LMPB_OK) return s;
  }
  return LMPB_OK;
}

}  // namespace
}  // namespace lmpb

extern "C" lmpb_status lmpb_adamw(int dtype, const lmpb_adamw_tensor* tensors, int count, double lr, double beta1,
                                  double beta2, double eps, double weight_decay, int64_t* step, void* stream) {
  using namespace lmpb;
  LMPB_CHECK_ARG(dtype == LMPB_FLOAT32 || dtype == LMPB_FLOAT64, "lmpb_adamw: float32 or float64 only");
  LMPB_CHECK_ARG(count >= 0 && (count == 0 || tensors), "lmpb_adamw: bad tensor list");
  LMPB_CHECK_ARG(std::isfinite(lr) && lr >= 0.0, "lmpb_adamw: lr must be finite and not negative");
  LMPB_CHECK_ARG(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "lmpb_adamw: betas must lie in [0, 1)");
  LMPB_CHECK_ARG(std::isfinite(eps) && eps >= 0.0, "lmpb_adamw: eps must be finite and not negative");
  LMPB_CHECK_ARG(std::isfinite(weight_decay) && weight_decay >= 0.0,
                 "lmpb_adamw: weight_decay must be finite and not negative");
  LMPB_CHECK_ARG(step, "lmpb_adamw: null step count");
  for (int i = 0; i < count; ++i) {
    const lmpb_adamw_tensor& t = tensors[i];
    LMPB_CHECK_ARG(t.n >= 0 && t.n <= (int64_t)1 << 40, "lmpb_adamw: bad tensor size");
    LMPB_CHECK_ARG(t.n == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq), "lmpb_adamw: null pointer");
  }
  const Rates r{lr, beta1, beta2, eps, weight_decay};
  return dtype == LMPB_FLOAT32 ? run<float>(tensors, count, r, step, as_stream(stream))
                               : run<double>(tensors, count, r, step, as_stream(stream));
}
