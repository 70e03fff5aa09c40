// Causal attention for a few short sequences, float32: one launch forward,
// one backward.
//
// With 32 tokens and fewer the work is nothing and the time is latency: a
// CTA takes a sequence and a head (backward: a key/value head, walking its
// group's query heads), holds all its rows in shared memory, and never waits
// for another kernel.  A warp walks query rows; a lane is a key for the
// scores and four columns for what is summed over keys, the weights going
// round by shuffles.  Shared rows are 4 floats longer than a multiple of 4,
// so that 32 lanes reading 16 bytes of 32 rows meet no bank twice.  In the backward the weights and dS stay in
// shared memory, where the keys' sums then read them by columns.  Everything
// is plain fp32, and a masked position never enters a sum.
#include <cuda_runtime.h>

#include <algorithm>

#include "attention.cuh"

namespace lmpb {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kRows = kShortRows / kWarps;  // of a warp, at most
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__host__ __device__ __forceinline__ int pitch_of(int dim) { return ((dim + 3) & ~3) + 4; }

// Rows of head `head` of a [*, heads, dim] tensor, 0 from `dim` up to a
// multiple of 4.  All of a thread's loads are on their way at once.
__device__ __forceinline__ void load_rows(float* __restrict__ dst, const float* __restrict__ src, int64_t row0, int n,
                                          int heads, int head, int dim, int pitch) {
  const float* base = src + (row0 * heads + head) * dim;
  const int64_t step = (int64_t)heads * dim;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float v[kRows][4];
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int row = warp + r * kWarps, col = lane + 32 * c;
      v[r][c] = row < n && col < dim ? __ldg(base + row * step + col) : 0.f;
    }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int row = warp + r * kWarps, col = lane + 32 * c;
      if (row < n && col < pitch - 4) dst[row * pitch + col] = v[r][c];
    }
}

__device__ __forceinline__ float4 at4(const float* p) { return *reinterpret_cast<const float4*>(p); }

__device__ __forceinline__ void add4(float4& s, float w, const float4& v) {
  s.x = fmaf(w, v.x, s.x);
  s.y = fmaf(w, v.y, s.y);
  s.z = fmaf(w, v.z, s.z);
  s.w = fmaf(w, v.w, s.w);
}

// a . b over `width` columns; `a` is one address for the warp, `b` each lane's own row.
__device__ __forceinline__ float dot(const float* a, const float* b, int width) {
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = 0; c < width; c += 4) {
    const float4 x = at4(a + c), y = at4(b + c);
    s.x = fmaf(x.x, y.x, s.x);
    s.y = fmaf(x.y, y.y, s.y);
    s.z = fmaf(x.z, y.z, s.z);
    s.w = fmaf(x.w, y.w, s.w);
  }
  return (s.x + s.y) + (s.z + s.w);
}

// Columns 4 lane .. of a result row.
__device__ __forceinline__ void store4(float* p, const float4& v, int col, int dim) {
  if (col < dim) p[col] = v.x;
  if (col + 1 < dim) p[col + 1] = v.y;
  if (col + 2 < dim) p[col + 2] = v.z;
  if (col + 3 < dim) p[col + 3] = v.w;
}

__global__ void __launch_bounds__(kThreads) forward_kernel(const AttentionArgs a, int cap) {
  extern __shared__ __align__(16) float smem[];
  const int4 t = a.tile[blockIdx.x];
  const int n = t.y, head = blockIdx.y, kv_head = head / (a.heads / a.kv_heads), pitch = pitch_of(a.dim), width = pitch - 4;
  float *q = smem, *k = q + cap * pitch, *v = k + cap * pitch;
  load_rows(q, a.q, t.x, n, a.heads, head, a.dim, pitch);
  load_rows(k, a.k, t.x, n, a.kv_heads, kv_head, a.dim, pitch);
  load_rows(v, a.v, t.x, n, a.kv_heads, kv_head, a.dim, pitch);
  __syncthreads();
  const int lane = threadIdx.x & 31, col = 4 * lane;
  const float c = a.scale * kLog2e;
  for (int i = threadIdx.x >> 5; i < n; i += kWarps) {
    const float s = lane <= i ? __fmul_rn(dot(q + i * pitch, k + lane * pitch, width), c) : -INFINITY;
    float m = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float p = lane <= i ? exp2f(s - (m == -INFINITY ? 0.f : m)) : 0.f;  // all weights 0: the row is 0 / 0
    const float l = warp_sum(p);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j <= i; ++j) {
      const float w = __shfl_sync(0xffffffffu, p, j);
      if (col < width) add4(o, w, at4(v + j * pitch + col));
    }
    float* out = a.out + ((int64_t)(t.x + i) * a.heads + head) * a.dim;
    store4(out, make_float4(__fdiv_rn(o.x, l), __fdiv_rn(o.y, l), __fdiv_rn(o.z, l), __fdiv_rn(o.w, l)), col, a.dim);
    if (lane == 0) a.lse[(int64_t)head * a.tokens + t.x + i] = m + log2f(l);
  }
}

__global__ void __launch_bounds__(kThreads) backward_kernel(const AttentionArgs a, int cap) {
  extern __shared__ __align__(16) float smem[];
  const int4 t = a.tile[blockIdx.x];
  const int n = t.y, kv_head = blockIdx.y, group = a.heads / a.kv_heads, pitch = pitch_of(a.dim), width = pitch - 4;
  float *k = smem, *v = k + cap * pitch, *q = v + cap * pitch, *g = q + cap * pitch;
  float *out = g + cap * pitch, *p = out + cap * pitch, *ds = p + cap * 33, *lse = ds + cap * 33;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = 4 * lane;
  load_rows(k, a.k, t.x, n, a.kv_heads, kv_head, a.dim, pitch);
  load_rows(v, a.v, t.x, n, a.kv_heads, kv_head, a.dim, pitch);
  float4 dk[kRows], dv[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) dk[r] = dv[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int head = kv_head * group; head < (kv_head + 1) * group; ++head) {
    load_rows(q, a.q, t.x, n, a.heads, head, a.dim, pitch);
    load_rows(g, a.grad, t.x, n, a.heads, head, a.dim, pitch);
    load_rows(out, a.out, t.x, n, a.heads, head, a.dim, pitch);
    if (threadIdx.x < n) lse[threadIdx.x] = __ldg(a.lse + (int64_t)head * a.tokens + t.x + threadIdx.x);
    __syncthreads();
    for (int i = warp; i < n; i += kWarps) {
      float delta = 0.f;
      for (int c = lane; c < a.dim; c += 32) delta = fmaf(g[i * pitch + c], out[i * pitch + c], delta);
      delta = warp_sum(delta);
      float w = 0.f, d = 0.f;
      if (lane <= i) {
        w = exp2f(__fsub_rn(__fmul_rn(dot(q + i * pitch, k + lane * pitch, width), a.scale * kLog2e), lse[i]));
        d = w * (dot(g + i * pitch, v + lane * pitch, width) - delta);
      }
      p[i * 33 + lane] = w;
      ds[i * 33 + lane] = d;
    }
    __syncthreads();
    if (a.dq) {
      for (int i = warp; i < n; i += kWarps) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (col < width) {
#pragma unroll 4
          for (int j = 0; j <= i; ++j) add4(o, ds[i * 33 + j], at4(k + j * pitch + col));
        }
        const float4 r = make_float4(o.x * a.scale, o.y * a.scale, o.z * a.scale, o.w * a.scale);
        store4(a.dq + ((int64_t)(t.x + i) * a.heads + head) * a.dim, r, col, a.dim);
      }
    }
    if (a.dk && col < width) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int j = warp + r * kWarps;
#pragma unroll 4
        for (int i = j; i < n; ++i) {
          add4(dv[r], p[i * 33 + j], at4(g + i * pitch + col));
          add4(dk[r], ds[i * 33 + j], at4(q + i * pitch + col));
        }
      }
    }
    __syncthreads();  // q and g are loaded anew
  }
  if (!a.dk) return;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int j = warp + r * kWarps;
    if (j >= n) break;
    const int64_t at = ((int64_t)(t.x + j) * a.kv_heads + kv_head) * a.dim;
    store4(a.dk + at, make_float4(dk[r].x * a.scale, dk[r].y * a.scale, dk[r].z * a.scale, dk[r].w * a.scale), col, a.dim);
    store4(a.dv + at, dv[r], col, a.dim);
  }
}

}  // namespace

// a.tile: one tile a sequence, none over kShortRows tokens; `longest`: the longest.
lmpb_status attention_short(const AttentionArgs& a, int longest, cudaStream_t st) {
  const size_t smem = (size_t)3 * longest * pitch_of(a.dim) * sizeof(float);  // at most 49.5 KB
  if (smem > 48 * 1024)
    LMPB_CUDA_TRY(cudaFuncSetAttribute(forward_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  forward_kernel<<<dim3((unsigned)a.tiles, (unsigned)a.heads), kThreads, smem, st>>>(a, longest);
  return launch_status("attention (short)");
}

lmpb_status attention_short_backward(const AttentionArgs& a, int longest, cudaStream_t st) {
  const size_t smem = ((size_t)5 * longest * pitch_of(a.dim) + longest * 67) * sizeof(float);  // at most 91 KB
  if (smem > 48 * 1024)
    LMPB_CUDA_TRY(cudaFuncSetAttribute(backward_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  backward_kernel<<<dim3((unsigned)a.tiles, (unsigned)a.kv_heads), kThreads, smem, st>>>(a, longest);
  return launch_status("attention_backward (short)");
}

}  // namespace lmpb
