// Layer norm over the last axis, forward and backward.
//
//   mean = sum(x) / F,  rstd = 1 / sqrt(sum((x - mean)^2) / F + eps)
//   h = (x - mean) * rstd,  y = h * w + b
//   a = g * w,  dx = rstd * (a - sum(a) / F - h * sum(a * h) / F)
//   dw = sum over rows of g * h,  db = sum over rows of g
//
// Bound: HBM.  A row is read once into registers and everything that needs
// the whole row (the mean, then the centred square sum; in the backward both
// sums at once) is a reduction over those registers, so the forward moves
// x + y and the backward x + g + dx and nothing twice.  The centred second
// pass costs no traffic and has no cancellation for a large mean.
//
// A row of up to 512 values, or 1024 in float32, belongs to one warp (8 rows a
// CTA, no barrier); a row of up to 8192 to a CTA of 256 or 512 threads.
// Longer rows, and in the backward doubles past 4096, are walked in memory
// (the *_long kernels).  The backward's CTAs stay resident and walk
// rows with a stride; each thread keeps its columns' share of dw and db in
// registers, writes it once at its end as one row of a partial table, and a
// second kernel adds the table's rows in their order, so the same call gives
// the same bits.
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"

namespace lmpb {
namespace {

constexpr int kThreads = 256;
// Threads of a CTA whose rows belong to TPR threads each.
constexpr int block_of(int tpr) { return tpr > kThreads ? tpr : kThreads; }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Packet {
  T v[VEC];
};

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the TPR threads of a row, returned to all of them.  For a whole
// CTA, `red` is two alternating buffers of a partial a warp per value (`phase`
// flips), so one barrier per call is enough: a thread can only reach the
// buffer again two barriers later.
template <typename T, int TPR, int N>
__device__ __forceinline__ void row_sum(T (&v)[N], T* red, int& phase) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    T* r = red + phase * (N * W);
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) r[k * W + (threadIdx.x >> 5)] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      T s = r[k * W];
#pragma unroll
      for (int w = 1; w < W; ++w) s += r[k * W + w];
      v[k] = s;
    }
  }
}

__device__ __forceinline__ float inv_sqrt(float v) { return __frcp_rn(__fsqrt_rn(v)); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// NV packets of VEC values a thread: columns (i * TPR + lane) * VEC.
template <typename T, int VEC, int NV, int TPR>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int lane, int F, T (&x)[NV * VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    Packet<T, VEC> u;
    if (c < F) {
      u = *reinterpret_cast<const Packet<T, VEC>*>(p + c);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) u.v[j] = T(0);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[i * VEC + j] = u.v[j];
  }
}

template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(block_of(TPR))
    forward_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, T* __restrict__ y,
                   T* __restrict__ mean_out, T* __restrict__ rstd_out, int64_t rows, int F, T inv_f, T eps) {
  constexpr int RPC = block_of(TPR) / TPR, E = NV * VEC;
  __shared__ T red[2 * (TPR / 32)];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  int phase = 0;
  for (int64_t row = (int64_t)blockIdx.x * RPC + sub; row < rows; row += (int64_t)gridDim.x * RPC) {
    T v[E];
    load_row<T, VEC, NV, TPR>(x + row * F, lane, F, v);
    T s[1] = {T(0)};
#pragma unroll
    for (int i = 0; i < E; ++i) s[0] += v[i];
    row_sum<T, TPR, 1>(s, red, phase);
    const T mean = s[0] * inv_f;
    s[0] = T(0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = (i * TPR + lane) * VEC < F;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i * VEC + j] -= mean;
        if (in) s[0] += v[i * VEC + j] * v[i * VEC + j];
      }
    }
    row_sum<T, TPR, 1>(s, red, phase);
    const T rstd = inv_sqrt(s[0] * inv_f + eps);
    if (lane == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c >= F) continue;
      Packet<T, VEC> u, pw, pb;
      if (w) pw = *reinterpret_cast<const Packet<T, VEC>*>(w + c);
      if (b) pb = *reinterpret_cast<const Packet<T, VEC>*>(b + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        T h = v[i * VEC + j] * rstd;
        if (w) h *= pw.v[j];
        if (b) h += pb.v[j];
        u.v[j] = h;
      }
      *reinterpret_cast<Packet<T, VEC>*>(y + row * F + c) = u;
    }
  }
}

// CTAs an SM must hold of a tile of E values a thread: two where the four
// tiles of a row (x and g, and the next row's) and the two running sums leave
// room for it in registers.
template <typename T, int E, int TPR>
constexpr int resident() { return TPR <= 256 && E * sizeof(T) <= 64 ? 2 : 1; }

// part: [gridDim.x, 2, F] of dw and db, or with one CTA the results
// themselves; null when neither is wanted.  The next row's x and g are loaded
// before this row's sums are awaited ([8192, 4096], with a slower fold than now:
// 77.6 us, without 88, and 109 with the rows fetched by bulk copies into a
// ring in shared memory, since fewer threads are then there to add).
template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(block_of(TPR), resident<T, NV * VEC, TPR>())
    backward_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ mean,
                    const T* __restrict__ rstd, const T* __restrict__ g, T* __restrict__ dx, T* __restrict__ part,
                    T* __restrict__ dw_out, T* __restrict__ db_out, int64_t rows, int F, T inv_f) {
  constexpr int RPC = block_of(TPR) / TPR, E = NV * VEC;
  __shared__ T red[4 * (TPR / 32)];
  extern __shared__ __align__(16) unsigned char fold_raw[];  // at most 8 rows of 4 KB
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  int phase = 0;
  T dw[E], db[E], h[E], a[E];
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = T(0);
  const int64_t step = (int64_t)gridDim.x * RPC;
  int64_t row = (int64_t)blockIdx.x * RPC + sub;
  T mu = T(0), rs = T(0);
  if (row < rows) {
    load_row<T, VEC, NV, TPR>(x + row * F, lane, F, h);
    load_row<T, VEC, NV, TPR>(g + row * F, lane, F, a);
    mu = mean[row], rs = rstd[row];
  }
  for (; row < rows; row += step) {
    T s[2] = {T(0), T(0)};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c >= F) continue;  // h and a are 0 there and stay so
      Packet<T, VEC> pw;
      if (w) pw = *reinterpret_cast<const Packet<T, VEC>*>(w + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int k = i * VEC + j;
        h[k] = (h[k] - mu) * rs;
        dw[k] += a[k] * h[k];
        db[k] += a[k];
        if (w) a[k] *= pw.v[j];
        s[0] += a[k];
        s[1] += a[k] * h[k];
      }
    }
    T nh[E], na[E], nmu = T(0), nrs = T(0);
    const int64_t next = row + step;
    if (next < rows) {
      load_row<T, VEC, NV, TPR>(x + next * F, lane, F, nh);
      load_row<T, VEC, NV, TPR>(g + next * F, lane, F, na);
      nmu = mean[next], nrs = rstd[next];
    }
    if (dx) {  // uniform
      row_sum<T, TPR, 2>(s, red, phase);
      const T m0 = s[0] * inv_f, m1 = s[1] * inv_f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * VEC;
        if (c >= F) continue;
        Packet<T, VEC> u;
#pragma unroll
        for (int j = 0; j < VEC; ++j) u.v[j] = rs * (a[i * VEC + j] - m0 - h[i * VEC + j] * m1);
        *reinterpret_cast<Packet<T, VEC>*>(dx + row * F + c) = u;
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) h[i] = nh[i], a[i] = na[i];
    mu = nmu, rs = nrs;
  }
  T* const prow[2] = {part ? part + (int64_t)blockIdx.x * 2 * F : dw_out, part ? part + ((int64_t)blockIdx.x * 2 + 1) * F : db_out};
  if (!prow[0] && !prow[1]) return;
  if constexpr (RPC == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c >= F) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (prow[0]) prow[0][c + j] = dw[i * VEC + j];
        if (prow[1]) prow[1][c + j] = db[i * VEC + j];
      }
    }
  } else {  // the CTA's rows' owners, added in their order
    T* fold = reinterpret_cast<T*>(fold_raw);  // [RPC, F]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (!prow[which]) continue;  // uniform
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * VEC;
        if (c >= F) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) fold[sub * F + c + j] = which ? db[i * VEC + j] : dw[i * VEC + j];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < F; c += kThreads) {
        T t = fold[c];
#pragma unroll
        for (int r = 1; r < RPC; ++r) t += fold[r * F + c];
        prow[which][c] = t;
      }
      __syncthreads();
    }
  }
}

// out[c] = sum over the table's rows of column c: 32 columns a CTA, 32 row
// lanes folded in order (8 lanes of four times the rows waited 13 us for
// [296, 2 x 4096], these 6.5).  It is launched while the rows' CTAs run and starts as the last one ends: 2.5 us less.
// Columns [0, F) go to dw, [F, 2F) to db.
template <typename T>
__global__ void __launch_bounds__(1024)
    fold_kernel(const T* part, int rows, int F, T* dw, T* db) {
  __shared__ T s[32][33];
  after_previous();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + tx, W = 2 * (int64_t)F;
  T t = T(0);
  if (col < W) {
#pragma unroll 5
    for (int r = ty; r < rows; r += 32) t += part[r * W + col];
  }
  s[ty][tx] = t;
  __syncthreads();
  if (ty == 0 && col < W) {
#pragma unroll
    for (int k = 1; k < 32; ++k) t += s[k][tx];
    T* out = col < F ? dw : db;
    if (out) out[col < F ? col : col - F] = t;
  }
}

// ------------------------------------------------ rows past the tiles

template <typename T>
__global__ void __launch_bounds__(kThreads)
    forward_long_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, T* __restrict__ y,
                        T* __restrict__ mean_out, T* __restrict__ rstd_out, int64_t rows, int64_t F, T inv_f, T eps) {
  __shared__ T red[16];
  int phase = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* p = x + row * F;
    T s[1] = {T(0)};
    for (int64_t c = threadIdx.x; c < F; c += kThreads) s[0] += p[c];
    row_sum<T, kThreads, 1>(s, red, phase);
    const T mean = s[0] * inv_f;
    s[0] = T(0);
    for (int64_t c = threadIdx.x; c < F; c += kThreads) s[0] += (p[c] - mean) * (p[c] - mean);
    row_sum<T, kThreads, 1>(s, red, phase);
    const T rstd = inv_sqrt(s[0] * inv_f + eps);
    if (threadIdx.x == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    for (int64_t c = threadIdx.x; c < F; c += kThreads) {
      T h = (p[c] - mean) * rstd;
      if (w) h *= w[c];
      if (b) h += b[c];
      y[row * F + c] = h;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    backward_long_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ mean,
                         const T* __restrict__ rstd, const T* __restrict__ g, T* __restrict__ dx, int64_t rows,
                         int64_t F, T inv_f) {
  __shared__ T red[32];
  int phase = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *p = x + row * F, *q = g + row * F;
    const T mu = mean[row], rs = rstd[row];
    T s[2] = {T(0), T(0)};
    for (int64_t c = threadIdx.x; c < F; c += kThreads) {
      const T a = w ? q[c] * w[c] : q[c];
      s[0] += a;
      s[1] += a * ((p[c] - mu) * rs);
    }
    row_sum<T, kThreads, 2>(s, red, phase);
    const T m0 = s[0] * inv_f, m1 = s[1] * inv_f;
    for (int64_t c = threadIdx.x; c < F; c += kThreads) {
      const T a = w ? q[c] * w[c] : q[c];
      dx[row * F + c] = rs * (a - m0 - (p[c] - mu) * rs * m1);
    }
  }
}

// dw and db shares of rows [y * chunk, (y + 1) * chunk), one column a thread.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    columns_long_kernel(const T* __restrict__ x, const T* __restrict__ mean, const T* __restrict__ rstd,
                        const T* __restrict__ g, T* __restrict__ part, int64_t rows, int64_t F, int64_t chunk) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= F) return;
  const int64_t r0 = blockIdx.y * chunk, r1 = min(rows, r0 + chunk);
  T dw = T(0), db = T(0);
  for (int64_t r = r0; r < r1; ++r) {
    const T gv = g[r * F + c];
    dw += gv * ((x[r * F + c] - mean[r]) * rstd[r]);
    db += gv;
  }
  T* prow = part + (int64_t)blockIdx.y * 2 * F;
  prow[c] = dw;
  prow[F + c] = db;
}

// ------------------------------------------------------------ host side

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// CTAs of the row walks: enough to fill the GPU, no more than there are rows.
unsigned grid_of(int64_t rows, int rows_per_cta, int ctas_per_sm) {
  const int64_t need = (rows + rows_per_cta - 1) / rows_per_cta;
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(need, (int64_t)sm_count() * ctas_per_sm));
}

// Whether a warp walks a row.  Up to 512 values always; up to 1024 floats
// where there are rows for 8 warps of 8 CTAs on every SM, otherwise a CTA a
// row is there sooner (forward: [16384, 1024] 27 us by warps, 41 by CTAs;
// [1023, 1001] 10.8 and 6.9).
template <typename T>
bool by_warps(int64_t rows, int64_t features) {
  return features <= 512 || (sizeof(T) == 4 && features <= 1024 && rows > 8 * (int64_t)sm_count());
}

// Calls f.run<VEC, NV, TPR>() for the tile that holds a row of F values;
// false when none does.  SUMS: the backward, whose two rows and two sums per
// value have to stay in registers, so doubles spread over 512 threads ([2048,
// 4096]: 50 us, 62 over 256; the forward has less to hold: 33 and 29).  More
// than 4096 values take 512 threads too ([4096, 8192]: forward 52 us, backward
// 76; over 1024 threads 91 and 102).
template <typename T, int VEC, bool SUMS, typename F>
bool with_tile(int64_t rows, int64_t features, F&& f) {
  if (by_warps<T>(rows, features)) {
    if (features <= 32 * 4) f.template run<VEC, 4 / VEC, 32>();
    else if (features <= 32 * 8) f.template run<VEC, 8 / VEC, 32>();
    else if (features <= 32 * 16) f.template run<VEC, 16 / VEC, 32>();
    else if constexpr (sizeof(T) == 4) f.template run<VEC, 32 / VEC, 32>();
    return true;
  }
  if (features <= 256 * 4) {
    f.template run<VEC, 4 / VEC, 256>();
    return true;
  }
  if constexpr (SUMS && sizeof(T) == 8) {
    if (features > 512 * 8) return false;
    if (features <= 512 * 4) f.template run<VEC, 4 / VEC, 512>();
    else f.template run<VEC, 8 / VEC, 512>();
  } else {
    if (features > 8192) return false;
    if (features <= 256 * 8) f.template run<VEC, 8 / VEC, 256>();
    else if (features <= 256 * 16) f.template run<VEC, 16 / VEC, 256>();
    else f.template run<VEC, 16 / VEC, 512>();
  }
  return true;
}

template <typename T>
struct Forward {
  const T *x, *w, *b;
  T *y, *mean, *rstd;
  int64_t rows, F;
  double eps;
  cudaStream_t st;
  template <int VEC, int NV, int TPR>
  void run() const {
    constexpr int B = block_of(TPR);
    forward_kernel<T, VEC, NV, TPR><<<grid_of(rows, B / TPR, 2048 / B), B, 0, st>>>(
        x, w, b, y, mean, rstd, rows, (int)F, T(1.0 / (double)F), T(eps));
  }
};

template <typename T>
struct Backward {
  const T *x, *w, *mean, *rstd, *g;
  T *dx, *part, *dw, *db;
  int64_t rows, F;
  unsigned grid;
  cudaStream_t st;
  template <int VEC, int NV, int TPR>
  void run() const {
    const size_t fold = TPR == 32 && (dw || db) ? (size_t)(kThreads / 32) * F * sizeof(T) : 0;
    backward_kernel<T, VEC, NV, TPR><<<grid, block_of(TPR), fold, st>>>(x, w, mean, rstd, g, dx, part, dw, db, rows, (int)F,
                                                                        T(1.0 / (double)F));
  }
};

template <typename T>
lmpb_status forward(const void* x, const void* w, const void* b, int64_t rows, int64_t F, double eps, void* y,
                    void* mean, void* rstd, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  Forward<T> f{(const T*)x, (const T*)w, (const T*)b, (T*)y, (T*)mean, (T*)rstd, rows, F, eps, st};
  const bool vec = F % V == 0 && aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b);
  if (!(vec ? with_tile<T, V, false>(rows, F, f) : with_tile<T, 1, false>(rows, F, f)))
    forward_long_kernel<T><<<grid_of(rows, 1, 8), kThreads, 0, st>>>(f.x, f.w, f.b, f.y, f.mean, f.rstd, rows, F,
                                                                     T(1.0 / (double)F), T(eps));
  return launch_status("layer_norm");
}

template <typename T>
lmpb_status backward(const void* x, const void* w, const void* mean, const void* rstd, const void* g, int64_t rows,
                     int64_t F, void* dx, void* dw, void* db, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // past the tiles ([20000, 4100] double: 0.63 ms; in a tile of 1024 threads, which spills, 1.43)
  const bool columns = dw || db, lng = F > (sizeof(T) == 8 ? 4096 : 8192);
  const bool vec = F % V == 0 && aligned16(x) && aligned16(g) && aligned16(dx) && aligned16(w);
  const bool warps = by_warps<T>(rows, F);
  // as many CTAs as fit at once, two where resident() allows ([2048, 4096] double: 42 us, 47.5 with twice the CTAs)
  const int fit = F > (warps ? 2048 / (int)sizeof(T) : sizeof(T) == 8 ? 1024 : 4096) ? 1 : 2;
  // a few rows, 8 an owner (warp or CTA): one CTA, whose sums over rows are the results, and one launch instead of
  // two (us: [32, 256] 6.0 and 6.8, [64, 64] 6.1 and 7.0; more rows wait on one another: [128, 64] 8.3 and 6.9,
  // [512, 16] 23 and 6.9, [8192, 1] 354 and 10.3)
  const unsigned grid = !lng && rows * F <= 8192 && rows <= (warps ? 64 : 8) ? 1 : grid_of(rows, warps ? kThreads / 32 : 1, fit);
  const bool table = columns && (lng || grid > 1);
  const int64_t chunk = std::max<int64_t>(32, (rows + 63) / 64);
  const int prows = lng ? (int)((rows + chunk - 1) / chunk) : (int)grid;
  T* part = nullptr;
  if (table) LMPB_CUDA_TRY(stream_alloc((void**)&part, (size_t)prows * 2 * F * sizeof(T), st));
  lmpb_status s = LMPB_OK;
  if (!lng) {
    Backward<T> f{(const T*)x, (const T*)w, (const T*)mean, (const T*)rstd, (const T*)g,
                  (T*)dx,      part,        (T*)dw,         (T*)db,         rows, F, grid, st};
    if (vec) with_tile<T, V, true>(rows, F, f);
    else with_tile<T, 1, true>(rows, F, f);
    s = launch_status("layer_norm_backward");
  } else {
    if (dx) {
      backward_long_kernel<T><<<grid_of(rows, 1, 8), kThreads, 0, st>>>((const T*)x, (const T*)w, (const T*)mean,
                                                                        (const T*)rstd, (const T*)g, (T*)dx, rows, F,
                                                                        T(1.0 / (double)F));
      s = launch_status("layer_norm_backward");
    }
    if (s == LMPB_OK && columns) {
      columns_long_kernel<T><<<dim3((unsigned)((F + kThreads - 1) / kThreads), (unsigned)prows), kThreads, 0, st>>>(
          (const T*)x, (const T*)mean, (const T*)rstd, (const T*)g, part, rows, F, chunk);
      s = launch_status("layer_norm_backward (columns)");
    }
  }
  if (s == LMPB_OK && table) {
    s = launch_early("layer_norm_backward (fold)", fold_kernel<T>, dim3((unsigned)((2 * F + 31) / 32)), 1024, 0, st, part, prows,
                     (int)F, (T*)dw, (T*)db);
  }
  if (part) {
    const cudaError_t e = cudaFreeAsync(part, st);
    if (s == LMPB_OK && e != cudaSuccess)
      return set_error(LMPB_ERR_CUDA, std::string("cudaFreeAsync: ") + cudaGetErrorString(e));
  }
  return s;
}

lmpb_status check(const char* what, int dtype, int64_t rows, int64_t features) {
  const std::string w(what);
  LMPB_CHECK_ARG(dtype == LMPB_FLOAT32 || dtype == LMPB_FLOAT64, w + ": float32 or float64 only");
  LMPB_CHECK_ARG(rows >= 0 && features >= 1, w + ": rows must be >= 0 and features >= 1");
  LMPB_CHECK_ARG(features <= (1 << 30), w + ": at most 2^30 features");
  return LMPB_OK;
}

}  // namespace

}  // namespace lmpb

extern "C" lmpb_status lmpb_layer_norm(int dtype, const void* x, const void* weight, const void* bias, int64_t rows,
                                       int64_t features, double eps, void* y, void* mean, void* rstd, void* stream) {
  using namespace lmpb;
  lmpb_status s = check("lmpb_layer_norm", dtype, rows, features);
  if (s != LMPB_OK) return s;
  LMPB_CHECK_ARG(eps >= 0.0 && std::isfinite(eps), "lmpb_layer_norm: eps must be finite and not negative");
  LMPB_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "lmpb_layer_norm: mean and rstd go together");
  if (rows == 0) return LMPB_OK;
  LMPB_CHECK_ARG(x && y, "lmpb_layer_norm: null pointer");
  return dtype == LMPB_FLOAT32 ? forward<float>(x, weight, bias, rows, features, eps, y, mean, rstd, as_stream(stream))
                               : forward<double>(x, weight, bias, rows, features, eps, y, mean, rstd, as_stream(stream));
}

extern "C" lmpb_status lmpb_layer_norm_backward(int dtype, const void* x, const void* weight, const void* mean,
                                                const void* rstd, const void* grad, int64_t rows, int64_t features,
                                                void* dx, void* dweight, void* dbias, void* stream) {
  using namespace lmpb;
  lmpb_status s = check("lmpb_layer_norm_backward", dtype, rows, features);
  if (s != LMPB_OK) return s;
  if (!dx && !dweight && !dbias) return LMPB_OK;
  const size_t bytes = (size_t)features * dtype_size(dtype);
  if (rows == 0) {  // sums over no rows
    if (dweight) LMPB_CUDA_TRY(cudaMemsetAsync(dweight, 0, bytes, as_stream(stream)));
    if (dbias) LMPB_CUDA_TRY(cudaMemsetAsync(dbias, 0, bytes, as_stream(stream)));
    return LMPB_OK;
  }
  LMPB_CHECK_ARG(x && mean && rstd && grad, "lmpb_layer_norm_backward: null pointer");
  return dtype == LMPB_FLOAT32
             ? backward<float>(x, weight, mean, rstd, grad, rows, features, dx, dweight, dbias, as_stream(stream))
             : backward<double>(x, weight, mean, rstd, grad, rows, features, dx, dweight, dbias, as_stream(stream));
}
