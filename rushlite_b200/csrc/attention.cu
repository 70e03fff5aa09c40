// Causal attention over packed sequences, float32: the C entries, the
// packed-sequence handle and the fp32 kernels.
//
//   S = scale * q k^T,  row i of a sequence sees its keys j <= i
//   P = exp(S) / sum_j exp(S),  o = P v;  kept for the backward: lse = log2(sum_j exp(S))
//   backward, with delta_i = sum(grad_i * o_i):
//   dP = grad v^T,  dS = P * (dP - delta),  dq = scale * dS k,  dk = scale * dS^T q,  dv = P^T grad
//
// Query head h reads key/value head h / (heads / kv_heads); dk and dv sum
// over the query heads of their group.
//
// The kernels here compute in plain fp32 (FFMA) with 64 x 64 tiles of S: a
// running row maximum and sum forward; backward dq by query tile, then dk and
// dv by key tile, walking the group's heads in order, so no sum depends on an
// order of atomics.  They serve the sequences and head groups whose values the
// fp16 split of the tensor-core path cannot carry (one launch behind that
// path's reads its flags and mostly ends there, 3 us), and more heads than its
// grids hold.  Masked positions never enter a sum, so a NaN or infinity in a
// row that a query does not see does not reach it.  Bound: FFMA and the
// shared-memory loads that feed it, [16384] x 8 heads (2) of 128: forward
// 16 ms, backward 65, against 1.15 and 4.8 on the tensor cores; 36 and 81 for
// flagged sequences, as that launch is one CTA an SM.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <numeric>
#include <vector>

#include "attention.cuh"

namespace lmpb {
namespace {

constexpr int kB = 64;        // rows and columns of an S tile
constexpr int kThreads = 256;  // 16 x 16, a 4 x 4 block of S each
constexpr int kPad = 4;
constexpr float kLog2e = 1.4426950408889634f;

// Rows [row0, row0 + 64) of head `head` of a [*, heads, dim] tensor, zero
// behind `n` rows and `dim` columns.
template <int DP>
__device__ __forceinline__ void load_tile(float (*dst)[DP + kPad], const float* __restrict__ src, int64_t row0, int n,
                                          int heads, int head, int dim, bool vec) {
  const float* base = src + (row0 * heads + head) * dim;
  const int64_t pitch = (int64_t)heads * dim;
  if (vec) {
    for (int i = threadIdx.x; i < kB * (DP / 4); i += kThreads) {
      const int r = i / (DP / 4), c = (i % (DP / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < n && c < dim) v = __ldg(reinterpret_cast<const float4*>(base + r * pitch + c));
      *reinterpret_cast<float4*>(&dst[r][c]) = v;
    }
  } else {
    for (int i = threadIdx.x; i < kB * DP; i += kThreads) {
      const int r = i / DP, c = i % DP;
      dst[r][c] = r < n && c < dim ? __ldg(base + r * pitch + c) : 0.f;
    }
  }
}

// s[i][j] = a[4 ty + i] . b[tx + 16 j]
template <int DP>
__device__ __forceinline__ void dot_tile(const float (*a)[DP + kPad], const float (*b)[DP + kPad], int ty, int tx,
                                         float (&s)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
  for (int c = 0; c < DP; c += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(&a[4 * ty + i][c]);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(&b[tx + 16 * j][c]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s[i][j] += x[i].x * y[j].x + x[i].y * y[j].y + x[i].z * y[j].z + x[i].w * y[j].w;
  }
}

// acc[i][c] += sum_j w(i, j) * b[j][column c of this thread]: columns
// 4 tx + 64 c.. (DP >= 64) or 2 tx (DP = 32).  `w` is read through `get`;
// where `masked`, only pairs that `see(i, j)` allows are added.
template <int DP, typename Get, typename See>
__device__ __forceinline__ void mul_tile(const float (*b)[DP + kPad], int tx, float (&acc)[4][DP / 16], Get get,
                                         bool masked, See see) {
  constexpr int W = DP >= 64 ? 4 : 2, NC = DP / 16 / W;
#pragma unroll 2
  for (int j = 0; j < kB; ++j) {
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = get(i, j);
    float y[DP / 16];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < W; ++k) y[c * W + k] = b[j][c * 16 * W + W * tx + k];
    if (masked) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (see(i, j)) {
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) acc[i][c] += w[i] * y[c];
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) acc[i][c] += w[i] * y[c];
    }
  }
}

// Column of acc[.][c].
template <int DP>
__device__ __forceinline__ int column(int tx, int c) {
  constexpr int W = DP >= 64 ? 4 : 2;
  return (c / W) * 16 * W + W * tx + c % W;
}

__device__ __forceinline__ float over16(float v, bool maximum) {
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = maximum ? fmaxf(v, u) : v + u;
  }
  return v;
}

// Flagged tiles.  Planes: query heads, then key heads, value heads and
// (backward) gradient heads.
__device__ __forceinline__ bool any_flag(const AttentionArgs& a) {
  if (!a.flags) return true;
  const int64_t n = ((int64_t)(a.grad ? 2 : 1) * a.heads + 2 * a.kv_heads) * a.flag_tiles;
  unsigned any = 0;
  for (int64_t i = threadIdx.x; i < n / 16; i += kThreads) {  // the array starts on a 16-byte boundary
    const uint4 f = reinterpret_cast<const uint4*>(a.flags)[i];
    any |= f.x | f.y | f.z | f.w;
  }
  for (int64_t i = n / 16 * 16 + threadIdx.x; i < n; i += kThreads) any |= a.flags[i];
  return __syncthreads_or(any != 0) != 0;
}

// Whether the sequence of tile t needs this group of heads computed: always
// without flags; with them, if any of its tiles in any of the group's planes is flagged.
__device__ __forceinline__ bool wanted(const AttentionArgs& a, const int4& t, int kv_head) {
  if (!a.flags) return true;
  const int n = (t.y + kTileRows - 1) / kTileRows, g = a.heads / a.kv_heads;
  const int planes = a.grad ? 2 * g + 2 : g + 2;
  int any = 0;
  for (int64_t i = threadIdx.x; i < (int64_t)n * planes; i += kThreads) {
    const int p = (int)(i / n);
    const int plane = p < g          ? kv_head * g + p
                      : p < g + 2    ? a.heads + (p - g) * a.kv_heads + kv_head
                                     : a.heads + 2 * a.kv_heads + kv_head * g + (p - g - 2);
    any |= a.flags[(int64_t)plane * a.flag_tiles + t.w + i % n];
  }
  return __syncthreads_or(any) != 0;
}

// Calls body(tile, first row, head) for this CTA's 64-row half tiles: heads
// of one half tile next to each other, those with the most work first.
template <typename F>
__device__ __forceinline__ void for_halves(const AttentionArgs& a, const int* order, int heads, F body) {
  const int64_t items = 2 * (int64_t)a.tiles * heads;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t i = item / heads;
    const int4 t = a.tile[order[i >> 1]];
    const int row0 = t.z * kTileRows + (int)(i & 1) * kB, head = (int)(item % heads);
    if (row0 < t.y && wanted(a, t, head / (heads / a.kv_heads))) body(t, row0, head);
  }
}

template <int DP>
struct ForwardSmem {
  float q[kB][DP + kPad];
  float kv[kB][DP + kPad];
  float p[kB][kB + kPad];
};

// One 64-row query tile of one head; k and v take turns in one buffer.
template <int DP>
__global__ void __launch_bounds__(kThreads) forward_kernel(const AttentionArgs a, bool vec) {
  extern __shared__ __align__(16) unsigned char raw[];
  ForwardSmem<DP>& s = *reinterpret_cast<ForwardSmem<DP>*>(raw);
  after_previous();
  if (!any_flag(a)) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float c = a.scale * kLog2e;
  for_halves(a, a.by_queries, a.heads, [&](const int4& t, int q0, int head) {
    const int kv_head = head / (a.heads / a.kv_heads);
    load_tile<DP>(s.q, a.q, t.x + q0, t.y - q0, a.heads, head, a.dim, vec);
    float acc[4][DP / 16] = {}, m[4], l[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY;
    for (int k0 = 0; k0 <= q0; k0 += kB) {
      const bool diag = k0 == q0;
      load_tile<DP>(s.kv, a.k, t.x + k0, t.y - k0, a.kv_heads, kv_head, a.dim, vec);
      __syncthreads();
      float z[4][4];
      dot_tile<DP>(s.q, s.kv, ty, tx, z);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool see = !diag || tx + 16 * j <= 4 * ty + i;
          z[i][j] = see ? __fmul_rn(z[i][j], c) : -INFINITY;  // rounded as in the backward, so that a weight of 1 is 1
          mx = fmaxf(mx, z[i][j]);  // drops a NaN: exp2f below keeps it in the row's sum
        }
        const float mn = fmaxf(m[i], over16(mx, true));
        const float base = mn == -INFINITY ? 0.f : mn;  // nothing finite yet: all weights 0
        const float alpha = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(z[i][j] - base);
          s.p[4 * ty + i][tx + 16 * j] = p;
          sum += p;
        }
        m[i] = mn;
        l[i] = l[i] * alpha + over16(sum, false);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) acc[i][k] *= alpha;
      }
      __syncthreads();
      load_tile<DP>(s.kv, a.v, t.x + k0, t.y - k0, a.kv_heads, kv_head, a.dim, vec);
      __syncthreads();
      mul_tile<DP>(s.kv, tx, acc, [&](int i, int j) { return s.p[4 * ty + i][j]; }, diag,
                   [&](int i, int j) { return j <= 4 * ty + i; });
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = q0 + 4 * ty + i;
      if (row >= t.y) continue;
      float* o = a.out + ((int64_t)(t.x + row) * a.heads + head) * a.dim;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (column<DP>(tx, k) < a.dim) o[column<DP>(tx, k)] = __fdiv_rn(acc[i][k], l[i]);
      if (tx == 0) a.lse[(int64_t)head * a.tokens + t.x + row] = m[i] + log2f(l[i]);
    }
  });
}

// delta[h, t] = sum(grad * out): a warp per row.
__global__ void __launch_bounds__(kThreads)
    delta_kernel(const float* __restrict__ grad, const float* __restrict__ out, float* __restrict__ delta,
                 int64_t rows, int64_t tokens, int heads, int dim) {
  const int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (i >= rows * heads) return;
  float s = 0.f;
  for (int c = threadIdx.x & 31; c < dim; c += 32) s += grad[i * dim + c] * out[i * dim + c];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) delta[(i % heads) * tokens + i / heads] = s;
}

template <int DP>
struct BackwardSmem {
  float q[kB][DP + kPad];
  float g[kB][DP + kPad];
  float k[kB][DP + kPad];
  float v[kB][DP + kPad];
  float p[kB][kB + kPad];
  float ds[kB][kB + kPad];
};

// P and dS of a 64 x 64 tile from the four tiles in shared memory: rows are
// queries q0.., columns keys k0...
template <int DP, bool kWithP>
__device__ __forceinline__ void probabilities(const AttentionArgs& a, BackwardSmem<DP>& s, const int4& t, int head,
                                              int q0, int k0, int ty, int tx) {
  float z[4][4], d[4][4];
  dot_tile<DP>(s.q, s.k, ty, tx, z);
  dot_tile<DP>(s.g, s.v, ty, tx, d);
  const float c = a.scale * kLog2e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = q0 + 4 * ty + i;
    const bool in = row < t.y;
    const int64_t at = (int64_t)head * a.tokens + t.x + row;
    const float lse = in ? a.lse[at] : 0.f, delta = in ? a.delta[at] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = k0 + tx + 16 * j;
      const bool see = in && key <= row;
      const float p = see ? exp2f(__fsub_rn(__fmul_rn(z[i][j], c), lse)) : 0.f;
      if (kWithP) s.p[4 * ty + i][tx + 16 * j] = p;
      s.ds[4 * ty + i][tx + 16 * j] = see ? p * (d[i][j] - delta) : 0.f;
    }
  }
}

template <int DP>
__device__ __forceinline__ void dq_halves(const AttentionArgs& a, BackwardSmem<DP>& s, bool vec) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for_halves(a, a.by_queries, a.heads, [&](const int4& t, int q0, int head) {
    const int kv_head = head / (a.heads / a.kv_heads);
    load_tile<DP>(s.q, a.q, t.x + q0, t.y - q0, a.heads, head, a.dim, vec);
    load_tile<DP>(s.g, a.grad, t.x + q0, t.y - q0, a.heads, head, a.dim, vec);
    float acc[4][DP / 16] = {};
    for (int k0 = 0; k0 <= q0; k0 += kB) {
      load_tile<DP>(s.k, a.k, t.x + k0, t.y - k0, a.kv_heads, kv_head, a.dim, vec);
      load_tile<DP>(s.v, a.v, t.x + k0, t.y - k0, a.kv_heads, kv_head, a.dim, vec);
      __syncthreads();
      probabilities<DP, false>(a, s, t, head, q0, k0, ty, tx);
      __syncthreads();
      mul_tile<DP>(s.k, tx, acc, [&](int i, int j) { return s.ds[4 * ty + i][j]; }, k0 == q0,
                   [&](int i, int j) { return j <= 4 * ty + i; });
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = q0 + 4 * ty + i;
      if (row >= t.y) continue;
      float* o = a.dq + ((int64_t)(t.x + row) * a.heads + head) * a.dim;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (column<DP>(tx, k) < a.dim) o[column<DP>(tx, k)] = acc[i][k] * a.scale;
    }
  });
}

template <int DP>
__device__ __forceinline__ void dkv_halves(const AttentionArgs& a, BackwardSmem<DP>& s, bool vec) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, group = a.heads / a.kv_heads;
  for_halves(a, a.by_keys, a.kv_heads, [&](const int4& t, int k0, int kv_head) {
    load_tile<DP>(s.k, a.k, t.x + k0, t.y - k0, a.kv_heads, kv_head, a.dim, vec);
    load_tile<DP>(s.v, a.v, t.x + k0, t.y - k0, a.kv_heads, kv_head, a.dim, vec);
    float dk[4][DP / 16] = {}, dv[4][DP / 16] = {};
    for (int head = kv_head * group; head < (kv_head + 1) * group; ++head) {
      for (int q0 = k0; q0 < t.y; q0 += kB) {
        load_tile<DP>(s.q, a.q, t.x + q0, t.y - q0, a.heads, head, a.dim, vec);
        load_tile<DP>(s.g, a.grad, t.x + q0, t.y - q0, a.heads, head, a.dim, vec);
        __syncthreads();
        probabilities<DP, true>(a, s, t, head, q0, k0, ty, tx);
        __syncthreads();
        const bool diag = q0 == k0;
        const auto see = [&](int i, int j) { return 4 * ty + i <= j; };  // row i: the key, j: the query
        mul_tile<DP>(s.g, tx, dv, [&](int i, int j) { return s.p[j][4 * ty + i]; }, diag, see);
        mul_tile<DP>(s.q, tx, dk, [&](int i, int j) { return s.ds[j][4 * ty + i]; }, diag, see);
        __syncthreads();
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = k0 + 4 * ty + i;
      if (row >= t.y) continue;
      const int64_t at = ((int64_t)(t.x + row) * a.kv_heads + kv_head) * a.dim;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const int col = column<DP>(tx, k);
        if (col >= a.dim) continue;
        a.dk[at + col] = dk[i][k] * a.scale;
        a.dv[at + col] = dv[i][k];
      }
    }
  });
}

template <int DP>
__global__ void __launch_bounds__(kThreads) backward_kernel(const AttentionArgs a, bool vec) {
  extern __shared__ __align__(16) unsigned char raw[];
  BackwardSmem<DP>& s = *reinterpret_cast<BackwardSmem<DP>*>(raw);
  after_previous();
  if (!any_flag(a)) return;
  if (a.dq) dq_halves<DP>(a, s, vec);
  if (a.dk) dkv_halves<DP>(a, s, vec);
}

// A CTA per half tile and head; where flags pick the few that are wanted, no
// more than fill the GPU once, since reading the flags is then all most do.
template <typename K>
lmpb_status launch(K kernel, size_t smem, int heads, const AttentionArgs& a, bool vec, const char* what,
                   cudaStream_t st) {
  LMPB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int64_t items = 2 * (int64_t)a.tiles * heads;
  const int64_t grid = std::min<int64_t>(items, a.flags ? sm_count() : INT32_MAX);
  if (a.flags) return launch_early(what, kernel, dim3((unsigned)grid), kThreads, (int)smem, st, a, vec);
  kernel<<<(unsigned)grid, kThreads, smem, st>>>(a, vec);
  return launch_status(what);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

lmpb_status attention_simt(const AttentionArgs& a, cudaStream_t st) {
  const bool vec = a.dim % 4 == 0 && aligned16(a.q) && aligned16(a.k) && aligned16(a.v);
  if (a.dim <= 32) return launch(forward_kernel<32>, sizeof(ForwardSmem<32>), a.heads, a, vec, "attention", st);
  if (a.dim <= 64) return launch(forward_kernel<64>, sizeof(ForwardSmem<64>), a.heads, a, vec, "attention", st);
  return launch(forward_kernel<128>, sizeof(ForwardSmem<128>), a.heads, a, vec, "attention", st);
}

lmpb_status attention_simt_backward(const AttentionArgs& a, cudaStream_t st) {
  const bool vec = a.dim % 4 == 0 && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.grad);
  const char* what = "attention_backward";
  const int heads = a.dq ? a.heads : a.kv_heads;
  if (a.dim <= 32) return launch(backward_kernel<32>, sizeof(BackwardSmem<32>), heads, a, vec, what, st);
  if (a.dim <= 64) return launch(backward_kernel<64>, sizeof(BackwardSmem<64>), heads, a, vec, what, st);
  return launch(backward_kernel<128>, sizeof(BackwardSmem<128>), heads, a, vec, what, st);
}

void use_tiles(AttentionArgs& a, const lmpb_sequences_s* seqs, const lmpb_sequences_s::Tiles& t) {
  a.tile = t.tile, a.by_queries = t.by_queries, a.by_keys = t.by_keys, a.tiles = t.count;
  a.pack = seqs->pack, a.flag_tiles = seqs->packed.count;
}

namespace {

lmpb_status check(const char* what, int64_t tokens, int heads, int kv_heads, int dim, float scale,
                  const lmpb_sequences_s* seqs) {
  const std::string w(what);
  LMPB_CHECK_ARG(seqs, w + ": null sequences");
  LMPB_CHECK_ARG(tokens >= 0 && heads >= 1 && kv_heads >= 1 && dim >= 1, w + ": bad sizes");
  LMPB_CHECK_ARG(dim <= 128, w + ": head_dim " + std::to_string(dim) + " is over 128");
  LMPB_CHECK_ARG(heads % kv_heads == 0, w + ": heads must be a multiple of kv_heads");
  LMPB_CHECK_ARG(heads <= 65535, w + ": at most 65535 heads");
  LMPB_CHECK_ARG(scale > 0.f && scale <= 0x1p64f, w + ": scale must be positive and at most 2^64");
  LMPB_CHECK_ARG(seqs->tokens <= tokens, w + ": the sequences have " + std::to_string(seqs->tokens) +
                                             " tokens, the tensors " + std::to_string(tokens));
  int dev = 0;
  if (seqs->plain.count) {
    LMPB_CUDA_TRY(cudaGetDevice(&dev));
    LMPB_CHECK_ARG(dev == seqs->device, w + ": the sequences are on device " + std::to_string(seqs->device) +
                                            ", the current device is " + std::to_string(dev));
  }
  return LMPB_OK;
}

// Which kernels: the short ones where one CTA a sequence and head is there
// first, the tensor cores' otherwise.
enum class Path { kShort, kTensor, kSimt };

Path path_of(const AttentionArgs& a, const lmpb_sequences_s* seqs) {
  static const char* force = getenv("LMPB_ATTENTION");  // A/B switch: simt, tensor or short
  const bool fits = attention_fits_sm100(a), brief = seqs->longest <= kShortRows;
  if (force && !strcmp(force, "simt")) return Path::kSimt;
  if (force && !strcmp(force, "tensor") && fits) return Path::kTensor;
  if (force && !strcmp(force, "short") && brief) return Path::kShort;
  // About where they meet ([32] x 150, 8 heads of 64: 42 + 88 us short, 39 + 87 on tensor cores; [20] x 10:
  // 8.4 + 11 and 21 + 37; [16] x 1000: 130 + 273 and 98 + 208).
  if (brief && (double)seqs->plain.count * a.heads * seqs->longest * seqs->longest <= 8192.0 * sm_count()) return Path::kShort;
  return fits ? Path::kTensor : Path::kSimt;
}

// Rows behind the last sequence belong to nobody: 0.
lmpb_status clear_tail(float* p, int64_t used, int64_t tokens, int64_t row, cudaStream_t st) {
  if (p && used < tokens) LMPB_CUDA_TRY(cudaMemsetAsync(p + used * row, 0, (size_t)((tokens - used) * row) * 4, st));
  return LMPB_OK;
}

}  // namespace
}  // namespace lmpb

extern "C" lmpb_status lmpb_sequences_create(const int64_t* lengths, int count, lmpb_sequences* handle) {
  using namespace lmpb;
  LMPB_CHECK_ARG(handle, "lmpb_sequences_create: null pointer");
  *handle = nullptr;
  LMPB_CHECK_ARG(count >= 0 && (count == 0 || lengths), "lmpb_sequences_create: bad list of lengths");
  int64_t tokens = 0, tiles = 0, longest = 0;
  for (int i = 0; i < count; ++i) {
    LMPB_CHECK_ARG(lengths[i] >= 0, "lmpb_sequences_create: length " + std::to_string(lengths[i]) + " is negative");
    LMPB_CHECK_ARG(lengths[i] <= INT32_MAX / 2 && tokens + lengths[i] <= INT32_MAX / 2,
                   "lmpb_sequences_create: over 2^30 tokens");
    tokens += lengths[i];
    longest = std::max(longest, lengths[i]);
    tiles += (lengths[i] + kTileRows - 1) / kTileRows;
  }
  lmpb_sequences_s* h = nullptr;
  try {
    h = new lmpb_sequences_s;
    h->tokens = tokens;
    h->longest = longest;
    std::vector<int4> plain, packed;
    std::vector<uchar2> pack;
    int64_t start = 0;
    for (int i = 0; i < count;) {
      // whole sequences that fit one tile together, or one longer sequence
      int end = i;
      int64_t rows = 0;
      while (end < count && (end == i || rows + lengths[end] <= kTileRows)) rows += lengths[end++];
      const int first = (int)packed.size(), n = (int)((rows + kTileRows - 1) / kTileRows);
      const bool shared = end - i > 1;
      for (int k = 0; k < n; ++k) packed.push_back(make_int4((int)start, (int)rows, k, shared ? ~(int)(pack.size() / kTileRows) : first));
      h->pair_tiles += (int64_t)n * (n + 1) / 2;
      if (shared && n) {
        const size_t at = pack.size();
        pack.resize(at + kTileRows, make_uchar2(0, 0));
        int64_t low = 0;
        for (int q = i; q < end; low += lengths[q++])
          for (int64_t r = low; r < low + lengths[q]; ++r) pack[at + r] = make_uchar2((unsigned char)low, (unsigned char)(low + lengths[q]));
      }
      for (; i < end; start += lengths[i++])
        for (int k = 0; k < (int)((lengths[i] + kTileRows - 1) / kTileRows); ++k)
          plain.push_back(make_int4((int)start, (int)lengths[i], k, first));
    }
    // both lists of tiles with their two orders, then the bounds
    std::vector<int> host;
    size_t at[2];
    for (int which = 0; which < 2; ++which) {
      const std::vector<int4>& tile = which ? packed : plain;
      const int n = (int)tile.size();
      at[which] = host.size();
      for (const int4& t : tile) host.insert(host.end(), {t.x, t.y, t.z, t.w});
      std::vector<int> order(n);
      std::iota(order.begin(), order.end(), 0);
      std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return tile[x].z > tile[y].z; });
      host.insert(host.end(), order.begin(), order.end());
      std::iota(order.begin(), order.end(), 0);
      const auto queries = [&](int x) { return (tile[x].y + kTileRows - 1) / kTileRows - tile[x].z; };
      std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return queries(x) > queries(y); });
      host.insert(host.end(), order.begin(), order.end());
      host.resize((host.size() + 3) / 4 * 4);  // int4 boundary
    }
    const size_t pack_at = host.size();
    host.resize(pack_at + pack.size() * sizeof(uchar2) / sizeof(int));
    if (!pack.empty()) std::memcpy(host.data() + pack_at, pack.data(), pack.size() * sizeof(uchar2));
    if (tiles) {
      const size_t bytes = host.size() * sizeof(int);
      cudaError_t e = cudaGetDevice(&h->device);
      if (e == cudaSuccess) e = cudaMalloc(&h->block, bytes);
      if (e == cudaSuccess) e = cudaMemcpy(h->block, host.data(), bytes, cudaMemcpyHostToDevice);
      // a copy from pageable memory may return with its last part under way, and the user's stream need not wait for it
      if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
      if (e != cudaSuccess) {
        cudaGetLastError();
        if (h->block) cudaFree(h->block);
        delete h;
        return set_error(LMPB_ERR_CUDA, std::string("lmpb_sequences_create: ") + cudaGetErrorString(e));
      }
      const int* dev = static_cast<const int*>(h->block);
      for (int which = 0; which < 2; ++which) {
        lmpb_sequences_s::Tiles& t = which ? h->packed : h->plain;
        t.count = (int)(which ? packed : plain).size();
        t.tile = reinterpret_cast<const int4*>(dev + at[which]);
        t.by_queries = dev + at[which] + 4 * t.count;
        t.by_keys = t.by_queries + t.count;
      }
      h->pack = reinterpret_cast<const uchar2*>(dev + pack_at);
    }
  } catch (const std::exception& e) {
    delete h;
    return set_error(LMPB_ERR_INVALID, std::string("lmpb_sequences_create: ") + e.what());
  }
  *handle = h;
  return LMPB_OK;
}

extern "C" lmpb_status lmpb_sequences_release(lmpb_sequences handle) {
  using namespace lmpb;
  if (!handle) return LMPB_OK;
  cudaError_t e = cudaSuccess;
  if (handle->block) {
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev != handle->device) e = cudaSetDevice(handle->device);
    if (e == cudaSuccess) e = cudaFree(handle->block);
    cudaSetDevice(dev);
  }
  delete handle;
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(LMPB_ERR_CUDA, std::string("lmpb_sequences_release: ") + cudaGetErrorString(e));
  }
  return LMPB_OK;
}

extern "C" lmpb_status lmpb_attention(const float* q, const float* k, const float* v, float* out, float* lse,
                                      int64_t tokens, int heads, int kv_heads, int head_dim, float scale,
                                      lmpb_sequences seqs, void* stream) {
  using namespace lmpb;
  lmpb_status s = check("lmpb_attention", tokens, heads, kv_heads, head_dim, scale, seqs);
  if (s != LMPB_OK) return s;
  if (tokens == 0) return LMPB_OK;
  LMPB_CHECK_ARG(q && k && v && out && lse, "lmpb_attention: null pointer");
  cudaStream_t st = as_stream(stream);
  s = clear_tail(out, seqs->tokens, tokens, (int64_t)heads * head_dim, st);
  if (s != LMPB_OK || seqs->plain.count == 0) return s;
  AttentionArgs a{};
  a.q = q, a.k = k, a.v = v, a.out = out, a.lse = lse;
  a.tokens = tokens, a.heads = heads, a.kv_heads = kv_heads, a.dim = head_dim, a.scale = scale;
  a.pair_tiles = seqs->pair_tiles, a.longest_tiles = (seqs->longest + kTileRows - 1) / kTileRows, a.splits = 1, a.share = 1 << 30;
  use_tiles(a, seqs, seqs->packed);
  const Path path = path_of(a, seqs);
  if (path == Path::kTensor) return attention_sm100(a, seqs, st);
  use_tiles(a, seqs, seqs->plain);
  if (path == Path::kShort) return attention_short(a, (int)seqs->longest, st);
  return attention_simt(a, st);
}

extern "C" lmpb_status lmpb_attention_backward(const float* q, const float* k, const float* v, const float* out,
                                               const float* lse, const float* grad, float* dq, float* dk, float* dv,
                                               int64_t tokens, int heads, int kv_heads, int head_dim, float scale,
                                               lmpb_sequences seqs, void* stream) {
  using namespace lmpb;
  lmpb_status s = check("lmpb_attention_backward", tokens, heads, kv_heads, head_dim, scale, seqs);
  if (s != LMPB_OK) return s;
  LMPB_CHECK_ARG((dk == nullptr) == (dv == nullptr), "lmpb_attention_backward: dk and dv go together");
  if (tokens == 0 || (!dq && !dk)) return LMPB_OK;
  LMPB_CHECK_ARG(q && k && v && out && lse && grad, "lmpb_attention_backward: null pointer");
  cudaStream_t st = as_stream(stream);
  s = clear_tail(dq, seqs->tokens, tokens, (int64_t)heads * head_dim, st);
  if (s == LMPB_OK) s = clear_tail(dk, seqs->tokens, tokens, (int64_t)kv_heads * head_dim, st);
  if (s == LMPB_OK) s = clear_tail(dv, seqs->tokens, tokens, (int64_t)kv_heads * head_dim, st);
  if (s != LMPB_OK || seqs->plain.count == 0) return s;
  AttentionArgs a{};
  a.q = q, a.k = k, a.v = v, a.out = const_cast<float*>(out), a.lse = const_cast<float*>(lse), a.grad = grad;
  a.dq = dq, a.dk = dk, a.dv = dv;
  a.tokens = tokens, a.heads = heads, a.kv_heads = kv_heads, a.dim = head_dim, a.scale = scale;
  a.pair_tiles = seqs->pair_tiles, a.longest_tiles = (seqs->longest + kTileRows - 1) / kTileRows, a.splits = 1, a.share = 1 << 30;
  use_tiles(a, seqs, seqs->packed);
  const Path path = path_of(a, seqs);
  if (path == Path::kTensor) return attention_sm100_backward(a, seqs, st);
  use_tiles(a, seqs, seqs->plain);
  if (path == Path::kShort) return attention_short_backward(a, (int)seqs->longest, st);
  float* delta = nullptr;
  LMPB_CUDA_TRY(stream_alloc((void**)&delta, (size_t)tokens * heads * 4, st));
  const int64_t rows = seqs->tokens * heads;
  delta_kernel<<<(unsigned)((rows + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, st>>>(
      grad, out, delta, seqs->tokens, tokens, heads, head_dim);
  s = launch_status("attention_backward (delta)");
  a.delta = delta;
  if (s == LMPB_OK) s = attention_simt_backward(a, st);
  const cudaError_t e = cudaFreeAsync(delta, st);
  if (s == LMPB_OK && e != cudaSuccess)
    return set_error(LMPB_ERR_CUDA, std::string("cudaFreeAsync: ") + cudaGetErrorString(e));
  return s;
}
