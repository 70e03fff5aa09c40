// Causal attention over packed sequences on the B200 tensor cores, float32 in
// and out: fp16 hi/lo split operands, tcgen05.mma, TMEM.
//
// fp32 accuracy.  A 128-row tile of q, k or v, and each row of grad, is scaled
// by the power of two that puts its largest magnitude into [2^14, 2^15) and
// each element x of it becomes hi = fp16(x), lo = fp16(x - hi); a product of
// two operands is the three MMAs lo.hi + hi.lo + hi.hi (lo.lo is 2^-22 of it).
// hi and lo together hold 22 bits of any x down to 2^-18 of the tile's (row's)
// maximum, and 2^-40 of that maximum below.  Weights and their gradients are
// split the same way on the fly, under a scale for each row of the result that
// they are summed into (see below).  The MMA's fp32 accumulator truncates, so
// nothing accumulates in it for longer than one 128-row block: each block's
// product is drained into registers, where the running sums round to nearest.
//
// Gradients of a loss differ by many powers of two from row to row, and a
// small row is not lost in a larger one: dq of a row depends on its own grad
// alone, and a key may be seen by rows with a small grad only.  So grad has an
// exponent a row; in dq it is that row's, and in dk, dv it joins the weights,
// whose scale is then the largest of a key's row of them in the block.  In the
// forward and in dq, too, a row's weights are scaled by their largest in the
// block: next to values far apart a small weight counts as much as a large one.
//
// Tiles whose values that cannot carry (infinities, NaN, q, k or v with rows
// over 2^18 apart or magnitudes below 2^-60, grad below 2^-110, magnitudes over 2^40, q or k so
// long that a score may pass 2^14, where the rounding of lse moves a weight by
// 2^-10; in the backward also rows of v, or outputs above them, and rows of q
// or k that are together over 2^18 apart) are flagged by the split and the
// backward; the fp32 kernels of attention.cu then redo the sequences and head
// groups that hold one.
//
// 1. Split pass: a CTA per tile and head plane writes the tile's hi and lo as
//    one block in the very layout the MMAs read from shared memory (128-byte
//    swizzled rows of 64 halves), so the kernels fetch operands with plain
//    bulk copies, no tensor maps.  Tiles never span sequences and rows
//    behind a sequence are 0.  For v and grad it also finds the largest row
//    norm, for grad the rows' exponents and the sums delta = sum(grad * out).
// 2. forward_kernel, backward_kernel: one CTA per tile and head (dk and dv: per
//    share of a key tile's work), one CTA per SM.  Warp 0 feeds a ring of
//    parts (the hi or lo half of a block, 16 or 32 KB), warp 1 issues the MMAs,
//    8 (128 columns) or 16 (64) warps compute.  A row of the 128 x 128 score
//    tile lives in one TMEM lane; two or four threads of different warps
//    share it.
//    Scores are overwritten in place by the split weights, which are then the
//    next MMA's A operand straight from TMEM.
//    Every mbarrier wait is bounded; after one expires the thread stops
//    waiting and issuing, runs its loops out and the kernel returns with its
//    TMEM freed and lmpb_device_error set.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"
#include "tcgen05.cuh"

namespace lmpb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kWeightBits = 14.f;  // weights enter the MMA times 2^14

__device__ unsigned int g_attention_error = 0;

// Wait that gives up for good: false from the first expiry on.
struct Waiter {
  bool ok = true;
  unsigned code;
  __device__ __forceinline__ explicit Waiter(unsigned c) : code(c) {}
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) {
    if (ok) ok = mbar_wait_bounded(bar, parity, &g_attention_error, code);
    return ok;
  }
};

// Bytes of one part (hi or lo) and of one tile's block.
template <int DP>
constexpr int part_bytes() { return DP / 64 * 128 * 128; }
template <int DP>
constexpr int block_bytes() { return 2 * part_bytes<DP>(); }

constexpr int kMaxSplits = 16;

// The first tile of tile t's sequence.
__device__ __forceinline__ int first_tile(const int4& tile, int t) { return tile.w < 0 ? t : tile.w; }

// Where the split pass puts things.  Planes: query heads, key heads, value
// heads, gradient heads; a plane's tile t is block plane * tiles + t.
struct Split {
  unsigned char* blocks;
  int* expo;             // the tile was scaled by 2^expo (q, k, v)
  float* norm;           // largest row norm (v; grad: of the scaled rows)
  float* dmax;           // largest |delta| of the scaled rows (grad)
  int* span;             // the tile's rows lie within 2^span (q, k, v)
  unsigned char* flags;
  int* row_expo;         // [heads, tokens]: grad's row was scaled by 2^row_expo; kZeroRow where it is 0
};
// By how many powers of two, together, two operands of a product may exceed
// what the row of a result takes most of its sum from: the halves' step,
// 2^-39 of the largest, is then 2^-21 of that.
constexpr int kMaxSpan = 18;
constexpr int kMaxRowExpo = 110, kZeroRow = 127;  // rows of grad below 2^-110, which this would not carry, are flagged

// ------------------------------------------------------------ split pass

// Two floats in one 64-bit register: sm_100 multiplies and adds them in one
// instruction, and the computing warps are bound by instructions and by the
// power that these take.
struct Two {
  unsigned long long v;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Two bits2(uint32_t a, uint32_t b) { return Two(__uint_as_float(a), __uint_as_float(b)); }

// hi and lo of two values, packed.
__device__ __forceinline__ void split2(Two x, uint32_t& hi, uint32_t& lo) {
  const float2 a = x.get();
  const __half2 h = __floats2half2_rn(a.x, a.y);
  const float2 f = __half22float2(h);
  const float2 d = fma2(Two(f.x, f.y), Two(-1.f), x).get();  // x - hi, exact
  const __half2 l = __floats2half2_rn(d.x, d.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ float two_to(int e) { return __int_as_float((e + 127) << 23); }  // e in [-126, 127]

// Grid: tiles x planes; a warp holds 8 rows (DP = 128) or 16 in registers.
// Lane l holds columns 4 l.. of a row (DP = 128), or lanes l and l + 16 hold
// one of two rows (DP = 64).  Bound by HBM and, one tile a CTA, by latency:
// 32 warps an SM are needed ([1500, 31, 700, 1, 1865] x 24 planes of 128: 27
// us with 16 rows a warp, 25 with 8; 40 planes of the backward: 64 and 50;
// with fold_rows in place of a tree for each row then 22 and 46).
template <int DP>
constexpr int split_warps() { return DP / 8; }

// Eight rows' partial results, one of each in every of their LANES lanes, into
// one row's result a lane: of row lane % LANES / (LANES / 8).  9 shuffles
// (LANES = 32) where a tree for each row takes 40.
template <int LANES, typename F>
__device__ __forceinline__ float fold_rows(float (&x)[8], int lane, F f) {
#pragma unroll
  for (int n = 4, off = LANES / 2; n; n >>= 1, off >>= 1) {
    const bool upper = lane & off;
#pragma unroll
    for (int i = 0; i < n; ++i)
      x[i] = f(upper ? x[i + n] : x[i], __shfl_xor_sync(0xffffffffu, upper ? x[i] : x[i + n], off));
  }
#pragma unroll
  for (int off = LANES / 16; off; off >>= 1) x[0] = f(x[0], __shfl_xor_sync(0xffffffffu, x[0], off));
  return x[0];
}

template <int DP>
__global__ void __launch_bounds__(32 * split_warps<DP>(), 2048 / (64 * split_warps<DP>())) split_kernel(const AttentionArgs a, const Split o, float* __restrict__ delta, bool vec) {
  constexpr int WARPS = split_warps<DP>(), ROWS = 128 / WARPS;  // of a warp
  constexpr int RPS = 128 / DP, STEPS = ROWS / RPS, LANES = 32 / RPS;  // rows a step, steps, lanes a row
  static_assert(STEPS == 8, "fold_rows");
  let_next_start();
  const int64_t plane = blockIdx.y;
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 tile = a.tile[t];
  const int row0 = tile.z * kTileRows, rows = min(kTileRows, tile.y - row0);
  const float* src;
  int heads = a.kv_heads, head;
  bool is_v = false, is_g = false;
  if (plane < a.heads) src = a.q, heads = a.heads, head = (int)plane;
  else if (plane < a.heads + a.kv_heads) src = a.k, head = (int)plane - a.heads;
  else if (plane < a.heads + 2 * a.kv_heads) src = a.v, head = (int)plane - a.heads - a.kv_heads, is_v = true;
  else src = a.grad, heads = a.heads, head = (int)plane - a.heads - 2 * a.kv_heads, is_g = true;
  const int64_t first = (int64_t)(tile.x + row0), pitch = (int64_t)heads * a.dim;
  const float* base = src + first * pitch + (int64_t)head * a.dim;
  const float* obase = is_g ? a.out + first * pitch + (int64_t)head * a.dim : nullptr;
  const int sub = lane / LANES, col = (lane % LANES) * 4;
  auto load4 = [&](const float* p, int r) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r >= rows || col >= a.dim) return v;
    p += r * pitch + col;
    if (vec) return __ldg(reinterpret_cast<const float4*>(p));
    v.x = __ldg(p);
    if (col + 1 < a.dim) v.y = __ldg(p + 1);
    if (col + 2 < a.dim) v.z = __ldg(p + 2);
    if (col + 3 < a.dim) v.w = __ldg(p + 3);
    return v;
  };
  float4 v[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) v[i] = load4(base, warp * ROWS + i * RPS + sub);
  const auto more = [](float x, float y) { return fmaxf(x, y); };
  const auto sum = [](float x, float y) { return x + y; };
  const int r1 = warp * ROWS + lane % LANES / (LANES / 8) * RPS + sub;  // the row whose result fold_rows leaves here
  float part[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
    part[i] = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
  float mx = fold_rows<LANES>(part, lane, more), mn = mx > 0.f ? mx : INFINITY;
  int er = 0;  // of row r1
  if (is_g) {  // each row by its own power of two
    er = min(row_exp(mx), kMaxRowExpo);
    const float f = two_to(er);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const float s = __shfl_sync(0xffffffffu, f, sub * LANES + i * (LANES / 8));
      v[i] = make_float4(v[i].x * s, v[i].y * s, v[i].z * s, v[i].w * s);
    }
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) part[i] = v[i].x * v[i].x + v[i].y * v[i].y + v[i].z * v[i].z + v[i].w * v[i].w;
  float nrm = fold_rows<LANES>(part, lane, sum), dmx = 0.f;
  bool bad = !(nrm < INFINITY);  // infinities and NaN, and values past the range anyway
  if (is_g) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const float4 u = load4(obase, warp * ROWS + i * RPS + sub);
      part[i] = v[i].x * u.x + v[i].y * u.y + v[i].z * u.z + v[i].w * u.w;
    }
    const float d = fold_rows<LANES>(part, lane, sum);
    dmx = fabsf(d);
    bad |= !(dmx < INFINITY);
    if (lane % (LANES / 8) == 0 && r1 < rows) {
      const int64_t at = (int64_t)head * a.tokens + first + r1;
      delta[at] = d * two_to(-er);
      o.row_expo[at] = mx > 0.f ? er : kZeroRow;
    }
  }
  __shared__ float red[4][WARPS];
#pragma unroll
  for (int s = 16; s >= LANES / 8; s >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, s));
    nrm = fmaxf(nrm, __shfl_xor_sync(0xffffffffu, nrm, s));
    dmx = fmaxf(dmx, __shfl_xor_sync(0xffffffffu, dmx, s));
  }
  if (lane == 0) red[0][warp] = mx, red[1][warp] = mn, red[2][warp] = nrm, red[3][warp] = dmx;
  const int bads = __syncthreads_or(bad);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    mx = fmaxf(mx, red[0][w]);
    mn = fminf(mn, red[1][w]);
    nrm = fmaxf(nrm, red[2][w]);
    dmx = fmaxf(dmx, red[3][w]);
  }
  const bool range = mx > 0x1p40f || (is_g ? mn < 0x1p-110f : mx > 0.f && (mx < 0x1p-60f || mn < mx * 0x1p-18f));
  const bool far = !is_v && !is_g && !(nrm * a.scale <= 0x1p14f);  // so |q| |k| scale <= 2^14 of unflagged tiles
  const bool flag = bads || range || far;
  const int e = flag || is_g ? 0 : row_exp(mx);
  const int64_t block = plane * a.tiles + t;
  if (threadIdx.x == 0) {
    o.expo[block] = e;
    o.span[block] = mx > 0.f ? row_exp(mn) - row_exp(mx) : 0;
    o.flags[block] = flag;
    if (is_v || is_g) {
      o.norm[block] = sqrtf(nrm) * 1.0001f;  // rounded sums: never below the norm
      o.dmax[block] = dmx;
    }
  }
  const float s = two_to(e);  // unflagged: e in [-26, 75]
  unsigned char* out = o.blocks + block * block_bytes<DP>();
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int r = warp * ROWS + i * RPS + sub;
    uint2 hi, lo;
    split2(Two(v[i].x * s, v[i].y * s), hi.x, lo.x);
    split2(Two(v[i].z * s, v[i].w * s), hi.y, lo.y);
    // 16-byte chunk c of row r sits at chunk c ^ (r & 7) of its 128 bytes
    const int byte = (col & 63) * 2, at = (col >> 6) * 16384 + r * 128 + ((((byte >> 4) ^ (r & 7)) << 4) | (byte & 15));
    *reinterpret_cast<uint2*>(out + at) = hi;
    *reinterpret_cast<uint2*>(out + part_bytes<DP>() + at) = lo;
  }
}

// ------------------------------------------------------------ PTX helpers

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Descriptors of 128-byte swizzled operand tiles with 8-row atoms 1024 bytes
// apart.  The high word is always the same; the low one holds the address and
// `lbo`, the stride between 64-column groups of an operand whose rows are the K axis.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr & 0x3FFFF) >> 4 | (lbo >> 4) << 16; }
constexpr uint32_t kDescHi = (1024 >> 4) | 1u << 14 | 2u << 29;

// f16 operands, fp32 accumulators, M = 128; B K-major, or with K as its rows.
constexpr uint32_t idesc_of(int n, bool b_rows) {
  return (1u << 4) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// a and b: low descriptor words, or a TMEM address for a.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}

// One lane of a converged warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 2^x to 2^-22 of it; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ Two exp2_fast(Two x) {
  const float2 f = x.get();
  return Two(exp2_fast(f.x), exp2_fast(f.y));
}

// A computing warp's wait: all its lanes go on together, with what the
// barrier orders before them visible to their tcgen05 operations.
__device__ __forceinline__ void warp_wait(Waiter& wait, uint32_t bar, uint32_t parity) {
  wait(bar, parity);
  __syncwarp();
  tc_fence_after();
}

// Barrier of the WARPS computing warps.
template <int WARPS>
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); }

// ------------------------------------------------------------ operand feed
//
// The ring carries parts: all of a tile's lo, then all of its hi, one bulk
// copy each.  The same bytes serve as an operand contracted over D (its rows
// are the product's columns) and as one contracted over tokens (its rows are
// the K axis); only the descriptors differ.  The lo part comes first: the
// accumulator is still small while the two cross products are added, so
// their roundings are, and the lo part is free again after one product.

// Position in a ring of N parts; full and empty barriers are 8 bytes each,
// all full ones first.
template <int DP, int N>
struct Ring {
  uint32_t parts, bars;  // shared addresses
  uint32_t slot = 0, phase = 0, started = 0;
  __device__ __forceinline__ uint32_t part() const { return parts + slot * part_bytes<DP>(); }
  __device__ __forceinline__ uint32_t full() const { return bars + slot * 8; }
  __device__ __forceinline__ uint32_t empty() const { return bars + (N + slot) * 8; }
  __device__ __forceinline__ void next() {
    if (++slot == N) slot = 0, phase ^= 1;
  }
};

template <int DP, int N>
__device__ __forceinline__ void feed(Ring<DP, N>& ring, Waiter& wait, const unsigned char* block) {
#pragma unroll
  for (int part = 1; part >= 0; --part) {
    if (!wait(ring.empty(), ring.phase ^ 1)) return;
    mbar_expect_tx(ring.full(), part_bytes<DP>());
    bulk_load(ring.part(), block + part * part_bytes<DP>(), part_bytes<DP>(), ring.full());
    ring.next();
    ++ring.started;
  }
}

// After the last feed: every copy that was started has landed.
template <int DP, int N>
__device__ __forceinline__ void feed_done(Ring<DP, N> ring) {
  const uint32_t n = min(ring.started, (uint32_t)N);
  for (uint32_t k = 0; k < n; ++k) {
    if (ring.slot == 0) ring.slot = N, ring.phase ^= 1;
    --ring.slot;
    Waiter wait(31);
    wait(ring.full(), ring.phase);
  }
}

// The MMA warp.  An elected lane issues; the whole warp runs along, so that
// addresses stay in uniform registers.  The tensor core's queue holds a few
// MMAs of 64 clocks, and a wait costs the issuing warp 100 clocks and more
// even where nothing is to be waited for, so waits are done while MMAs are
// still queued: the next operand's barrier (and what `ahead` tests) is looked
// at before the last third of a product is issued.  With each wait at the
// place of its need the tensor core idled 1,300 of 4,300 clocks a key block.
template <int DP, int N>
struct Issuer {
  Ring<DP, N> ring;
  Waiter wait;
  bool landed = false;  // what take() waits for, as far as is known

  __device__ __forceinline__ Issuer(uint32_t parts, uint32_t bars, unsigned code) : ring{parts, bars}, wait(code) {}

  // Lanes agree on the outcome; what the barrier orders is visible to the MMAs.
  __device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
    wait(bar, parity);
    wait.ok = __all_sync(0xffffffffu, wait.ok);
    tc_fence_after();
    return wait.ok;
  }
  __device__ __forceinline__ bool test(uint32_t bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, mbar_test(bar, parity));
  }
  // The next operand: with DP = 64 both its parts, else the first.
  __device__ __forceinline__ bool take() {
    if (landed) tc_fence_after();
    else if (!wait_for(ring.full(), ring.phase)) return false;
    if (DP == 64 && !landed) {
      Ring<DP, N> second = ring;
      second.next();
      if (!wait_for(second.full(), second.phase)) return false;
    }
    landed = false;
    return true;
  }

  // D[128, 128] = A (shared, resident block) . B^T, B the ring's next tile.
  // `done`, if not 0, is signalled when this and all products before are done.
  template <typename Ahead>
  __device__ __forceinline__ void columns(uint32_t d, uint32_t a_block, uint32_t done, Ahead ahead) {
    constexpr uint32_t idesc = idesc_of(128, false);
    constexpr int U = DP / 64;
    const uint32_t ah = desc_lo(a_block, 16), al = ah + (part_bytes<DP>() >> 4);
    product<4 * U>([&](uint32_t b, int k, bool lo_a, uint32_t acc) {  // 16 columns = 32 bytes a step, 64 a swizzle atom
      const uint32_t o = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
      mma_ss(d, (lo_a ? al : ah) + o, b + o, idesc, acc);
    }, 16, done, ahead);
  }

  // D[128, DP] = W . B, W the split weights in TMEM (16 columns for 16
  // tokens: 8 of hi, 8 of lo), B the ring's next tile.
  template <typename Ahead>
  __device__ __forceinline__ void rows(uint32_t d, uint32_t w, uint32_t done, Ahead ahead) {
    constexpr uint32_t idesc = idesc_of(DP, true);
    product<8>([&](uint32_t b, int k, bool lo_w, uint32_t acc) {  // 16 rows = 2048 bytes a step
      mma_ts(d, w + k * 16 + (lo_w ? 8 : 0), b + k * (2048 >> 4), idesc, acc);
    }, 16384, done, ahead);
  }

  // With DP = 64 a product is 768 clocks of MMAs, against which three separate
  // runs of the issuing lane weigh too much: both parts are awaited at once.
  // With DP = 128 it is 1,536, and the ring is too short to hold them so long.
  template <int STEPS, typename Mma, typename Ahead>
  __device__ __forceinline__ void product(Mma mma, uint32_t lbo, uint32_t done, Ahead ahead) {
    if (!take()) return;
    const uint32_t lo = desc_lo(ring.part(), lbo), lo_free = ring.empty();
    ring.next();
    if (DP == 128) {
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) mma(lo, k, false, k != 0);
        mma_commit(lo_free);
      }
      __syncwarp();
      if (!wait_for(ring.full(), ring.phase)) return;
    }
    const uint32_t hi = desc_lo(ring.part(), lbo), hi_free = ring.empty();
    ring.next();
    if (DP == 128) {
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) mma(hi, k, true, 1);
      }
      __syncwarp();
      landed = test(ring.full(), ring.phase);
      ahead();
    }
    if (elect_one()) {
      if (DP == 64) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) mma(lo, k, false, k != 0);
        mma_commit(lo_free);
#pragma unroll
        for (int k = 0; k < STEPS; ++k) mma(hi, k, true, 1);
      }
#pragma unroll
      for (int k = 0; k < STEPS; ++k) mma(hi, k, false, 1);
      mma_commit(hi_free);
      if (done) mma_commit(done);
    }
    __syncwarp();
    if (DP == 64) {
      Ring<DP, N> second = ring;
      second.next();
      landed = test(ring.full(), ring.phase) && test(second.full(), second.phase);
      ahead();
    }
  }
};

// Signals `bar` when every product issued so far is done.
__device__ __forceinline__ void commit(uint32_t bar) {
  if (elect_one()) mma_commit(bar);
  __syncwarp();
}

// ------------------------------------------------------------ shared memory

constexpr int kBars = 48;

// A kernel's warps: four that feed, issue or idle, then W that compute, four
// of them to each share of a score row's columns.  The launch gives every
// warp the same registers (what __launch_bounds__ leaves, LAUNCH); the first
// four keep LOW of theirs so that the others can have HIGH.
template <int W, int LAUNCH, int LOW, int HIGH>
struct Warps {
  static constexpr int kWarps = W, kParts = W / 4, kCols = 128 / kParts, kThreads = (4 + W) * 32;
  static_assert(4 * LOW + W * HIGH <= (4 + W) * LAUNCH, "more registers than the launch has");
  static __device__ __forceinline__ void few() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(LOW)); }
  static __device__ __forceinline__ void many() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(HIGH)); }
};
using Warps8 = Warps<8, 168, 88, 208>;
using Warps16 = Warps<16, 96, 64, 104>;
// With DP = 64, where the weights' arithmetic weighs as much as the MMAs, 16
// warps (backward of [8192] x 16 heads (4) 1.65 ms, of [1024] x 4 x 8 heads (2) 89 us, with 8
// warps 1.68 and 97; forward 0.392 ms and 33.0 us, with 8 warps 0.382 and 31.1;
// a forward of two pipelines of 8 that take the key blocks in turn 0.42).
// With DP = 128, where the MMAs outweigh it, 8 warps of twice the registers.
template <int DP>
using WarpsOf = std::conditional_t<DP == 64, Warps16, Warps8>;

template <int DP, int RESIDENT, int RING, int SCRATCH>
struct Layout {
  static constexpr int kRing = RESIDENT * block_bytes<DP>();
  static constexpr int kBarsAt = kRing + RING * part_bytes<DP>();
  static constexpr int kScratch = kBarsAt + kBars * 8 + 16;
  static constexpr int kBytes = kScratch + SCRATCH;
  static_assert(kBytes <= 232448, "over 227 KB of shared memory");
};

template <int DP>
constexpr int forward_ring() { return DP == 64 ? 8 : 5; }
template <int DP>
constexpr int backward_ring() { return DP == 64 ? 8 : 3; }
template <int DP>
using ForwardLayout = Layout<DP, 1, forward_ring<DP>(), 2 * WarpsOf<DP>::kParts * 128 * 4>;
template <int DP>
using BackwardLayout = Layout<DP, 2, backward_ring<DP>(), 5 * 128 * 4>;

// Sets up the barriers and all of TMEM, then waits for the kernel ahead; every thread calls it.  False (for
// all) when the shared memory does not start on a swizzle atom.
__device__ __forceinline__ bool setup(unsigned char* smem, uint32_t bars, uint32_t* slot, int ring, const int* counts, int n) {
  const int warp = threadIdx.x >> 5;
  const bool aligned = (smem_u32(smem) & 1023u) == 0;
  if (!aligned) {
    after_previous();
    if (threadIdx.x == 0) atomicCAS(&g_attention_error, 0u, 99u);
    return false;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * ring; ++i) mbar_init(bars + 8 * i, 1);
    for (int i = 0; i < n; ++i) mbar_init(bars + 8 * (2 * ring + i), counts[i]);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_start();
  after_previous();
  if (*slot != 0) {  // 512 columns can only start at 0
    if (warp == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(*slot) : "memory");
    if (threadIdx.x == 0) atomicCAS(&g_attention_error, 0u, 98u);
    return false;
  }
  return true;
}

__device__ __forceinline__ void teardown(uint32_t tmem) {
  tc_fence_before();
  __syncthreads();
  if ((threadIdx.x >> 5) == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// What a computing thread is.  TMEM lane quarter warp % 4, so rows quarter * 32
// + lane; each four warps in a row take the next PARTS-th of a score row's
// columns and of D.
template <int PARTS>
struct Who {
  int row, part;
  uint32_t lanes;  // TMEM lane offset of this warp's quarter
  __device__ __forceinline__ explicit Who(int first_warp) {
    const int warp = threadIdx.x >> 5;
    row = (warp & 3) * 32 + (threadIdx.x & 31);
    part = (warp - first_warp) >> 2;
    lanes = (uint32_t)((warp & 3) * 32) << 16;
  }
};

// A computing warp is done with what `bar` guards (one arrival a warp).
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// acc = acc (* alpha) + f * this thread's C columns of a drained block.
template <int C, bool RESCALE>
__device__ __forceinline__ void drain(uint32_t taddr, float (&acc)[C], float alpha, float f) {
#pragma unroll
  for (int c = 0; c < C; c += 16) {
    uint32_t r[16];
    tmem_ld16_issue(taddr + c, r);
    tmem_ld_wait();
    tmem_regs_ready(r);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const Two x(acc[c + i], acc[c + i + 1]);
      const float2 s = fma2(bits2(r[i], r[i + 1]), Two(f), RESCALE ? mul2(x, Two(alpha)) : x).get();
      acc[c + i] = s.x, acc[c + i + 1] = s.y;
    }
  }
}

// One row's share of a result: columns [c0, c0 + C).
template <int C>
__device__ __forceinline__ void store_row(float* p, const float (&acc)[C], int c0, int dim, float f, bool vec) {
  if (vec) {
#pragma unroll
    for (int c = 0; c < C; c += 4)
      if (c0 + c < dim)
        *reinterpret_cast<float4*>(p + c0 + c) = make_float4(acc[c] * f, acc[c + 1] * f, acc[c + 2] * f, acc[c + 3] * f);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c0 + c < dim) p[c0 + c] = acc[c] * f;
  }
}

// ------------------------------------------------------------ forward
//
// TMEM: scores of even and odd key blocks in columns [0, 128) and [128, 256),
// their products with v in [256, 256 + DP) and [384, 384 + DP).  While the computing warps
// turn block j's scores into weights, the MMAs of block j + 1's scores run.

template <int DP>
__global__ void __launch_bounds__(WarpsOf<DP>::kThreads, 1) forward_kernel(const AttentionArgs a, const Split sp, bool vec_out) {
  extern __shared__ __align__(1024) unsigned char smem[];
  using L = ForwardLayout<DP>;
  using W = WarpsOf<DP>;
  constexpr int WARPS = W::kWarps, PARTS = W::kParts, COLS = W::kCols;
  constexpr int RING = forward_ring<DP>();
  const uint32_t base = smem_u32(smem), bars = base + L::kBarsAt;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + L::kBarsAt + kBars * 8);
  // q, scores of each parity, weights, product of each parity, end
  const int counts[7] = {1, 1, 1, WARPS, 1, 1, 1};
  if (!setup(smem, bars, slot, RING, counts, 7)) return;
  const uint32_t qfull = bars + 16 * RING, sfull = qfull + 8, pfull = qfull + 24, ofull = qfull + 32, done = qfull + 48;
  const auto phase2 = [](int j) { return (uint32_t)(j >> 1) & 1; };  // of a barrier that every other block uses
  constexpr uint32_t tmem = 0;  // all of it was allocated
  const int order = blockIdx.x / a.heads, head = blockIdx.x % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const int t = a.by_queries[order];
  const int4 tile = a.tile[t];
  const int n = tile.z + 1;  // key blocks
  const int64_t kplane = (int64_t)(a.heads + kv_head) * a.tiles + first_tile(tile, t);
  const int64_t vplane = kplane + (int64_t)a.kv_heads * a.tiles;
  const int64_t qblock = (int64_t)head * a.tiles + t;
  const int warp = threadIdx.x >> 5;
  if (warp < 4) {
    W::few();
    const unsigned char *kblocks = sp.blocks + kplane * block_bytes<DP>(), *vblocks = sp.blocks + vplane * block_bytes<DP>();
    if (warp == 0 && (threadIdx.x & 31) == 0) {
      Ring<DP, RING> ring{base + L::kRing, bars};
      Waiter wait(1);
      mbar_expect_tx(qfull, block_bytes<DP>());
      bulk_load(base, sp.blocks + qblock * block_bytes<DP>(), block_bytes<DP>(), qfull);
      feed(ring, wait, kblocks);
      for (int j = 0; j < n; ++j) {
        if (j + 1 < n) feed(ring, wait, kblocks + (j + 1) * block_bytes<DP>());
        feed(ring, wait, vblocks + j * block_bytes<DP>());
      }
      feed_done(ring);
      Waiter last(32);
      last(qfull, 0);
    } else if (warp == 1) {
      Issuer<DP, RING> mma(base + L::kRing, bars, 2);
      const auto nothing = [] {};
      mma.wait_for(qfull, 0);
      mma.columns(tmem, base, sfull, nothing);
      for (int j = 0; j < n && mma.wait.ok; ++j) {
        // block j's weights; that they are there also says that block j - 2's product is drained
        bool weights = false;
        if (j + 1 < n)
          mma.columns(tmem + ((j + 1) & 1) * 128, base, sfull + 8 * ((j + 1) & 1), [&] { weights = mma.test(pfull, j & 1); });
        if (!weights) mma.wait_for(pfull, j & 1);
        else tc_fence_after();
        if (mma.wait.ok) mma.rows(tmem + 256 + (j & 1) * 128, tmem + (j & 1) * 128, ofull + 8 * (j & 1), nothing);
      }
      Waiter last(33);  // nothing of this CTA is in flight when it ends
      commit(done);
      last(done, 0);
    }
  } else {
    W::many();
    constexpr int C = DP / PARTS;
    const Who<PARTS> me(4);
    Waiter wait(3);
    float acc[C], m = -INFINITY, l = 0.f, alpha = 0.f, of = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    const int eq = sp.expo[qblock];
    int ek = sp.expo[kplane], ev = sp.expo[vplane];
    // of the last block a row sees columns low..row, low its sequence's first:
    // this thread's column i if unsigned(col0 + i) < span
    const int low = a.low_of(tile, me.row), col0 = me.part * COLS - low;
    const unsigned span = me.row - low + 1;
    const uint32_t own = tmem + me.lanes + me.part * COLS, oown = tmem + 256 + me.lanes + me.part * C;
    float* xch = reinterpret_cast<float*>(smem + L::kScratch) + me.row;  // [2][PARTS][128]
    const auto drain_block = [&](int j) {
      warp_wait(wait, ofull + 8 * (j & 1), phase2(j));
      drain<C, true>(oown + (j & 1) * 128, acc, alpha, of);
    };
    const auto block = [&](int j, auto diagonal) {
      constexpr bool diag = decltype(diagonal)::value;
      const float c = ldexpf(a.scale * kLog2e, -(eq + ek));
      const float f = two_to(-ev);
      if (j + 1 < n) ek = sp.expo[kplane + j + 1], ev = sp.expo[vplane + j + 1];
      const uint32_t s = own + (j & 1) * 128;
      warp_wait(wait, sfull + 8 * (j & 1), phase2(j));
      // scores are read twice, for the maximum and for the weights: kept, they
      // would spill, and with all of L1 given to shared memory that costs more
      float mx = -INFINITY;
#pragma unroll 2
      for (int k = 0; k < COLS; k += 16) {
        uint32_t r[16];
        tmem_ld16(s + k, r);
        if (diag) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (unsigned(col0 + k + i) >= span) r[i] = 0xff800000u;  // -inf
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, __uint_as_float(r[i]));
      }
      float* x = xch + (j & 1) * (128 * PARTS);
      x[me.part * 128] = mx;
      compute_sync<WARPS>();
#pragma unroll
      for (int k = 0; k < PARTS; ++k) mx = fmaxf(mx, x[k * 128]);
      // The weights are split relative to the block's own largest (finite: every row sees a key of every block):
      // relative to the row's, those of a block of large v but small weights would lose their bits.
      const float mb = mx * c, mn = fmaxf(m, mb), next = exp2_fast(m - mn), up = exp2_fast(mb - mn);
      const float bias = kWeightBits - mb;
      Two sums(0.f);
#pragma unroll 2
      for (int k = 0; k < COLS; k += 16) {
        uint32_t r[16], w[16];
        tmem_ld16(s + k, r);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          Two p = exp2_fast(fma2(bits2(r[i], r[i + 1]), Two(c), Two(bias)));
          if (diag) {  // by index: a scale of 0 makes NaN of -inf
            float2 q = p.get();
            if (unsigned(col0 + k + i) >= span) q.x = 0.f;
            if (unsigned(col0 + k + i + 1) >= span) q.y = 0.f;
            p = Two(q.x, q.y);
          }
          sums = add2(sums, p);
          split2(p, w[i / 2], w[8 + i / 2]);
        }
        tmem_st16(s + k, w);
      }
      tmem_st_wait();
      warp_arrive(pfull);
      l = l * next + (sums.get().x + sums.get().y) * up;
      m = mn;
      if (j > 0) drain_block(j - 1);
      alpha = next;
      of = f * up;
    };
    for (int j = 0; j + 1 < n; ++j) block(j, std::false_type{});
    block(n - 1, std::true_type{});
    drain_block(n - 1);
    float* x = xch + (n & 1) * (128 * PARTS);
    x[me.part * 128] = l;
    compute_sync<WARPS>();
    l = 0.f;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) l += x[k * 128];
    const int row = tile.z * kTileRows + me.row;
    if (row < tile.y && wait.ok) {
      const int64_t at = tile.x + row;
      store_row<C>(a.out + (at * a.heads + head) * a.dim, acc, me.part * C, a.dim, __frcp_rn(l), vec_out);
      if (me.part == 0) a.lse[(int64_t)head * a.tokens + at] = m + (log2f(l) - kWeightBits);
    }
  }
  teardown(tmem);
}

// ------------------------------------------------------------ backward
//
// Below, grad and delta are those of the scaled rows, 2^row_expo times the real
// ones.  |dP_ij| <= |grad_i| |v_j|, so with a weight W_ij <= 1 in place of P
// |W (dP - delta)| <= max|grad_i| max|v_j| + |delta_i|, which gives the power
// of two under which it is split into fp16.
//   dq: W_ij = P_ij 2^-M_i, M_i the exponent of the power of two at or above the largest
//   P_ij of row i in the block, and delta is the row's own; each block's product
//   is drained times 2^(M_i - row_expo_i).
//   dk, dv: W_ij = P_ij 2^(-row_expo_i - M_j), M_j the exponent of the power of two at or
//   above the largest P_ij 2^-row_expo_i of key j in the block.  W is dv's
//   operand and the row of dS's; each block's product is drained times 2^M_j.

struct DsScale {
  int e;        // dS enters the MMA times 2^e
  float dp, d;  // dS 2^e = W (dp * dP' - d * delta), dP' the scaled operands' product
};

__device__ __forceinline__ DsScale ds_scale(float gnorm, float vnorm, float dmax, int ev, float weight_bits) {
  DsScale s;
  s.e = min(100, row_exp(fmaf(gnorm, vnorm, dmax)));
  s.dp = ldexpf(1.f, s.e - ev - (int)weight_bits);
  s.d = ldexpf(1.f, s.e - (int)weight_bits);
  return s;
}

// dq of one query tile and head.  TMEM: scores of even and odd key blocks in
// columns [0, 256), overwritten by dS; dP in [256, 384); the block's product
// with k in [384, 384 + DP).  Block j + 1's scores run while the computing
// warps turn block j's scores and dP into dS.
template <int DP>
__device__ __forceinline__ void dq_tile(const AttentionArgs& a, const Split& sp, int cta, bool vec_out) {
  extern __shared__ __align__(1024) unsigned char smem[];
  using L = BackwardLayout<DP>;
  using W = WarpsOf<DP>;
  constexpr int WARPS = W::kWarps, PARTS = W::kParts, COLS = W::kCols;
  constexpr int RING = backward_ring<DP>();
  const uint32_t base = smem_u32(smem), bars = base + L::kBarsAt;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + L::kBarsAt + kBars * 8);
  // q and grad, scores and dP, dS, product, product drained, end
  const int counts[6] = {1, 1, WARPS, 1, WARPS, 1};
  if (!setup(smem, bars, slot, RING, counts, 6)) return;
  const uint32_t resident = bars + 16 * RING, spfull = resident + 8, dsfull = resident + 16, ofull = resident + 24,
                 oempty = resident + 32, done = resident + 40;
  constexpr uint32_t tmem = 0;  // all of it was allocated
  const int order = cta / a.heads, head = cta % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const int t = a.by_queries[order];
  const int4 tile = a.tile[t];
  const int n = tile.z + 1;  // key blocks
  const int64_t kplane = (int64_t)(a.heads + kv_head) * a.tiles + first_tile(tile, t);
  const int64_t vplane = kplane + (int64_t)a.kv_heads * a.tiles;
  const int64_t qblock = (int64_t)head * a.tiles + t;
  const int64_t gblock = qblock + (int64_t)(a.heads + 2 * a.kv_heads) * a.tiles;
  const int warp = threadIdx.x >> 5;
  constexpr int64_t BB = block_bytes<DP>();
  if (warp < 4) {
    W::few();
    if (warp == 0 && (threadIdx.x & 31) == 0) {
      Ring<DP, RING> ring{base + L::kRing, bars};
      Waiter wait(11);
      mbar_expect_tx(resident, 2 * BB);
      bulk_load(base, sp.blocks + qblock * BB, BB, resident);
      bulk_load(base + BB, sp.blocks + gblock * BB, BB, resident);
      feed(ring, wait, sp.blocks + kplane * BB);
      feed(ring, wait, sp.blocks + vplane * BB);
      for (int j = 0; j < n; ++j) {
        if (j + 1 < n) {
          feed(ring, wait, sp.blocks + (kplane + j + 1) * BB);
          feed(ring, wait, sp.blocks + (vplane + j + 1) * BB);
        }
        feed(ring, wait, sp.blocks + (kplane + j) * BB);
      }
      feed_done(ring);
      Waiter last(32);
      last(resident, 0);
    } else if (warp == 1) {
    Issuer<DP, RING> mma(base + L::kRing, bars, 12);
    const auto nothing = [] {};
    mma.wait_for(resident, 0);
    mma.columns(tmem, base, 0, nothing);
    mma.columns(tmem + 256, base + BB, spfull, nothing);
    for (int j = 0; j < n && mma.wait.ok; ++j) {
      bool ds = false, drained = false;
      if (j + 1 < n) mma.columns(tmem + ((j + 1) & 1) * 128, base, 0, [&] { ds = mma.test(dsfull, j & 1); });
      if (!ds) mma.wait_for(dsfull, j & 1);
      else tc_fence_after();
      if (j + 1 < n && mma.wait.ok) {
        mma.columns(tmem + 256, base + BB, spfull, [&] { drained = mma.test(oempty, (j & 1) ^ 1); });
      }
      if (!drained) mma.wait_for(oempty, (j & 1) ^ 1);
      else tc_fence_after();
      if (mma.wait.ok) mma.rows(tmem + 384, tmem + (j & 1) * 128, ofull, nothing);
    }
    Waiter last(33);
    commit(done);
    last(done, 0);
    } else if (warp == 2) {  // dS follows the size of v and is multiplied by k: both far apart are a case for the fp32 kernels
      bool far = false;
#pragma unroll 1
      for (int j = threadIdx.x & 31; j < n; j += 32) far |= sp.span[kplane + j] + sp.span[vplane + j] > kMaxSpan;
      if (far) sp.flags[qblock] = 1;
    }
  } else {
    W::many();
    constexpr int C = DP / PARTS;
    const Who<PARTS> me(4);
    Waiter wait(13);
    float acc[C], of = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    const int row = tile.z * kTileRows + me.row;
    const int64_t at = (int64_t)head * a.tokens + tile.x + row;
    const float lse = row < tile.y ? a.lse[at] : INFINITY;  // rows behind the sequence: no weight
    int eg = row < tile.y ? sp.row_expo[at] : kZeroRow;
    if (eg == kZeroRow) eg = 0;
    const float delta = row < tile.y ? a.delta[at] * two_to(eg) : 0.f;
    const int eq = sp.expo[qblock];
    const float gnorm = sp.norm[gblock];
    int ek = sp.expo[kplane], ev = sp.expo[vplane];
    float vnorm = sp.norm[vplane];
    const int low = a.low_of(tile, me.row), col0 = me.part * COLS - low;
    const unsigned span = me.row - low + 1;
    const uint32_t own = tmem + me.lanes + me.part * COLS, oown = tmem + 384 + me.lanes + me.part * C;
    float* xch = reinterpret_cast<float*>(smem + L::kScratch) + me.row;  // [PARTS][128]
    const auto block = [&](int j, auto diagonal) {
      constexpr bool diag = decltype(diagonal)::value;
      const float c = ldexpf(a.scale * kLog2e, -(eq + ek));
      const DsScale ds = ds_scale(gnorm, vnorm, fabsf(delta), ev, 0.f);
      const float dd = delta * ds.d;
      const int expo = ds.e + eg + ek;
      if (j + 1 < n) ek = sp.expo[kplane + j + 1], ev = sp.expo[vplane + j + 1], vnorm = sp.norm[vplane + j + 1];
      const uint32_t s = own + (j & 1) * 128, dp = own + 256;
      warp_wait(wait, spfull, j & 1);
      float mx = -INFINITY;
#pragma unroll 1
      for (int k = 0; k < COLS; k += 16) {
        uint32_t r[16];
        tmem_ld16(s + k, r);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!diag || unsigned(col0 + k + i) < span) mx = fmaxf(mx, __uint_as_float(r[i]));
      }
      xch[me.part * 128] = mx;  // all warps have read the last block's: dP, which spfull tells of, is written after their dsfull
      compute_sync<WARPS>();
#pragma unroll
      for (int k = 0; k < PARTS; ++k) mx = fmaxf(mx, xch[k * 128]);
      const float top = fminf(fmaxf(ceilf(fmaf(mx, c, -lse)), -112.f), 112.f), bias = -lse - top;
      const float f = ldexpf(a.scale, (int)top - expo);
#pragma unroll
      for (int k = 0; k < COLS; k += 16) {
        uint32_t r[16], u[16], w[16];
        tmem_ld16_issue(s + k, r);
        tmem_ld16_issue(dp + k, u);
        tmem_ld_wait();
        tmem_regs_ready(r);
        tmem_regs_ready(u);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const Two p = exp2_fast(fma2(bits2(r[i], r[i + 1]), Two(c), Two(bias)));
          Two d = mul2(p, fma2(bits2(u[i], u[i + 1]), Two(ds.dp), Two(-dd)));
          if (diag) {
            float2 q = d.get();
            if (unsigned(col0 + k + i) >= span) q.x = 0.f;
            if (unsigned(col0 + k + i + 1) >= span) q.y = 0.f;
            d = Two(q.x, q.y);
          }
          split2(d, w[i / 2], w[8 + i / 2]);
        }
        tmem_st16(s + k, w);
      }
      tmem_st_wait();
      warp_arrive(dsfull);
      if (j > 0) {
        warp_wait(wait, ofull, (j - 1) & 1);
        drain<C, false>(oown, acc, 1.f, of);
        warp_arrive(oempty);
      }
      of = f;
    };
    for (int j = 0; j + 1 < n; ++j) block(j, std::false_type{});
    block(n - 1, std::true_type{});
    warp_wait(wait, ofull, (n - 1) & 1);
    drain<C, false>(oown, acc, 1.f, of);
    if (row < tile.y && wait.ok)
      store_row<C>(a.dq + ((int64_t)(tile.x + row) * a.heads + head) * a.dim, acc, me.part * C, a.dim, 1.f, vec_out);
  }
  teardown(tmem);
}

// Shares of a key tile whose head has `per_head` query blocks; a.splits at most.
__device__ __forceinline__ int shares_of(const AttentionArgs& a, int per_head) {
  return min(a.splits, (per_head * (a.heads / a.kv_heads) + a.share - 1) / a.share);
}

// dk and dv of one key tile and key/value head, over the group's query heads
// and their tiles from the diagonal on: one list of blocks, cut into shares of
// about a.share blocks.  Where a tile has more than one share, their results
// go to a.part [splits, 2, tokens, kv_heads, dim], which join_kernel adds in
// their order.  Rows are keys, columns queries.
// TMEM: scores in columns [0, 128), overwritten by the weights; dP in
// [128, 256), overwritten by dS; the block's shares of dv and dk in
// [256, 256 + DP) and [384, 384 + DP).  The MMAs of a block run scores, dP,
// dv, dk: weights are computed under dP, dS under dv.
//
// Both running sums are held in registers, 2 x DP / PARTS a thread.
template <int DP>
__device__ __forceinline__ void dkv_tile(const AttentionArgs& a, const Split& sp, int cta, bool vec_out) {
  extern __shared__ __align__(1024) unsigned char smem[];
  using L = BackwardLayout<DP>;
  using W = WarpsOf<DP>;
  constexpr int WARPS = W::kWarps, PARTS = W::kParts, COLS = W::kCols;
  constexpr int RING = backward_ring<DP>();
  const uint32_t base = smem_u32(smem), bars = base + L::kBarsAt;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + L::kBarsAt + kBars * 8);
  // of the block's queries [128] each: -lse, -lse - row_expo, 2^-row_expo; then of even and odd blocks: -scaled delta
  float* const stat = reinterpret_cast<float*>(smem + L::kScratch);
  const int per_order = a.kv_heads * a.splits, order = cta / per_order, kv_head = cta % per_order / a.splits;
  const int split = cta % a.splits, group = a.heads / a.kv_heads;
  const int t = a.by_keys[order];
  const int4 tile = a.tile[t];
  const int per_head = (tile.y + kTileRows - 1) / kTileRows - tile.z;  // query blocks of a head
  const int shares = shares_of(a, per_head);
  if (split >= shares) return after_previous();
  const int first = (int)((int64_t)per_head * group * split / shares);
  const int n = (int)((int64_t)per_head * group * (split + 1) / shares) - first;
  // k and v, scores, dP, weights, dS, dv, dv drained, dk, dk drained, end
  const int counts[10] = {1, 1, 1, WARPS, WARPS, 1, WARPS, 1, WARPS, 1};
  if (!setup(smem, bars, slot, RING, counts, 10)) return;
  const uint32_t resident = bars + 16 * RING, sfull = resident + 8, dpfull = resident + 16, pfull = resident + 24,
                 dsfull = resident + 32, vfull = resident + 40, vempty = resident + 48, kfull = resident + 56,
                 kempty = resident + 64, done = resident + 72;
  constexpr uint32_t tmem = 0;  // all of it was allocated
  const int64_t kblock = (int64_t)(a.heads + kv_head) * a.tiles + t;
  const int64_t vblock = kblock + (int64_t)a.kv_heads * a.tiles;
  const int64_t gplanes = (int64_t)(a.heads + 2 * a.kv_heads) * a.tiles;
  // the blocks of this share: query head and tile, counted from the diagonal
  struct Walk {
    int head, x, per_head;
    __device__ __forceinline__ void next() {
      if (++x == per_head) x = 0, ++head;
    }
  };
  const Walk begin{kv_head * group + first / per_head, first % per_head, per_head};
  const auto qblock = [&](const Walk& w) { return (int64_t)w.head * a.tiles + t + w.x; };  // of the q planes
  const int warp = threadIdx.x >> 5;
  constexpr int64_t BB = block_bytes<DP>();
  if (warp < 4) {
    W::few();
    if (warp == 0 && (threadIdx.x & 31) == 0) {
      Ring<DP, RING> ring{base + L::kRing, bars};
      Waiter wait(21);
      mbar_expect_tx(resident, 2 * BB);
      bulk_load(base, sp.blocks + kblock * BB, BB, resident);
      bulk_load(base + BB, sp.blocks + vblock * BB, BB, resident);
      Walk at = begin;
      for (int i = 0; i < n; ++i, at.next()) {
        const unsigned char *q = sp.blocks + qblock(at) * BB, *g = q + gplanes * BB;
        feed(ring, wait, q);
        feed(ring, wait, g);
        feed(ring, wait, g);
        feed(ring, wait, q);
      }
      feed_done(ring);
      Waiter last(32);
      last(resident, 0);
    } else if (warp == 1) {
      Issuer<DP, RING> mma(base + L::kRing, bars, 22);
      const auto nothing = [] {};
      mma.wait_for(resident, 0);
      for (int i = 0; i < n && mma.wait.ok; ++i) {
        bool p = false, v = false, ds = false, k = false;
        mma.columns(tmem, base, sfull, nothing);
        mma.columns(tmem + 128, base + BB, dpfull, [&] { p = mma.test(pfull, i & 1), v = mma.test(vempty, (i & 1) ^ 1); });
        if (!p) mma.wait_for(pfull, i & 1);
        if (!v) mma.wait_for(vempty, (i & 1) ^ 1);
        tc_fence_after();
        if (mma.wait.ok) mma.rows(tmem + 256, tmem, vfull, [&] { ds = mma.test(dsfull, i & 1), k = mma.test(kempty, (i & 1) ^ 1); });
        if (!ds) mma.wait_for(dsfull, i & 1);
        if (!k) mma.wait_for(kempty, (i & 1) ^ 1);
        tc_fence_after();
        if (mma.wait.ok) mma.rows(tmem + 384, tmem + 128, kfull, nothing);
      }
      Waiter last(33);
      commit(done);
      last(done, 0);
    } else if (warp == 2) {
      // dS has one bound for all queries of a block, and is multiplied by q.  Where the bound comes from
      // larger rows of v, or from outputs, and deltas, far above these keys' v (all 0: the sequence's
      // least), and q lies apart too, a query with a small q and dS could lose its bits: a case for the
      // fp32 kernels.
      float vnorm = sp.norm[vblock];
      if (!(vnorm > 0.f)) {
        vnorm = INFINITY;
#pragma unroll 1
        for (int k = (tile.y + kTileRows - 1) / kTileRows; k-- > 0;) {
          const float x = sp.norm[vblock - t + first_tile(tile, t) + k];
          if (x > 0.f) vnorm = fminf(vnorm, x);
        }
      }
      bool far = false;
#pragma unroll 1
      for (int i = threadIdx.x & 31; i < n; i += 32) {
        const int64_t qb = (int64_t)(kv_head * group + (first + i) / per_head) * a.tiles + t + (first + i) % per_head, gb = qb + gplanes;
        const float gv = sp.norm[gb] * vnorm;
        far |= sp.dmax[gb] + gv > two_to(kMaxSpan - sp.span[qb] - sp.span[vblock]) * gv;
      }
      if (far) sp.flags[kblock] = 1;
    }
  } else {
    W::many();
    constexpr int C = DP / PARTS;
    const Who<PARTS> me(4);
    Waiter wait(23);
    float dk[C], dv[C], fk = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) dk[i] = dv[i] = 0.f;
    const int ek = sp.expo[kblock], ev = sp.expo[vblock];
    const float vnorm = sp.norm[vblock];
    // in the diagonal block a key is seen by queries row..high - 1, high its
    // sequence's end: by this thread's column i if unsigned(col0 + i) < span
    const int col0 = me.part * COLS - me.row;
    const unsigned span = a.high_of(tile, me.row) - me.row;
    const uint32_t own = tmem + me.lanes + me.part * COLS, oown = tmem + 256 + me.lanes + me.part * C;
    // the next block's row statistics, a query a thread: lse (first half) or delta, and the exponent
    const int tid = threadIdx.x - 128;
    const float* source = tid < 128 ? a.lse : a.delta;
    float next = 0.f;
    int enext = kZeroRow;
    const auto fetch = [&](const Walk& w) {
      const int r = (tile.z + w.x) * kTileRows + (tid & 127);
      const bool in = tid < 256 && r < tile.y;
      const int64_t from = (int64_t)w.head * a.tokens + tile.x + r;
      next = in ? source[from] : 0.f;
      enext = in ? sp.row_expo[from] : kZeroRow;
    };
    Walk at = begin, ahead = begin;
    fetch(ahead);
    for (int i = 0; i < n; ++i, at.next()) {
      const int64_t qb = qblock(at), gb = qb + gplanes;
      const int eq = sp.expo[qb];
      const float c = ldexpf(a.scale * kLog2e, -(eq + ek));
      const DsScale ds = ds_scale(sp.norm[gb], vnorm, sp.dmax[gb], ev, kWeightBits);
      // All warps are past the last block's weights (vfull was waited for, which
      // their arrival at pfull precedes), so only delta has two buffers.
      float* const st = stat + 384 + (i & 1) * 128;
      if (tid < 128) {  // a gradient of 0, or no query: no weight
        const bool none = enext == kZeroRow;
        stat[tid] = none ? -INFINITY : -next;
        stat[128 + tid] = none ? -INFINITY : -next - (float)enext;
        stat[256 + tid] = none ? 0.f : two_to(-enext);
      } else if (tid < 256) {
        st[tid - 128] = enext == kZeroRow ? 0.f : -(next * two_to(enext)) * ds.d;
      }
      compute_sync<WARPS>();
      ahead.next();
      if (i + 1 < n) fetch(ahead);
      const bool diag = at.x == 0;
      const float4* bias = reinterpret_cast<const float4*>(stat + me.part * COLS);
      const float4* dd = reinterpret_cast<const float4*>(st + me.part * COLS);
      // the other block's delta is done with: here the parts of a row tell each other their M
      signed char* const xch = reinterpret_cast<signed char*>(stat + 384 + (~i & 1) * 128) + 4 * me.row;
      int top = 0;  // M of this thread's key
      warp_wait(wait, sfull, i & 1);
      const auto weights = [&](auto diagonal) {
        float mx = -INFINITY;
#pragma unroll 1
        for (int k = 0; k < COLS; k += 16) {
          uint32_t r[16];
          tmem_ld16(own + k, r);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 b = bias[32 + (k + j) / 4];
            const float2 x[2] = {fma2(bits2(r[j], r[j + 1]), Two(c), Two(b.x, b.y)).get(),
                                 fma2(bits2(r[j + 2], r[j + 3]), Two(c), Two(b.z, b.w)).get()};
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              if (!decltype(diagonal)::value || unsigned(col0 + k + j + 2 * y) < span) mx = fmaxf(mx, x[y].x);
              if (!decltype(diagonal)::value || unsigned(col0 + k + j + 2 * y + 1) < span) mx = fmaxf(mx, x[y].y);
            }
          }
        }
        xch[me.part] = (signed char)(int)fminf(fmaxf(ceilf(mx), -112.f), 112.f);  // none, or next to nothing: -112
        compute_sync<WARPS>();
        top = max((int)xch[0], (int)xch[1]);
        if (PARTS == 4) top = max(top, max((int)xch[2], (int)xch[3]));
        const Two f(two_to((int)kWeightBits - top));
#pragma unroll
        for (int k = 0; k < COLS; k += 16) {
          uint32_t r[16], w[16];
          tmem_ld16_issue(own + k, r);
          tmem_ld_wait();
          tmem_regs_ready(r);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 b = bias[(k + j) / 4], g = bias[64 + (k + j) / 4];
            Two p[2] = {mul2(mul2(exp2_fast(fma2(bits2(r[j], r[j + 1]), Two(c), Two(b.x, b.y))), Two(g.x, g.y)), f),
                        mul2(mul2(exp2_fast(fma2(bits2(r[j + 2], r[j + 3]), Two(c), Two(b.z, b.w))), Two(g.z, g.w)), f)};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (decltype(diagonal)::value) {
                float2 q = p[x].get();
                if (unsigned(col0 + k + j + 2 * x) >= span) q.x = 0.f;
                if (unsigned(col0 + k + j + 2 * x + 1) >= span) q.y = 0.f;
                p[x] = Two(q.x, q.y);
              }
              split2(p[x], w[j / 2 + x], w[8 + j / 2 + x]);
            }
          }
          tmem_st16(own + k, w);
        }
      };
      if (diag) weights(std::true_type{});
      else weights(std::false_type{});
      tmem_st_wait();
      warp_arrive(pfull);
      if (i > 0) {
        warp_wait(wait, kfull, (i - 1) & 1);
        drain<C, false>(oown + 128, dk, 1.f, fk);
        warp_arrive(kempty);
      }
      warp_wait(wait, dpfull, i & 1);
#pragma unroll
      for (int k = 0; k < COLS; k += 16) {
        uint32_t r[16], u[16], w[16];
        tmem_ld16_issue(own + k, r);
        tmem_ld16_issue(own + 128 + k, u);
        tmem_ld_wait();
        tmem_regs_ready(r);
        tmem_regs_ready(u);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 d = dd[(k + j) / 4];
          const Two nd[2] = {Two(d.x, d.y), Two(d.z, d.w)};
#pragma unroll
          for (int x = 0; x < 2; ++x) {  // the weight is exactly hi + lo
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&r[j / 2 + x]));
            const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&r[8 + j / 2 + x]));
            const Two p = add2(Two(h.x, h.y), Two(l.x, l.y));
            split2(mul2(p, fma2(bits2(u[j + 2 * x], u[j + 2 * x + 1]), Two(ds.dp), nd[x])), w[j / 2 + x], w[8 + j / 2 + x]);
          }
        }
        tmem_st16(own + 128 + k, w);
      }
      tmem_st_wait();
      warp_arrive(dsfull);
      warp_wait(wait, vfull, i & 1);
      drain<C, false>(oown, dv, 1.f, two_to(top - (int)kWeightBits));
      warp_arrive(vempty);
      fk = ldexpf(a.scale, top - (ds.e + eq));
    }
    warp_wait(wait, kfull, (n - 1) & 1);
    drain<C, false>(oown + 128, dk, 1.f, fk);
    const int row = tile.z * kTileRows + me.row;
    if (row < tile.y && wait.ok) {
      const int64_t to = ((int64_t)(tile.x + row) * a.kv_heads + kv_head) * a.dim;
      const int64_t values = a.tokens * a.kv_heads * a.dim;
      store_row<C>((shares > 1 ? a.part + 2 * split * values : a.dk) + to, dk, me.part * C, a.dim, 1.f, vec_out);
      store_row<C>((shares > 1 ? a.part + (2 * split + 1) * values : a.dv) + to, dv, me.part * C, a.dim, 1.f, vec_out);
    }
  }
  teardown(tmem);
}

// One launch for both, dk and dv's larger CTAs first.
template <int DP>
__global__ void __launch_bounds__(WarpsOf<DP>::kThreads, 1)
    backward_kernel(const AttentionArgs a, const Split sp, int dkv_ctas, bool vec_dkv, bool vec_dq) {
  if ((int)blockIdx.x < dkv_ctas) dkv_tile<DP>(a, sp, blockIdx.x, vec_dkv);
  else dq_tile<DP>(a, sp, blockIdx.x - dkv_ctas, vec_dq);
}

// dk and dv of the tiles that have several shares, added in their order.
// Grid: tiles x key/value heads, and kJoin shares of a tile's rows.  Latency
// bound, so V = 4 floats a load where rows allow it ([4096] x 8 heads (2) of
// 128 with 8 shares of rows: 9 us, 22 with one float), and one load a thread.
constexpr int kJoin = 16;

template <int V>
__global__ void __launch_bounds__(256) join_kernel(const AttentionArgs a) {
  struct alignas(4 * V) Pack {
    float x[V];
  };
  let_next_start();
  after_previous();
  const int t = blockIdx.x / a.kv_heads, kv_head = blockIdx.x % a.kv_heads;
  const int4 tile = a.tile[t];
  const int shares = shares_of(a, (tile.y + kTileRows - 1) / kTileRows - tile.z);
  if (shares == 1) return;
  const int row0 = blockIdx.y * (kTileRows / kJoin), rows = min(kTileRows / kJoin, tile.y - tile.z * kTileRows - row0);
  const int64_t values = a.tokens * a.kv_heads * a.dim;
  const int packs = a.dim / V;
  for (int i = threadIdx.x; i < rows * packs; i += 256) {
    const int64_t at = ((int64_t)(tile.x + tile.z * kTileRows + row0 + i / packs) * a.kv_heads + kv_head) * a.dim + i % packs * V;
    Pack k{}, v{};
#pragma unroll 4
    for (int s = 0; s < shares; ++s) {
      const Pack x = *reinterpret_cast<const Pack*>(a.part + 2 * s * values + at);
      const Pack y = *reinterpret_cast<const Pack*>(a.part + (2 * s + 1) * values + at);
#pragma unroll
      for (int c = 0; c < V; ++c) k.x[c] += x.x[c], v.x[c] += y.x[c];
    }
    *reinterpret_cast<Pack*>(a.dk + at) = k;
    *reinterpret_cast<Pack*>(a.dv + at) = v;
  }
}

// ------------------------------------------------------------ host side

template <typename K>
lmpb_status allow_smem(K kernel, int bytes) {
  LMPB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return LMPB_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// One allocation for the split blocks and what goes with them.
lmpb_status make_split(AttentionArgs& a, bool backward, int dp, Split& s, float** delta, void** ws, cudaStream_t st) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const size_t planes = (size_t)(backward ? 2 : 1) * a.heads + 2 * a.kv_heads, n = planes * a.tiles;
  const size_t blocks = n * (dp == 64 ? block_bytes<64>() : block_bytes<128>());
  const size_t dbytes = backward ? up((size_t)a.tokens * a.heads * 4) : 0;  // of delta, and of the rows' exponents
  const size_t pbytes = a.splits > 1 ? (size_t)a.splits * 2 * a.tokens * a.kv_heads * a.dim * 4 : 0;
  LMPB_CUDA_TRY(stream_alloc(ws, blocks + 4 * up(4 * n) + up(n) + 2 * dbytes + pbytes, st));
  unsigned char* p = static_cast<unsigned char*>(*ws);
  s.blocks = p;
  s.expo = reinterpret_cast<int*>(p + blocks);
  s.norm = reinterpret_cast<float*>(p + blocks + up(4 * n));
  s.dmax = reinterpret_cast<float*>(p + blocks + 2 * up(4 * n));
  s.span = reinterpret_cast<int*>(p + blocks + 3 * up(4 * n));
  s.flags = p + blocks + 4 * up(4 * n);
  *delta = reinterpret_cast<float*>(s.flags + up(n));
  s.row_expo = reinterpret_cast<int*>(s.flags + up(n) + dbytes);
  if (pbytes) a.part = reinterpret_cast<float*>(s.flags + up(n) + 2 * dbytes);
  return LMPB_OK;
}

template <int DP>
lmpb_status split(const AttentionArgs& a, const Split& s, float* delta, cudaStream_t st) {
  const unsigned planes = (a.grad ? 2 : 1) * a.heads + 2 * a.kv_heads;
  const bool vec = a.dim % 4 == 0 && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.grad) &&
                   (!a.grad || aligned16(a.out));
  split_kernel<DP><<<dim3((unsigned)a.tiles, planes), 32 * split_warps<DP>(), 0, st>>>(a, s, delta, vec);
  return launch_status("attention (split)");
}

template <int DP>
lmpb_status forward(const AttentionArgs& a, const Split& s, cudaStream_t st) {
  lmpb_status r = split<DP>(a, s, nullptr, st);
  if (r == LMPB_OK) r = allow_smem(forward_kernel<DP>, ForwardLayout<DP>::kBytes);
  if (r != LMPB_OK) return r;
  const bool vec = a.dim % 4 == 0 && aligned16(a.out);
  return launch_early("attention", forward_kernel<DP>, dim3((unsigned)(a.tiles * a.heads)), WarpsOf<DP>::kThreads,
                      ForwardLayout<DP>::kBytes, st, a, s, vec);
}

template <int DP>
lmpb_status backward(const AttentionArgs& a, const Split& s, float* delta, cudaStream_t st) {
  lmpb_status r = split<DP>(a, s, delta, st);
  constexpr int bytes = BackwardLayout<DP>::kBytes;
  if (r == LMPB_OK) r = allow_smem(backward_kernel<DP>, bytes);
  if (r != LMPB_OK) return r;
  const int dkv = a.dk ? a.tiles * a.kv_heads * a.splits : 0, dq = a.dq ? a.tiles * a.heads : 0;
  const bool vec_dkv = a.dim % 4 == 0 && aligned16(a.dk) && aligned16(a.dv) && (!a.part || a.tokens * a.kv_heads * a.dim % 4 == 0);
  const bool vec_dq = a.dim % 4 == 0 && aligned16(a.dq);
  r = launch_early("attention_backward", backward_kernel<DP>, dim3((unsigned)(dkv + dq)), WarpsOf<DP>::kThreads, bytes, st, a,
                   s, dkv, vec_dkv, vec_dq);
  if (r == LMPB_OK && dkv > 0 && a.splits > 1)
    r = launch_early("attention_backward (join)", vec_dkv ? join_kernel<4> : join_kernel<1>, dim3((unsigned)(a.tiles * a.kv_heads), kJoin), 256, 0, st, a);
  return r;
}

}  // namespace

bool attention_fits_sm100(const AttentionArgs& a) {
  return (int64_t)a.tiles * a.heads * (kMaxSplits + 1) <= 0x7fffffff && 2 * a.heads + 2 * a.kv_heads <= 65535;
}

// Cuts the dk, dv work of the key tiles into shares, so that no SM ends long
// after the others (one key/value head, or a long sequence): five quarters of
// what an SM gets on average, as dq's CTAs fill what is left, and 2 blocks
// for what starting a CTA and joining the shares cost.  Backward, us:
//                                             2 + 1.25   2 + 1   3 + 1.25
//   [300] x 4 heads (1) of 64                    28        28       32
//   [2500] x 4 (1) of 64                         78        84       77
//   [1024] x 4, 8 (2) of 64                      89        94       93
//   [600, 300, 900] x 12 (1) of 128             102       102      104
//   [1500, 31, 700, 1, 1865] x 16 (4) of 128    320       328      318
void cut_dkv(AttentionArgs& a) {
  const int64_t group = a.heads / a.kv_heads, most = a.longest_tiles * group;
  const double average = (double)a.pair_tiles * a.heads / sm_count();
  a.share = (int)std::min<int64_t>(most, (int64_t)(2 + 1.25 * average));
  a.share = (int)std::max<int64_t>(a.share, (most + kMaxSplits - 1) / kMaxSplits);
  a.splits = (int)((most + a.share - 1) / a.share);
}

lmpb_status attention_sm100(const AttentionArgs& args, const lmpb_sequences_s* seqs, cudaStream_t st) {
  AttentionArgs a = args;
  Split s{};
  float* unused = nullptr;
  void* ws = nullptr;
  const int dp = a.dim <= 64 ? 64 : 128;
  lmpb_status r = make_split(a, false, dp, s, &unused, &ws, st);
  if (r != LMPB_OK) return r;
  r = dp == 64 ? forward<64>(a, s, st) : forward<128>(a, s, st);
  a.flags = s.flags;
  use_tiles(a, seqs, seqs->plain);  // the fp32 kernels for what was flagged
  if (r == LMPB_OK) r = attention_simt(a, st);
  const cudaError_t e = cudaFreeAsync(ws, st);
  if (r == LMPB_OK && e != cudaSuccess)
    return set_error(LMPB_ERR_CUDA, std::string("cudaFreeAsync: ") + cudaGetErrorString(e));
  return r;
}

lmpb_status attention_sm100_backward(const AttentionArgs& args, const lmpb_sequences_s* seqs, cudaStream_t st) {
  AttentionArgs a = args;
  Split s{};
  float* delta = nullptr;
  void* ws = nullptr;
  const int dp = a.dim <= 64 ? 64 : 128;
  if (a.dk) cut_dkv(a);
  lmpb_status r = make_split(a, true, dp, s, &delta, &ws, st);
  if (r != LMPB_OK) return r;
  a.delta = delta;
  r = dp == 64 ? backward<64>(a, s, delta, st) : backward<128>(a, s, delta, st);
  a.flags = s.flags;
  use_tiles(a, seqs, seqs->plain);  // the fp32 kernels for what was flagged
  if (r == LMPB_OK) r = attention_simt_backward(a, st);
  const cudaError_t e = cudaFreeAsync(ws, st);
  if (r == LMPB_OK && e != cudaSuccess)
    return set_error(LMPB_ERR_CUDA, std::string("cudaFreeAsync: ") + cudaGetErrorString(e));
  return r;
}

// Reads and clears the attention kernels' error word (0 = none).
unsigned int attention_take_error() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_attention_error, sizeof v) != cudaSuccess) return 0xFFFFFFFFu;
  if (v) cudaMemcpyToSymbol(g_attention_error, &zero, sizeof zero);
  return v;
}

}  // namespace lmpb
