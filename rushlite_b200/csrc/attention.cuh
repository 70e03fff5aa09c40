// What the attention kernels share: the packed-sequence handle and the call
// of each path.
#pragma once

#include "common.cuh"

// Packed sequences, cut into tiles for the two paths.  One device block holds
// all tables.
//   fp32 kernels: tiles of 128 tokens, the last of a sequence shorter:
//     {sequence's first token, its length, tile within it, its first tensor-core tile}.
//   Tensor cores: the same, except that whole sequences that follow one
//     another and fit 128 rows together share a tile: {first token, rows, 0, ~p},
//     with their rows' bounds in pack[128 p ..].
struct lmpb_sequences_s {
  int device = 0;
  int64_t tokens = 0;
  int64_t longest = 0;
  void* block = nullptr;
  struct Tiles {
    int count = 0;
    const int4* tile = nullptr;
    const int* by_queries = nullptr;  // those with the most keys to visit first
    const int* by_keys = nullptr;     // those with the most queries to visit first
  } plain, packed;
  const uchar2* pack = nullptr;  // of each row: its sequence's first row, and the row behind its last
  int64_t pair_tiles = 0;        // query tile, key tile pairs of the packed tiles
};

namespace lmpb {

constexpr int kTileRows = 128;

// One call's arguments.  q, out, grad, dq: [tokens, heads, dim]; k, v, dk,
// dv: [tokens, kv_heads, dim]; lse, delta: [heads, tokens].
struct AttentionArgs {
  const float *q, *k, *v;
  float *out, *lse;
  const float *grad, *delta;
  float *dq, *dk, *dv;
  int64_t tokens;
  int heads, kv_heads, dim;
  float scale;
  const int4* tile;
  const int *by_queries, *by_keys;
  int tiles;
  const uchar2* pack;
  int64_t pair_tiles;     // query tile, key tile pairs
  int64_t longest_tiles;  // of one sequence
  // dk, dv work of a key tile in shares of `share` blocks, `splits` at most.
  int splits, share;
  float* part;
  // Per head plane and tile: not 0 where the tensor-core path's fp16 split
  // cannot carry the tile's values.  Null: every tile is computed here.
  const unsigned char* flags;
  int flag_tiles;  // tiles a plane of them

  // Where row `row` of a tensor-core tile's sequence starts and ends in the tile.
  __device__ __forceinline__ int low_of(const int4& t, int row) const { return t.w < 0 && row < t.y ? pack[128 * ~t.w + row].x : 0; }
  __device__ __forceinline__ int high_of(const int4& t, int row) const { return t.w < 0 && row < t.y ? pack[128 * ~t.w + row].y : 128; }
};

// Tensor-core kernels (attention_sm100.cu), for sequences that fill tiles.
bool attention_fits_sm100(const AttentionArgs& a);
lmpb_status attention_sm100(const AttentionArgs& a, const lmpb_sequences_s* seqs, cudaStream_t st);
// Computes delta itself.
lmpb_status attention_sm100_backward(const AttentionArgs& a, const lmpb_sequences_s* seqs, cudaStream_t st);
// Points `a` at one of the sequences' lists of tiles.
void use_tiles(AttentionArgs& a, const lmpb_sequences_s* seqs, const lmpb_sequences_s::Tiles& t);

// A few sequences of at most kShortRows tokens (attention_short.cu).
constexpr int kShortRows = 32;
lmpb_status attention_short(const AttentionArgs& a, int longest, cudaStream_t st);
lmpb_status attention_short_backward(const AttentionArgs& a, int longest, cudaStream_t st);  // computes delta itself

// fp32 kernels for any values and lengths (attention.cu).
lmpb_status attention_simt(const AttentionArgs& a, cudaStream_t st);
lmpb_status attention_simt_backward(const AttentionArgs& a, cudaStream_t st);

}  // namespace lmpb
