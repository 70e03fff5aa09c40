// What the attention kernels share: the packed-sequence handle and the call
// of each path.
#pragma once

#include "common.cuh"

// Packed sequences cut into tiles of 128 tokens, the last of a sequence
// shorter; tiles never span sequences.  One device block holds the table.
struct lmpb_sequences_s {
  int device = 0;
  int count = 0;
  int64_t tokens = 0;
  int64_t longest = 0;
  int tiles = 0;
  void* block = nullptr;
  const int4* tile = nullptr;        // {sequence's first token, its length, tile within it, its first tile}
  const int* by_queries = nullptr;   // tiles, those with the most keys to visit first
  const int* by_keys = nullptr;      // tiles, those with the most queries to visit first
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
  // Per head plane and tile: not 0 where the tensor-core path's fp16 split
  // cannot carry the tile's values.  Null: every tile is computed here.
  const unsigned char* flags;
};

// Tensor-core kernels (attention_sm100.cu), for sequences that fill tiles.
bool attention_fits_sm100(const AttentionArgs& a);
lmpb_status attention_sm100(const AttentionArgs& a, cudaStream_t st);
lmpb_status attention_sm100_backward(const AttentionArgs& a, cudaStream_t st);  // computes delta itself

// fp32 kernels for any values and lengths (attention.cu).
lmpb_status attention_simt(const AttentionArgs& a, cudaStream_t st);
lmpb_status attention_simt_backward(const AttentionArgs& a, cudaStream_t st);

}  // namespace lmpb
