// Speculative decoding over a tree of drafted tokens: attention of the tree's
// nodes over a cache, and the small kernels around it.
//
// A sequence b holds n_b = lengths[b] committed keys in its cache rows
// [0, n_b); the tree's nodes 0 .. T-1 (T <= 64, parents before children) hold
// rows n_b .. n_b + T - 1.  Bit j of a node's 64-bit `ancestors` word is set
// where node j is the node itself or lies on its path to the root.
#pragma once

#include "common.cuh"

namespace m5 {

constexpr int kTreeMax = 64;       // nodes of a tree (one bit each)
constexpr int kTreeLayers = 128;   // layers of one commit launch

struct TreeAttnArgs {
  const bf16* q;                   // element strides below, dims contiguous
  int64_t q_sb, q_sh, q_sl;
  bf16* out;
  int64_t o_sb, o_sh, o_sl;
  int B, Hq, Hkv, L, T, D, bits;   // L queries: any nodes of the tree
  m5_kv_view k, v;
  int64_t capacity;                // rows per head
  const int32_t* lengths;          // [B]
  const unsigned long long* anc;   // [B, L], batch stride below
  int64_t anc_sb;
  float scale;
  void* ws;
};

size_t tree_attn_ws_bytes(int B, int Hq, int Hkv, int L, int D);
int tree_attn_check(const TreeAttnArgs& a);
int tree_attn_launch(const TreeAttnArgs& a, cudaStream_t stream);
int tree_attn_error(int reset);

}  // namespace m5
