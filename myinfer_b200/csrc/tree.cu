// The small kernels of speculative decoding over a tree, and the C entry
// points of the tree operators.
//
//  tree_plan    a node's ancestors word is its own bit or'ed with its parent's
//               word.  The path is walked by doubling: after k rounds a thread
//               holds 2^k nodes of its path and the node above them, so 64
//               nodes take 6 rounds instead of 64 dependent steps.
//  tree_accept  from node 0, the first child whose drafted token is the one the
//               model chose after its parent, until there is none.  Matching
//               is one comparison per node; the first matching child of each
//               node is the minimum over an integer atomic in shared memory
//               (independent of order), and one thread follows the chain.
//  tree_commit  cache rows n + path[i] -> n + i of every layer, in place: all
//               rows of one (layer, K or V, head) go through registers of one
//               CTA, loads before stores, so sources and destinations may
//               overlap in any way.  All layers are one launch: the table of
//               their buffers travels as the kernel's parameter (of 32, 64 or 128
//               layers: 8 KB of it cost the host 0.5 us more than 2).
// None of them moves enough bytes to matter (a commit of 20 rows over 64 layers
// is 5 MB): they are bound by their launch and by one to three dependent trips to
// memory.  Accepting, one tree of 8 or 64 trees of 64 nodes: 1.9-2.0 us on the device.  A
// commit of 28 layers, 8 heads, 8 bits: 3.0 us; of 64 layers for 4 requests, 4 bits: 5.8 us
// (11 MB, 1.9 TB/s).
#include <algorithm>

#include "tree.cuh"

namespace m5 {
namespace {

__global__ void __launch_bounds__(kTreeMax) tree_plan_kernel(const int32_t* parents, int T, long long* anc, int32_t* depth) {
  __shared__ unsigned long long s_bits[kTreeMax];
  __shared__ int s_up[kTreeMax];
  const int i = threadIdx.x, b = blockIdx.x;
  // up: the next node above the ones in `bits`; -1 above a root, -2 for a node of no tree
  int up = i < T ? parents[size_t(b) * T + i] : -2;
  if (up < -1 || up >= i) up = -2;
  unsigned long long bits = up == -2 ? 0ull : 1ull << i;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    s_bits[i] = bits;
    s_up[i] = up;
    __syncthreads();
    if (up >= 0) {
      bits |= s_bits[up];
      up = s_up[up];
    }
    __syncthreads();
  }
  if (up == -2) bits = 0;  // hangs below a node of no tree
  if (i < T) {
    anc[size_t(b) * T + i] = (long long)bits;
    if (depth) depth[size_t(b) * T + i] = max(0, __popcll(bits) - 1);
  }
}

__global__ void __launch_bounds__(kTreeMax) tree_accept_kernel(const int32_t* parents, const int32_t* tokens,
                                                               const int32_t* picks, int T, int32_t* path,
                                                               int32_t* accepted, int32_t* next, int32_t* counts,
                                                               int64_t counts_ld, int V) {
  __shared__ int s_pick[kTreeMax], s_tok[kTreeMax], s_child[kTreeMax], s_path[kTreeMax], s_n;
  const int i = threadIdx.x, b = blockIdx.x;
  const size_t at = size_t(b) * T + i;
  const int par = i < T ? parents[at] : -2;
  const int tok = i < T ? tokens[at] : -1;
  s_pick[i] = i < T ? picks[at] : -1;
  s_tok[i] = tok;
  s_child[i] = kTreeMax;
  s_path[i] = -1;
  __syncthreads();
  if (par >= 0 && par < i && s_pick[par] == tok) atomicMin(&s_child[par], i);
  __syncthreads();
  if (i == 0) {
    int n = 0, cur = 0;
    while (cur < kTreeMax) {  // a child's index is above its parent's: at most 64 steps
      s_path[n++] = cur;
      cur = s_child[cur];
    }
    s_n = n;
    accepted[b] = n;
    next[b] = s_pick[s_path[n - 1]];
  }
  __syncthreads();
  if (i < T) path[at] = s_path[i];
  if (counts && i < s_n) {
    const int t = s_tok[s_path[i]];
    if (t >= 0 && t < V) atomicAdd(counts + b * counts_ld + t, 1);
  }
}

template <int LAYERS>
struct CommitTable {
  struct {
    void* p[6];        // K data, scales, biases, V data, scales, biases
    int64_t capacity;
    int32_t row;       // bytes of a data row
    int32_t group;     // bytes of a scale row (0: bf16 cache)
  } layer[LAYERS];
};

constexpr int kCommitThreads = 128;

// UNITS: 16-byte units per thread of 64 of the widest rows (256 bytes: 8).  The registers they take
// decide how many of the small CTAs an SM holds (4 requests x 64 layers are 4096).
template <int UNITS, int LAYERS>
__global__ void __launch_bounds__(kCommitThreads, UNITS == 2 ? 16 : UNITS == 4 ? 10 : 7) tree_commit_kernel(const __grid_constant__ CommitTable<LAYERS> t, int Hkv,
                                                                     const int32_t* lengths, const int32_t* path,
                                                                     int T, const int32_t* accepted) {
  __shared__ int s_path[kTreeMax];
  const int tid = threadIdx.x, b = blockIdx.x / Hkv;
  const auto& ly = t.layer[blockIdx.y];
  const int kv = 3 * blockIdx.z;
  const int64_t len = lengths[b];
  const int n = min(accepted[b], T);
  if (tid < n) {
    // rows that stay, or that no cache row backs, are marked -1
    const int p = path[size_t(b) * T + tid];
    s_path[tid] = (p >= 0 && p < T && p != tid && len >= 0 && len + max(p, tid) < ly.capacity) ? p : -1;
  }
  __syncthreads();
  const size_t base = size_t(blockIdx.x) * ly.capacity + len;
  uint4* data = reinterpret_cast<uint4*>(ly.p[kv]);
  const int per = ly.row / 16;  // 16-byte units of a row: 2 to 16, a power of two
  uint4 u[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int e = tid + k * kCommitThreads, r = e / per;
    if (r < n && s_path[r] >= 0) u[k] = data[(base + s_path[r]) * per + e % per];
  }
  uint16_t s[2];
  const int gr = ly.group / 2, sr = gr ? tid / gr : n;
  const bool sm = sr < n && s_path[sr] >= 0;
  if (sm) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      s[k] = reinterpret_cast<const uint16_t*>(ly.p[kv + 1 + k])[(base + s_path[sr]) * gr + tid % gr];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int e = tid + k * kCommitThreads, r = e / per;
    if (r < n && s_path[r] >= 0) data[(base + r) * per + e % per] = u[k];
  }
  if (sm) {
#pragma unroll
    for (int k = 0; k < 2; ++k) reinterpret_cast<uint16_t*>(ly.p[kv + 1 + k])[(base + sr) * gr + tid % gr] = s[k];
  }
}

// One launch for the first layers (as many as the table holds).
template <int LAYERS>
int commit_some(const m5_layer_kv* layers, int left, int B, int Hkv, int D, const int32_t* lengths, const int32_t* path,
                int T, const int32_t* accepted, void* stream) {
  CommitTable<LAYERS> t;
  int row = 0;  // widest
  const int nl = std::min(LAYERS, left);
  for (int i = 0; i < nl; ++i) {
    const m5_layer_kv& l = layers[i];
    void* const p[6] = {l.k, l.k_scales, l.k_biases, l.v, l.v_scales, l.v_biases};
    std::copy(p, p + 6, t.layer[i].p);
    t.layer[i].capacity = l.capacity;
    t.layer[i].row = l.bits ? D * l.bits / 8 : 2 * D;
    t.layer[i].group = l.bits ? D / 64 * 2 : 0;
    row = std::max(row, t.layer[i].row);
  }
  const auto kernel = row <= 64 ? tree_commit_kernel<2, LAYERS> : row <= 128 ? tree_commit_kernel<4, LAYERS>
                                                                             : tree_commit_kernel<8, LAYERS>;
  kernel<<<dim3(B * Hkv, nl, 2), kCommitThreads, 0, (cudaStream_t)stream>>>(t, Hkv, lengths, path, T, accepted);
  M5_LAUNCH_CHECK("tree commit launch");
  return M5_OK;
}

}  // namespace
}  // namespace m5

using namespace m5;

extern "C" int m5_tree_plan(const int32_t* parents, int B, int T, int64_t* ancestors, int32_t* depths, void* stream) {
  M5_CHECK_ARG(parents && ancestors, "m5_tree_plan: null pointer");
  M5_CHECK_ARG(B > 0 && T > 0, "m5_tree_plan: empty shape");
  M5_CHECK_ARG(T <= kTreeMax, "m5_tree_plan: more than 64 nodes");
  tree_plan_kernel<<<B, kTreeMax, 0, (cudaStream_t)stream>>>(parents, T, (long long*)ancestors, depths);
  M5_LAUNCH_CHECK("tree plan launch");
  return M5_OK;
}

extern "C" int m5_tree_accept(const int32_t* parents, const int32_t* tokens, const int32_t* picks, int B, int T,
                              int32_t* path, int32_t* accepted, int32_t* next, int32_t* counts, int64_t counts_ld,
                              int64_t vocab, void* stream) {
  M5_CHECK_ARG(parents && tokens && picks && path && accepted && next, "m5_tree_accept: null pointer");
  M5_CHECK_ARG(B > 0 && T > 0, "m5_tree_accept: empty shape");
  M5_CHECK_ARG(T <= kTreeMax, "m5_tree_accept: more than 64 nodes");
  M5_CHECK_ARG(!counts || (vocab > 0 && vocab < (1LL << 31) && counts_ld >= vocab), "m5_tree_accept: counts shape");
  tree_accept_kernel<<<B, kTreeMax, 0, (cudaStream_t)stream>>>(parents, tokens, picks, T, path, accepted, next, counts,
                                                              counts_ld, (int)vocab);
  M5_LAUNCH_CHECK("tree accept launch");
  return M5_OK;
}

extern "C" int m5_tree_commit(const m5_layer_kv* layers, int num_layers, int B, int Hkv, int D, const int32_t* lengths,
                              const int32_t* path, int T, const int32_t* accepted, void* stream) {
  M5_CHECK_ARG(layers && lengths && path && accepted, "m5_tree_commit: null pointer");
  M5_CHECK_ARG(num_layers > 0 && B > 0 && Hkv > 0 && T > 0, "m5_tree_commit: empty shape");
  M5_CHECK_ARG(T <= kTreeMax, "m5_tree_commit: more than 64 nodes");
  M5_CHECK_ARG(D == 64 || D == 128, "m5_tree_commit: head_dim must be 64 or 128");
  for (int i = 0; i < num_layers; ++i) {
    const m5_layer_kv& l = layers[i];
    M5_CHECK_ARG(l.k && l.v && l.capacity > 0, "m5_tree_commit: cache layer");
    M5_CHECK_ARG(l.bits == 0 || l.bits == 4 || l.bits == 8, "m5_tree_commit: bits must be 0, 4 or 8");
    M5_CHECK_ARG(!l.bits || (l.k_scales && l.k_biases && l.v_scales && l.v_biases && l.group_size == 64),
                 "m5_tree_commit: packed cache needs scales/biases and group 64");
    M5_CHECK_ARG((reinterpret_cast<uintptr_t>(l.k) | reinterpret_cast<uintptr_t>(l.v)) % 16 == 0,
                 "m5_tree_commit: K/V rows must be 16-byte aligned");
  }
  for (int l0 = 0; l0 < num_layers;) {
    const int left = num_layers - l0;
    const auto some = left <= 32 ? commit_some<32> : left <= 64 ? commit_some<64> : commit_some<kTreeLayers>;
    if (int rc = some(layers + l0, left, B, Hkv, D, lengths, path, T, accepted, stream)) return rc;
    l0 += kTreeLayers;
  }
  return M5_OK;
}

int m5::tree_attn_check(const TreeAttnArgs& a) {
  M5_CHECK_ARG(a.q && a.out && a.k.data && a.v.data && a.lengths && a.anc, "m5_tree_attention: null pointer");
  M5_CHECK_ARG(a.B > 0 && a.Hq > 0 && a.Hkv > 0 && a.L > 0 && a.T > 0 && a.capacity > 0, "m5_tree_attention: empty shape");
  M5_CHECK_ARG(a.Hq % a.Hkv == 0, "m5_tree_attention: Hq must be a multiple of Hkv");
  M5_CHECK_ARG(a.L <= kTreeMax && a.T <= kTreeMax, "m5_tree_attention: more than 64 nodes");
  M5_CHECK_ARG(a.D == 64 || a.D == 128, "m5_tree_attention: head_dim must be 64 or 128");
  M5_CHECK_ARG(a.bits == 0 || a.bits == 4 || a.bits == 8, "m5_tree_attention: bits must be 0, 4 or 8");
  M5_CHECK_ARG(!a.bits || (a.k.scales && a.k.biases && a.v.scales && a.v.biases),
               "m5_tree_attention: packed K/V need scales and biases");
  M5_CHECK_ARG(a.capacity + kTreeMax < (1LL << 31), "m5_tree_attention: capacity must stay below 2^31 rows");
  const int64_t blocks = (int64_t(a.L) * (a.Hq / a.Hkv) + 127) / 128;
  M5_CHECK_ARG(int64_t(a.B) * a.Hkv < (1LL << 31) / blocks / ((a.capacity + 63) / 64),
               "m5_tree_attention: more than 2^31 tiles of 128 rows and 64 keys");
  M5_CHECK_ARG((reinterpret_cast<uintptr_t>(a.k.data) | reinterpret_cast<uintptr_t>(a.v.data)) % 16 == 0,
               "m5_tree_attention: K/V rows must be 16-byte aligned");
  M5_CHECK_ARG(!a.bits || (reinterpret_cast<uintptr_t>(a.k.scales) | reinterpret_cast<uintptr_t>(a.k.biases) |
                           reinterpret_cast<uintptr_t>(a.v.scales) | reinterpret_cast<uintptr_t>(a.v.biases)) %
                                  (a.D / 32) == 0,
               "m5_tree_attention: a row's scales and biases must be aligned to their size");
  M5_CHECK_ARG((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out)) % 16 == 0 &&
                   (a.q_sb | a.q_sh | a.q_sl | a.o_sb | a.o_sh | a.o_sl) % 8 == 0,
               "m5_tree_attention: query and output rows must be 16-byte aligned");
  return M5_OK;
}

extern "C" int m5_tree_attention_workspace(int B, int Hq, int Hkv, int L, int D, size_t* bytes) {
  M5_CHECK_ARG(bytes, "m5_tree_attention_workspace: null pointer");
  M5_CHECK_ARG(B > 0 && Hq > 0 && Hkv > 0 && L > 0 && Hq % Hkv == 0 && (D == 64 || D == 128),
               "m5_tree_attention_workspace: shape");
  *bytes = tree_attn_ws_bytes(B, Hq, Hkv, L, D);
  return M5_OK;
}

extern "C" int m5_tree_attention(const void* q, const int64_t* q_strides, int B, int Hq, int L, int D, m5_kv_view keys,
                                 m5_kv_view values, int Hkv, int64_t capacity, const int32_t* lengths, int tree_len,
                                 const int64_t* ancestors, int64_t ancestors_stride, float scale, int group_size,
                                 int bits, void* out, const int64_t* out_strides, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  M5_CHECK_ARG(q_strides && out_strides, "m5_tree_attention: null pointer");
  M5_CHECK_ARG(bits == 0 || group_size == 64, "m5_tree_attention: group_size must be 64");
  TreeAttnArgs a{};
  a.q = (const bf16*)q;
  a.q_sb = q_strides[0];
  a.q_sh = q_strides[1];
  a.q_sl = q_strides[2];
  a.out = (bf16*)out;
  a.o_sb = out_strides[0];
  a.o_sh = out_strides[1];
  a.o_sl = out_strides[2];
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.L = L;
  a.T = tree_len;
  a.D = D;
  a.bits = bits;
  a.k = keys;
  a.v = values;
  a.capacity = capacity;
  a.lengths = lengths;
  a.anc = (const unsigned long long*)ancestors;
  a.anc_sb = ancestors_stride;
  a.scale = scale;
  a.ws = workspace;
  if (int rc = tree_attn_check(a)) return rc;
  const size_t need = tree_attn_ws_bytes(B, Hq, Hkv, L, D);
  M5_CHECK_ARG(!need || (workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               "m5_tree_attention: workspace too small or not 16-byte aligned");
  return tree_attn_launch(a, (cudaStream_t)stream);
}
