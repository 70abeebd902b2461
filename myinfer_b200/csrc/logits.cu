// Logits processors of constrained and penalised decoding, as one pass:
//
//   c = counts[b][w] + occurrences of w on the row's own path of drafted tokens
//   c > 0:  v = v < 0 ? v * rep : v / rep,  v -= presence,  v -= frequency * c
//   v += bias[w];   v = -inf where the grammar's bit of w is 0
//
// in fp32 with one rounding to the logits' type at the end, and the first
// index of the row's largest value (NaN is never chosen; -1 where nothing is
// left).  A batch of trees has one row per node; the counts and penalties
// belong to the node's sequence.
//
// One cluster of up to 8 CTAs per row.  Penalties and the mask act on every
// entry alike: 8 consecutive entries per thread and step, with 16-byte loads;
// entries whose mask byte is 0 are written without a load.  The few entries with
// a bias or on the path are marked in a shared bitmap first, skipped by the
// pass and finished one thread each: the last bias entry of a token is the one
// that counts, and it (else the token's last path entry) is the one that
// writes, so no order of threads matters.  The row's choice is a maximum over
// (value, lowest index) words, joined over the cluster in shared memory.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "tree.cuh"

namespace m5 {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 512;
constexpr int kLpCluster = 8;
constexpr int64_t kLpMaxVocab = 524288;
constexpr int kLpMaxBias = 1024;

struct LogitsArgs {
  const void* in;
  void* out;
  int64_t in_ld, out_ld;
  int T, V, per;  // nodes per sequence, vocabulary, entries per CTA (a multiple of 32)
  const int32_t* counts;
  int64_t counts_ld;
  const float* penalties;               // [B, 3]
  const int32_t* tokens;                // [B, T]
  const unsigned long long* anc;        // [B, T]
  const int32_t* bias_ids;              // [B, n_bias]
  const float* bias_values;
  int n_bias;
  const uint32_t* mask;                 // [rows, mask_ld]
  int64_t mask_ld;
  int32_t* choices;
};

template <typename T>
struct Lp;
template <>
struct Lp<bf16> {
  static __device__ __forceinline__ float get(bf16 x) { return bf2f(x); }
  static __device__ __forceinline__ bf16 put(float x) { return f2bf(x); }
};
template <>
struct Lp<float> {
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};

__device__ __forceinline__ float lp_penalise(float v, int c, float rep, float pres, float freq) {
  if (c > 0) {
    v = v < 0.f ? __fmul_rn(v, rep) : __fdiv_rn(v, rep);
    v = __fsub_rn(v, pres);
    v = __fsub_rn(v, __fmul_rn(freq, float(c)));
  }
  return v;
}

// (value, lowest index first) as one word; 0 for NaN and -inf
__device__ __forceinline__ unsigned long long lp_key(float v, int w) {
  if (!(v > -INFINITY)) return 0ull;
  uint32_t u = __float_as_uint(v + 0.f);  // -0 and 0 tie
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xFFFFFFFFu - (uint32_t)w);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) process_logits_kernel(const LogitsArgs a) {
  __shared__ uint32_t s_mark[kLpMaxVocab / kLpCluster / 32 + 1];
  __shared__ unsigned long long s_best[kLpThreads / 32], s_join[kLpCluster];
  const int tid = threadIdx.x, r = blockIdx.y, b = r / a.T, t = r % a.T;
  const int v0 = blockIdx.x * a.per, v1 = min(a.V, v0 + a.per);
  const T* in = reinterpret_cast<const T*>(a.in) + r * a.in_ld;
  T* out = reinterpret_cast<T*>(a.out) + r * a.out_ld;
  const int32_t* counts = a.counts ? a.counts + b * a.counts_ld : nullptr;
  const uint32_t* mask = a.mask ? a.mask + r * a.mask_ld : nullptr;
  const float rep = a.penalties ? a.penalties[3 * b] : 1.f, pres = a.penalties ? a.penalties[3 * b + 1] : 0.f,
              freq = a.penalties ? a.penalties[3 * b + 2] : 0.f;
  const int32_t* toks = a.tokens ? a.tokens + size_t(b) * a.T : nullptr;
  const unsigned long long anc = a.tokens ? a.anc[size_t(b) * a.T + t] : 0ull;
  const int32_t* ids = a.bias_ids + size_t(b) * a.n_bias;
  const int n_path = a.tokens ? a.T : 0, n_special = a.n_bias + n_path;

  for (int i = tid; i < (v1 - v0 + 31) / 32; i += kLpThreads) s_mark[i] = 0;
  __syncthreads();
  for (int e = tid; e < n_special; e += kLpThreads) {
    const int j = e - a.n_bias;
    const int w = e < a.n_bias ? ids[e] : ((anc >> j) & 1 ? toks[j] : -1);
    if (w >= v0 && w < v1) atomicOr(&s_mark[(w - v0) >> 5], 1u << ((w - v0) & 31));
  }
  __syncthreads();

  unsigned long long best = 0;
  for (int w = v0 + tid; w < v1; w += kLpThreads) {
    if ((s_mark[(w - v0) >> 5] >> ((w - v0) & 31)) & 1) continue;
    float v = -INFINITY;
    if (!mask || ((mask[w >> 5] >> (w & 31)) & 1)) v = lp_penalise(Lp<T>::get(in[w]), counts ? counts[w] : 0, rep, pres, freq);
    const T x = Lp<T>::put(v);
    out[w] = x;
    best = max(best, lp_key(Lp<T>::get(x), w));
  }
  for (int e = tid; e < n_special; e += kLpThreads) {
    const int j = e - a.n_bias;
    const int w = e < a.n_bias ? ids[e] : ((anc >> j) & 1 ? toks[j] : -1);
    if (w < v0 || w >= v1) continue;
    // the token's last bias entry writes it, else its last path entry
    bool last = true;
    for (int f = e < a.n_bias ? e + 1 : 0; f < a.n_bias && last; ++f) last = ids[f] != w;
    int c = counts ? counts[w] : 0;
    for (int i = 0; i < n_path; ++i) {
      if (!((anc >> i) & 1) || toks[i] != w) continue;
      ++c;
      if (e >= a.n_bias && i > j) last = false;
    }
    if (!last) continue;
    float v = -INFINITY;
    if (!mask || ((mask[w >> 5] >> (w & 31)) & 1)) {
      v = lp_penalise(Lp<T>::get(in[w]), c, rep, pres, freq);
      if (e < a.n_bias) v = __fadd_rn(v, a.bias_values[size_t(b) * a.n_bias + e]);
    }
    const T x = Lp<T>::put(v);
    out[w] = x;
    best = max(best, lp_key(Lp<T>::get(x), w));
  }
  if (!a.choices) return;  // the same for every CTA of the cluster
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) s_best[tid >> 5] = best;
  __syncthreads();
  cg::cluster_group cl = cg::this_cluster();
  if (tid == 0) {
    for (int i = 1; i < kLpThreads / 32; ++i) best = max(best, s_best[i]);
    *cl.map_shared_rank(&s_join[blockIdx.x], 0) = best;
  }
  cl.sync();
  if (blockIdx.x == 0 && tid == 0) {
    for (int i = 0; i < int(gridDim.x); ++i) best = max(best, s_join[i]);
    a.choices[r] = best ? int32_t(0xFFFFFFFFu - uint32_t(best)) : -1;
  }
}

template <typename T>
cudaError_t lp_launch(const LogitsArgs& a, int ctas, int rows, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, rows);
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, process_logits_kernel<T>, a);
}

}  // namespace
}  // namespace m5

using namespace m5;

extern "C" int m5_process_logits(const void* logits, int64_t ld, void* out, int64_t out_ld, int dtype, int B, int T,
                                 int64_t vocab, const int32_t* counts, int64_t counts_ld, const float* penalties,
                                 const int32_t* tokens, const int64_t* ancestors, const int32_t* bias_ids,
                                 const float* bias_values, int n_bias, const int32_t* mask, int64_t mask_ld,
                                 int32_t* choices, void* stream) {
  M5_CHECK_ARG(logits && out, "m5_process_logits: null pointer");
  M5_CHECK_ARG(dtype == M5_DTYPE_BF16 || dtype == M5_DTYPE_F32, "m5_process_logits: dtype");
  M5_CHECK_ARG(B > 0 && T > 0 && vocab > 0, "m5_process_logits: empty shape");
  M5_CHECK_ARG(T <= kTreeMax, "m5_process_logits: more than 64 nodes");
  M5_CHECK_ARG(int64_t(B) * T <= 65535, "m5_process_logits: more than 65535 rows");
  M5_CHECK_ARG(vocab <= kLpMaxVocab, "m5_process_logits: vocabulary above 524288");
  M5_CHECK_ARG(ld >= vocab && out_ld >= vocab && (!counts || counts_ld >= vocab), "m5_process_logits: row stride below the vocabulary");
  M5_CHECK_ARG(!(counts || tokens) || penalties, "m5_process_logits: counts and tokens need penalties");
  M5_CHECK_ARG(!tokens || ancestors, "m5_process_logits: tokens need ancestors");
  M5_CHECK_ARG(n_bias >= 0 && n_bias <= kLpMaxBias, "m5_process_logits: 0 to 1024 bias entries");
  M5_CHECK_ARG(!n_bias || (bias_ids && bias_values), "m5_process_logits: bias entries need ids and values");
  M5_CHECK_ARG(!mask || mask_ld >= (vocab + 31) / 32, "m5_process_logits: mask rows need a bit per token");
  LogitsArgs a{};
  a.in = logits;
  a.out = out;
  a.in_ld = ld;
  a.out_ld = out_ld;
  a.T = T;
  a.V = (int)vocab;
  const int ctas = (int)std::min<int64_t>(kLpCluster, (vocab + 4095) / 4096);
  a.per = (int)(((vocab + ctas - 1) / ctas + 31) / 32 * 32);
  a.counts = counts;
  a.counts_ld = counts_ld;
  a.penalties = penalties;
  a.tokens = tokens;
  a.anc = (const unsigned long long*)ancestors;
  a.bias_ids = bias_ids;
  a.bias_values = bias_values;
  a.n_bias = n_bias;
  a.mask = (const uint32_t*)mask;
  a.mask_ld = mask_ld;
  a.choices = choices;
  M5_CUDA(dtype == M5_DTYPE_BF16 ? lp_launch<bf16>(a, ctas, B * T, (cudaStream_t)stream)
                                 : lp_launch<float>(a, ctas, B * T, (cudaStream_t)stream));
  return M5_OK;
}
