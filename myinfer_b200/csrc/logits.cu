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
// One cluster of up to 16 CTAs per row, so that a single row already uses 16 SMs.
// The pass is bound by the loads in flight: a thread takes 8 consecutive
// entries with 16-byte loads, two such groups at once (rows that are not
// 16-byte aligned: 8 entries a warp apart, coalesced).  Entries whose mask byte
// is 0 are written without a load, groups nothing applies to are copied as they
// are (in place: left alone), and the choice looks at a group's maximum only.
// The few entries with a bias or on the path are marked in a shared bitmap
// first, skipped by the pass and finished by a warp together: the last bias entry
// of a token is the one that counts, and it (else the token's last path entry)
// is the one that writes, so no order of threads matters.  The row's choice is a
// maximum over (value, lowest index) words, joined over the cluster in shared memory.
//
// On the device: one bf16 row of 151936 with penalties 5.9 us (latency: loads, cluster join);
// a tree of 64 such rows with 300 biases and masks 28.6 us (40.7 MB from and to memory, 1.42 TB/s;
// the counts, read again for every row from L2, take 7 us of it, the biases 6.5, the masks 2.5,
// a plain copy 10); 40 fp32 rows of 32001, unaligned, 12.9 us.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "tree.cuh"

namespace m5 {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 512;
constexpr int kLpCluster = 16;
constexpr int kLpPer = 65536;  // most entries of one CTA
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

// A row's penalties; y = 1 / rep rounded to nearest.
struct Pen {
  float rep, pres, freq, y;
  bool plain;  // rep far from the ends of fp32's range
};
// The division for any operands.
__device__ __noinline__ float lp_div(float v, float rep) { return __fdiv_rn(v, rep); }
// One entry that has occurred c > 0 times.  v / rep takes three operations from
// the row's reciprocal: q = v y, then q + (v - q rep) y with the remainder exact
// in one fma, which is the quotient rounded to nearest (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", IBM J. Res. Dev. 34, 1990) while
// nothing comes near the ends of the range; else the divide itself.
__device__ __forceinline__ float lp_penalise(float v, int c, const Pen& p) {
  const float m = fabsf(v);
  float d;
  if (v < 0.f) {
    d = __fmul_rn(v, p.rep);
  } else {
    const float q = __fmul_rn(v, p.y);
    d = __fmaf_rn(__fmaf_rn(-q, p.rep, v), p.y, q);
    if (!(p.plain && m > 0x1p-60f && m < 0x1p60f)) d = lp_div(v, p.rep);
  }
  d = __fsub_rn(d, p.pres);
  return __fsub_rn(d, __fmul_rn(p.freq, float(c)));
}

// (value, lowest index first) as one word; 0 for NaN and -inf
__device__ __forceinline__ unsigned long long lp_key(float v, int w) {
  if (!(v > -INFINITY)) return 0ull;
  uint32_t u = __float_as_uint(v + 0.f);  // -0 and 0 tie
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xFFFFFFFFu - (uint32_t)w);
}

// All CTAs of a cluster have arrived before any thread passes the wait (nothing is ordered by it).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// 8 entries of a thread: raw bits of consecutive ones (VEC), or of entries 32 apart.
template <typename T, bool VEC>
struct Group {
  float v[8];
  uint32_t raw[sizeof(T) * 2];  // VEC: as loaded
  int c[8];
  uint32_t on, mark;            // allowed, special: a bit per entry
};

// Loads the group at entry w0 (VEC: its first; else the warp's first of 256, this lane's k-th is w0 + 32 k + lane).
template <typename T, bool VEC>
__device__ __forceinline__ void lp_load(Group<T, VEC>& g, const LogitsArgs& a, const T* in, const int32_t* counts,
                                        const uint32_t* mask, const uint32_t* mark, int w0, int v0, int v1, int lane) {
  if constexpr (VEC) {
    g.on = mask ? (mask[w0 >> 5] >> (w0 & 31)) & 0xFFu : 0xFFu;
    g.mark = mark ? (mark[(w0 - v0) >> 5] >> ((w0 - v0) & 31)) & 0xFFu : 0u;
    if (g.on) {
      const uint4* p = reinterpret_cast<const uint4*>(in + w0);
#pragma unroll
      for (int k = 0; k < int(sizeof(T)) / 2; ++k) {
        const uint4 u = p[k];
        g.raw[4 * k] = u.x;
        g.raw[4 * k + 1] = u.y;
        g.raw[4 * k + 2] = u.z;
        g.raw[4 * k + 3] = u.w;
      }
      if (counts) {
        const int4 x = reinterpret_cast<const int4*>(counts + w0)[0], y = reinterpret_cast<const int4*>(counts + w0)[1];
        g.c[0] = x.x; g.c[1] = x.y; g.c[2] = x.z; g.c[3] = x.w;
        g.c[4] = y.x; g.c[5] = y.y; g.c[6] = y.z; g.c[7] = y.w;
      }
    }
  } else {
    // lane k holds the mask and mark words of the warp's k-th 32 entries
    const int k0 = w0 + 32 * lane;
    const uint32_t mw = k0 < v1 && lane < 8 ? (mask ? mask[k0 >> 5] : ~0u) : 0u;
    const uint32_t sw = mark && k0 < v1 && lane < 8 ? mark[(k0 - v0) >> 5] : 0u;
    g.on = g.mark = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int w = w0 + 32 * k + lane;
      const bool on = ((__shfl_sync(0xffffffffu, mw, k) >> lane) & 1) && w < v1;
      g.mark |= ((__shfl_sync(0xffffffffu, sw, k) >> lane) & 1) << k;
      g.on |= uint32_t(on) << k;
      g.v[k] = on ? Lp<T>::get(in[w]) : 0.f;
      g.c[k] = on && counts ? counts[w] : 0;
    }
  }
}

// Finishes a group: writes it and takes it into the thread's best value.
template <typename T, bool VEC>
__device__ __forceinline__ void lp_finish(Group<T, VEC>& g, const LogitsArgs& a, T* out, bool counts, bool in_place,
                                          int w0, int v1, int lane, const Pen& pen, float& best, int& at) {
  if constexpr (VEC) {
    if (!g.on && !g.mark) {
      const uint32_t ninf = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
#pragma unroll
      for (int k = 0; k < int(sizeof(T)) / 2; ++k) reinterpret_cast<uint4*>(out + w0)[k] = make_uint4(ninf, ninf, ninf, ninf);
      return;
    }
    int any = 0;
    if (g.on) {
      if (counts) {
#pragma unroll
        for (int k = 0; k < 8; ++k) any |= g.c[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (sizeof(T) == 2) g.v[k] = (k & 1) ? bf16_hi(g.raw[k / 2]) : bf16_lo(g.raw[k / 2]);
        else g.v[k] = __uint_as_float(g.raw[k]);
      }
    }
    if (!g.mark && !any) {
      // nothing but the mask applies: the bits as they are, or -inf's
      if (g.on != 0xFFu) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t keep = ((g.on >> (2 * k)) & 1u) * 0xFFFFu | ((g.on >> (2 * k + 1)) & 1u) * 0xFFFF0000u;
            g.raw[k] = (g.raw[k] & keep) | (0xFF80FF80u & ~keep);
            g.v[2 * k] = bf16_lo(g.raw[k]);
            g.v[2 * k + 1] = bf16_hi(g.raw[k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (!((g.on >> k) & 1)) g.v[k] = -INFINITY;
            g.raw[k] = __float_as_uint(g.v[k]);
          }
        }
      }
      if (!in_place || g.on != 0xFFu) {
#pragma unroll
        for (int k = 0; k < int(sizeof(T)) / 2; ++k)
          reinterpret_cast<uint4*>(out + w0)[k] = make_uint4(g.raw[4 * k], g.raw[4 * k + 1], g.raw[4 * k + 2], g.raw[4 * k + 3]);
      }
    } else {
      T x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (any && g.c[k] > 0) g.v[k] = lp_penalise(g.v[k], g.c[k], pen);
        x[k] = Lp<T>::put(((g.on >> k) & 1) ? g.v[k] : -INFINITY);
        g.v[k] = ((g.mark >> k) & 1) ? -INFINITY : Lp<T>::get(x[k]);
      }
      if (!g.mark) {
#pragma unroll
        for (int k = 0; k < int(sizeof(T)) / 2; ++k)
          reinterpret_cast<uint4*>(out + w0)[k] = reinterpret_cast<const uint4*>(x)[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (!((g.mark >> k) & 1)) out[w0 + k] = x[k];
      }
    }
    // ascending entries and a strict comparison: the lowest index stays (NaN never wins)
    const float top = fmaxf(fmaxf(fmaxf(g.v[0], g.v[1]), fmaxf(g.v[2], g.v[3])),
                            fmaxf(fmaxf(g.v[4], g.v[5]), fmaxf(g.v[6], g.v[7])));
    if (top > best) {
      best = top;
#pragma unroll
      for (int k = 7; k >= 0; --k)
        if (g.v[k] == top) at = w0 + k;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int w = w0 + 32 * k + lane;
      if (w >= v1 || ((g.mark >> k) & 1)) continue;
      float v = g.v[k];
      if (g.c[k] > 0) v = lp_penalise(v, g.c[k], pen);
      const T x = Lp<T>::put(((g.on >> k) & 1) ? v : -INFINITY);
      out[w] = x;
      v = Lp<T>::get(x);
      if (v > best) {
        best = v;
        at = w;
      }
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kLpThreads, 2) process_logits_kernel(const LogitsArgs a) {
  __shared__ uint32_t s_mark[kLpPer / 32];
  __shared__ unsigned long long s_best[kLpThreads / 32], s_join[kLpCluster];
  __shared__ int32_t s_tok[kLpMaxBias + kTreeMax];   // special tokens: biases, then the row's path (-1: unused)
  __shared__ uint16_t s_list[kLpMaxBias + kTreeMax]; // those in this CTA's part, in any order
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, r = blockIdx.y, b = r / a.T, t = r - b * a.T;
  const int v0 = blockIdx.x * a.per, v1 = min(a.V, v0 + a.per);
  if (a.choices) cluster_arrive();  // this CTA has started: the others' join may write to its shared memory
  const T* in = reinterpret_cast<const T*>(a.in) + r * a.in_ld;
  T* out = reinterpret_cast<T*>(a.out) + r * a.out_ld;
  const int32_t* counts = a.counts ? a.counts + b * a.counts_ld : nullptr;
  const uint32_t* mask = a.mask ? a.mask + r * a.mask_ld : nullptr;
  Pen pen{1.f, 0.f, 0.f, 1.f, true};
  if (a.penalties) {
    pen.rep = a.penalties[3 * b];
    pen.pres = a.penalties[3 * b + 1];
    pen.freq = a.penalties[3 * b + 2];
    pen.y = __frcp_rn(pen.rep);
    pen.plain = fabsf(pen.rep) > 0x1p-20f && fabsf(pen.rep) < 0x1p20f;
  }
  const int32_t* toks = a.tokens ? a.tokens + size_t(b) * a.T : nullptr;
  const unsigned long long anc = a.tokens ? a.anc[size_t(b) * a.T + t] : 0ull;
  const int32_t* ids = a.bias_ids + size_t(b) * a.n_bias;
  const int n_path = a.tokens ? a.T : 0, n_special = a.n_bias + n_path;
  const bool in_place = (const void*)in == (const void*)out;

  if (n_special) {
    if (tid == 0) s_n = 0;
    for (int i = tid; i < (v1 - v0 + 31) / 32; i += kLpThreads) s_mark[i] = 0;
    __syncthreads();
    for (int e = tid; e < n_special; e += kLpThreads) {
      const int j = e - a.n_bias;
      const int w = e < a.n_bias ? ids[e] : ((anc >> j) & 1 ? toks[j] : -1);
      s_tok[e] = w;
      if (w >= v0 && w < v1) {
        atomicOr(&s_mark[(w - v0) >> 5], 1u << ((w - v0) & 31));
        s_list[atomicAdd(&s_n, 1)] = uint16_t(e);
      }
    }
    __syncthreads();
  }
  const uint32_t* mark = n_special ? s_mark : nullptr;

  float top = -INFINITY;
  int at = 0;
  // VEC: thread after thread; else warp after warp, 256 entries each
  const int w_first = VEC ? v0 + 8 * tid : v0 + 256 * (tid >> 5);
  constexpr int STEP = 8 * kLpThreads;
#pragma unroll 1
  for (int w = w_first; w < v1; w += 2 * STEP) {
    Group<T, VEC> g0, g1;
    const bool two = w + STEP < v1;
    lp_load<T, VEC>(g0, a, in, counts, mask, mark, w, v0, v1, lane);
    if (two) lp_load<T, VEC>(g1, a, in, counts, mask, mark, w + STEP, v0, v1, lane);
    lp_finish<T, VEC>(g0, a, out, counts != nullptr, in_place, w, v1, lane, pen, top, at);
    if (two) lp_finish<T, VEC>(g1, a, out, counts != nullptr, in_place, w + STEP, v1, lane, pen, top, at);
  }
  unsigned long long best = lp_key(top, at);
  if (n_special) {
    // A warp takes every 16th special entry: lane l loads what its l-th one needs, the warp looks
    // through the list for each (is it the token's last bias entry, else its last path entry?), and
    // the lanes finish theirs at once.
    constexpr int WARPS = kLpThreads / 32;
    for (int i0 = tid >> 5; i0 < s_n; i0 += 32 * WARPS) {
      const int i = i0 + WARPS * lane;
      const bool have = i < s_n;
      const int e = have ? s_list[i] : 0, w = have ? s_tok[e] : 0;
      const bool on = have && (!mask || ((mask[w >> 5] >> (w & 31)) & 1));
      float v = on ? Lp<T>::get(in[w]) : 0.f;
      int c = on && counts ? counts[w] : 0;
      const float bias = have && e < a.n_bias ? a.bias_values[size_t(b) * a.n_bias + e] : 0.f;
      bool mine = have;
      for (int l = 0; l < 32 && i0 + WARPS * l < s_n; ++l) {
        const int le = __shfl_sync(0xffffffffu, e, l), lw = __shfl_sync(0xffffffffu, w, l);
        const bool path = le >= a.n_bias;
        bool later = false;
        for (int f = (path ? 0 : le + 1) + lane; f < a.n_bias; f += 32) later |= s_tok[f] == lw;
        int occ = 0;
        for (int f = a.n_bias + lane; f < n_special; f += 32) {
          const bool same = s_tok[f] == lw;
          occ += same;
          later |= same && path && f > le;
        }
        later = __any_sync(0xffffffffu, later);
        occ = __reduce_add_sync(0xffffffffu, occ);
        if (lane == l) {
          mine = !later;
          c += occ;
        }
      }
      if (mine) {
        if (on && c > 0) v = lp_penalise(v, c, pen);
        if (e < a.n_bias) v = __fadd_rn(v, bias);
        const T x = Lp<T>::put(on ? v : -INFINITY);
        out[w] = x;
        best = max(best, lp_key(Lp<T>::get(x), w));
      }
    }
  }
  if (!a.choices) return;  // the same for every CTA of the cluster
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) s_best[tid >> 5] = best;
  __syncthreads();
  cluster_wait();  // rank 0 has started (a part with nothing to do gets here before it)
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
  // 16-byte groups of 8 entries: every row of every array starts on 16 bytes and no group passes the vocabulary's end
  const uintptr_t align = reinterpret_cast<uintptr_t>(a.in) | reinterpret_cast<uintptr_t>(a.out) |
                          uintptr_t(a.in_ld * sizeof(T)) | uintptr_t(a.out_ld * sizeof(T)) |
                          reinterpret_cast<uintptr_t>(a.counts) | uintptr_t(a.counts ? a.counts_ld * 4 : 0);
  const bool vec = align % 16 == 0 && a.V % 8 == 0;
  static DeviceOnce once;  // clusters above 8
  cudaError_t e = once.run([&] {
    cudaError_t x = cudaFuncSetAttribute(process_logits_kernel<T, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return x ? x : cudaFuncSetAttribute(process_logits_kernel<T, false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (e != cudaSuccess) return e;
  return vec ? cudaLaunchKernelEx(&cfg, process_logits_kernel<T, true>, a)
             : cudaLaunchKernelEx(&cfg, process_logits_kernel<T, false>, a);
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
  // CTAs of a row: all rows at once on the SMs (two CTAs each), a power of two up to the cluster's
  // 16 (7 CTAs for 40 rows of 32001 left SMs without a whole cluster: 17.8 us, 4 CTAs 12.9), parts
  // of 4096 to 65536 entries.  One row of 151936: 8 CTAs 8.0 us, 16 CTAs 5.9.
  const int64_t fit = 2 * sm_count() / (int64_t(B) * T);
  int ctas = 1;
  while (ctas < kLpCluster && (vocab > int64_t(ctas) * kLpPer || (2 * ctas <= fit && int64_t(ctas) * 4096 < vocab))) ctas *= 2;
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
