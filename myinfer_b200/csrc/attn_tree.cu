// Attention of a drafted tree's nodes over an 8/4-bit or bf16 cache.
//
//   o_i = sum_s p_is v_s / sum_s p_is,  p_is = exp(scale q_i . k_s - max_i)
//
// over the keys s < n_b and the tree keys whose bit is set in node i's word; a
// row that sees no key is zero.  One CTA per (sequence, head, node): each
// warp takes every eighth key with its own running maximum and sum in fp32, and
// the eight states are joined at the end.
#include <cmath>

#include "tree.cuh"

namespace m5 {

constexpr int TA_WARPS = 8;

template <int BITS, int D>
__device__ __forceinline__ void ta_row(const m5_kv_view& w, int64_t row, int lane, float (&x)[D / 32]) {
  constexpr int N = D / 32;
  const int d0 = lane * N;
  if constexpr (BITS == 0) {
    const bf16* p = reinterpret_cast<const bf16*>(w.data) + row * D + d0;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = bf2f(p[i]);
  } else {
    const uint32_t wd = reinterpret_cast<const uint32_t*>(w.data)[row * (D * BITS / 32) + d0 * BITS / 32];
    const float s = bf2f(reinterpret_cast<const bf16*>(w.scales)[row * (D / 64) + d0 / 64]);
    const float b = bf2f(reinterpret_cast<const bf16*>(w.biases)[row * (D / 64) + d0 / 64]);
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[i] = fmaf(float((wd >> ((d0 * BITS) % 32 + i * BITS)) & ((1u << BITS) - 1)), s, b);
  }
}

template <int BITS, int D>
__global__ void __launch_bounds__(TA_WARPS * 32) tree_attn_kernel(const TreeAttnArgs a) {
  constexpr int N = D / 32;
  __shared__ float s_m[TA_WARPS], s_l[TA_WARPS], s_o[TA_WARPS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x % a.L, h = blockIdx.x / a.L % a.Hq, b = blockIdx.x / a.L / a.Hq;
  const int hk = h / (a.Hq / a.Hkv);
  const int64_t n = a.lengths[b];
  const unsigned long long bits = a.anc[b * a.anc_sb + i];
  const int64_t end = min(n + a.T, a.capacity);
  float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    q[j] = bf2f(a.q[b * a.q_sb + h * a.q_sh + i * a.q_sl + lane * N + j]) * a.scale;
    o[j] = 0.f;
  }
  for (int64_t s = warp; s < end; s += TA_WARPS) {
    if (s >= n && !((bits >> (s - n)) & 1)) continue;
    float x[N], d = 0.f;
    ta_row<BITS, D>(a.k, b * a.k.batch_stride + hk * a.k.head_stride + s, lane, x);
#pragma unroll
    for (int j = 0; j < N; ++j) d = fmaf(q[j], x[j], d);
    d = warp_sum(d);
    const float mn = fmaxf(m, d), c = m == -INFINITY ? 0.f : expf(m - mn), p = expf(d - mn);
    m = mn;
    l = l * c + p;
    ta_row<BITS, D>(a.v, b * a.v.batch_stride + hk * a.v.head_stride + s, lane, x);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = fmaf(p, x[j], o[j] * c);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) s_o[warp][lane * N + j] = o[j];
  __syncthreads();
  float M = -INFINITY;
  for (int w = 0; w < TA_WARPS; ++w) M = fmaxf(M, s_m[w]);
  for (int d = threadIdx.x; d < D; d += TA_WARPS * 32) {
    float num = 0.f, den = 0.f;
    for (int w = 0; w < TA_WARPS; ++w) {
      const float c = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - M);
      num = fmaf(c, s_o[w][d], num);
      den = fmaf(c, s_l[w], den);
    }
    a.out[b * a.o_sb + h * a.o_sh + i * a.o_sl + d] = f2bf(den > 0.f ? num / den : 0.f);
  }
}

size_t tree_attn_ws_bytes(int, int, int, int, int) { return 0; }

template <int D>
static void ta_launch(const TreeAttnArgs& a, cudaStream_t st) {
  const dim3 grid(a.B * a.Hq * a.L);
  if (a.bits == 8) tree_attn_kernel<8, D><<<grid, TA_WARPS * 32, 0, st>>>(a);
  else if (a.bits == 4) tree_attn_kernel<4, D><<<grid, TA_WARPS * 32, 0, st>>>(a);
  else tree_attn_kernel<0, D><<<grid, TA_WARPS * 32, 0, st>>>(a);
}

int tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st) {
  if (a.D == 64) ta_launch<64>(a, st);
  else ta_launch<128>(a, st);
  M5_LAUNCH_CHECK("tree attention launch");
  return M5_OK;
}

int tree_attn_error(int) { return 0; }

}  // namespace m5
