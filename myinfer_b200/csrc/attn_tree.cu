// Attention of a drafted tree's nodes over an 8/4-bit or bf16 cache, on the
// fifth-generation tensor cores.
//
//   o_i = sum_s p_is v_s / sum_s p_is,  p_is = exp(scale q_i . k_s - max_i)
//
// over the keys s < n_b and the tree keys whose bit is set in node i's word.  The
// L nodes and the G = Hq / Hkv heads of a kv head are L * G rows over the same keys;
// up to 128 of them are the M side of the MMAs, so each key is converted once
// for all of them.  Rows x tiles of 64 keys over all sequences, kv heads and row
// blocks form one line of tiles, cut into equal parts, one CTA per SM each: any
// mix of lengths is balanced without the host knowing them.  A part that ends
// inside a (sequence, head, row block) leaves a partial (max, sum, O) in the
// workspace, joined by tree_join_kernel.
//
// Roles of a CTA (480 threads):
//   warp 13      producer: bulk copies of 64-key tiles of K / V rows and of their
//                scales and biases (as the 16-byte blocks around them, so any
//                2-byte alignment will do) into a ring;
//   warp 14      scales: per tile and operand the exponent that puts the tile's largest value
//                into [2^7, 2^8), and scale and bias in fp16 under it;
//   warps 8-11   conversion to fp16, K and V alike: [key][dim] rows of 128 bytes,
//                128-byte swizzle (K is read K-major, V MN-major: no transpose);
//   warp 12      one thread issues the MMAs:  S = Q K^T  (Q, K in shared memory) and
//                O += P V  (P in tensor memory);
//   warps 0-7    softmax.  Even and odd tiles are two independent streams of four
//                warps each, with their own running maximum, sum and O, so that one's exponentials
//                run beside the other's MMAs; S is double buffered within a
//                stream and P overwrites the S it came from.
// Rounding: K, V and P are fp16 (2^-12 of the value or less; bf16 would cost as
// much as the output's own rounding).  The exponents make that safe for
// any range: values keep full precision down to 2^-22 of their tile's largest
// one.  Q is scaled per row in the same way, which is exact.  Scores, maxima,
// sums and O are fp32.  A row's maximum is only moved when a new score exceeds
// it by 2^8 (p <= 256 in fp16): O is rescaled rarely.
// With 64 rows or fewer, the idle rows repeat the rows and take a part of each
// tile's keys (64 rows: halves, 32: quarters), which divides the exponentials
// of a warp by 2 or 4; their states are joined like those of other CTAs.
// TMEM columns: S / P [stream][2] 64 each, O [stream] 128 each.
#include <algorithm>
#include <cmath>

#include "tcgen05.cuh"
#include "tree.cuh"

namespace m5 {

static __device__ int g_attn_tree_err = 0;

namespace atr {

constexpr int TK = 64;      // keys per tile
constexpr int ROWS = 128;   // MMA M
constexpr int SMX_WARPS = 8, DQ_WARPS = 4;
constexpr int MMA_WARP = SMX_WARPS + DQ_WARPS, PROD_WARP = MMA_WARP + 1, PREP_WARP = MMA_WARP + 2;
constexpr int THREADS = (PREP_WARP + 1) * 32;
constexpr int NOP = 3;      // converted K and V tiles held
constexpr int EXPS = 32;    // tile exponents held: more than the tiles between conversion and softmax
constexpr uint32_t TMEM_COLS = 512, S_COL = 0, O_COL = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAZY = 8.f; // log2 growth of a row's maximum that is left in p
constexpr int TOP = 7;      // exponent of a tile's largest value in fp16
constexpr int MIN_TILES = 2;  // per CTA: one per stream

template <int BITS, int D>
struct Cfg {
  static constexpr int G = D / 64;                              // scale groups
  static constexpr int KROW = BITS ? D * BITS / 8 : 2 * D;      // bytes of a packed row
  static constexpr int SROW = BITS ? 2 * G : 0;                 // bytes of a row's scales
  static constexpr int SWIN = BITS ? TK * 2 * G + 32 : 0;       // a tile's scales with the 16-byte blocks around them
  static constexpr int K_OFF = 0, V_OFF = TK * KROW;
  static constexpr int S_OFF = 2 * TK * KROW;                   // K scales, K biases, V scales, V biases
  static constexpr int H_OFF = S_OFF + 4 * SWIN;                // fp16 (s, s), (b, b) per key and group, K then V
  static constexpr int STAGE = (H_OFF + (BITS ? 2 * TK * G * 8 : 0) + 127) / 128 * 128;
  static constexpr int OPER = TK * D * 2;                       // a converted tile
  static constexpr int QBYTES = ROWS * D * 2;
  static constexpr int FIXED = QBYTES + 2 * NOP * OPER + 1024 + 1024;  // + alignment, barriers
  static constexpr int ST = (227 * 1024 - 4096 - FIXED) / STAGE < 8 ? (227 * 1024 - 4096 - FIXED) / STAGE : 8;
  static constexpr int SMEM = FIXED + ST * STAGE;
};

// Barriers, in the order of the array.
template <int ST>
struct Bars {
  uint64_t full[ST], empty[ST], prep[ST];
  uint64_t kfull[NOP], kempty[NOP], vfull[NOP], vempty[NOP];
  uint64_t sfull[4];   // [stream][buffer]
  uint64_t pfull[2], pvdone[2];
  uint64_t qready, idle;
  uint64_t dqmax;      // bf16 caches: the conversion warps' maxima of a tile are in shared memory
};

__device__ __forceinline__ uint32_t sw128(int n, int j) {
  return uint32_t((n >> 3) * 1024 + (n & 7) * 128 + ((j ^ (n & 7)) << 4));
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t hsub1024(uint32_t x) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64006400u));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }  // |e| <= 126
// e with max / 2^e in [2^TOP, 2^(TOP + 1)), kept to exponents pow2 can hold
__device__ __forceinline__ int top_exp(float max) {
  const int e = int(__float_as_uint(max) >> 23) - 127 - TOP;
  return ::min(120, ::max(-120, e));
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// kind::f16 with fp16 operands, fp32 D; B MN-major when `bmn`.
__host__ __device__ constexpr uint32_t idesc(int N, bool bmn) {
  return (1u << 4) | (bmn ? 1u << 16 : 0u) | (uint32_t(N >> 3) << 17) | (uint32_t(ROWS >> 4) << 24);
}
// 128-byte-swizzled operand: 8 x 128-byte atoms `stride` 1 KB apart along the
// row index; `lead` bytes between 64-element blocks along the rows (MN-major).
__device__ __forceinline__ uint64_t sdesc(uint32_t addr, uint32_t lead) {
  return tc_sdesc_sw128(addr) & ~(uint64_t(0x3FFF) << 16) | (uint64_t(lead >> 4) << 16);
}

__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Bounded wait by one thread (~2 s); a failure is shared by the CTA.
__device__ __forceinline__ bool wait1(uint64_t* bar, uint32_t par, volatile int* fail) {
  if (mbar_try_wait_fast(bar, par)) return true;
  const uint64_t t0 = now_ns();
  for (;;) {
    if (mbar_try_wait(bar, par)) return true;
    if (*fail) return false;
    if (now_ns() - t0 > 2000000000ull) break;
  }
  *fail = 1;
  atomicExch(&g_attn_tree_err, M5_DEV_ERR_WAIT_TIMEOUT);
  return false;
}
// Bounded wait by a warp: every lane polls, the result is the same for all.
__device__ __forceinline__ bool waitw(uint64_t* bar, uint32_t par, volatile int* fail) {
  return __all_sync(0xffffffffu, wait1(bar, par, fail));
}

// The line of tiles: sequences in order, each with `pairs` (kv head, row
// block) runs of tiles(b) tiles.
struct Line {
  long long total, begin, end;  // all tiles; this CTA's part
  int b;                        // sequence of `begin` and where its tiles start
  long long base;
};
__device__ __forceinline__ int seq_len(const TreeAttnArgs& a, int b) {
  return (int)::min((long long)::max(a.lengths[b], 0), (long long)a.capacity);
}
__device__ __forceinline__ int seq_end(const TreeAttnArgs& a, int n) {
  return (int)::min((long long)n + a.T, (long long)a.capacity);
}
__device__ __forceinline__ int seq_tiles(const TreeAttnArgs& a, int b) {
  return (seq_end(a, seq_len(a, b)) + TK - 1) / TK;
}
__device__ __forceinline__ long long part_of(long long total, int ctas, long long c) { return total * c / ctas; }
__device__ __forceinline__ int parts(const TreeAttnArgs& a, long long total, int ctas) {
  return (int)::min((long long)ctas, ::max(1LL, total / MIN_TILES));
}
// by one warp: the sum over all sequences, and the sequence that holds tile `at`
// (at < 0: none wanted)
__device__ __forceinline__ void scan_line(const TreeAttnArgs& a, int pairs, int lane, long long at, long long& total,
                                          int& b_at, long long& base_at) {
  long long sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    const long long w = b < a.B ? (long long)seq_tiles(a, b) * pairs : 0;
    long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const bool here = at >= sum + inc - w && at < sum + inc;
    const unsigned m = __ballot_sync(0xffffffffu, here);
    if (m) {
      const int src = __ffs(m) - 1;
      b_at = b0 + src;
      base_at = sum + __shfl_sync(0xffffffffu, inc - w, src);
    }
    sum += __shfl_sync(0xffffffffu, inc, 31);
  }
  total = sum;
}

// Walks a CTA's part run by run; every role holds one and steps it alike.
struct Walk {
  long long at, end, base;
  int b, n, kend, tiles;                      // sequence: committed keys, end of its keys, tiles
  int hk, rb, t0, nt, pair;                   // run: kv head, row block, first tile, tiles of this part; pair = its number
  bool whole;                                 // the part holds all of the run
  __device__ __forceinline__ Walk(const Line& l, const TreeAttnArgs& a) : at(l.begin), end(l.end), base(l.base), b(l.b) {
    load(a);
  }
  __device__ __forceinline__ void load(const TreeAttnArgs& a) {
    n = seq_len(a, b);
    kend = seq_end(a, n);
    tiles = (kend + TK - 1) / TK;
  }
  __device__ __forceinline__ bool next(const TreeAttnArgs& a, int nrb) {
    if (at >= end) return false;
    const int pairs = a.Hkv * nrb;
    if (at - base >= (long long)tiles * pairs) {
      base += (long long)tiles * pairs;
      ++b;
      load(a);
    }
    const long long in = at - base;
    const int p = (int)(in / tiles);
    t0 = (int)(in - (long long)p * tiles);
    nt = (int)::min((long long)(tiles - t0), end - at);
    hk = p / nrb;
    rb = p % nrb;
    pair = b * pairs + p;
    whole = t0 == 0 && nt == tiles;
    at += nt;
    return true;
  }
};

// Rows of a block (nrows of 128) repeat 4, 2 or 1 times over the lanes.
__device__ __forceinline__ int repeats(int nrows) { return nrows <= 32 ? 4 : nrows <= 64 ? 2 : 1; }

// Tree keys that some query of sequence b sees (by one warp).
__device__ __forceinline__ unsigned long long seen_by_any(const TreeAttnArgs& a, int b, int lane) {
  unsigned long long w = 0;
  for (int i = lane; i < a.L; i += 32) w |= a.anc[b * a.anc_sb + i];
  const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)w), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(w >> 32));
  return ((unsigned long long)hi << 32) | lo;
}
// Visible keys of the 64 from `key0` on, as bits: all below n, then the bits of
// `word` (tree keys below T and the cache's end).
__device__ __forceinline__ unsigned long long visible(unsigned long long word, int key0, int n, int kend) {
  const int rel = key0 - n, t = kend - n;
  if (t < 64) word &= (1ull << t) - 1;
  if (rel >= 64) return 0;
  if (rel >= 0) return word >> rel;
  if (rel <= -64) return ~0ull;
  return (word << -rel) | ((1ull << -rel) - 1);
}

// fp16 (K, V): 8 consecutive dims of a row into one 16-byte chunk.
// 8-bit: (1024 + code) - 1024 is exact, as are s and b (bf16 values), so code * s + b is rounded
// once.  Folding an offset of the code into b instead would round b, which errs alike for
// all 64 dims of a group: 1 % of the output where the scores reach 50.
__device__ __forceinline__ uint4 conv8(uint2 w, uint32_t s, uint32_t b) {
  uint4 o;
  o.x = hfma2(hsub1024(__byte_perm(w.x, 0x64u, 0x4140)), s, b);
  o.y = hfma2(hsub1024(__byte_perm(w.x, 0x64u, 0x4342)), s, b);
  o.z = hfma2(hsub1024(__byte_perm(w.y, 0x64u, 0x4140)), s, b);
  o.w = hfma2(hsub1024(__byte_perm(w.y, 0x64u, 0x4342)), s, b);
  return o;
}
// 4-bit: the same.  Position 2 i + h of the chunk is dim i + 4 h.
__device__ __forceinline__ uint4 conv4(uint32_t w, uint32_t s, uint32_t b) {
  constexpr uint32_t M = 0x000F000Fu, X = 0x64006400u;
  uint4 o;
  o.x = hfma2(hsub1024((w & M) | X), s, b);
  o.y = hfma2(hsub1024(((w >> 4) & M) | X), s, b);
  o.z = hfma2(hsub1024(((w >> 8) & M) | X), s, b);
  o.w = hfma2(hsub1024(((w >> 12) & M) | X), s, b);
  return o;
}
__device__ __forceinline__ uint4 conv16(uint4 w, float f) {
  return make_uint4(h2(bf16_lo(w.x) * f, bf16_hi(w.x) * f), h2(bf16_lo(w.y) * f, bf16_hi(w.y) * f),
                    h2(bf16_lo(w.z) * f, bf16_hi(w.z) * f), h2(bf16_lo(w.w) * f, bf16_hi(w.w) * f));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

// State of one row in one stream.
struct Row {
  float m, l;  // maximum in log2 units (-inf: nothing seen), sum of p
  int ev;      // O holds its sum divided by 2^ev
};

// One tile of a softmax thread: N of the tile's 64 keys, from `off` on.  P of the
// other keys is zero.  Returns false when a wait failed.
template <int N, int D>
__device__ __forceinline__ bool softmax_tile(Row& r, uint32_t s_addr, uint32_t o_addr, int off, float c, int ev,
                                             bool edge, unsigned long long vis, bool first, uint64_t* pvdone,
                                             uint32_t pv_par, volatile int* fail) {
  float s[N];
#pragma unroll
  for (int i = 0; i < N; i += 16) tmem_ld16(s_addr + off + i, *reinterpret_cast<float(*)[16]>(s + i));
  tmem_ld_wait();
  if (edge) {
    vis >>= off;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!((vis >> i) & 1)) s[i] = -INFINITY;
  }
  float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int i = 4; i < N; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mx[j] = i + 4 + j < N ? max3(mx[j], s[i + j], s[i + 4 + j]) : fmaxf(mx[j], s[i + j]);
  }
  const float tmax = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
  const float mt = tmax == -INFINITY ? -INFINITY : tmax * c;
  float corr = 1.f;
  if (mt > r.m + LAZY || (r.m == -INFINITY && mt != -INFINITY)) {
    corr = r.m == -INFINITY ? 0.f : ex2(r.m - mt);
    r.m = mt;
    r.l *= corr;
  }
  if (!first && ev != r.ev) corr *= pow2(::max(r.ev - ev, -126));
  r.ev = ev;
  const float neg = r.m == -INFINITY ? 0.f : -r.m;
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint32_t p[N / 2];
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 x = ffma2(make_float2(s[i], s[i + 1]), make_float2(c, c), make_float2(neg, neg));
    const float2 e = make_float2(ex2(x.x), ex2(x.y));
    sum[(i >> 1) & 1] = ffma2(e, make_float2(1.f, 1.f), sum[(i >> 1) & 1]);
    p[i / 2] = h2(e.x, e.y);
  }
  r.l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
  if constexpr (N == 64) {
    tmem_st32(s_addr, p);
  } else {
    uint32_t z[16];
#pragma unroll
    for (int k = 0; k < 64; k += 32) {  // 32 keys = 16 columns at a time
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if constexpr (N == 32) z[i] = k == off ? p[i] : 0u;
        else z[i] = k + (i >= 8 ? 16 : 0) == off ? p[i & 7] : 0u;
      }
      tmem_st16(s_addr + k / 2, z);
    }
  }
  if (!first && __any_sync(0xffffffffu, corr != 1.f)) {
    if (!waitw(pvdone, pv_par, fail)) return false;
    tc_fence_after();
#pragma unroll
    for (int d = 0; d < D; d += 16) {
      float o[16];
      uint32_t u[16];
      tmem_ld16(o_addr + d, o);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(o[i] * corr);
      tmem_st16(o_addr + d, u);
    }
  }
  tmem_st_wait();
  return true;
}

template <int BITS, int D>
__global__ void __launch_bounds__(THREADS, 1) tree_attn_kernel(const TreeAttnArgs a, const int nrb, float* part_o,
                                                               float2* part_ml) {
  using C = Cfg<BITS, D>;
  constexpr int ST = C::ST, G = C::G;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = base;                         // [G][128 rows][128 bytes]
  uint8_t* kop = qs + C::QBYTES;              // [NOP][G][64 keys][128 bytes]
  uint8_t* vop = kop + NOP * C::OPER;
  uint8_t* ring = vop + NOP * C::OPER;
  Bars<ST>& bar = *reinterpret_cast<Bars<ST>*>(ring + ST * C::STAGE);
  static_assert(sizeof(Bars<ST>) <= 1024, "barriers");
  __shared__ Row s_row[2][ROWS];
  __shared__ float s_kmul[EXPS];
  __shared__ int s_ev[EXPS];
  __shared__ float s_dqmax[2][2][DQ_WARPS];  // [tile parity][K, V]
  __shared__ Line s_line;
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail, s_stop;
  volatile int* fail = &s_fail;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = a.Hq / a.Hkv, R = a.L * grp;  // heads of a kv head, rows

  if (tid == 0) {
    s_fail = 0;
    for (int i = 0; i < ST; ++i) {
      mbar_init(&bar.full[i], 1);
      mbar_init(&bar.empty[i], DQ_WARPS);
      mbar_init(&bar.prep[i], 1);
    }
    for (int i = 0; i < NOP; ++i) {
      mbar_init(&bar.kfull[i], DQ_WARPS);
      mbar_init(&bar.vfull[i], DQ_WARPS);
      mbar_init(&bar.kempty[i], 1);
      mbar_init(&bar.vempty[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bar.sfull[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.pfull[i], SMX_WARPS / 2);
      mbar_init(&bar.pvdone[i], 1);
    }
    mbar_init(&bar.qready, SMX_WARPS);
    mbar_init(&bar.idle, 1);
    mbar_init(&bar.dqmax, DQ_WARPS);
    fence_mbar_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&s_tmem, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0) {
    Line l;
    scan_line(a, a.Hkv * nrb, lane, -1, l.total, l.b, l.base);
    const int np = parts(a, l.total, gridDim.x), c = blockIdx.x;
    l.begin = c < np ? part_of(l.total, np, c) : l.total;
    l.end = c < np ? part_of(l.total, np, c + 1) : l.total;
    l.b = a.B - 1;
    l.base = 0;
    long long t;
    scan_line(a, a.Hkv * nrb, lane, l.begin, t, l.b, l.base);
    if (lane == 0) s_line = l;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const Line line = s_line;
  const int cta_slot = blockIdx.x;

  if (warp == PROD_WARP) {
    // ------------------------------------------------------------- producer
    if (lane == 0) {
      Walk w(line, a);
      int g = 0;
      bool ok = true;
      while (ok && w.next(a, nrb)) {
        const int64_t kb = w.b * a.k.batch_stride + w.hk * a.k.head_stride;
        const int64_t vb = w.b * a.v.batch_stride + w.hk * a.v.head_stride;
        for (int t = 0; t < w.nt; ++t, ++g) {
          const int st = g % ST, key0 = (w.t0 + t) * TK, nk = min(TK, w.kend - key0);
          if (!(ok = wait1(&bar.empty[st], ((g / ST) & 1) ^ 1, fail))) break;
          uint8_t* sb = ring + size_t(st) * C::STAGE;
          uint32_t bytes = 2 * nk * C::KROW;
          uintptr_t src[4];
          uint32_t len[4];
          if constexpr (BITS != 0) {
            const void* const arr[4] = {a.k.scales, a.k.biases, a.v.scales, a.v.biases};
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // the 16-byte blocks that hold the tile's values
              const uintptr_t p = reinterpret_cast<uintptr_t>(arr[i]) + uintptr_t((i < 2 ? kb : vb) + key0) * C::SROW;
              src[i] = p & ~uintptr_t(15);
              len[i] = uint32_t(((p + nk * C::SROW + 15) & ~uintptr_t(15)) - src[i]);
              bytes += len[i];
            }
          }
          mbar_arrive_expect_tx(&bar.full[st], bytes);
          bulk_g2s(sb + C::K_OFF, reinterpret_cast<const uint8_t*>(a.k.data) + (kb + key0) * C::KROW, nk * C::KROW,
                   &bar.full[st]);
          bulk_g2s(sb + C::V_OFF, reinterpret_cast<const uint8_t*>(a.v.data) + (vb + key0) * C::KROW, nk * C::KROW,
                   &bar.full[st]);
          if constexpr (BITS != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              bulk_g2s(sb + C::S_OFF + i * C::SWIN, reinterpret_cast<const void*>(src[i]), len[i], &bar.full[st]);
          }
        }
      }
      // the copies in flight land before the CTA may exit
      for (int t = max(0, g - ST); t < g; ++t) (void)wait1(&bar.full[t % ST], (t / ST) & 1, fail);
    }
  } else if (warp == PREP_WARP) {
    // --------------------------------------------------------------- scales
    if constexpr (BITS != 0) {
      Walk w(line, a);
      int g = 0;
      bool ok = true;
      while (ok && w.next(a, nrb)) {
        int ev[2] = {-127, -127};  // running exponent of V in each stream
        const int64_t kb = w.b * a.k.batch_stride + w.hk * a.k.head_stride;
        const int64_t vb = w.b * a.v.batch_stride + w.hk * a.v.head_stride;
        for (int t = 0; t < w.nt; ++t, ++g) {
          const int st = g % ST, key0 = (w.t0 + t) * TK;
          unsigned long long vis = ~0ull;
          if (key0 + TK > w.n) vis = visible(seen_by_any(a, w.b, lane), key0, w.n, w.kend);
          if (!(ok = waitw(&bar.full[st], (g / ST) & 1, fail))) break;
          uint8_t* sb = ring + size_t(st) * C::STAGE;
          const void* const arr[4] = {a.k.scales, a.k.biases, a.v.scales, a.v.biases};
          float s[2][2 * G], b[2][2 * G], mx[2] = {0.f, 0.f};
#pragma unroll
          for (int o = 0; o < 2; ++o) {  // K, V
            const uint32_t at = uint32_t(o ? vb + key0 : kb + key0) * C::SROW;
            const uint8_t* sp = sb + C::S_OFF + 2 * o * C::SWIN + ((uint32_t(reinterpret_cast<uintptr_t>(arr[2 * o])) + at) & 15);
            const uint8_t* bp = sb + C::S_OFF + (2 * o + 1) * C::SWIN +
                                ((uint32_t(reinterpret_cast<uintptr_t>(arr[2 * o + 1])) + at) & 15);
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) {  // element e of the tile's [64][G]
              const int e = lane + 32 * i;
              const bool in = (vis >> (e / G)) & 1;
              s[o][i] = in ? bf2f(reinterpret_cast<const bf16*>(sp)[e]) : 0.f;
              b[o][i] = in ? bf2f(reinterpret_cast<const bf16*>(bp)[e]) : 0.f;
              mx[o] = max3(mx[o], fabsf(b[o][i]), fabsf(fmaf(s[o][i], float((1 << BITS) - 1), b[o][i])));
            }
            mx[o] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx[o])));
          }
          const int ek = top_exp(mx[0]);
          const int e2 = max(ev[g & 1], top_exp(mx[1]));
          ev[g & 1] = e2;
          if (lane == 0) {
            s_kmul[g % EXPS] = pow2(ek);
            s_ev[g % EXPS] = e2;
          }
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const float f = pow2(-(o ? e2 : ek));
            uint2* dst = reinterpret_cast<uint2*>(sb + C::H_OFF + o * TK * G * 8);
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) {
              const float sf = s[o][i] * f, bfv = b[o][i] * f;
              dst[lane + 32 * i] = make_uint2(h2(sf, sf), h2(bfv, bfv));
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.prep[st]);
        }
      }
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t id_s = idesc(TK, false), id_o = idesc(D, true);
      const uint32_t q_addr = smem_addr(qs), k_addr = smem_addr(kop), v_addr = smem_addr(vop);
      Walk w(line, a);
      int g0 = 0, seg = 0;
      bool ok = true;
      while (ok && w.next(a, nrb)) {
        ok = wait1(&bar.qready, seg & 1, fail);
        auto issue_s = [&](int g) -> bool {
          const int j = g & 1, u = g >> 1, ob = g % NOP;
          if (!wait1(&bar.kfull[ob], (g / NOP) & 1, fail)) return false;
          // P of tile g - 4 sits in this buffer until its PV is done (a run's first two tiles: it is, and the phase is past)
          if (g >= g0 + 2 && u >= 2 && !wait1(&bar.pvdone[j], (u - 2) & 1, fail)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t blk = kk / 4, in = 2u * (kk % 4);
            tc_mma_ss(tmem + S_COL + 64u * (2 * j + (u & 1)), sdesc(q_addr + blk * (ROWS * 128), 16) + in,
                      sdesc(k_addr + ob * C::OPER + blk * (TK * 128), 16) + in, id_s, kk > 0 ? 1u : 0u);
          }
          tc_commit(&bar.sfull[2 * j + (u & 1)]);
          tc_commit(&bar.kempty[ob]);
          return true;
        };
        if (ok) ok = issue_s(g0);
        if (ok && w.nt > 1) ok = issue_s(g0 + 1);
        for (int t = 0; t < w.nt && ok; ++t) {
          const int g = g0 + t, j = g & 1, u = g >> 1, ob = g % NOP;
          if (t + 2 < w.nt && !(ok = issue_s(g + 2))) break;
          if (!(ok = wait1(&bar.vfull[ob], (g / NOP) & 1, fail) && wait1(&bar.pfull[j], u & 1, fail))) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < TK / 16; ++kk)
            tc_mma_ts(tmem + O_COL + 128u * j, tmem + S_COL + 64u * (2 * j + (u & 1)) + 8u * kk,
                      sdesc(v_addr + ob * C::OPER + kk * 2048, TK * 128), id_o, (t > 1 || kk > 0) ? 1u : 0u);
          tc_commit(&bar.pvdone[j]);
          tc_commit(&bar.vempty[ob]);
        }
        g0 += w.nt;
        ++seg;
      }
      // every MMA issued has completed before TMEM may be freed
      tc_commit(&bar.idle);
      (void)wait1(&bar.idle, 0, fail);
    }
  } else if (warp >= SMX_WARPS) {
    // ------------------------------------------------------------ conversion
    const int d = tid - SMX_WARPS * 32;
    constexpr int PIECES = D / 16, PER = TK * PIECES / (DQ_WARPS * 32);  // 16-dim pieces of a row; per thread and operand
    Walk w(line, a);
    int g = 0;
    bool ok = true;
    while (ok && w.next(a, nrb)) {
      int ev[2] = {-127, -127};
      for (int t = 0; t < w.nt; ++t, ++g) {
        const int st = g % ST, ob = g % NOP;
        const uint8_t* sb = ring + size_t(st) * C::STAGE;
        unsigned long long vis = ~0ull;
        if constexpr (BITS == 0) {
          const int key0 = (w.t0 + t) * TK;
          if (key0 + TK > w.n) vis = visible(seen_by_any(a, w.b, lane), key0, w.n, w.kend);
        } else {
          if (!(ok = waitw(&bar.prep[st], (g / ST) & 1, fail))) break;
        }
        if (!(ok = waitw(&bar.full[st], (g / ST) & 1, fail))) break;
        // bf16 caches: both operands' values and largest exponents first (the softmax reads them with S)
        uint4 x[BITS == 0 ? 2 : 1][PER][2];
        float scale16[2];
        if constexpr (BITS == 0) {
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const uint8_t* src = sb + (o ? C::V_OFF : C::K_OFF);
            uint32_t mx = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int e = d + i * DQ_WARPS * 32, key = e / PIECES, c = e % PIECES;
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                // halves of the row's upper group in the other order: the 8 lanes of a phase hit 8 bank groups
                const int h = G == 2 ? hh ^ (c >> 2) : hh;
                const uint4 y = ((vis >> key) & 1) ? *reinterpret_cast<const uint4*>(src + key * C::KROW + (2 * c + h) * 16)
                                                   : make_uint4(0, 0, 0, 0);
                x[o][i][hh] = y;
                mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(y.x & 0x7FFF7FFFu, y.y & 0x7FFF7FFFu),
                                           __vmaxu2(y.z & 0x7FFF7FFFu, y.w & 0x7FFF7FFFu)));
              }
            }
            mx = __reduce_max_sync(0xffffffffu, max(mx & 0xFFFFu, mx >> 16));
            if (lane == 0) s_dqmax[g & 1][o][warp - SMX_WARPS] = __uint_as_float(mx << 16);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.dqmax);
          if (!(ok = waitw(&bar.dqmax, g & 1, fail))) break;
          float m[2] = {0.f, 0.f};
#pragma unroll
          for (int i = 0; i < DQ_WARPS; ++i) {
            m[0] = fmaxf(m[0], s_dqmax[g & 1][0][i]);
            m[1] = fmaxf(m[1], s_dqmax[g & 1][1][i]);
          }
          const int ek = top_exp(m[0]);
          ev[g & 1] = max(ev[g & 1], top_exp(m[1]));
          if (d == 0) {
            s_kmul[g % EXPS] = pow2(ek);
            s_ev[g % EXPS] = ev[g & 1];
          }
          scale16[0] = pow2(-ek);
          scale16[1] = pow2(-ev[g & 1]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.empty[st]);
        }
#pragma unroll
        for (int o = 0; o < 2; ++o) {  // K, V
          uint64_t* fullb = o ? bar.vfull : bar.kfull;
          uint64_t* emptyb = o ? bar.vempty : bar.kempty;
          uint8_t* dst = (o ? vop : kop) + ob * C::OPER;
          const uint8_t* src = sb + (o ? C::V_OFF : C::K_OFF);
          if constexpr (BITS == 0) {
            if (!(ok = waitw(&emptyb[ob], ((g / NOP) & 1) ^ 1, fail))) break;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int e = d + i * DQ_WARPS * 32, key = e / PIECES, c = e % PIECES;
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const int ch = 2 * c + (G == 2 ? hh ^ (c >> 2) : hh);
                *reinterpret_cast<uint4*>(dst + (ch >> 3) * (TK * 128) + sw128(key, ch & 7)) = conv16(x[o][i][hh], scale16[o]);
              }
            }
          } else {
            const uint2* sc = reinterpret_cast<const uint2*>(sb + C::H_OFF + o * TK * G * 8);
            if (!(ok = waitw(&emptyb[ob], ((g / NOP) & 1) ^ 1, fail))) break;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int e = d + i * DQ_WARPS * 32, key = e / PIECES, c = e % PIECES;
              const uint2 sbv = sc[key * G + (G == 2 ? c >> 2 : 0)];
              uint4 v[2];
              if constexpr (BITS == 8) {
                const uint4 x = *reinterpret_cast<const uint4*>(src + key * C::KROW + c * 16);
                v[0] = conv8(make_uint2(x.x, x.y), sbv.x, sbv.y);
                v[1] = conv8(make_uint2(x.z, x.w), sbv.x, sbv.y);
              } else {
                const uint2 x = *reinterpret_cast<const uint2*>(src + key * C::KROW + c * 8);
                v[0] = conv4(x.x, sbv.x, sbv.y);
                v[1] = conv4(x.y, sbv.x, sbv.y);
              }
              const bool sw = G == 2 && (c >> 2);  // upper group: halves in the other order (bank groups)
#pragma unroll
              for (int hh = 0; hh < 2; ++hh) {
                const int ch = 2 * c + (sw ? hh ^ 1 : hh);
                *reinterpret_cast<uint4*>(dst + (ch >> 3) * (TK * 128) + sw128(key, ch & 7)) = sw ? v[hh ^ 1] : v[hh];
              }
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&fullb[ob]);
            if (BITS != 0 && o) mbar_arrive(&bar.empty[st]);
          }
        }
        if (!ok) break;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int j = warp >> 2, r = tid & 127;      // stream, lane of tensor memory
    const uint32_t lrow = uint32_t(32 * (warp & 3)) << 16;
    Walk w(line, a);
    int g0 = 0;
    bool ok = true;
    while (ok && w.next(a, nrb)) {
      const int row0 = w.rb * ROWS, nrows = min(ROWS, R - row0);
      const int rep = repeats(nrows), per = ROWS / rep;
      const int lr = r % per, off = r / per * (TK / rep);  // row of the block, first of this lane's keys
      const bool row_ok = lr < nrows;
      const bool idle = lr - lane >= nrows;                // the whole warp has no row (per is a multiple of 32)
      const int row = row0 + (row_ok ? lr : 0), qi = row / grp, h = w.hk * grp + row % grp;
      const unsigned long long word = a.anc[w.b * a.anc_sb + qi];
      // Q, scaled by a power of two per row; the sign of `scale` goes with it
      float c_row;
      {
        const uint4* qr = reinterpret_cast<const uint4*>(a.q + w.b * a.q_sb + h * a.q_sh + qi * a.q_sl);
        uint4 x[D / 8];
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = row_ok ? qr[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu),
                                     __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu)));
        const int eq = top_exp(__uint_as_float(max(mx & 0xFFFFu, mx >> 16) << 16));
        const float f = a.scale < 0.f ? -pow2(-eq) : pow2(-eq);
        c_row = fmaxf(fabsf(a.scale) * LOG2E * pow2(eq), 1e-37f);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {  // stream j stores half of the chunks
          const int ch = j * (D / 16) + i;
          const uint4 y = j ? x[D / 16 + i] : x[i];
          uint4 o = conv16(y, f);
          if constexpr (BITS == 4)  // positions 2 i + h hold dims i + 4 h, as the codes come
            o = make_uint4(__byte_perm(o.x, o.z, 0x5410), __byte_perm(o.x, o.z, 0x7632), __byte_perm(o.y, o.w, 0x5410),
                           __byte_perm(o.y, o.w, 0x7632));
          *reinterpret_cast<uint4*>(qs + (ch >> 3) * (ROWS * 128) + sw128(r, ch & 7)) = o;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.qready);
      }
      Row st{-INFINITY, 0.f, 0};
      int last = -1;  // this stream's last tile
      for (int g = g0 + ((g0 & 1) ^ j); g < g0 + w.nt && ok; g += 2) {
        const int u = g >> 1, buf = 2 * j + (u & 1), key0 = (w.t0 + g - g0) * TK;
        if (!(ok = waitw(&bar.sfull[buf], (u >> 1) & 1, fail))) break;
        if (!idle) {
          tc_fence_after();
          const bool edge = key0 + TK > w.n;
          const unsigned long long vis = edge ? visible(word, key0, w.n, w.kend) : 0ull;
          const float c = c_row * s_kmul[g % EXPS];
          const int ev = s_ev[g % EXPS];
          const uint32_t sa = tmem + lrow + S_COL + 64u * buf, oa = tmem + lrow + O_COL + 128u * j;
          if (rep == 1)
            ok = softmax_tile<64, D>(st, sa, oa, 0, c, ev, edge, vis, last < 0, &bar.pvdone[j], (u - 1) & 1, fail);
          else if (rep == 2)
            ok = softmax_tile<32, D>(st, sa, oa, off, c, ev, edge, vis, last < 0, &bar.pvdone[j], (u - 1) & 1, fail);
          else
            ok = softmax_tile<16, D>(st, sa, oa, off, c, ev, edge, vis, last < 0, &bar.pvdone[j], (u - 1) & 1, fail);
          if (!ok) break;
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.pfull[j]);
        last = u;
      }
      // ---- end of the run: both streams' O are complete
      if (ok && last >= 0) ok = waitw(&bar.pvdone[j], last & 1, fail);
      s_row[j][r] = st;
      tc_fence_before();
      named_sync(1, SMX_WARPS * 32);
      tc_fence_after();
      if (tid == 0) s_stop = *fail;
      if (ok && !idle) {
        const Row x = s_row[0][r], y = s_row[1][r];
        const float M = fmaxf(x.m, y.m);
        const float wx = x.m == -INFINITY ? 0.f : ex2(x.m - M), wy = y.m == -INFINITY ? 0.f : ex2(y.m - M);
        const float l = x.l * wx + y.l * wy;
        const bool direct = w.whole && rep == 1;
        const float inv = direct ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
        const float fx = wx * pow2(x.ev) * inv, fy = wy * pow2(y.ev) * inv;
        const size_t slot = size_t(cta_slot + w.pair) * ROWS + r;
        bf16* out = a.out + w.b * a.o_sb + h * a.o_sh + qi * a.o_sl;
#pragma unroll
        for (int i = 0; i < D / 2; i += 16) {  // stream j's warps write half of the dims
          const int d0 = j * (D / 2) + i;
          float o0[16], o1[16];
          tmem_ld16(tmem + lrow + O_COL + d0, o0);
          tmem_ld16(tmem + lrow + O_COL + 128u + d0, o1);
          tmem_ld_wait();
          float o[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int dim = BITS == 4 ? (k & 8) + ((k & 7) >> 1) + 4 * (k & 1) : k;
            o[dim] = (wx > 0.f ? o0[k] * fx : 0.f) + (wy > 0.f ? o1[k] * fy : 0.f);
          }
          if (!row_ok) continue;
          if (direct) {
            uint4 v[2];
            uint32_t* p = reinterpret_cast<uint32_t*>(v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const __nv_bfloat162 z = __floats2bfloat162_rn(o[2 * k], o[2 * k + 1]);
              p[k] = *reinterpret_cast<const uint32_t*>(&z);
            }
            reinterpret_cast<uint4*>(out + d0)[0] = v[0];
            reinterpret_cast<uint4*>(out + d0)[1] = v[1];
          } else {
            float4* po = reinterpret_cast<float4*>(part_o + slot * D + d0);
#pragma unroll
            for (int k = 0; k < 4; ++k) po[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
        }
        if (!direct && row_ok && j == 0) part_ml[slot] = make_float2(M, l);
      }
      tc_fence_before();
      named_sync(1, SMX_WARPS * 32);  // O and Q may be overwritten
      tc_fence_after();
      ok = !s_stop;  // one answer for the eight warps: they meet at the barriers of the next run or leave together
      g0 += w.nt;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Joins the partial states of the rows whose run was cut: one CTA per (row block of a
// kv head, row): o = sum_i w_i O_i / sum_i w_i l_i, w_i = 2^(m_i - max).
// The parts of a run are consecutive CTAs, each with `rep` repeats of the row.
constexpr int JOIN_WARPS = 4;
template <int D>
__global__ void __launch_bounds__(JOIN_WARPS * 32) tree_join_kernel(const TreeAttnArgs a, const int nrb, const int ctas,
                                                                    const float* part_o, const float2* part_ml) {
  constexpr int N = D / 32;
  __shared__ float s_m[JOIN_WARPS], s_l[JOIN_WARPS], s_o[JOIN_WARPS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = a.Hq / a.Hkv, R = a.L * grp, pairs = a.Hkv * nrb;
  const int row = blockIdx.x % R, hk = blockIdx.x / R % a.Hkv, b = blockIdx.x / R / a.Hkv;
  const int rb = row / ROWS, lr = row % ROWS, rep = repeats(min(ROWS, R - rb * ROWS)), per = ROWS / rep;
  long long total, base = 0;
  {
    // tiles before sequence b, and in all
    long long before = 0, all = 0;
    for (int i = lane; i < a.B; i += 32) {
      const long long t = (long long)seq_tiles(a, i) * pairs;
      all += t;
      if (i < b) before += t;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      all += __shfl_xor_sync(0xffffffffu, all, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    total = all;
    base = before;
  }
  const int tiles = seq_tiles(a, b), p = hk * nrb + rb, np = parts(a, total, ctas);
  const long long t0 = base + (long long)p * tiles, t1 = t0 + tiles - 1;
  // part c holds tile t: total * c / np <= t
  const int c0 = (int)(((t0 + 1) * np - 1) / total), c1 = (int)(((t1 + 1) * np - 1) / total);
  if (c0 == c1 && rep == 1) return;  // written by the attention kernel
  const int n = (c1 - c0 + 1) * rep;
  const size_t slot0 = size_t(c0 + b * pairs + p) * ROWS + lr;
  float m = -INFINITY, l = 0.f, o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  for (int i = warp; i < n; i += JOIN_WARPS) {
    const size_t slot = slot0 + size_t(i / rep) * ROWS + (i % rep) * per;
    const float2 ml = part_ml[slot];
    if (ml.x == -INFINITY) continue;
    const float mn = fmaxf(m, ml.x), c = m == -INFINITY ? 0.f : exp2f(m - mn), e = exp2f(ml.x - mn);
    m = mn;
    l = l * c + ml.y * e;
    const float* po = part_o + slot * D + lane * N;
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = fmaf(po[k], e, o[k] * c);
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s_o[warp][lane * N + i] = o[i];
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < JOIN_WARPS; ++i) M = fmaxf(M, s_m[i]);
  const int qi = row / grp, h = hk * grp + row % grp;
  for (int d = threadIdx.x; d < D; d += JOIN_WARPS * 32) {
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int i = 0; i < JOIN_WARPS; ++i) {
      const float c = s_m[i] == -INFINITY ? 0.f : exp2f(s_m[i] - M);
      num = fmaf(c, s_o[i][d], num);
      den = fmaf(c, s_l[i], den);
    }
    a.out[b * a.o_sb + h * a.o_sh + qi * a.o_sl + d] = f2bf(den == 0.f ? 0.f : num / den);
  }
}

struct Plan {
  int nrb, ctas;
  size_t slots;
};
static Plan plan(int B, int Hq, int Hkv, int L) {
  const int nrb = ceil_div((long long)L * (Hq / Hkv), ROWS);
  const int ctas = sm_count();
  return {nrb, ctas, size_t(ctas) + size_t(B) * Hkv * nrb};
}

template <int BITS, int D>
static cudaError_t launch(const TreeAttnArgs& a, const Plan& p, cudaStream_t st) {
  using C = Cfg<BITS, D>;
  static DeviceOnce once;
  cudaError_t e = once.run([&] {
    return cudaFuncSetAttribute(tree_attn_kernel<BITS, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (e != cudaSuccess) return e;
  float* po = reinterpret_cast<float*>(a.ws);
  float2* ml = reinterpret_cast<float2*>(po + p.slots * ROWS * D);
  tree_attn_kernel<BITS, D><<<p.ctas, THREADS, C::SMEM, st>>>(a, p.nrb, po, ml);
  tree_join_kernel<D><<<a.B * a.Hq * a.L, JOIN_WARPS * 32, 0, st>>>(a, p.nrb, p.ctas, po, ml);
  return cudaGetLastError();
}

}  // namespace atr

size_t tree_attn_ws_bytes(int B, int Hq, int Hkv, int L, int D) {
  return atr::plan(B, Hq, Hkv, L).slots * atr::ROWS * (size_t(D) + 2) * sizeof(float);
}

int tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st) {
  const atr::Plan p = atr::plan(a.B, a.Hq, a.Hkv, a.L);
  cudaError_t e;
  if (a.D == 64) e = a.bits == 8 ? atr::launch<8, 64>(a, p, st) : a.bits == 4 ? atr::launch<4, 64>(a, p, st) : atr::launch<0, 64>(a, p, st);
  else e = a.bits == 8 ? atr::launch<8, 128>(a, p, st) : a.bits == 4 ? atr::launch<4, 128>(a, p, st) : atr::launch<0, 128>(a, p, st);
  M5_CUDA(e);
  return M5_OK;
}

int tree_attn_error(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_tree_err, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v) {
    const int z = 0;
    cudaMemcpyToSymbol(g_attn_tree_err, &z, sizeof(int));
  }
  return v;
}

}  // namespace m5
