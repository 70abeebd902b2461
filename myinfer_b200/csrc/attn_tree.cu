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
// Roles of a CTA (896 threads, registers moved to the softmax by setmaxnreg):
//   warp 25      producer: bulk copies of 64-key tiles of K / V rows and of their
//                scales and biases (as the 16-byte blocks around them, since a head's may
//                start anywhere) into a ring;
//   warps 26-27  scales, even and odd tiles: per tile and operand the exponent that puts the tile's largest value
//                under 2^-2, and scale and bias in fp16 under it;
//   warps 16-23  conversion to fp16, four warps for K and four for V, both into [key][dim] rows of
//                128 bytes, 128-byte swizzle (K is read K-major, V MN-major: no transpose);
//   warp 24      one thread issues the MMAs:  S = Q K^T  (Q, K in shared memory) and
//                O += P V  (P in tensor memory);
//   warps 0-15   softmax.  Two independent streams of eight warps, each with its own running
//                maximum, sum and O, so that one's exponentials run beside the other's
//                MMAs: the even and the odd tiles of one block of 128 rows, or, above 128
//                rows, the same tiles for two blocks.  Two warps share 32 rows of a
//                stream and take half of a tile's keys each; they only exchange maxima when
//                one of them moves (a barrier with an OR tells).  S is double buffered
//                within a stream and P overwrites the S it came from.
// Rounding: K, V and P are fp16 (2^-11 of the value; bf16 would cost as
// much as the output's own rounding).  The exponents make that safe for any range:
// below fp16's normal numbers an element is off by half a unit, 2^-25, where the
// largest of K's tile, and of V's tiles in this run so far (O can follow an exponent
// up, not down: it might overflow), is held at 2^-3 or more for codes and 2^7 for bf16.
// That is 2^-22 of the largest, twice for codes with the rounding of their bias, and 2^-32 for bf16:
// a value 2^12 below another one of its run is right to 2^-9 of itself, a bf16's rounding.
// Q is scaled per row in the same way, which is exact.  Scores, maxima,
// sums and O are fp32.  Infinities and NaN stay what they are and have no part in the
// exponents; the V of a tree key that holds one is zeroed and the queries that see the key
// are made NaN at the run's end, so that the others do not meet 0 times it (512 rows over
// 32768 keys 98.9 us with it, 97.5 without; bf16 127.4, 123.2).  A row's maximum is only
// moved when a new score exceeds it by 2^8 (p <= 256 in fp16): O is rescaled rarely.
// TMEM columns: S / P [stream][2] 64 each, O [stream] 128 each (all 512).
//
// Time on the device (launches in a graph, inputs of 3 sets in turn): 2 rows a kv head over
// 512 keys 13.0 us (two launches, one tile per CTA and a join: latency); 128 rows x 8 kv heads over
// 131072 keys, 4 bits: 105 us = 654 TFLOP/s, 1.44 TB/s; 512 rows x 8 kv heads over 32768 keys, 8
// bits: 98.9 us = 696 TFLOP/s.  Long calls are bound by the chain of hand-overs of a tile (a
// poll of a complete barrier takes 80-190 cycles, commit to wait 230) together with the issue
// slots: at 512 rows 61 % of the slots, tensor cores 56 % of the cycles, DRAM 10 %; a copy without any
// arithmetic in conversion and softmax still took 64-70 us.  What did not pay, at 512 rows (96 us then):
// 8 softmax warps (110), one lane polling for its warp (166), S and PV from two warps (113), one
// thread as MMA warp with its waits polled ahead (104), 128 keys per hand-over (104: a stream's
// next S then waits for its PV).  Few rows: repeated over the idle lanes of a tile, 8 rows over
// 32768 keys 38.7 (36.2 then; 37.5 now).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tcgen05.cuh"
#include "tree.cuh"

namespace m5 {

static __device__ int g_attn_tree_err = 0;

namespace atr {

constexpr int TK = 64;      // keys per tile
constexpr int ROWS = 128;   // MMA M
constexpr int SMX_WARPS = 16, DQ_WARPS = 4;  // conversion: DQ_WARPS for K and as many for V
constexpr int MMA_WARP = SMX_WARPS + 2 * DQ_WARPS, PROD_WARP = MMA_WARP + 1, PREP_WARP = MMA_WARP + 2;
constexpr int THREADS = (PREP_WARP + 2) * 32;
constexpr int EXPS = 32;    // tile exponents held: more than the tiles between conversion and softmax
constexpr uint32_t TMEM_COLS = 512, S_COL = 0, O_COL = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAZY = 8.f; // log2 growth of a row's maximum that is left in p
// Exponent of the largest value in fp16: of a bf16 row or tile, and of a packed
// tile.  Codes are used as fp16 subnormals (code * 2^-24, 4-bit: * 2^-20), an
// exact operand without a conversion; scale * 2^24 stays finite when the tile's values,
// hence 255 scales, stay below 2^-1.
constexpr int TOP16 = 7, TOPQ = -3;

// TWO: a CTA holds two blocks of 128 rows, one per softmax stream; else one
template <int BITS, int D, bool TWO>
struct Cfg {
  static constexpr int G = D / 64;                              // scale groups
  static constexpr int KROW = BITS ? D * BITS / 8 : 2 * D;      // bytes of a packed row
  static constexpr int SROW = BITS ? 2 * G : 0;                 // bytes of a row's scales
  static constexpr int SWIN = BITS ? TK * 2 * G + 32 : 0;       // a tile's scales with the 16-byte blocks around them
  static constexpr int K_OFF = 0, V_OFF = TK * KROW;
  static constexpr int S_OFF = 2 * TK * KROW;                   // K scales, K biases, V scales, V biases
  static constexpr int H_OFF = (S_OFF + 4 * SWIN + 15) / 16 * 16;                // fp16 (s, s), (b, b) per key and group, K then V
  static constexpr int STAGE = (H_OFF + (BITS ? 2 * TK * G * 8 : 0) + 127) / 128 * 128;
  static constexpr int OPER = TK * D * 2;                       // a converted tile
  static constexpr int NOP = TWO && BITS == 0 && D == 128 ? 2 : 3;  // converted K and V tiles held
  static constexpr int CW = BITS ? DQ_WARPS / 2 : DQ_WARPS;     // conversion warps per tile and operand
  static constexpr int BLOCKS = TWO ? 2 : 1;
  static constexpr int QBLOCK = ROWS * D * 2, QBYTES = BLOCKS * QBLOCK;
  // registers per thread after setmaxnreg: 4 + 2 + 1 warpgroups out of 896 x 72 at launch.  A spill
  // in the single warps costs most, it is on every tile's path.
  static constexpr int SMX_REGS = 80, DQ_REGS = BITS ? 56 : 64, MISC_REGS = BITS ? 72 : 56;
  static_assert(512 * SMX_REGS + 256 * DQ_REGS + 128 * MISC_REGS <= THREADS * 72, "register split");
  static constexpr int FIXED = QBYTES + 2 * NOP * OPER + 1024 + 1024;  // + alignment, barriers
  static constexpr int ST = (227 * 1024 - 6656 - FIXED) / STAGE < 8 ? (227 * 1024 - 6656 - FIXED) / STAGE : 8;
  static constexpr int SMEM = FIXED + ST * STAGE;
};

// Barriers, in the order of the array.
template <int ST, int NOP>
struct Bars {
  uint64_t full[ST], empty[ST], prep[ST];
  uint64_t kfull[NOP], kempty[NOP], vfull[NOP], vempty[NOP];
  // [stream][buffer].  P and PV need one per buffer too.  S of the next tile is there ahead, so a
  // warp may hand over that tile's P before its neighbours have handed over this one's; and a
  // stream may be two PVs ahead of the last finished one, which one phase bit cannot tell.
  uint64_t sfull[4], pfull[4], pvdone[4];
  uint64_t qready, idle;
  uint64_t dqmax[2];   // [K, V] bf16 caches: the conversion warps' maxima of a tile are in shared memory
  // Tree keys of a tile whose V holds a NaN or an infinity, a bit per key: P = 0 times it would be NaN for
  // queries that do not see it.  Packed caches [tile % EXPS]; bf16 [tile % 8][warp of V's four].  Read at
  // the run's end, for its last two tiles, when V's conversion is at most NOP tiles into the next run.
  unsigned long long broken[EXPS];
};
static_assert(EXPS == 8 * DQ_WARPS, "broken");

__device__ __forceinline__ uint32_t sw128(int n, int j) {
  return uint32_t((n >> 3) * 1024 + (n & 7) * 128 + ((j ^ (n & 7)) << 4));
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
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
// e with max / 2^e in [2^top, 2^(top + 1)), kept to exponents whose powers are finite
__device__ __forceinline__ int top_exp(float max, int top) {
  const int e = int(__float_as_uint(max) >> 23) - 127 - top;
  return ::min(120, ::max(-100, e));
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

template <int N>
__device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
// Bounded wait by one thread (M5_WAIT_LIMIT polls of up to ~2 us); a failure is shared by the CTA.
__device__ __forceinline__ bool wait1(uint64_t* bar, uint32_t par, volatile int* fail) {
#pragma unroll 1
  for (uint32_t i = 0; i < M5_WAIT_LIMIT; ++i) {
    if (mbar_try_wait(bar, par)) return true;
    if (*fail) return false;
  }
  *fail = 1;
  atomicExch(&g_attn_tree_err, M5_DEV_ERR_WAIT_TIMEOUT);
  return false;
}
// Waits by a warp, with one answer for all lanes.  A poll takes 80 cycles even when the phase is
// complete (110 with a suspend-time hint, 120 when one lane polls for the others), so what
// is needed together is polled together.
struct Ph {
  uint64_t* bar;
  uint32_t par;
};
__device__ __forceinline__ bool waitw(volatile int* fail, Ph a) {
  if (__all_sync(0xffffffffu, mbar_try_wait_fast(a.bar, a.par))) return true;
  return __all_sync(0xffffffffu, wait1(a.bar, a.par, fail));
}
__device__ __forceinline__ bool waitw(volatile int* fail, Ph a, Ph b) {
  const bool x = mbar_try_wait_fast(a.bar, a.par), y = mbar_try_wait_fast(b.bar, b.par);
  if (__all_sync(0xffffffffu, x && y)) return true;
  return __all_sync(0xffffffffu, wait1(a.bar, a.par, fail) && wait1(b.bar, b.par, fail));
}
__device__ __forceinline__ bool waitw(volatile int* fail, Ph a, Ph b, Ph c) {
  const bool x = mbar_try_wait_fast(a.bar, a.par), y = mbar_try_wait_fast(b.bar, b.par),
             z = mbar_try_wait_fast(c.bar, c.par);
  if (__all_sync(0xffffffffu, x && y && z)) return true;
  return __all_sync(0xffffffffu,
                    wait1(a.bar, a.par, fail) && wait1(b.bar, b.par, fail) && wait1(c.bar, c.par, fail));
}

// A slot of a ring of N buffers and the parity of its current use.
template <int N>
struct Slot {
  int i = 0;
  uint32_t par = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      par ^= 1;
    }
  }
};

// The line of tiles: sequences in order, each with `pairs` (kv head, row
// block) runs of tiles(b) tiles.  32-bit counts: the host refuses longer lines.
struct Line {
  int begin, end;  // this CTA's part
  int b, base, n;  // sequence of tile `begin`, that sequence's first tile and committed keys
};
__device__ __forceinline__ int seq_len(const TreeAttnArgs& a, int b) {
  return ::min(::max(a.lengths[b], 0), (int)a.capacity);
}
__device__ __forceinline__ int seq_end(const TreeAttnArgs& a, int n) { return ::min(n + a.T, (int)a.capacity); }
__device__ __forceinline__ int seq_tiles(const TreeAttnArgs& a, int b) {
  return (seq_end(a, seq_len(a, b)) + TK - 1) / TK;
}
// first tile of part c of `ctas`: floor(total * c / ctas), without a 64-bit division
__device__ __forceinline__ int part_of(int total, int ctas, int c) {
  const int q = total / ctas;
  return c * q + c * (total - q * ctas) / ctas;
}
// the part that holds tile t, from a rounded guess
__device__ __forceinline__ int part_with(int total, int ctas, int t) {
  int c = ::min(ctas - 1, (int)((float)t * (float)ctas / (float)total));
  while (part_of(total, ctas, c) > t) --c;
  while (c + 1 < ctas && part_of(total, ctas, c + 1) <= t) ++c;
  return c;
}
// parts of the line: down to one tile each (a CTA's second tile costs more than a part to join: one
// node over 512 keys 16.3 us with at least two tiles, 13.0 with one)
__device__ __forceinline__ int parts(int total, int ctas) { return ::min(ctas, total); }
// by one warp: this CTA's part of the line
__device__ __forceinline__ Line part_of_line(const TreeAttnArgs& a, int pairs, int lane, int c, int ctas) {
  Line l{0, 0, a.B - 1, 0, 0};
  // pass 0 adds up all tiles, pass 1 finds the sequence (one chunk of 32 sequences: from the registers)
  int total = 0, n = 0, w = 0, inc = 0;
  auto chunk = [&](int b0) {
    const int b = b0 + lane;
    n = b < a.B ? seq_len(a, b) : 0;
    w = b < a.B ? (seq_end(a, n) + TK - 1) / TK * pairs : 0;
    inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    return __shfl_sync(0xffffffffu, inc, 31);
  };
#pragma unroll 1
  for (int b0 = 0; b0 < a.B; b0 += 32) total += chunk(b0);
  const int np = parts(total, ctas);
  l.begin = c < np ? part_of(total, np, c) : total;
  l.end = c < np ? part_of(total, np, c + 1) : total;
#pragma unroll 1
  for (int b0 = 0, sum = 0; b0 < a.B; b0 += 32) {
    if (a.B > 32) chunk(b0);
    const unsigned m = __ballot_sync(0xffffffffu, l.begin >= sum + inc - w && l.begin < sum + inc);
    if (m) {
      const int src = __ffs(m) - 1;
      l.b = b0 + src;
      l.base = sum + __shfl_sync(0xffffffffu, inc - w, src);
      l.n = __shfl_sync(0xffffffffu, n, src);
      break;
    }
    sum += __shfl_sync(0xffffffffu, inc, 31);
  }
  return l;
}

// Walks a CTA's part run by run; every role holds one and steps it alike.
struct Walk {
  int at, end, base;
  int b, n, kend, tiles;        // sequence: committed keys, end of its keys, tiles
  int hk, rb, t0, nt, pair;     // run: kv head, row block, first tile, tiles of this part; pair = its number
  __device__ __forceinline__ Walk(const Line& l, const TreeAttnArgs& a)
      : at(l.begin), end(l.end), base(l.base), b(l.b), n(l.n) {
    kend = seq_end(a, n);
    tiles = (kend + TK - 1) / TK;
  }
  __device__ __forceinline__ bool next(const TreeAttnArgs& a, int nrb) {
    if (at >= end) return false;
    const int pairs = a.Hkv * nrb;
    if (at - base >= tiles * pairs) {
      base += tiles * pairs;
      ++b;
      n = seq_len(a, b);
      kend = seq_end(a, n);
      tiles = (kend + TK - 1) / TK;
    }
    const unsigned in = at - base, p = in / (unsigned)tiles;
    t0 = in - p * tiles;
    nt = ::min(tiles - t0, end - at);
    hk = nrb == 1 ? p : p / (unsigned)nrb;
    rb = p - hk * nrb;
    pair = b * pairs + p;
    at += nt;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return nt == tiles; }
};

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

// Does a query with this word see any key?
__device__ __forceinline__ bool sees_any(unsigned long long word, int n, int kend) {
  return n > 0 || visible(word, n, n, kend) != 0;
}

// fp16 (K, V): 8 consecutive dims of a row into one 16-byte chunk.
// 8-bit: byte c is the fp16 subnormal c * 2^-24; s (times 2^24) and b are exact
// (bf16 values), so code * s + b is rounded once.  An offset of the code folded into b
// instead would round b, which errs alike for all 64 dims of a group: 1 % of the
// output where the scores reach 50.
__device__ __forceinline__ uint4 conv8(uint2 w, uint32_t s, uint32_t b) {
  return make_uint4(hfma2(__byte_perm(w.x, 0u, 0x4140), s, b), hfma2(__byte_perm(w.x, 0u, 0x4342), s, b),
                    hfma2(__byte_perm(w.y, 0u, 0x4140), s, b), hfma2(__byte_perm(w.y, 0u, 0x4342), s, b));
}
// 4-bit: nibble c at bits 4-7 is c * 2^-20.  Position 2 i + h of the chunk is dim i + 4 h.
__device__ __forceinline__ uint4 conv4(uint32_t w, uint32_t s, uint32_t b) {
  constexpr uint32_t M = 0x00F000F0u;
  return make_uint4(hfma2((w << 4) & M, s, b), hfma2(w & M, s, b), hfma2((w >> 4) & M, s, b), hfma2((w >> 8) & M, s, b));
}
__device__ __forceinline__ uint4 conv16(uint4 w, float f) {
  return make_uint4(h2(bf16_lo(w.x) * f, bf16_hi(w.x) * f), h2(bf16_lo(w.y) * f, bf16_hi(w.y) * f),
                    h2(bf16_lo(w.z) * f, bf16_hi(w.z) * f), h2(bf16_lo(w.w) * f, bf16_hi(w.w) * f));
}


// O *= f over D dims of this thread's row.
template <int D>
__device__ __forceinline__ void scale_o(uint32_t o_addr, float f) {
#pragma unroll 1
  for (int d = 0; d < D; d += 16) {
    float o[16];
    tmem_ld16(o_addr + d, o);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] *= f;
    tmem_st16(o_addr + d, reinterpret_cast<const uint32_t(&)[16]>(o));
  }
}

// Meets the other warp of a row quarter; whether `p` holds for any of the 64 lanes.
__device__ __forceinline__ bool pair_or(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n barrier.cta.red.or.pred q, %1, 64, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(id), "r"(uint32_t(p))
      : "memory");
  return r != 0;
}

// State of one row in one stream, kept by both warps that share it.
struct Row {
  float m, l;  // maximum in log2 units (-inf: nothing seen); this warp's part of the sum of p
  int ev;      // O holds its sum divided by 2^ev
};

// One tile of a softmax thread: N of the tile's 64 keys, from `off` on, into the P
// columns of those keys.  pair: barrier of the two warps that share the
// rows, mine / other: where they exchange maxima.
// Returns the factor by which O has to change.
__device__ __forceinline__ float softmax_tile(Row& r, uint32_t s_addr, int off, float c, bool edge,
                                              unsigned long long vis, int pair, float* mine, const float* other) {
  constexpr int N = TK / 2;
  float s[N];
  tmem_ld32(s_addr + off, s);
  tmem_ld_wait();
  if (edge) {
    const uint32_t v = uint32_t(vis >> off);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!((v >> i) & 1)) s[i] = -INFINITY;
  }
  float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int i = 4; i < N; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) mx[j] = i + 4 + j < N ? max3(mx[j], s[i + j], s[i + 4 + j]) : fmaxf(mx[j], s[i + j]);
  }
  const float tmax = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
  float mt = tmax == -INFINITY ? -INFINITY : tmax * c, corr = 1.f;
  const bool up = mt > r.m + LAZY;  // also: the first score the row sees (r.m = -inf)
  // both warps have read their S here, so either's P may overwrite it
  if (pair_or(pair, up)) {
    *mine = mt;
    named_sync(pair, 64);
    mt = fmaxf(mt, *other);
    if (mt > r.m + LAZY) {
      corr = r.m == -INFINITY ? 0.f : ex2(r.m - mt);
      r.m = mt;
      r.l *= corr;
    }
  }
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
  __syncwarp();  // lanes whose maximum moved and those whose did not: the store is the whole warp's
  tmem_st16(s_addr + off / 2, p);
  return corr;
}

template <int BITS, int D, bool TWO>
__global__ void __launch_bounds__(THREADS, 1) tree_attn_kernel(const TreeAttnArgs a, const int nrb, float4* part_o,
                                                               float2* part_ml) {
  using C = Cfg<BITS, D, TWO>;
  constexpr int ST = C::ST, G = C::G, NOP = C::NOP;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = base;                         // [blocks][G][128 rows][128 bytes]
  uint8_t* kop = qs + C::QBYTES;              // [NOP][G][64 keys][128 bytes]
  uint8_t* vop = kop + NOP * C::OPER;
  uint8_t* ring = vop + NOP * C::OPER;
  Bars<ST, NOP>& bar = *reinterpret_cast<Bars<ST, NOP>*>(ring + ST * C::STAGE);
  static_assert(sizeof(Bars<ST, NOP>) <= 1024, "barriers");
  __shared__ float s_m[2][ROWS], s_xl[2][2][ROWS];  // at a run's end; s_xl [stream][half] also: maxima exchanged
  __shared__ int s_oev[2][ROWS];
  __shared__ uint32_t s_qmax[4][ROWS];
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
      mbar_init(&bar.empty[i], 2 * C::CW);
      mbar_init(&bar.prep[i], 1);
    }
    for (int i = 0; i < NOP; ++i) {
      mbar_init(&bar.kfull[i], C::CW);
      mbar_init(&bar.vfull[i], C::CW);
      mbar_init(&bar.kempty[i], 1);
      mbar_init(&bar.vempty[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bar.sfull[i], 1);
      mbar_init(&bar.pfull[i], SMX_WARPS / 2);
      mbar_init(&bar.pvdone[i], 1);
    }
    mbar_init(&bar.qready, SMX_WARPS);
    mbar_init(&bar.idle, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar.dqmax[i], DQ_WARPS);
    fence_mbar_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&s_tmem, TMEM_COLS);
    tmem_relinquish();
  }
  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    const Line l = part_of_line(a, a.Hkv * nrb, lane, blockIdx.x, gridDim.x);
    if (lane == 0) s_line = l;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const Line line = s_line;

  if (warp >= MMA_WARP) setmaxnreg_dec<C::MISC_REGS>();
  if (warp == PROD_WARP) {
    // ------------------------------------------------------------- producer
    // Lanes 0 and 1 copy the tile's K and V rows, lanes 2-5 the 16-byte blocks that hold its K
    // scales, K biases, V scales and V biases: each works out its own copy.
    constexpr int COPIES = BITS ? 6 : 2;
    const int op = lane < 2 ? lane : (lane - 2) >> 1;  // K, V
    const m5_kv_view& view = op ? a.v : a.k;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(lane < 2 ? view.data : (lane & 1) ? view.biases : view.scales);
    const int unit = lane < 2 ? C::KROW : C::SROW;     // bytes per key
    const int to = lane < 2 ? (op ? C::V_OFF : C::K_OFF) : C::S_OFF + (lane - 2) * C::SWIN;
    Walk w(line, a);
    Slot<ST> r;
    int issued = 0;
    bool ok = true;
    while (ok && w.next(a, nrb)) {
      int left = w.kend - w.t0 * TK;  // keys from the tile on
      const uint8_t* from = src + (w.b * view.batch_stride + w.hk * view.head_stride + w.t0 * TK) * unit;
#pragma unroll 1
      for (int t = 0; t < w.nt; ++t, from += TK * unit, left -= TK) {
        const uint32_t skew = lane < 2 ? 0u : uint32_t(reinterpret_cast<uintptr_t>(from)) & 15u;
        const uint32_t len = lane < COPIES ? (skew + min(TK, left) * unit + 15) & ~15u : 0u;  // rows are multiples of 16
        const uint32_t bytes = __reduce_add_sync(0xffffffffu, len);
        if (!(ok = waitw(fail, {&bar.empty[r.i], r.par ^ 1}))) break;
        if (lane == 0) mbar_arrive_expect_tx(&bar.full[r.i], bytes);
        __syncwarp();
        if (lane < COPIES) bulk_g2s(ring + r.i * C::STAGE + to, from - skew, len, &bar.full[r.i]);
        ++issued;
        r.next();
      }
    }
    // the copies in flight land before the CTA may exit: the last min(ST, issued) uses
    Slot<ST> f;
#pragma unroll 1
    for (int i = 0; i < issued; ++i, f.next())
      if (i >= issued - ST) (void)waitw(fail, {&bar.full[f.i], f.par});
  } else if (warp >= PREP_WARP) {
    // ---------------------------------------- scales: even tiles, odd tiles
    if constexpr (BITS != 0) {
      Walk w(line, a);
      Slot<ST> r;
      int g = 0;
      bool ok = true;
      constexpr float SUB = BITS == 8 ? 16777216.f : 1048576.f;  // codes are used as c / SUB
      using Pair = typename std::conditional<G == 2, uint32_t, uint16_t>::type;  // a key's scales (or biases)
      while (ok && w.next(a, nrb)) {
        const uint32_t kb = uint32_t(w.b * a.k.batch_stride + w.hk * a.k.head_stride);  // only its low bits matter
        const uint32_t vb = uint32_t(w.b * a.v.batch_stride + w.hk * a.v.head_stride);
#pragma unroll 1
        for (int t = 0; t < w.nt; ++t, ++g, r.next()) {
          if ((g & 1) != warp - PREP_WARP) continue;
          const int key0 = (w.t0 + t) * TK;
          unsigned long long vis = ~0ull;
          const bool edge = key0 + TK > w.n;
          if (edge) vis = visible(seen_by_any(a, w.b, lane), key0, w.n, w.kend);
          if (!(ok = waitw(fail, {&bar.full[r.i], r.par}))) break;
          uint8_t* sb = ring + r.i * C::STAGE;
          // keys lane and lane + 32: [K, V][key][group]
          float s[2][2][G], b[2][2][G];
          uint32_t mx[2];
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const m5_kv_view& view = o ? a.v : a.k;
            const uint32_t at = ((o ? vb : kb) + key0) * C::SROW;
            const uint8_t* sp = sb + C::S_OFF + 2 * o * C::SWIN + ((uint32_t(reinterpret_cast<uintptr_t>(view.scales)) + at) & 15);
            const uint8_t* bp = sb + C::S_OFF + (2 * o + 1) * C::SWIN + ((uint32_t(reinterpret_cast<uintptr_t>(view.biases)) + at) & 15);
            float m = 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t sw = reinterpret_cast<const Pair*>(sp)[lane + 32 * k], bw = reinterpret_cast<const Pair*>(bp)[lane + 32 * k];
              if (edge && !((vis >> (lane + 32 * k)) & 1)) sw = bw = 0;
#pragma unroll
              for (int q = 0; q < G; ++q) {
                s[o][k][q] = q ? bf16_hi(sw) : bf16_lo(sw);
                b[o][k][q] = q ? bf16_hi(bw) : bf16_lo(bw);
                m = max3(m, fabsf(b[o][k][q]), fabsf(fmaf(s[o][k][q], float((1 << BITS) - 1), b[o][k][q])));
              }
            }
            mx[o] = __float_as_uint(m);
          }
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            mx[o] = __reduce_max_sync(0xffffffffu, mx[o]);
            if (mx[o] == 0x7F800000u) {  // an infinity is what it is under any exponent: once more without it (NaN never counts)
              float m = 0.f;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int q = 0; q < G; ++q) {
                  const float z = fmaxf(fabsf(b[o][k][q]), fabsf(fmaf(s[o][k][q], float((1 << BITS) - 1), b[o][k][q])));
                  m = fmaxf(m, z < INFINITY ? z : 0.f);
                }
              }
              mx[o] = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
            }
          }
          if (edge) {  // broken V of tree keys: zeroed, the queries that see it are told
            unsigned long long br = 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              bool x = false;
#pragma unroll
              for (int q = 0; q < G; ++q)
                x = x || !(fabsf(fmaf(s[1][k][q], float((1 << BITS) - 1), b[1][k][q])) < INFINITY);
              x = x && key0 + lane + 32 * k >= w.n;
#pragma unroll
              for (int q = 0; q < G; ++q) {
                if (x) s[1][k][q] = b[1][k][q] = 0.f;
              }
              br |= (unsigned long long)__ballot_sync(0xffffffffu, x) << (32 * k);
            }
            if (lane == 0) bar.broken[g & (EXPS - 1)] = br;
          }
          const int ek = top_exp(__uint_as_float(mx[0]), TOPQ);
          int ev = top_exp(__uint_as_float(mx[1]), TOPQ);
          // V's exponent runs on within a stream: the tile before it (TWO: settled by the other warp)
          if (t >= (TWO ? 1 : 2)) {
            if constexpr (TWO) {
              static_assert(ST > 2, "the other warp is at most one tile ahead: the stage before is not in use again");
              const int pi = r.i ? r.i - 1 : ST - 1;
              if (!(ok = waitw(fail, {&bar.prep[pi], r.i ? r.par : r.par ^ 1}))) break;
            }
            ev = max(ev, s_ev[(g - (TWO ? 1 : 2)) & (EXPS - 1)]);
          }
          if (lane == 0) {
            s_kmul[g & (EXPS - 1)] = pow2(ek);
            s_ev[g & (EXPS - 1)] = ev;
          }
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const float f = pow2(-(o ? ev : ek)), fs = f * SUB;
            uint8_t* dst = sb + C::H_OFF + o * TK * G * 8;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t v[2 * G];
#pragma unroll
              for (int q = 0; q < G; ++q) {
                const float x = s[o][k][q] * fs, y = b[o][k][q] * f;
                v[2 * q] = h2(x, x);
                v[2 * q + 1] = h2(y, y);
              }
              if constexpr (G == 2) reinterpret_cast<uint4*>(dst)[lane + 32 * k] = make_uint4(v[0], v[1], v[2], v[3]);
              else reinterpret_cast<uint2*>(dst)[lane + 32 * k] = make_uint2(v[0], v[1]);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.prep[r.i]);
        }
      }
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------- MMA issuer
    // the whole warp walks and waits, one elected lane issues
    constexpr uint32_t id_s = idesc(TK, false), id_o = idesc(D, true);
    const bool issuer = elect_one();
    const uint64_t q_desc = sdesc(smem_addr(qs), 16), k_desc = sdesc(smem_addr(kop), 16),
                   v_desc = sdesc(smem_addr(vop), TK * 128);
    // Tiles go to the streams in turn, or (TWO) each to both: u counts a stream's tiles.  S runs
    // ahead of PV so that a softmax warp finds its next S in place when it has handed over P,
    // and each PV is followed by an S that waits for nothing recent:
    //   one block   PV(t), S(t + 3)                            (tiles t, t + 3 of different streams)
    //   TWO         PV_0(t), S_1(t + 1), PV_1(t), S_0(t + 2)
    Walk w(line, a);
    auto s_mma = [&](int j, int u, int slot, bool last_use) {
      if (issuer) {
        const uint32_t d = tmem + S_COL + 64u * (2 * j + (u & 1));
        const uint64_t qd = q_desc + (TWO ? j * (C::QBLOCK / 16) : 0), kd = k_desc + uint32_t(slot * (C::OPER / 16));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc_mma_ss(d, qd + (kk / 4) * (ROWS * 128 / 16) + 2 * (kk % 4),
                    kd + (kk / 4) * (TK * 128 / 16) + 2 * (kk % 4), id_s, kk > 0 ? 1u : 0u);
        tc_commit(&bar.sfull[2 * j + (u & 1)]);
        if (last_use) tc_commit(&bar.kempty[slot]);
      }
      __syncwarp();
    };
    auto pv_mma = [&](int j, int u, int slot, bool first, bool last_use) {
      if (issuer) {
        const uint32_t d = tmem + O_COL + 128u * j, p = tmem + S_COL + 64u * (2 * j + (u & 1));
        const uint64_t vd = v_desc + uint32_t(slot * (C::OPER / 16));
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk)
          tc_mma_ts(d, p + 8u * kk, vd + kk * (2048 / 16), id_o, (kk > 0 || !first) ? 1u : 0u);
        tc_commit(&bar.pvdone[2 * j + (u & 1)]);
        if (last_use) tc_commit(&bar.vempty[slot]);
      }
      __syncwarp();
    };
    // the phase of PV(u - 2), whose P sits in the buffer S(u) goes to (u < 2: complete at once)
    auto free_s = [&](int j, int u) { return Ph{&bar.pvdone[2 * j + (u & 1)], uint32_t((u >> 1) + 1) & 1}; };
    auto p_of = [&](int j, int u) { return Ph{&bar.pfull[2 * j + (u & 1)], uint32_t(u >> 1) & 1}; };
    Slot<NOP> ks, k1, vs;  // next K (TWO: of stream 0, of stream 1), next V
    int g0 = 0;            // tiles before the run
    uint32_t seg = 0;
    bool ok = true;
    while (ok && w.next(a, nrb)) {
      ok = waitw(fail, {&bar.qready, seg & 1});
      ++seg;
      constexpr int AHEAD = TWO ? 2 : 3;
#pragma unroll 1
      for (int t = -AHEAD; t < w.nt && ok; ++t) {
        const int g = g0 + t;
        if constexpr (TWO) {
          if (t >= 0) {
            if (!(ok = waitw(fail, {&bar.vfull[vs.i], vs.par}, p_of(0, g)))) break;
            tc_fence_after();
            pv_mma(0, g, vs.i, t == 0, false);
          }
          if (t >= -1 && t + 1 < w.nt) {  // its K is there: S_0(t + 1) has used it
            if (!(ok = waitw(fail, free_s(1, g + 1)))) break;
            tc_fence_after();
            s_mma(1, g + 1, k1.i, true);
            k1.next();
          }
          if (t >= 0) {
            if (!(ok = waitw(fail, p_of(1, g)))) break;
            tc_fence_after();
            pv_mma(1, g, vs.i, t == 0, true);
            vs.next();
          }
          if (t + 2 < w.nt) {
            if (!(ok = waitw(fail, {&bar.kfull[ks.i], ks.par}, free_s(0, g + 2)))) break;
            tc_fence_after();
            s_mma(0, g + 2, ks.i, false);
            ks.next();
          }
        } else {
          if (t >= 0) {
            if (!(ok = waitw(fail, {&bar.vfull[vs.i], vs.par}, p_of(g & 1, g >> 1)))) break;
            tc_fence_after();
            pv_mma(g & 1, g >> 1, vs.i, t < 2, true);
            vs.next();
          }
          if (t + 3 < w.nt) {
            if (!(ok = waitw(fail, {&bar.kfull[ks.i], ks.par}, free_s((g + 3) & 1, (g + 3) >> 1)))) break;
            tc_fence_after();
            s_mma((g + 3) & 1, (g + 3) >> 1, ks.i, true);
            ks.next();
          }
        }
      }
      g0 += w.nt;
    }
    // every MMA issued has completed before TMEM may be freed
    if (issuer) tc_commit(&bar.idle);
    __syncwarp();
    (void)waitw(fail, {&bar.idle, 0});
  } else if (warp >= SMX_WARPS && warp < MMA_WARP) {
    // ------------------------------------------------------------ conversion
    // A thread takes dims 16 c .. 16 c + 15 of every KSTEP-th key of a tile.  The 8
    // lanes of a shared-memory phase must read 8 different 16-byte columns and
    // write 8 different (chunk ^ key & 7): with two groups they hold the pieces 0-3 of
    // one key and 4-7 of its neighbour (8/4-bit rows), or all pieces of
    // one key with the halves of 4-7 in the other order (bf16 rows of 256 bytes).
    setmaxnreg_dec<C::DQ_REGS>();
    const int o = warp >= SMX_WARPS + DQ_WARPS;  // K, V
    // Packed caches: two warps convert the even tiles of an operand and two the odd ones (a tile's
    // chain of waits, loads, stores and fence is latency, which two tiles at once hide).
    // bf16 caches: all four every tile (they take its maximum first, and V's runs on).
    const int turn = (warp - SMX_WARPS) % DQ_WARPS / C::CW;
    const int d = (tid - SMX_WARPS * 32) % (C::CW * 32);
    constexpr int PIECES = D / 16, KSTEP = C::CW * 32 / PIECES, PER = TK / KSTEP;
    const int c = d % PIECES;
    const int key = G == 2 && BITS != 0 ? 2 * (d >> 4) + (((d >> 2) ^ (d >> 3)) & 1) : d / PIECES;
    const int swap = G == 2 && BITS == 0 ? c >> 2 : 0;  // order of the two 8-dim chunks
    uint32_t to[2];  // where they go; key & 7 is the same for all of a thread's keys
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int ch = 2 * c + (hh ^ swap);
      to[hh] = (ch >> 3) * (TK * 128) + sw128(key, ch & 7);
    }
    static_assert(KSTEP % 8 == 0, "a thread's keys share key & 7");
    uint64_t* const fullb = o ? bar.vfull : bar.kfull;
    uint64_t* const emptyb = o ? bar.vempty : bar.kempty;
    uint8_t* const oper = o ? vop : kop;
    const uint32_t from0 = (o ? C::V_OFF : C::K_OFF) + key * C::KROW + c * (BITS ? 2 * BITS : 32);
    Walk w(line, a);
    Slot<ST> r;
    Slot<NOP> q;
    int g = 0;
    bool ok = true;
    while (ok && w.next(a, nrb)) {
      int ev0 = -127, ev1 = -127;
#pragma unroll 1
      for (int t = 0; t < w.nt; ++t, ++g, r.next(), q.next()) {
        if (BITS != 0 && (g & 1) != turn) continue;
        const uint8_t* sb = ring + r.i * C::STAGE;
        const uint8_t* src = sb + from0;
        uint8_t* dst = oper + q.i * C::OPER;
        if constexpr (BITS == 0) {
          const int key0 = (w.t0 + t) * TK;
          unsigned long long vis = ~0ull;
          const bool edge = key0 + TK > w.n;
          if (edge) vis = visible(seen_by_any(a, w.b, lane), key0, w.n, w.kend) >> key;
          else vis >>= key;
          if (!(ok = waitw(fail, {&bar.full[r.i], r.par}))) break;
          uint4 x[PER][2];
          uint32_t mx = 0;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint4 y = ((vis >> (i * KSTEP)) & 1)
                                  ? *reinterpret_cast<const uint4*>(src + i * (KSTEP * C::KROW) + 16 * (hh ^ swap))
                                  : make_uint4(0, 0, 0, 0);
              x[i][hh] = y;
              mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(y.x & 0x7FFF7FFFu, y.y & 0x7FFF7FFFu),
                                         __vmaxu2(y.z & 0x7FFF7FFFu, y.w & 0x7FFF7FFFu)));
            }
          }
          mx = __reduce_max_sync(0xffffffffu, max(mx & 0xFFFFu, mx >> 16));
          uint32_t brk = 0;  // a bit per key of this thread
          if (mx >= 0x7F80u) {  // NaN and infinities are what they are under any exponent: once more without them
            mx = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              uint32_t y[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
              uint32_t any = 0, top = 0;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                y[k] &= 0x7FFF7FFFu;
                const uint32_t no = __vcmpgeu2(y[k], 0x7F807F80u);
                any |= no;
                top = __vmaxu2(top, y[k] & ~no);
              }
              // broken V of a tree key: zeroed, the queries that see it are told
              const uint32_t row = __ballot_sync(0xffffffffu, any != 0) >> (lane & ~(PIECES - 1));
              if (o && (row & ((1u << PIECES) - 1)) && key0 + key + i * KSTEP >= w.n) {
                x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
                brk |= 1u << i;
                top = 0;
              }
              mx = __vmaxu2(mx, top);
            }
            mx = __reduce_max_sync(0xffffffffu, max(mx & 0xFFFFu, mx >> 16));
          }
          if (lane == 0) {
            s_dqmax[g & 1][o][warp & (DQ_WARPS - 1)] = __uint_as_float(mx << 16);
            mbar_arrive(&bar.dqmax[o]);
            mbar_arrive(&bar.empty[r.i]);
          }
          if (!(ok = waitw(fail, {&bar.dqmax[o], uint32_t(g & 1)}))) break;
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < DQ_WARPS; ++i) m = fmaxf(m, s_dqmax[g & 1][o][i]);
          int e = top_exp(m, TOP16);
          if (o) {
            e = max(ev0, e);
            ev0 = TWO ? e : ev1;
            ev1 = e;
          }
          if (d == 0) {
            if (o) s_ev[g & (EXPS - 1)] = e;
            else s_kmul[g & (EXPS - 1)] = pow2(e);
          }
          const float f = pow2(-e);
          if (!(ok = waitw(fail, {&emptyb[q.i], q.par ^ 1}))) break;
          if (edge && o) {
            unsigned long long br = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) br |= (unsigned long long)((brk >> i) & 1) << (key + i * KSTEP);
            const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)br), hi = __reduce_or_sync(0xffffffffu, (uint32_t)(br >> 32));
            if (lane == 0) bar.broken[(g & 7) * DQ_WARPS + (warp & (DQ_WARPS - 1))] = ((unsigned long long)hi << 32) | lo;
          }
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            *reinterpret_cast<uint4*>(dst + to[0] + i * (KSTEP * 128)) = conv16(x[i][0], f);
            *reinterpret_cast<uint4*>(dst + to[1] + i * (KSTEP * 128)) = conv16(x[i][1], f);
          }
        } else {
          if (!(ok = waitw(fail, {&bar.prep[r.i], r.par}, {&bar.full[r.i], r.par}, {&emptyb[q.i], q.par ^ 1}))) break;
          const uint2* sc = reinterpret_cast<const uint2*>(sb + C::H_OFF + o * TK * G * 8) + key * G + (G == 2 ? c >> 2 : 0);
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const uint2 f = sc[i * KSTEP * G];
            uint4 v[2];
            if constexpr (BITS == 8) {
              const uint4 y = *reinterpret_cast<const uint4*>(src + i * (KSTEP * C::KROW));
              v[0] = conv8(make_uint2(y.x, y.y), f.x, f.y);
              v[1] = conv8(make_uint2(y.z, y.w), f.x, f.y);
            } else {
              const uint2 y = *reinterpret_cast<const uint2*>(src + i * (KSTEP * C::KROW));
              v[0] = conv4(y.x, f.x, f.y);
              v[1] = conv4(y.y, f.x, f.y);
            }
            *reinterpret_cast<uint4*>(dst + to[0] + i * (KSTEP * 128)) = v[0];
            *reinterpret_cast<uint4*>(dst + to[1] + i * (KSTEP * 128)) = v[1];
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&fullb[q.i]);
          if (BITS != 0) mbar_arrive(&bar.empty[r.i]);
        }
      }
    }
  } else if (warp < SMX_WARPS) {
    // ---------------------------------------------------------------- softmax
    setmaxnreg_inc<C::SMX_REGS>();
    const int j = warp >> 3, h = (warp >> 2) & 1, r = tid & 127;  // stream, half of the keys, lane of tensor memory
    const uint32_t lrow = uint32_t(32 * (warp & 3)) << 16;
    constexpr int QPARTS = TWO ? 2 : 4;           // warps that share a row: of its stream, of both
    const int qp = TWO ? h : 2 * j + h;
    const int pair_id = 2 + 4 * j + (warp & 3);   // barriers 2-9
    Walk w(line, a);
    int g0 = 0;
    bool ok = true;
    while (ok && w.next(a, nrb)) {
      const int row0 = (w.rb * C::BLOCKS + (TWO ? j : 0)) * ROWS, nrows = max(0, min(ROWS, R - row0));
      const bool row_ok = r < nrows, idle = r - lane >= nrows;  // idle: the whole warp has no row
      const int row = row_ok ? row0 + r : 0, qi = row / grp, hq = w.hk * grp + row % grp;
      const unsigned long long word = a.anc[w.b * a.anc_sb + qi];
      // Q, scaled by a power of two per row; the sign of `scale` goes with it
      float c_row;
      {
        constexpr int NQ = D / 8 / QPARTS;  // chunks of 8 dims per warp
        const uint4* qr = reinterpret_cast<const uint4*>(a.q + w.b * a.q_sb + hq * a.q_sh + qi * a.q_sl) + qp * NQ;
        uint4 x[NQ];
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < NQ; ++i) x[i] = row_ok ? qr[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu),
                                     __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu)));
        // the largest exponent of the whole row
        s_qmax[2 * j + h][r] = mx;
        __syncwarp();
        named_sync(1, SMX_WARPS * 32);
#pragma unroll
        for (int i = 0; i < QPARTS; ++i) mx = __vmaxu2(mx, s_qmax[TWO ? 2 * j + i : i][r]);
        const int eq = top_exp(__uint_as_float(max(mx & 0xFFFFu, mx >> 16) << 16), TOP16);
        const float f = a.scale < 0.f ? -pow2(-eq) : pow2(-eq);
        c_row = fabsf(a.scale) * LOG2E * pow2(eq);
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          const int ch = qp * NQ + i;
          uint4 o = conv16(x[i], f);
          if constexpr (BITS == 4)  // positions 2 i + h hold dims i + 4 h, as the codes come
            o = make_uint4(__byte_perm(o.x, o.z, 0x5410), __byte_perm(o.x, o.z, 0x7632), __byte_perm(o.y, o.w, 0x5410),
                           __byte_perm(o.y, o.w, 0x7632));
          *reinterpret_cast<uint4*>(qs + (TWO ? j * C::QBLOCK : 0) + (ch >> 3) * (ROWS * 128) + sw128(r, ch & 7)) = o;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.qready);
      }
      Row st{-INFINITY, 0.f, 0};
      int last = -1;  // this stream's last tile
      // After a wait that ran out the loop goes on without waiting: the warps of a pair meet in every tile.
#pragma unroll 1
      for (int g = TWO ? g0 : g0 + ((g0 & 1) ^ j); g < g0 + w.nt; g += TWO ? 1 : 2) {
        const int u = TWO ? g : g >> 1, buf = 2 * j + (u & 1), key0 = (w.t0 + g - g0) * TK;
        ok = ok && waitw(fail, {&bar.sfull[buf], uint32_t(u >> 1) & 1});
        if (!idle) {
          tc_fence_after();
          const bool edge = key0 + TK > w.n;
          const unsigned long long vis = edge ? visible(word, key0, w.n, w.kend) : 0ull;
          // Above 0, for a hidden score is -inf and times 0 NaN: rows and tiles of zeros (exponents of -100 both)
          // come to 1e-61, and so does a scale of 0.  S is below 2^23 here, times 1e-37 it is nothing.
          float c = c_row * s_kmul[g & (EXPS - 1)];
          if (c < 1e-37f) c = 1e-37f;  // (a NaN stays)
          const uint32_t sa = tmem + lrow + S_COL + 64u * buf;
          float corr = softmax_tile(st, sa, 32 * h, c, edge, vis, pair_id, &s_xl[j][h][r], &s_xl[j][h ^ 1][r]);
          // V's exponent in this stream; for bf16 caches it is there once the tile's V is (whose
          // buffer cannot be refilled before this P is used: its phase stands still)
          if (BITS == 0) ok = ok && waitw(fail, {&bar.vfull[g % NOP], uint32_t(g / NOP) & 1});
          const int ev = s_ev[g & (EXPS - 1)];
          if (last >= 0) {
            if (ev != st.ev) corr *= pow2(max(st.ev - ev, -126));
            if (__any_sync(0xffffffffu, corr != 1.f)) {  // the same for both warps: each takes half of the dims
              ok = ok && waitw(fail, {&bar.pvdone[buf ^ 1], uint32_t((u - 1) >> 1) & 1});
              tc_fence_after();
              scale_o<D / 2>(tmem + lrow + O_COL + 128u * j + h * (D / 2), corr);
            }
          }
          st.ev = ev;
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.pfull[buf]);
        last = u;
      }
      // ---- end of the run: both streams' O are complete
      if (ok && last >= 0) ok = waitw(fail, {&bar.pvdone[2 * j + (last & 1)], uint32_t(last >> 1) & 1});
      s_xl[j][h][r] = idle ? 0.f : st.l;
      if (h == 0) {
        s_m[j][r] = st.m;
        s_oev[j][r] = st.ev;
      }
      tc_fence_before();
      named_sync(1, SMX_WARPS * 32);
      tc_fence_after();
      if (tid == 0) s_stop = *fail;
      __syncwarp();  // the loads of tensor memory below are the whole warp's
      if (ok && r - lane < nrows) {
        // the two streams' states of the row, joined; TWO: the stream's own
        const int j0 = TWO ? j : 0;
        const float mx = s_m[j0][r], my = TWO ? -INFINITY : s_m[1][r], M = fmaxf(mx, my);
        const float wx = mx == -INFINITY ? 0.f : ex2(mx - M), wy = my == -INFINITY ? 0.f : ex2(my - M);
        float l = (s_xl[j0][0][r] + s_xl[j0][1][r]) * wx;
        if constexpr (!TWO) l += (s_xl[1][0][r] + s_xl[1][1][r]) * wy;
        // the tiles with tree keys, two at most: a query that sees a broken value has no number
        for (int t = ::max(0, w.n / TK - w.t0); t < w.nt; ++t) {
          const int g = g0 + t;
          unsigned long long br = 0;
#pragma unroll
          for (int i = 0; i < (BITS ? 1 : DQ_WARPS); ++i) br |= bar.broken[BITS ? g & (EXPS - 1) : (g & 7) * DQ_WARPS + i];
          if (br && (br & visible(a.anc[w.b * a.anc_sb + qi], (w.t0 + t) * TK, w.n, w.kend))) l = NAN;
        }
        const bool direct = w.whole();
        // no weight: the row sees no key (0), or its scores are all -inf (0 / 0)
        if (direct && l == 0.f && sees_any(a.anc[w.b * a.anc_sb + qi], w.n, w.kend)) l = NAN;
        const float inv = direct ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
        // a stream without a finite score has no O to add, but its NaN counts
        const bool ux = wx > 0.f || l != l, uy = !TWO && (wy > 0.f || l != l);
        const float fx = wx * pow2(s_oev[j0][r]) * inv, fy = TWO ? 0.f : wy * pow2(s_oev[1][r]) * inv;
        const size_t slot = size_t(blockIdx.x + w.pair) * C::BLOCKS + (TWO ? j : 0);
        bf16* out = a.out + w.b * a.o_sb + hq * a.o_sh + qi * a.o_sl;
#pragma unroll 1
        for (int d0 = qp * (D / QPARTS); d0 < (qp + 1) * (D / QPARTS); d0 += 16) {
          float o0[16], o1[16];
          tmem_ld16(tmem + lrow + O_COL + 128u * j0 + d0, o0);
          if constexpr (!TWO) tmem_ld16(tmem + lrow + O_COL + 128u + d0, o1);
          tmem_ld_wait();
          float o[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int dim = BITS == 4 ? (k & 8) + ((k & 7) >> 1) + 4 * (k & 1) : k;
            o[dim] = (ux ? o0[k] * fx : 0.f) + (uy ? o1[k] * fy : 0.f);
          }
          if (row_ok && direct) {
            uint4 v[2];
            uint32_t* p = reinterpret_cast<uint32_t*>(v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const __nv_bfloat162 z = __floats2bfloat162_rn(o[2 * k], o[2 * k + 1]);
              p[k] = *reinterpret_cast<const uint32_t*>(&z);
            }
            reinterpret_cast<uint4*>(out + d0)[0] = v[0];
            reinterpret_cast<uint4*>(out + d0)[1] = v[1];
          } else if (row_ok) {
            float4* po = part_o + (slot * (D / 4) + d0 / 4) * ROWS + r;  // [slot][dim / 4][row]: rows side by side
#pragma unroll
            for (int k = 0; k < 4; ++k) po[k * ROWS] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
          __syncwarp();  // lanes without a row meet the others before the next load
        }
        if (!direct && row_ok && qp == 0) part_ml[slot * ROWS + r] = make_float2(M, l);
      }
      __syncwarp();
      tc_fence_before();
      named_sync(1, SMX_WARPS * 32);  // O and Q may be overwritten
      tc_fence_after();
      ok = !s_stop;  // one answer for all warps: they meet at the barriers of the next run or leave together
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

// Joins the partial states of the rows whose run was cut:
//   o = sum_i w_i O_i / sum_i w_i l_i,  w_i = 2^(m_i - max).
// A part without a finite score has m = -inf and counts for nothing, but for a sum of NaN.
// One CTA per block of 128 rows and 8 dims; a thread takes one row of every
// fourth part (the parts of a run are consecutive CTAs), so all loads run along
// the rows and a run of 40 parts is three rounds of loads (the idle lanes of 32 rows or
// fewer as 16 ways: no faster).  The four quarters of a row's parts meet in shared memory.
constexpr int JOIN_DIMS = 8, JOIN_WAYS = 4;
__global__ void __launch_bounds__(JOIN_WAYS * ROWS) tree_join_kernel(const TreeAttnArgs a, const int nrb, const int blocks,
                                                                     const int ctas, const float4* part_o,
                                                                     const float2* part_ml) {
  __shared__ float s_m[JOIN_WAYS][ROWS], s_l[JOIN_WAYS][ROWS], s_o[JOIN_WAYS][ROWS][JOIN_DIMS + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, r = tid & (ROWS - 1), way = tid / ROWS;
  const int grp = a.Hq / a.Hkv, R = a.L * grp, pairs = a.Hkv * nrb;
  int x = blockIdx.x;
  const int blk = x % blocks;
  x /= blocks;
  const int p = x % pairs, b = x / pairs;
  const int row0 = (p % nrb * blocks + blk) * ROWS, nrows = min(ROWS, R - row0);
  if (nrows <= 0) return;
  int total = 0, base = 0;  // tiles of all sequences, and of those before b
  for (int i = lane; i < a.B; i += 32) {
    const int t = seq_tiles(a, i) * pairs;
    total += t;
    if (i < b) base += t;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  base = __reduce_add_sync(0xffffffffu, base);
  const int tiles = seq_tiles(a, b), np = parts(total, ctas);
  const int t0 = base + p * tiles, t1 = t0 + tiles - 1;
  const int c0 = part_with(total, np, t0), c1 = part_with(total, np, t1);
  if (c0 == c1) return;  // written by the attention kernel
  const int n = c1 - c0 + 1, d4 = blockIdx.y * (JOIN_DIMS / 4), D4 = a.D / 4;
  const size_t slot0 = size_t(c0 + b * pairs + p) * blocks + blk;
  const float2* ml = part_ml + slot0 * ROWS + r;
  const float4* po = part_o + (slot0 * D4 + d4) * ROWS + r;
  float m = -INFINITY, l = 0.f;
  float4 o[JOIN_DIMS / 4];
#pragma unroll
  for (int k = 0; k < JOIN_DIMS / 4; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (r < nrows) {
#pragma unroll 4
    for (int i = way; i < n; i += JOIN_WAYS) m = fmaxf(m, ml[size_t(i) * blocks * ROWS].x);
#pragma unroll 4
    for (int i = way; i < n; i += JOIN_WAYS) {
      const float2 e = ml[size_t(i) * blocks * ROWS];
      const float w = e.x == -INFINITY ? 0.f : ex2(e.x - m);
      l = fmaf(w, e.y, l);
#pragma unroll
      for (int k = 0; k < JOIN_DIMS / 4; ++k) {
        const float4 v = po[(size_t(i) * blocks * D4 + k) * ROWS];
        o[k].x = fmaf(w, v.x, o[k].x);
        o[k].y = fmaf(w, v.y, o[k].y);
        o[k].z = fmaf(w, v.z, o[k].z);
        o[k].w = fmaf(w, v.w, o[k].w);
      }
    }
  }
  s_m[way][r] = m;
  s_l[way][r] = l;
#pragma unroll
  for (int k = 0; k < JOIN_DIMS / 4; ++k) {
    s_o[way][r][4 * k] = o[k].x;
    s_o[way][r][4 * k + 1] = o[k].y;
    s_o[way][r][4 * k + 2] = o[k].z;
    s_o[way][r][4 * k + 3] = o[k].w;
  }
  __syncthreads();
  if (tid >= nrows) return;  // a thread per row from here on
  float M = -INFINITY;
#pragma unroll
  for (int y = 0; y < JOIN_WAYS; ++y) M = fmaxf(M, s_m[y][tid]);
  float den = 0.f, num[JOIN_DIMS];
#pragma unroll
  for (int k = 0; k < JOIN_DIMS; ++k) num[k] = 0.f;
#pragma unroll
  for (int y = 0; y < JOIN_WAYS; ++y) {
    const float w = s_m[y][tid] == -INFINITY ? 0.f : ex2(s_m[y][tid] - M);
    den = fmaf(w, s_l[y][tid], den);
#pragma unroll
    for (int k = 0; k < JOIN_DIMS; ++k) num[k] = fmaf(w, s_o[y][tid][k], num[k]);
  }
  const int row = row0 + tid, qi = row / grp, h = p / nrb * grp + row % grp;
  float inv = 1.f / den;
  if (den == 0.f) {  // as at the end of a run that was not cut
    const int sn = seq_len(a, b);
    inv = sees_any(a.anc[b * a.anc_sb + qi], sn, seq_end(a, sn)) ? NAN : 0.f;
  }
  uint32_t v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 z = __floats2bfloat162_rn(num[2 * k] * inv, num[2 * k + 1] * inv);
    v[k] = *reinterpret_cast<const uint32_t*>(&z);
  }
  *reinterpret_cast<uint4*>(a.out + b * a.o_sb + h * a.o_sh + qi * a.o_sl + 4 * d4) = make_uint4(v[0], v[1], v[2], v[3]);
}

// Launch that may begin while the kernel before it on the stream ends (both
// kernels wait for it before they read or write anything in global memory).
template <typename... KArgs, typename... Args>
static cudaError_t launch_early(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

struct Plan {
  int nrb, blocks, ctas;  // runs per kv head, row blocks of a run
  size_t slots;
};
static Plan plan(int B, int Hq, int Hkv, int L) {
  const long long rows = (long long)L * (Hq / Hkv);
  // Two blocks of rows per converted tile (one: two parts convert each tile) from 129 rows on, over
  // 32768 keys: 256 rows 61.8 us (one: 65.9), 512 rows 98.9 (118.4), bf16 127.4 (184.8); 128 rows
  // 51.3 (one: 43.9), the second stream idle.  Over 600 keys one would do: 256 rows 19.4 (16.0), 512
  // 26.1 (26.2); of the lengths only the capacity is known here, which a loop reserves ahead of them.
  const int blocks = rows > ROWS ? 2 : 1, nrb = ceil_div(rows, ROWS * blocks), ctas = sm_count();
  return {nrb, blocks, ctas, (size_t(ctas) + size_t(B) * Hkv * nrb) * blocks};
}

template <int BITS, int D, bool TWO>
static cudaError_t launch(const TreeAttnArgs& a, const Plan& p, cudaStream_t st) {
  using C = Cfg<BITS, D, TWO>;
  static DeviceOnce once;
  cudaError_t e = once.run([&] {
    return cudaFuncSetAttribute(tree_attn_kernel<BITS, D, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (e != cudaSuccess) return e;
  float4* po = reinterpret_cast<float4*>(a.ws);
  float2* ml = reinterpret_cast<float2*>(po + p.slots * ROWS * (D / 4));
  if ((e = launch_early(tree_attn_kernel<BITS, D, TWO>, dim3(p.ctas), dim3(THREADS), C::SMEM, st, a, p.nrb, po, ml)))
    return e;
  return launch_early(tree_join_kernel, dim3(a.B * a.Hkv * p.nrb * p.blocks, D / JOIN_DIMS), dim3(JOIN_WAYS * ROWS), 0, st, a,
                      p.nrb, p.blocks, p.ctas, po, ml);
}
template <int BITS, int D>
static cudaError_t launch(const TreeAttnArgs& a, const Plan& p, cudaStream_t st) {
  return p.blocks == 2 ? launch<BITS, D, true>(a, p, st) : launch<BITS, D, false>(a, p, st);
}
template <int BITS>
static cudaError_t launch(const TreeAttnArgs& a, const Plan& p, cudaStream_t st) {
  return a.D == 64 ? launch<BITS, 64>(a, p, st) : launch<BITS, 128>(a, p, st);
}

}  // namespace atr

size_t tree_attn_ws_bytes(int B, int Hq, int Hkv, int L, int D) {
  return atr::plan(B, Hq, Hkv, L).slots * atr::ROWS * (size_t(D) + 2) * sizeof(float);
}

int tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st) {
  const atr::Plan p = atr::plan(a.B, a.Hq, a.Hkv, a.L);
  M5_CUDA(a.bits == 8 ? atr::launch<8>(a, p, st) : a.bits == 4 ? atr::launch<4>(a, p, st) : atr::launch<0>(a, p, st));
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
