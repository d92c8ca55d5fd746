// Attention of a batch's new rows over the 8-bit paged KV cache: single tokens,
// chunks, prompts and draft trees (qwen3_tree.py:54-76, qwen35_tree.py:503-540,
// adapters.py:494-533), with a sliding window and sinks.
//
// A sequence's (new row, query head of the group) pairs are flattened, the head
// fastest: pair m = row * G + head. 32 pairs are the columns of S^T = K Q^T and
// O^T = V^T P^T on 32x32x16 fp16 MFMA, so a lane owns one pair and its softmax
// statistics are lane-local (one exchange with lane ^ 32).
//
// Scales. raw = q . k8 on the integers, exact in fp16; with the logits in log2
// units
//   t_j = raw_j * ks_j + log2(vs_j),  u_j = 2^(t_j - m),
//   o = sum_j u_j v8_j / sum_j u_j / vs_j,
// so a key's value scale joins its softmax weight in the exponent, u needs no
// further factor before its rounding to fp16, and the running maximum m keeps
// the largest weight times value scale of the row inside fp16's normal range
// whatever the scales are. q is moved by a power of two per workgroup, into the
// upper part of fp16's range, and taken back in ks; pairs of a workgroup too far
// apart for that by one of their own each, taken back in the pair's ks (raw alone
// is larger than the logit, by up to 127 / max |k|).
// A masked key's t is -inf, whatever its scales and bytes are (u = 0 exactly).
//
// Two kernels. Up to 32 pairs of a sequence and KV head (decoded tokens; 16 with
// 256 dims) are bound by the pages' bytes or, for short prefixes, by latency: the
// token kernel, pages straight to registers. More pairs are bound by the matrix and
// vector units together (neither alone is busy for more than 56 % of the time): the
// rows kernel, a page converted once for 128 or 256 pairs through LDS. Both split
// the keys into ranges where sequences are too few to fill the card, and a third
// joins them.
#include <algorithm>
#include <type_traits>

#include "kv_q8.h"

namespace dtree {
namespace {

constexpr float kFloor = -3.4e38f;      // m of a row that has seen no key
constexpr float kMinVs = 0x1p-80f;      // value scales below count as this
// Pairs without an RMSNorm whose largest values differ by more than this have an
// exponent each: fp16 has 2^27 from a workgroup's largest value down to its
// smallest normal one, so a pair keeps its 11 bits down to 2^-14 of its own largest.
constexpr float kFarApart = 0x1p12f;
constexpr float kTop = 6.f, kSlack = 8.f;  // u <= 2^kTop after a rescale, <= 2^(kTop + kSlack) before the next

struct AttnQ8Params {
  DtreeKvQ8 kv;
  DtreeAttnQ8Args a;
  float* part;    // [parts][total_rows][Hq][D], of every key range
  float* part_ml;  // and (m, l) of the same
  int G, blocks, pairs_wg;  // heads per group; row blocks per sequence, pairs of one
  int parts, per;           // key ranges the grid holds; pages of a range
  int sink_pages;
  float scale_log2;
  int tiled, h16;
  int plain;  // out: rows of bf16 alone, 16-byte aligned, no gate
};

// The pages that the rows from..to of a sequence see between them: the sink's,
// then a run that ends at the last row's own page.
struct Q8Range {
  int sink, first, tiles;
  __device__ __forceinline__ int page(int t) const { return t < sink ? t : first + t - sink; }
};
__device__ __forceinline__ Q8Range q8_range(const AttnQ8Params& p, const Q8Seq& q, int from, int to) {
  const int last = (q.past + (p.a.ancestors ? q.n - 1 : to)) / DTREE_PAGE;
  const int first = p.a.window > 0 ? max(0, q.past + from - p.a.window + 1) / DTREE_PAGE : 0;
  const int sink = min(p.sink_pages, first);
  return Q8Range{sink, first, sink + last - first + 1};
}

// Key ranges that a row block's pages are split into, and the pages of one.
__device__ __forceinline__ int q8_parts(const AttnQ8Params& p, int tiles) {
  return min(p.parts, (tiles + p.per - 1) / p.per);
}

// 4 int8 -> 4 fp16, exact: 1024 + 128 + q as fp16 bits, less 1152.
__device__ __forceinline__ void q8_word_to_h4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const f16x2_t bias = {(_Float16)1152.f, (_Float16)1152.f};
  const uint32_t x = w ^ 0x80808080u;
  lo = __builtin_bit_cast(uint32_t,
                          __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias);
  hi = __builtin_bit_cast(uint32_t,
                          __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias);
}
// 16 int8 -> two fragments of eight fp16.
__device__ __forceinline__ void q8_to_h16(u32x4_t w, u32x4_t& a, u32x4_t& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo, hi;
    q8_word_to_h4(w[i], lo, hi);
    (i < 2 ? a : b)[2 * (i & 1)] = lo;
    (i < 2 ? a : b)[2 * (i & 1) + 1] = hi;
  }
}

// max over the lane and lane ^ 32, without an LDS round trip: v_permlane32_swap of
// a value with its copy leaves one half's values in one register, the other's in
// the other. (s_nop: VALU write to permlane read.)
__device__ __forceinline__ float max_halves(float a) {
  float b;
  asm volatile("v_mov_b32 %1, %0\n\ts_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_max_f32 %0, %0, %1"
               : "+v"(a), "=&v"(b));
  return a;
}

// 2^e that takes a bound on the values into [2^13, 2^14), and its inverse.
__device__ __forceinline__ void q8_exponent(float amax, float& f, float& inv) {
  const int e = (int)(__float_as_uint(amax) >> 23);
  const int ef = amax > 0.f ? min(max(267 - e, 1), 253) : 127;
  f = __uint_as_float((uint32_t)ef << 23);
  inv = __uint_as_float((uint32_t)(254 - ef) << 23);
}

// Max over the TPR = D / 8 lanes of a pair.
template <int TPR>
__device__ __forceinline__ float q8_max_lanes(float a) {
  a = fmaxf(a, dpp<0xB1>(a));
  a = fmaxf(a, dpp<0x4E>(a));
  a = fmaxf(a, dpp<0x141>(a));
  if constexpr (TPR >= 16) a = fmaxf(a, dpp<0x140>(a));
  if constexpr (TPR >= 32) a = fmaxf(a, swz_xor16(a));
  return a;
}

// The queries of up to PAIRS pairs from pair0 on (q_norm, RoPE, the softmax scale
// in log2 units), in fp16 at qs[pair][D + 8] (past `pairs` anything, their
// results unread), moved by one power of two for the workgroup, whose inverse is
// returned: from a bound on the values, sqrt(2 D) max |w| behind an RMSNorm, else
// sqrt(2) times the largest finite one. `wide` (one value for the workgroup): the
// pairs' sizes are further apart than kFarApart, each is moved by a power of its
// own, whose inverse lies behind its values in qs, and 1 is returned. W waves;
// the barriers wait for LDS alone.
// No load is in a branch, so that a batch's loads go out together: lanes without a
// rotation read a table's first entries, calls without one the row.
template <int D, int PAIRS, int W, bool BF>
__device__ __forceinline__ float q8_queries_of(const AttnQ8Params& p, const Q8Seq& q, int g, int pair0, int pairs,
                                               uint16_t* qs, float (*wmax)[W], bool& wide) {
  constexpr int TPR = D / 8, NT = 64 * W, PPR = NT / TPR, kFlight = 8;  // PPR pairs a round
  constexpr int NR = (PAIRS + PPR - 1) / PPR, BR = NR < kFlight ? NR : kFlight;  // rounds; rounds in flight
  constexpr int SZ = BF ? 2 : 4;
  static_assert(NR % BR == 0, "whole batches of rounds");
  const int tid = threadIdx.x, j = tid % TPR;
  const int half = p.a.rope_dims / 2;
  const Q8Pieces pc = q8_pieces<D>(p.a.rope_dims, j);
  // Pair to pair in steps of PPR: dr rows and dh heads on, one row more where the
  // heads wrap; past the last row it stays there.
  const int dr = PPR / p.G, dh = PPR % p.G;
  const int r0 = (pair0 + tid / TPR) / p.G, h0 = pair0 + tid / TPR - r0 * p.G;
  const char* const base0 = static_cast<const char*>(p.a.q) + (size_t)q.start * p.a.ld_q * SZ;
  int r = r0, hd = h0;
  auto load = [&](u32x4_t& x0, u32x4_t& x1, size_t& row, const char*& base) {
    const int rr = min(r, q.n - 1);
    row = (size_t)q.start + rr;
    base = base0 + ((size_t)rr * (unsigned)p.a.ld_q + (unsigned)((g * p.G + hd) * p.a.q_stride)) * SZ;
    if constexpr (BF) {
      const u32x2_t a = *reinterpret_cast<const u32x2_t*>(base + 2 * pc.at[0]);
      const u32x2_t b = *reinterpret_cast<const u32x2_t*>(base + 2 * pc.at[1]);
      x0 = u32x4_t{a[0], a[1], 0, 0};
      x1 = u32x4_t{b[0], b[1], 0, 0};
    } else {
      x0 = ld_u32x4(base + 4 * pc.at[0]);
      x1 = ld_u32x4(base + 4 * pc.at[1]);
    }
    r += dr;
    hd += dh;
    const bool wrap = hd >= p.G;
    hd -= wrap ? p.G : 0;
    r += wrap ? 1 : 0;
  };
  auto value = [](u32x4_t x) {
    if constexpr (BF) return q8_bf4(u32x2_t{x[0], x[1]});
    else return __builtin_bit_cast(f32x4_t, x);
  };
  const int rounds = min(NR, (pairs - pair0 + PPR - 1) / PPR);  // (what is behind them stays as LDS has it)
  const bool norm = p.a.q_norm != nullptr;
  f32x4_t w0 = {p.scale_log2, p.scale_log2, p.scale_log2, p.scale_log2}, w1 = w0;
  float f, inv, bound = 0.f;
  wide = false;
  // the largest finite value of a lane's pieces (what is not finite stays in its row)
  auto largest = [](f32x4_t a, f32x4_t b) {
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t = fabsf(a[e]) < INFINITY ? fmaxf(t, fabsf(a[e])) : t;
      t = fabsf(b[e]) < INFINITY ? fmaxf(t, fabsf(b[e])) : t;
    }
    return t;
  };
  const float unit = p.scale_log2 * 1.4142136f;
  if (norm) {
    u32x2_t a, b;  // (tables and weights at any address of their type)
    __builtin_memcpy(&a, p.a.q_norm + pc.at[0], 8);
    __builtin_memcpy(&b, p.a.q_norm + pc.at[1], 8);
    w0 *= q8_bf4(a);
    w1 *= q8_bf4(b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float m = fmaxf(fabsf(w0[e]), fabsf(w1[e]));
      bound = m < INFINITY ? fmaxf(bound, m) : bound;
    }
    bound = q8_max_lanes<TPR>(bound) * sqrtf(2.f * D);
  } else {
    float least = -INFINITY;  // less the smallest pair's largest value (a pair of zeros has no size)
#pragma unroll 1
    for (int k = 0; k < rounds; ++k) {
      u32x4_t x0, x1;
      size_t row;
      const char* base;
      load(x0, x1, row, base);
      const float top = q8_max_lanes<TPR>(largest(value(x0), value(x1)));
      bound = fmaxf(bound, top);
      least = top > 0.f ? fmaxf(least, -top) : least;
    }
    r = r0;
    hd = h0;
    bound = max_halves(q8_max_lanes<32>(bound));
    least = max_halves(q8_max_lanes<32>(least));
    if ((tid & 63) == 0) {
      wmax[0][tid >> 6] = bound;
      wmax[1][tid >> 6] = least;
    }
    lds_barrier();
#pragma unroll
    for (int k = 0; k < W; ++k) {
      bound = fmaxf(bound, wmax[0][k]);
      least = fmaxf(least, wmax[1][k]);
    }
    wide = __builtin_amdgcn_readfirstlane(bound > -least * kFarApart);
    bound *= unit;
  }
  q8_exponent(bound, f, inv);
  auto load_all = [&](u32x4_t (&x)[2], f32x4_t& cs, f32x4_t& sn) {
    size_t row;
    const char* base;
    load(x[0], x[1], row, base);
    const size_t at = 4 * (row * half + (pc.turns ? 4 * j : 0));
    const char* tc = half ? reinterpret_cast<const char*>(p.a.rope_cos) + at : base;
    const char* ts = half ? reinterpret_cast<const char*>(p.a.rope_sin) + at : base;
    __builtin_memcpy(&cs, tc, 16);
    __builtin_memcpy(&sn, ts, 16);
  };
  // The pair of round k, rotated, times rs, to LDS.
  auto put = [&](int k, f32x4_t x0, f32x4_t x1, f32x4_t cs, f32x4_t sn, float rs) {
    f32x4_t y, z;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = x0[e] * w0[e], b = x1[e] * w1[e];
      // (a select, not sn = 0, which would carry an infinity to another dim)
      y[e] = (pc.turns ? a * cs[e] - b * sn[e] : a) * rs;
      z[e] = (pc.turns ? a * sn[e] + b * cs[e] : b) * rs;
    }
    const int pl = tid / TPR + k * PPR;
    if (PAIRS % PPR == 0 || pl < PAIRS) {
      *reinterpret_cast<u32x2_t*>(qs + pl * (D + 8) + pc.at[0]) = u32x2_t{pack_h2(y[0], y[1]), pack_h2(y[2], y[3])};
      *reinterpret_cast<u32x2_t*>(qs + pl * (D + 8) + pc.at[1]) = u32x2_t{pack_h2(z[0], z[1]), pack_h2(z[2], z[3])};
    }
  };
  if (wide) {  // (rare: one round at a time, little code)
#pragma unroll 1
    for (int k = 0; k < rounds; ++k) {
      u32x4_t x[2];
      f32x4_t cs, sn;
      load_all(x, cs, sn);
      const f32x4_t x0 = value(x[0]), x1 = value(x[1]);
      q8_exponent(q8_max_lanes<TPR>(largest(x0, x1)) * unit, f, inv);
      put(k, x0, x1, cs, sn, f);
      const int pl = tid / TPR + k * PPR;
      if (j == 0 && (PAIRS % PPR == 0 || pl < PAIRS)) *reinterpret_cast<float*>(qs + pl * (D + 8) + D) = inv;
    }
    lds_barrier();
    return 1.f;
  }
#pragma unroll 1
  for (int k0 = 0; k0 < rounds; k0 += BR) {
    u32x4_t x[BR][2];
    f32x4_t cs[BR], sn[BR];
#pragma unroll
    for (int k = 0; k < BR; ++k) load_all(x[k], cs[k], sn[k]);
#pragma unroll
    for (int k = 0; k < BR; ++k) {
      const f32x4_t x0 = value(x[k][0]), x1 = value(x[k][1]);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], ss));
      ss += dpp<0xB1>(ss);
      ss += dpp<0x4E>(ss);
      ss += dpp<0x141>(ss);
      if constexpr (TPR >= 16) ss += dpp<0x140>(ss);
      if constexpr (TPR >= 32) ss += swz_xor16(ss);
      const float rs = norm ? f * __builtin_amdgcn_rsqf(ss * (1.0f / D) + p.a.eps) : f;  // (1 ulp; fp16 follows)
      put(k0 + k, x0, x1, cs[k], sn[k], rs);
    }
  }
  lds_barrier();
  return inv;
}
template <int D, int PAIRS, int W>
__device__ __forceinline__ float q8_queries(const AttnQ8Params& p, const Q8Seq& q, int g, int pair0, int pairs,
                                            uint16_t* qs, float (*wmax)[W], bool& wide) {
  return p.a.q_type == DTREE_T_BF16 ? q8_queries_of<D, PAIRS, W, true>(p, q, g, pair0, pairs, qs, wmax, wide)
                                    : q8_queries_of<D, PAIRS, W, false>(p, q, g, pair0, pairs, qs, wmax, wide);
}

// (ks, log2 vs, 1 / vs) of a key. A NaN reaches a row that sees the key through
// ks and log2 vs; 1 / vs stays finite, since a masked key's u = 0 meets it.
__device__ __forceinline__ void q8_scales(float ks, float vs, float inv, float& k, float& lv, float& iv) {
  const float v = vs < kMinVs ? kMinVs : vs;
  k = ks * inv;
  lv = __builtin_amdgcn_logf(v);
  iv = v == v ? 1.f / v : 1.f;
}

// The keys key0 .. key0 + 31 that the pair at `pos` (-1: none) sees, a bit each.
// Draft tree: the cached prefix and `anc`, the pair's ancestor words in LDS.
__device__ __forceinline__ uint32_t q8_low_bits(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t q8_sees(const AttnQ8Params& p, const Q8Seq& q, int pos, int key0,
                                            const uint32_t* anc) {
  if (p.a.ancestors) {
    const int n = key0 - q.past;  // the new row that key0 is
    if (pos < 0) return 0u;
    if (n <= -32) return ~0u;
    if (n < 0) return q8_low_bits(-n) | ((anc[0] & q8_low_bits(q.n)) << -n);
    if (n >= q.n) return 0u;
    const int w = n >> 5;  // (at most 128 rows)
    const uint32_t lo = anc[w], hi = w + 1 < DTREE_MASK_WORDS ? anc[w + 1] : 0u;
    return __builtin_amdgcn_alignbit(hi, lo, n & 31) & q8_low_bits(q.n - n);
  }
  uint32_t bits = q8_low_bits(pos - key0 + 1);
  if (p.a.window > 0) bits &= ~q8_low_bits(pos - p.a.window + 1 - key0) | q8_low_bits(p.a.sink - key0);
  return bits;
}
// The ancestor words of pairs pair0 .. pair0 + n - 1 to LDS (a barrier follows).
__device__ __forceinline__ void q8_ancestors(const AttnQ8Params& p, const Q8Seq& q, int pair0, int n, int pairs,
                                             uint32_t (*anc)[DTREE_MASK_WORDS]) {
  if (!p.a.ancestors) return;
  for (int u = threadIdx.x; u < n * DTREE_MASK_WORDS; u += blockDim.x) {
    const int m = pair0 + u / DTREE_MASK_WORDS, w = u % DTREE_MASK_WORDS;
    anc[u / DTREE_MASK_WORDS][w] =
        m < pairs ? p.a.ancestors[((size_t)q.start + m / p.G) * DTREE_MASK_WORDS + w] : 0u;
  }
}

// The output gate's logits at dims d .. of a pair (0 without a gate, unused).
__device__ __forceinline__ f32x4_t q8_gate(const AttnQ8Params& p, size_t row, int head, int d) {
  if (!p.a.gated) return f32x4_t{0.f, 0.f, 0.f, 0.f};
  const size_t at = row * p.a.ld_q + (size_t)head * p.a.q_stride + p.kv.head_dim + d;
  if (p.a.q_type == DTREE_T_BF16)
    return q8_bf4(*reinterpret_cast<const u32x2_t*>(static_cast<const uint16_t*>(p.a.q) + at));
  return *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p.a.q) + at);
}
// Four values of dims d .. of a pair's output, gated, stored.
__device__ __forceinline__ void q8_store(const AttnQ8Params& p, size_t row, int head, int d, f32x4_t o, f32x4_t gate) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = p.a.gated ? o[e] * __builtin_amdgcn_rcpf(1.0f + __expf(-gate[e])) : o[e];
  const int col = head * p.kv.head_dim + d;
  const size_t oi = p.tiled ? tiled_index((int)row, col, p.a.ld_out) : row * p.a.ld_out + col;
  store_act4(p.a.out, p.a.out_lo, oi, y, p.h16);
}
__device__ __forceinline__ void q8_store_zero(const AttnQ8Params& p, size_t row, int head, int d) {
  const int col = head * p.kv.head_dim + d;
  const size_t oi = p.tiled ? tiled_index((int)row, col, p.a.ld_out) : row * p.a.ld_out + col;
  *reinterpret_cast<u32x2_t*>(p.a.out + oi) = u32x2_t{0, 0};  // (0 in bf16 and in fp16)
  if (p.a.out_lo) *reinterpret_cast<u32x2_t*>(p.a.out_lo + oi) = u32x2_t{0, 0};
}

// 1 / l, 0 where the row has seen no key.
__device__ __forceinline__ float q8_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Four values of a pair of one of several ranges, with the range's m and softmax
// sum l, to the partials.
__device__ __forceinline__ void q8_partial(const AttnQ8Params& p, int part, size_t row, int head, int d, f32x4_t o,
                                           float m, float l) {
  const size_t u = ((size_t)part * p.kv.total_rows + row) * p.a.num_heads + head;
  *reinterpret_cast<f32x4_t*>(p.part + u * p.kv.head_dim + d) = o;
  if (d == 0) *reinterpret_cast<f32x2_t*>(p.part_ml + 2 * u) = f32x2_t{m, l};
}

__device__ __forceinline__ f32x4_t mfma16_f16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                0);
}

// A workgroup: all pairs of a sequence and KV head, up to 16 NC, over one key
// range, its pages dealt to the W waves in turn. A wave loads its pages
// straight into registers, the next one during the current one; the waves'
// results meet in LDS.
//
// 16 pairs are the columns of 16x16x32 products: half the softmax of 32 columns
// that one decoded token leaves mostly empty. Lane 16 kq + c owns column c, and,
// with kq = 2 b + h, a page's keys 32 b + 8 i + 4 h + e (i, e < 4). So
// * S block i (accumulator e) has the key 32 (rho / 8) + 8 i + rho % 8 in its row
//   rho: K's lane rho reads 16 dims of that key (two steps, dims 64 JJ + 16 kq +
//   8 step + ..);
// * V's lane (dim % 16, kq) reads its 16 keys of one dim as they lie, i = 2 step,
//   2 step + 1, and P needs no exchange.
//
// Measured (8 KV heads of 128, 4 query heads each): one token over 65536 keys 27.7
// us, 138 MB at 5.0 TB/s, as a copy; 32 tokens over up to 8193 keys 27.1 us, 100 MB
// at 3.7 TB/s (half of them hold under 200 keys, a few long ones' ranges are what is
// left at the end); one over 1001 keys 10 us, all latency: lengths, page ids, the
// first page with the query rows, 3 pages a wave, the merge.
template <int D, int NC, int W>
__global__ __launch_bounds__(64 * W, 8 / W) void q8_token_kernel(AttnQ8Params p) {
  constexpr int NJ = D / 64, NK = 4 * NJ, ND = D / 16;  // K loads (block, 64 dims) and V loads (16 dims) per page
  constexpr int RS = D + 4;                             // a pair's row in `red`
  union Lds {
    uint16_t q[16 * NC * (D + 8)];
    float red[W * 16 * NC * RS];
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  __shared__ __attribute__((aligned(16))) float scl[W][192];
  __shared__ float mls[W][2][16 * NC];
  __shared__ float wmax[2][W];
  __shared__ uint32_t anc[16 * NC][DTREE_MASK_WORDS];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hkv = p.kv.num_kv_heads, g = blockIdx.x % Hkv, b0 = blockIdx.x / Hkv;
  const int part = b0 % p.parts, s = b0 / p.parts;
  const Q8Seq q = q8_seq(p.kv, s);
  if (part == 0 && q.n < p.a.rows_padded) {  // rows past the sequence's
    for (int e = tid; e < (p.a.rows_padded - q.n) * p.G * (D / 4); e += 64 * W)
      q8_store_zero(p, q.n + e / (D / 4) / p.G, g * p.G + e / (D / 4) % p.G, 4 * (e % (D / 4)));
  }
  if (q.n == 0) return;
  const Q8Range rg = q8_range(p, q, 0, q.n - 1);
  const int used = q8_parts(p, rg.tiles), per = (rg.tiles + used - 1) / used;
  const int t0 = part * per, t1 = min(rg.tiles, t0 + per);
  if (part >= used) return;
  const int pairs = q.n * p.G;

  u32x4_t kb[NK], vb[ND];
  float ksl, vsl;
  auto block = [&](int page) { return ((size_t)max(page, 0) * Hkv + g); };
  // The wave's i-th page is in lane i % 64 of `ids`: a load in the loop would
  // have to come back, and with it every load before it, to be used.
  int ids = -1;
  auto load_ids = [&](int i) {
    const int t = t0 + wave + W * (i + lane);
    ids = t < t1 ? q8_page(p.kv, s, rg.page(t)) : -1;
  };
  auto page_of = [&](int i) {
    if ((i & 63) == 0) load_ids(i);
    return __builtin_amdgcn_readlane(ids, i & 63);
  };
  // (a resource of no bytes reads as zeros without an access)
  const int koff = (c >> 3) * (32 * D) + (kq >> 1) * 1024 + ((kq & 1) * 32 + (c & 7)) * 16;
  const int voff = (kq >> 1) * (32 * D) + ((kq & 1) * 32 + c) * 16;
  auto load_k = [&](int page) {
    const auto rk = buf_rsrc(p.kv.k_pages + block(page) * (DTREE_PAGE * D), page < 0 ? 0 : DTREE_PAGE * D);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) kb[i * NJ + j] = buf_ld(rk, koff + 128 * i + 2048 * j);
    ksl = page < 0 ? 0.f : p.kv.k_scales[block(page) * DTREE_PAGE + lane];
    vsl = page < 0 ? 0.f : p.kv.v_scales[block(page) * DTREE_PAGE + lane];
  };
  auto load_v = [&](int page) {
    const auto rv = buf_rsrc(p.kv.v_pages + block(page) * (DTREE_PAGE * D), page < 0 ? 0 : DTREE_PAGE * D);
#pragma unroll
    for (int i = 0; i < ND; ++i) vb[i] = buf_ld(rv, voff + 1024 * (i >> 1) + 256 * (i & 1));
  };
  const int steps = max(0, (t1 - t0 - wave + W - 1) / W);  // the wave's pages
  int cur = page_of(0);
  if constexpr (NC == 1) load_k(cur);
  q8_ancestors(p, q, 0, 16 * NC, pairs, anc);
  bool wide;
  const float inv = q8_queries<D, 16 * NC, W>(p, q, g, 0, pairs, lds.q, wmax, wide);
  if constexpr (NC == 2) load_k(cur);
  load_v(cur);  // (not earlier: the queries' registers)
  // The queries' fragments in registers; of 128 dims the first block's alone, of 256
  // dims none, the others read from LDS in every step: two waves a SIMD have room for
  // no more (32 x 2 tokens over 8000 keys of 256 dims: 53.6 us, with one 62.7), and a
  // register spilled and read back waits for all loads before its own.
  constexpr int NQ = D == 256 ? 0 : D == 128 ? 1 : NC;
  auto q_frag = [&](int n, int i) {
    return *reinterpret_cast<const u32x4_t*>(lds.q + (16 * n + c) * (D + 8) + 64 * (i >> 1) + 16 * kq + 8 * (i & 1));
  };
  u32x4_t qf[NQ ? NQ : 1][2 * NJ];
  int pos[NC];  // the columns' positions; -1: no pair
  float own[NC];  // what takes a column's own power of two back (wide)
#pragma unroll
  for (int n = 0; n < NC; ++n) {
#pragma unroll
    for (int i = 0; i < 2 * NJ && n < NQ; ++i) qf[n][i] = q_frag(n, i);
    pos[n] = 16 * n + c < pairs ? q.past + (16 * n + c) / p.G : -1;
    own[n] = wide ? *reinterpret_cast<const float*>(lds.q + (16 * n + c) * (D + 8) + D) : 1.f;
  }
  f32x4_t o[NC][ND];
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int d = 0; d < ND; ++d) o[n][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m[NC], l[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    m[n] = kFloor;
    l[n] = 0.f;
  }
  const int kkey = 32 * (kq >> 1) + 4 * (kq & 1);  // the lane's keys: kkey + 8 i + e
  float* sc = scl[wave];
  for (int i = 0; i < steps; ++i) {
    const int next = page_of(i + 1);
    const int k0 = DTREE_PAGE * rg.page(t0 + wave + W * i);
    {
      float k, lv, iv;
      q8_scales(ksl, vsl, inv, k, lv, iv);
      sc[lane] = k;
      sc[64 + lane] = lv;
      sc[128 + lane] = iv;
    }
    f32x4_t st[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int b = 0; b < 4; ++b) st[n][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      u32x4_t qj[NC][2];
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) qj[n][k] = n < NQ ? qf[n < NQ ? n : 0][2 * j + k] : q_frag(n, 2 * j + k);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u32x4_t a0, a1;
        q8_to_h16(kb[b * NJ + j], a0, a1);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          st[n][b] = mfma16_f16(a0, qj[n][0], st[n][b]);
          st[n][b] = mfma16_f16(a1, qj[n][1], st[n][b]);
        }
      }
    }
    load_k(next);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (cur >= 0) {
      const bool masked = p.a.ancestors ? k0 + DTREE_PAGE > q.past
                                        : k0 + DTREE_PAGE - 1 > q.past ||
                                              (p.a.window > 0 && k0 + DTREE_PAGE - 1 >= p.a.sink &&
                                               q.past + q.n - 1 - k0 >= p.a.window);
      u32x4_t ph[NC][2];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        float mx = kFloor;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const f32x4_t ks = *reinterpret_cast<const f32x4_t*>(sc + kkey + 8 * b);
          const f32x4_t lv = *reinterpret_cast<const f32x4_t*>(sc + 64 + kkey + 8 * b);
#pragma unroll
          for (int e = 0; e < 4; ++e) st[n][b][e] = fmaf(st[n][b][e], ks[e] * own[n], lv[e]);
        }
        if (masked) {
          const uint32_t sees = q8_sees(p, q, pos[n], k0 + (kkey & 32), anc[16 * n + c]) >> (kkey & 31);
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) st[n][b][e] = sees & (1u << (8 * b + e)) ? st[n][b][e] : -INFINITY;
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, st[n][b][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m[n] + (kTop + kSlack))) {
          const float mn = mx > m[n] + (kTop + kSlack) ? mx - kTop : m[n], alpha = fast_exp2(m[n] - mn);
          m[n] = mn;
          l[n] *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][d][e] *= alpha;
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const f32x4_t iv = *reinterpret_cast<const f32x4_t*>(sc + 128 + kkey + 8 * b);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            st[n][b][e] = fast_exp2(st[n][b][e] - m[n]);
            l[n] = fmaf(st[n][b][e], iv[e], l[n]);
          }
          ph[n][b >> 1][2 * (b & 1)] = pack_h2(st[n][b][0], st[n][b][1]);
          ph[n][b >> 1][2 * (b & 1) + 1] = pack_h2(st[n][b][2], st[n][b][3]);
        }
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        u32x4_t a0, a1;
        q8_to_h16(vb[d], a0, a1);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          o[n][d] = mfma16_f16(a0, ph[n][0], o[n][d]);
          o[n][d] = mfma16_f16(a1, ph[n][1], o[n][d]);
        }
      }
    }
    load_v(next);
    cur = next;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // the waves' results
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    l[n] += __shfl_xor(l[n], 16);
    l[n] += __shfl_xor(l[n], 32);
    if (kq == 0) {
      mls[wave][0][16 * n + c] = m[n];
      mls[wave][1][16 * n + c] = l[n];
    }
  }
  lds_barrier();  // also: every wave has read its queries
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int pr = 16 * n + c;
    if (pr >= pairs) continue;
    float mt = kFloor;
#pragma unroll
    for (int w = 0; w < W; ++w) mt = fmaxf(mt, mls[w][0][pr]);
    const float fac = fast_exp2(m[n] - mt);
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<f32x4_t*>(lds.red + (wave * 16 * NC + pr) * RS + 16 * d + 4 * kq) =
          f32x4_t{o[n][d][0] * fac, o[n][d][1] * fac, o[n][d][2] * fac, o[n][d][3] * fac};
  }
  lds_barrier();
  for (int u = tid; u < pairs * (D / 4); u += 64 * W) {
    const int pr = u / (D / 4), d = 4 * (u % (D / 4)), head = g * p.G + pr % p.G;
    const size_t row = (size_t)q.start + pr / p.G;
    const f32x4_t gate = q8_gate(p, row, head, d);
    float mt = kFloor, lt = 0.f;
    f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) mt = fmaxf(mt, mls[w][0][pr]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      lt += mls[w][1][pr] * fast_exp2(mls[w][0][pr] - mt);
      y += *reinterpret_cast<const f32x4_t*>(lds.red + (w * 16 * NC + pr) * RS + d);
    }
    if (used > 1) q8_partial(p, part, row, head, d, y, mt, lt);
    else q8_store(p, row, head, d, y * q8_inverse(lt), gate);
  }
}

// A workgroup: W waves of 32 pairs of one KV head over one key range. A page is
// converted to fp16 once for all of them, on its way from memory to LDS, the
// next one while the current one is used.
//
// A step is 32 keys, half a page: S^T = K Q^T, softmax, O^T += V^T P^T. The matrix
// cores run S of the next step (block2) while the weights of this step's first 16
// keys are taken, then PV (block1): of the first 16 keys while the weights of the
// others are taken, of the others while the next step's logits are scaled, with
// the next page's conversion in every second block1. A slot is one MFMA, the loads
// that a later slot needs and a share of the VALU work, and the code is written in
// that order: with each product before or behind all of its softmax, neither unit
// was busy for half the time. Two waves a SIMD: one of 64 pairs, with half the LDS
// reads, took 8 % longer, since a wave alone issues one instruction at a time.
//
// Measured: 4096 rows, 32 heads of 128 on 8: 165 to 173 us, 0.8 PFLOP/s (a large library
// product 1.2), MFMA busy 42 %, VALU 56 %, LDS 44 % of the time, waves waiting 31 %:
// no unit is full, and what the waits are for was not found. 1000 gated rows after
// 8192 keys, 16 heads of 256, one wave a SIMD: 186 us without the join, 0.76 PFLOP/s.
template <int D, int W>
__global__ __launch_bounds__(64 * W, D <= 128 ? 8 / W : 1) void q8_rows_kernel(AttnQ8Params p) {
  constexpr int NB = D / 32, PB = DTREE_PAGE * D;  // bytes of a page's K (or V) as int8
  constexpr int NT = 64 * W, NP = PB / 16 / NT;    // 16-byte pieces of it per thread
  constexpr int NF = D / 16;                       // fragments of K (or V) in a step, MFMAs of a block
  constexpr int RF = 4;                            // fragments loaded ahead
  constexpr int WP = 32 * W;                       // pairs of the workgroup
  constexpr int RS = D + 4;  // a pair's row in `red`
  // Three pages where LDS has room beside the outputs: the next page can then be
  // staged while the last one's V is read, with one barrier a page, and its K read
  // ahead; with two it waits for that between two barriers.
  constexpr int NBUF = D == 64 || W == 8 ? 3 : 2;
  union Lds {
    unsigned char kv[NBUF][4 * PB];  // fp16 K, then V
    uint16_t q[WP * (D + 8)];
    float red[WP * RS];
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  __shared__ __attribute__((aligned(16))) float scl[NBUF][192];
  __shared__ float wmax[2][W];
  __shared__ uint32_t anc[WP][DTREE_MASK_WORDS];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hkv = p.kv.num_kv_heads, g = blockIdx.x % Hkv;
  int bx = blockIdx.x / Hkv;
  const int part = bx % p.parts;
  bx /= p.parts;
  const int w = p.blocks - 1 - bx % p.blocks, s = bx / p.blocks;  // longest ranges first
  const Q8Seq q = q8_seq(p.kv, s);
  const int pairs = q.n * p.G, pair0 = WP * w;
  if (part == 0 && p.a.rows_padded > 0) {  // rows past the sequence's
    const int end = min(pair0 + WP, p.a.rows_padded * p.G);
    for (int e = max(pairs - pair0, 0) * (D / 4) + tid; e < (end - pair0) * (D / 4); e += NT) {
      const int m = pair0 + e / (D / 4);
      q8_store_zero(p, m / p.G, g * p.G + m % p.G, 4 * (e % (D / 4)));
    }
  }
  if (pair0 >= pairs) return;
  const int from = pair0 / p.G, to = min(q.n - 1, (pair0 + WP - 1) / p.G);  // the workgroup's rows
  const Q8Range rg = q8_range(p, q, from, to);
  const int used = q8_parts(p, rg.tiles), per = (rg.tiles + used - 1) / used;
  const int t0 = part * per, t1 = min(rg.tiles, t0 + per);
  if (part >= used) return;
  const int wpair = pair0 + 32 * wave;
  // the wave's rows (a wave past the last pair works on zero queries, unread)
  const int wfrom = min(wpair / p.G, q.n - 1), wto = min(q.n - 1, (wpair + 31) / p.G);

  u32x4_t raw[2 * NP];
  float ksl = 0.f, vsl = 0.f;
  // The range's i-th page is in lane i % 64 of `ids` (a load in the loop would
  // have to come back to be used).
  int ids = -1;
  auto load = [&](int i) {  // this thread's pieces of the i-th page; false: the page is absent
    i = min(i, t1 - t0 - 1);
    if ((i & 63) == 0) ids = t0 + i + lane < t1 ? q8_page(p.kv, s, rg.page(t0 + i + lane)) : -1;
    const int page = __builtin_amdgcn_readlane(ids, i & 63);
    const size_t blk = (size_t)max(page, 0) * Hkv + g;
    const auto rk = buf_rsrc(p.kv.k_pages + blk * PB, page < 0 ? 0 : PB);
    const auto rv = buf_rsrc(p.kv.v_pages + blk * PB, page < 0 ? 0 : PB);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      raw[i] = buf_ld(rk, 16 * tid + 16 * NT * i);
      raw[NP + i] = buf_ld(rv, 16 * tid + 16 * NT * i);
    }
    const auto sk = buf_rsrc(p.kv.k_scales + blk * DTREE_PAGE, page < 0 ? 0 : 4 * DTREE_PAGE);
    const auto sv = buf_rsrc(p.kv.v_scales + blk * DTREE_PAGE, page < 0 ? 0 : 4 * DTREE_PAGE);
    ksl = buf_ldf(sk, 4 * tid);  // (threads past the page's positions read 0)
    vsl = buf_ldf(sv, 4 * tid);
    return page >= 0;
  };
  bool here = load(0);
  q8_ancestors(p, q, pair0, WP, pairs, anc);
  bool wide;
  const float inv = q8_queries<D, WP, W>(p, q, g, pair0, pairs, lds.q, wmax, wide);
  u32x4_t qf[NF];
  const int pos = wpair + c < pairs ? q.past + (wpair + c) / p.G : -1;  // -1: the lane has no pair
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    qf[i] = *reinterpret_cast<const u32x4_t*>(lds.q + (32 * wave + c) * (D + 8) + 32 * (i >> 1) + 16 * h + 8 * (i & 1));
    // (an MFMA reads its B operand from either file: not the one the softmax needs)
    if constexpr (D == 256) asm("" : "+a"(qf[i]));
  }
  // what takes the lane's own power of two back (wide)
  const float own = wide ? *reinterpret_cast<const float*>(lds.q + (32 * wave + c) * (D + 8) + D) : 1.f;
  lds_barrier();
  auto stage_scales = [&](int buf) {
    if (tid < DTREE_PAGE) {
      float k, lv, iv;
      q8_scales(ksl, vsl, inv, k, lv, iv);
      scl[buf][tid] = k;
      scl[buf][64 + tid] = lv;
      scl[buf][128 + tid] = iv;
    }
  };
  // Word j of piece i (K's pieces, then V's) of the raw page; its fragments go out
  // when they are whole.
  u32x4_t half;
  auto stage_word = [&](int buf, int i, int j) {
    const int u = tid + NT * (i % NP);
    uint32_t lo, hi;
    q8_word_to_h4(raw[i][j], lo, hi);
    half[2 * (j & 1)] = lo;
    half[2 * (j & 1) + 1] = hi;
    if (j & 1)
      *reinterpret_cast<u32x4_t*>(
          &lds.kv[buf][(i / NP) * 2 * PB + (u >> 6) * 2048 + (j >> 1) * 1024 + (u & 63) * 16]) = half;
  };
  f32x16_t o[NB], sa, sb;  // sa, sb: the logits of even and odd steps
  u32x4_t ph[2], kf[RF], vf[RF];
  f32x4_t ks[4], lv[4], iv[4];
  float m = kFloor, l = 0.f, mx;
  ph[0] = ph[1] = u32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) sb[i] = -INFINITY;  // the step before the first: no keys
#pragma unroll
  for (int db = 0; db < NB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  // Fragment f of a half page: K's dims 16 f ..; V's keys 16 (f / NB) .., dims 32 (f % NB) ..
  auto k_frag = [&](int buf, int b, int f) {
    return *reinterpret_cast<const u32x4_t*>(&lds.kv[buf][b * PB + 1024 * f + 16 * lane]);
  };
  auto v_frag = [&](int buf, int b, int f) {
    return *reinterpret_cast<const u32x4_t*>(&lds.kv[buf][2 * PB + b * PB + 1024 * (2 * (f % NB) + f / NB) + 16 * lane]);
  };
  auto consts = [&](f32x4_t (&x)[4], int buf, int which, int b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const f32x4_t*>(&scl[buf][64 * which + 32 * b + 8 * i + 4 * h]);
  };
  auto weight = [&](f32x16_t& x, int r) {
    x[r] = fast_exp2(x[r] - m);
    l = fmaf(x[r], iv[r / 4][r % 4], l);
    if (r & 1) ph[r >> 3][(r >> 1) & 3] = pack_h2(x[r - 1], x[r]);
  };
  // PV of the last step (its V: half vh of buffer vbuf; its logits `old`), the logits
  // `cur` of this one (half b of buffer buf, whose 1 / vs it loads). STAGE: the raw
  // page to buffer sbuf. AHEAD: the first K fragments (half kh of kbuf) of block2.
  auto block1 = [&](f32x16_t& old, f32x16_t& cur, int vbuf, int vh, int buf, int b, auto stage, int sbuf, auto ahead,
                    int kbuf, int kh) {
    constexpr int ST = NF / 2 > 2 ? NF / 2 - 1 : 1;  // slots of the logits
    constexpr int SW = 8 * NP / NF;                  // words converted per slot
    mx = kFloor;
#pragma unroll
    for (int k = 0; k < NF; ++k) {
      o[k % NB] = mfma32_f16(vf[k % RF], ph[k / NB], o[k % NB]);
      if (k + RF < NF) vf[k % RF] = v_frag(vbuf, vh, k + RF);
      else if constexpr (decltype(ahead)::value) kf[k + RF - NF] = k_frag(kbuf, kh, k + RF - NF);
      if constexpr (decltype(stage)::value) {
#pragma unroll
        for (int i = k * SW; i < (k + 1) * SW; ++i) stage_word(sbuf, i / 4, i % 4);
      }
      if (k < NF / 2) {
#pragma unroll
        for (int r = 8 + k * 16 / NF; r < 8 + (k + 1) * 16 / NF; ++r) weight(old, r);
      } else {
        const int j = k - NF / 2;
        if (j < ST) {
#pragma unroll
          for (int r = j * 16 / ST; r < (j + 1) * 16 / ST; ++r) {
            cur[r] = fmaf(cur[r], ks[r / 4][r % 4], lv[r / 4][r % 4]);
            mx = fmaxf(mx, cur[r]);
          }
        }
        if (j == 0) consts(iv, buf, 2, b);
        if (j == NF / 2 - 1) mx = max_halves(mx);
      }
    }
  };
  // What the rows may not see; the output rescaled where a row's maximum has grown.
  auto limits = [&](f32x16_t& cur, bool masked, bool there, int key0) {
    if (masked) {
      const uint32_t sees = there ? q8_sees(p, q, pos, key0, anc[32 * wave + c]) >> (4 * h) : 0u;
      mx = kFloor;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        cur[r] = sees & (1u << acc_row(r, 0)) ? cur[r] : -INFINITY;
        mx = fmaxf(mx, cur[r]);
      }
      mx = max_halves(mx);
    }
    if (__any(mx > m + (kTop + kSlack))) {
      const float mn = mx > m + (kTop + kSlack) ? mx - kTop : m, alpha = fast_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
    }
  };
  auto k_ahead = [&](int buf, int b) {
#pragma unroll
    for (int f = 0; f < RF; ++f) kf[f] = k_frag(buf, b, f);
  };
  // S of the next step (half b of buffer buf, whose ks and log2 vs it loads) to
  // `next`, the weights of `cur`'s first 16 keys, the first V fragments (half vh of
  // vbuf) of the next block1.
  auto block2 = [&](f32x16_t& cur, f32x16_t& next, int buf, int b, int vbuf, int vh) {
#pragma unroll
    for (int r = 0; r < 16; ++r) next[r] = 0.f;
#pragma unroll
    for (int k = 0; k < NF; ++k) {
      next = mfma32_f16(kf[k % RF], qf[k], next);
      if (k + RF < NF) kf[k % RF] = k_frag(buf, b, k + RF);
      else vf[k + RF - NF] = v_frag(vbuf, vh, k + RF - NF);
      if (k == 0) consts(ks, buf, 0, b);
      if (k == NF / 4) consts(lv, buf, 1, b);
#pragma unroll
      for (int r = k * 8 / NF; r < (k + 1) * 8 / NF; ++r) weight(cur, r);
    }
    asm volatile("" : "+v"(ph[0]), "+v"(l));  // taken here, not sunk to their use
    if (wide) {
#pragma unroll
      for (int i = 0; i < 4; ++i) ks[i] *= own;
    }
  };
  auto hidden = [&](int k0) {  // does a page hold keys that some row may not see
    return p.a.ancestors ? k0 + DTREE_PAGE > q.past
                         : k0 + DTREE_PAGE - 1 > q.past + wfrom ||
                               (p.a.window > 0 && k0 + DTREE_PAGE - 1 >= p.a.sink && q.past + wto - k0 >= p.a.window);
  };
  stage_scales(0);
#pragma unroll
  for (int i = 0; i < 2 * NP; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) stage_word(0, i, j);
  bool next = load(1);
  lds_barrier();
  // S of the first step. PV of none before it: zero weights times the first page.
  consts(iv, 0, 2, 0);
  k_ahead(0, 0);
  block2(sb, sa, 0, 0, 0, 0);
  int vbuf = 0, vh = 0, buf = 0;  // where the last step's V is; this page
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  for (int t = t0; t < t1; ++t) {
    const int k0 = DTREE_PAGE * rg.page(t), then = buf + 1 == NBUF ? 0 : buf + 1;  // the next page's buffer
    const bool masked = !here || hidden(k0);
    bool soon;
    if constexpr (NBUF == 3) {
      stage_scales(then);
      block1(sb, sa, vbuf, vh, buf, 0, yes, then, yes, buf, 1);
      soon = load(t + 2 - t0);
      limits(sa, masked, here, k0);
      block2(sa, sb, buf, 1, buf, 0);
      lds_barrier();  // page t + 1 is there, and the last readers of page t - 1 are done
      block1(sa, sb, buf, 0, buf, 1, no, 0, yes, then, 0);
    } else {
      block1(sb, sa, vbuf, vh, buf, 0, no, 0, yes, buf, 1);
      limits(sa, masked, here, k0);
      block2(sa, sb, buf, 1, buf, 0);
      lds_barrier();  // the other buffer's last readers are done
      stage_scales(then);
      block1(sa, sb, buf, 0, buf, 1, yes, then, no, 0, 0);
      lds_barrier();  // page t + 1 is there
      k_ahead(then, 0);
      soon = load(t + 2 - t0);
    }
    limits(sb, masked, here, k0 + 32);
    block2(sb, sa, then, 0, buf, 1);
    vbuf = buf;
    vh = 1;
    buf = then;
    here = next;
    next = soon;
  }
  block1(sb, sa, vbuf, vh, vbuf, 0, no, 0, no, 0, 0);
  lds_barrier();  // every wave has read the pages
  // The outputs through LDS: rows of D values, 8 a thread, whichever wave they are of.
  constexpr int U = 4;
  const bool plain = used == 1 && p.plain;
  const float lt = l + __shfl_xor(l, 32);
  float* red = lds.red + 32 * wave * RS;
#pragma unroll
  for (int db = 0; db < NB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4_t*>(red + c * RS + 32 * db + 8 * i + 4 * h) =
          f32x4_t{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
  if (h == 0) {  // the pair's row, head, m and l or 1 / l behind its values
    const int row = (wpair + c) / p.G;
    *reinterpret_cast<f32x4_t*>(red + c * RS + D) = f32x4_t{m, used > 1 ? lt : q8_inverse(lt), __int_as_float(row),
                                                            __int_as_float(wpair + c - row * p.G)};
  }
  lds_barrier();
  red = lds.red;
  const int nl = min(WP, pairs - pair0) * (D / 8);
  for (int e0 = tid; e0 < nl; e0 += NT * U) {
    f32x4_t gate[U][2];
    if (used == 1 && p.a.gated) {  // U pieces' gates at once: a store holds back the loads behind it
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int e = min(e0 + NT * k, nl - 1), pl = e / (D / 8), d = 8 * (e % (D / 8));
        const f32x4_t of = *reinterpret_cast<const f32x4_t*>(red + pl * RS + D);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          gate[k][i] = q8_gate(p, (size_t)q.start + __float_as_int(of[2]), g * p.G + __float_as_int(of[3]), d + 4 * i);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int e = e0 + NT * k, pl = e / (D / 8), d = 8 * (e % (D / 8));
      if (e >= nl) break;
      const f32x4_t x0 = *reinterpret_cast<const f32x4_t*>(red + pl * RS + d);
      const f32x4_t x1 = *reinterpret_cast<const f32x4_t*>(red + pl * RS + d + 4);
      const f32x4_t of = *reinterpret_cast<const f32x4_t*>(red + pl * RS + D);
      const size_t row = (size_t)q.start + __float_as_int(of[2]);
      const int head = g * p.G + __float_as_int(of[3]);
      if (plain) {  // rows of bf16, 16 bytes a lane
        const f32x4_t y0 = x0 * of[1], y1 = x1 * of[1];
        *reinterpret_cast<u32x4_t*>(p.a.out + row * p.a.ld_out + head * D + d) =
            u32x4_t{pack_bf2(y0[0], y0[1]), pack_bf2(y0[2], y0[3]), pack_bf2(y1[0], y1[1]), pack_bf2(y1[2], y1[3])};
      } else if (used > 1) {
        q8_partial(p, part, row, head, d, x0, of[0], of[1]);
        q8_partial(p, part, row, head, d + 4, x1, of[0], of[1]);
      } else {
        q8_store(p, row, head, d, x0 * of[1], gate[k][0]);
        q8_store(p, row, head, d + 4, x1 * of[1], gate[k][1]);
      }
    }
  }
}

// Adds the ranges' partial results (4 to 5 us for a few tokens, latency; 1000 gated
// rows of 16 heads of 256 in two ranges 12.5 us, 58 MB at 4.6 TB/s: 33 of partials and
// 16 of gate logits in, 8 out): D / 4 threads for a pair's dims, NG groups of them
// take its ranges in turn (many ranges of few pairs), and meet in LDS.
template <int D, bool TOKENS, int NG>
__global__ __launch_bounds__(256) void q8_join_kernel(AttnQ8Params p) {
  constexpr int TPP = D / 4, PPB = 256 / TPP / NG;  // pairs of a workgroup
  __shared__ __attribute__((aligned(16))) float sums[NG > 1 ? NG : 1][TPP * PPB][4];
  __shared__ float stat[NG > 1 ? NG : 1][PPB][2];
  const int tid = threadIdx.x, d = 4 * (tid % TPP), pl = tid / TPP % PPB, grp = tid / (TPP * PPB);
  const int s = blockIdx.y, u = blockIdx.x * PPB + pl;
  const Q8Seq q = q8_seq(p.kv, s);
  const int r = u / p.a.num_heads, head = u % p.a.num_heads;
  if (blockIdx.x * PPB >= q.n * p.a.num_heads) return;
  int from = 0, to = q.n - 1;  // the rows of its workgroup
  if constexpr (!TOKENS) {
    const int pair0 = (r * p.G + head % p.G) / p.pairs_wg * p.pairs_wg;
    from = min(pair0 / p.G, q.n - 1);
    to = min(q.n - 1, (pair0 + p.pairs_wg - 1) / p.G);
  }
  const int tiles = q8_range(p, q, from, to).tiles, used = q8_parts(p, tiles);
  const bool live = r < q.n && used > 1;
  const size_t row = (size_t)q.start + (live ? r : 0), at = row * p.a.num_heads + head;
  const size_t step = (size_t)p.kv.total_rows * p.a.num_heads;
  float m = kFloor, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  f32x4_t gate = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    gate = q8_gate(p, row, head, d);
    constexpr int U = 4;  // ranges in flight
    for (int i0 = grp; i0 < used; i0 += U * NG) {
      f32x2_t ml[U];
      f32x4_t v[U];
      float mx = m;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = min(i0 + k * NG, used - 1);
        ml[k] = *reinterpret_cast<const f32x2_t*>(p.part_ml + 2 * (at + i * step));
        v[k] = *reinterpret_cast<const f32x4_t*>(p.part + (at + i * step) * D + d);
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i0 + k * NG < used) mx = fmaxf(mx, ml[k][0]);
      const float a = fast_exp2(m - mx);
      m = mx;
      l *= a;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= a;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (i0 + k * NG >= used) continue;
        const float f = fast_exp2(ml[k][0] - m);
        l = fmaf(f, ml[k][1], l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(f, v[k][e], o[e]);
      }
    }
  }
  if constexpr (NG > 1) {
    if (tid % TPP == 0) {
      stat[grp][pl][0] = m;
      stat[grp][pl][1] = l;
    }
    *reinterpret_cast<f32x4_t*>(sums[grp][tid % (TPP * PPB)]) = f32x4_t{o[0], o[1], o[2], o[3]};
    __syncthreads();
    if (grp) return;
    float mt = kFloor;
#pragma unroll
    for (int k = 0; k < NG; ++k) mt = fmaxf(mt, stat[k][pl][0]);
    m = mt;
    l = o[0] = o[1] = o[2] = o[3] = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      const float f = fast_exp2(stat[k][pl][0] - mt);
      l = fmaf(f, stat[k][pl][1], l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, sums[k][tid % (TPP * PPB)][e], o[e]);
    }
  }
  if (live) q8_store(p, row, head, d, f32x4_t{o[0], o[1], o[2], o[3]} * q8_inverse(l), gate);
}

// The launch for a record: which kernel, its grid and key ranges.
struct Plan {
  bool tokens;
  int nc;     // tokens: column blocks of 16 pairs
  int waves;  // of a workgroup
  int blocks, parts, per;
};

size_t part_bytes(const DtreeKvQ8& kv, const DtreeAttnQ8Args& a) {
  return (size_t)kv.total_rows * a.num_heads * (kv.head_dim + 2) * sizeof(float);
}

// Pages of a key range. Tokens: up to kOneRange pages are one range (17 pages, 8
// workgroups: 10.2 us, in two ranges 11.0 with the join; 16 x 20 pages 12.1, 12.8).
// More are cut so that the ranges are as many as the CUs hold at once, two
// workgroups each, if all sequences are as long as the longest (1 x 1025 pages:
// 32.9 us with 16 pages a range, 36.8 with 8; 1 x 125: 13.0 with 8, 16.3 with 32),
// but not longer than kRagged in a batch, where sequences may differ (the host knows
// bounds alone) and short ones leave their ranges empty (32 of up to 129 pages: 30.8
// us, with 16 a range 31.2, with 8 32.1; 64 of up to 32: 19.9, 23.5, 32.0), and no
// more of them than kMost. Rows: as many workgroups as the CUs hold, each sequence
// counted with max_rows rows: a single token beside a chunk has the chunk's ranges
// (one over 65536 keys beside 1000 rows: 1.8 ms, the two in calls of their own 92 us).
constexpr int kOneRange = 24, kMinTokens = 8, kRagged = 12, kMost = 4096, kResident = 512;
// A row block's few pages are one range (4 pages, 128 dims: 14.6 us, in two 15.3;
// 256 dims, with twice the work a page: 3 pages in two 23.3, in one 29.8). More are
// cut down to kMinRows (25 tree rows, 33 pages: 18.4 us, with 4 pages a range 20.2),
// with many row blocks to twice that (128 of 10 pages: 20.8 us, cut finer 22.1).
constexpr int kMinRows = 2, kOneRows = 4, kOneRows256 = 2, kManyRows = 64;
// 8 waves share a page's conversion where they read many (64 pages: 171 us, 4 waves
// 181); 4 start sooner and leave less of a CU idle at the end (20: 45 us, 8 waves 50).
constexpr int kLongPages = 32;

Plan make_plan(const DtreeKvQ8& kv, const DtreeAttnQ8Args& a) {
  const int G = a.num_heads / kv.num_kv_heads, D = kv.head_dim;
  Plan pl{};
  const int64_t pairs = (int64_t)std::max(kv.max_rows, a.rows_padded) * G;
  pl.tokens = pairs <= (D == 256 ? 16 : 32);  // (registers: 32 columns of 256 dims do not fit)
  pl.nc = pairs <= 16 ? 1 : 2;
  // pages that one workgroup's rows can see
  const int64_t end = std::min((int64_t)kv.max_past_length + kv.max_rows, (int64_t)kv.ld_page_table * DTREE_PAGE);
  const int64_t all = (end + DTREE_PAGE - 1) / DTREE_PAGE;
  auto pages = [&](int64_t rows) {
    if (a.window == 0) return all;
    return std::min(all, ((int64_t)a.sink + DTREE_PAGE - 1) / DTREE_PAGE + (a.window + rows) / DTREE_PAGE + 2);
  };
  pl.waves = D == 128 && pairs > 128 && pages(256 / G + 2) >= kLongPages ? 8 : 4;
  const int wp = 32 * pl.waves;  // pairs of a workgroup of rows
  pl.blocks = pl.tokens ? 1 : (int)((pairs + wp - 1) / wp);
  const int64_t tiles = pages(pl.tokens ? kv.max_rows : std::min(kv.max_rows, wp / G + 2));
  const int64_t units = (int64_t)kv.num_seqs * kv.num_kv_heads * pl.blocks;
  auto cut = [](int64_t n, int64_t into) { return (n + into - 1) / into; };
  int64_t per;
  if (pl.tokens) {
    per = std::max<int64_t>(kMinTokens, cut(tiles * units, kResident));
    if (kv.num_seqs > 1) per = std::min<int64_t>(per, kRagged);
    per = tiles <= kOneRange ? tiles : std::max(per, cut(tiles, std::max<int64_t>(1, kMost / units)));
  } else {
    const int64_t fill = D == 256 || pl.waves == 8 ? kResident / 2 : kResident;
    const int64_t least = units > kManyRows ? 2 * kMinRows : kMinRows;
    per = tiles <= (D == 256 ? kOneRows256 : kOneRows)
              ? tiles
              : std::max(least, cut(tiles, std::max<int64_t>(1, fill / units)));
  }
  pl.per = (int)per;
  pl.parts = (int)((tiles + pl.per - 1) / pl.per);
  // Tokens that leave CUs to spare: 8 waves, fewer pages for each (128 workgroups of
  // 20 pages: 11.7 us, 4 waves 12.3; with 256 dims no gain).
  if (pl.tokens && D != 256 && pl.parts * units <= kResident / 2) pl.waves = 8;
  return pl;
}

template <int D, bool TOKENS>
int launch_join(const AttnQ8Params& p, hipStream_t stream) {
  constexpr int NG = 1024 / D;  // groups with one pair a workgroup
  const int64_t pairs = (int64_t)p.kv.max_rows * p.a.num_heads;
  const bool groups = p.parts >= NG;  // a range for each
  const dim3 grid((unsigned)(groups ? pairs : (pairs + NG - 1) / NG), (unsigned)p.kv.num_seqs);
  if (groups) q8_join_kernel<D, TOKENS, NG><<<grid, 256, 0, stream>>>(p);
  else q8_join_kernel<D, TOKENS, 1><<<grid, 256, 0, stream>>>(p);
  DTREE_LAUNCH_CHECK("attention_q8 join launch");
  return DTREE_OK;
}

template <int D>
int launch(const AttnQ8Params& p, const Plan& pl, unsigned grid, hipStream_t stream) {
  if (pl.tokens) {
    if constexpr (D == 256) {
      q8_token_kernel<D, 1, 4><<<grid, 256, 0, stream>>>(p);
    } else if (pl.waves == 8) {
      if (pl.nc == 1) q8_token_kernel<D, 1, 8><<<grid, 512, 0, stream>>>(p);
      else q8_token_kernel<D, 2, 8><<<grid, 512, 0, stream>>>(p);
    } else if (pl.nc == 1) {
      q8_token_kernel<D, 1, 4><<<grid, 256, 0, stream>>>(p);
    } else {
      q8_token_kernel<D, 2, 4><<<grid, 256, 0, stream>>>(p);
    }
  } else if (pl.waves == 4) {
    q8_rows_kernel<D, 4><<<grid, 256, 0, stream>>>(p);
  } else if constexpr (D == 128) {
    q8_rows_kernel<D, 8><<<grid, 512, 0, stream>>>(p);
  }
  DTREE_LAUNCH_CHECK("attention_q8 launch");
  if (p.parts == 1) return DTREE_OK;
  return pl.tokens ? launch_join<D, true>(p, stream) : launch_join<D, false>(p, stream);
}

bool q8_geometry(const DtreeKvQ8& kv, const DtreeAttnQ8Args& a) {
  return kv.num_kv_heads > 0 && a.num_heads > 0 && a.num_heads % kv.num_kv_heads == 0 && a.num_heads <= 1024 &&
         kv.max_rows > 0 && kv.max_rows <= (1 << 24) && kv.num_seqs > 0 && kv.total_rows > 0 && kv.head_dim > 0 &&
         kv.max_past_length >= 0 && kv.ld_page_table > 0 && a.window >= 0 && a.sink >= 0;
}

}  // namespace
}  // namespace dtree

using namespace dtree;

extern "C" size_t dtree_attn_q8_args_bytes(void) { return sizeof(DtreeAttnQ8Args); }

extern "C" size_t dtree_attention_q8_workspace_bytes(const DtreeKvQ8* kv, const DtreeAttnQ8Args* a) {
  if (!kv || !a || !q8_geometry(*kv, *a)) return 0;
  const Plan pl = make_plan(*kv, *a);
  return pl.parts > 1 ? pl.parts * part_bytes(*kv, *a) : 0;
}

extern "C" int dtree_attention_q8(const DtreeKvQ8* kv, const DtreeAttnQ8Args* a, hipStream_t stream) {
  if (int rc = q8_check(kv, "attention_q8")) return rc;
  DTREE_REQUIRE(a, "attention_q8: null args");
  DTREE_REQUIRE(a->q && a->out, "attention_q8: null pointer");
  const int D = kv->head_dim;
  DTREE_REQUIRE(a->window >= 0 && a->sink >= 0 && a->window <= (1 << 28) && a->sink <= (1 << 28),
                "attention_q8: sink and window in [0, 2^28]");
  DTREE_REQUIRE(q8_geometry(*kv, *a), "attention_q8: num_heads a multiple of num_kv_heads, at most 1024");
  DTREE_REQUIRE(a->q_type == DTREE_T_F32 || a->q_type == DTREE_T_BF16, "attention_q8: element type");
  const int run = a->q_type == DTREE_T_BF16 ? 8 : 4, hw = a->gated ? 2 * D : D;
  DTREE_REQUIRE(((uintptr_t)a->q & 15) == 0 && a->q_stride >= hw && a->q_stride % run == 0 && a->q_stride <= (1 << 20) &&
                    a->ld_q % run == 0 && (int64_t)a->ld_q >= (int64_t)(a->num_heads - 1) * a->q_stride + hw,
                "attention_q8: q rows of num_heads heads q_stride apart, 16-byte aligned");
  DTREE_REQUIRE(a->rope_dims >= 0 && a->rope_dims % 32 == 0 && a->rope_dims <= D,
                "attention_q8: rope_dims must be a multiple of 32, at most head_dim");
  DTREE_REQUIRE(a->rope_dims == 0 || (a->rope_cos && a->rope_sin), "attention_q8: null RoPE table");
  DTREE_REQUIRE(a->eps >= 0.f && a->scale > 0.f && a->scale <= 3.4e38f, "attention_q8: eps or scale");
  DTREE_REQUIRE(!a->ancestors || (a->window == 0 && kv->max_rows <= DTREE_MAX_NODES),
                "attention_q8: a draft tree has no window and at most 128 rows");
  const int od = a->num_heads * D;
  const bool tiled = a->out_layout == DTREE_W_TILED || a->out_layout == DTREE_W_TILED_F16;
  DTREE_REQUIRE(((uintptr_t)a->out & 7) == 0 && ((uintptr_t)a->out_lo & 7) == 0 &&
                    (a->out_layout == DTREE_W_ROWMAJOR ? a->ld_out >= od && a->ld_out % 4 == 0
                                                       : tiled && a->ld_out == od),
                "attention_q8: out layout (8-byte aligned; tiled needs ld_out == num_heads * head_dim)");
  DTREE_REQUIRE(a->rows_padded >= 0 && a->rows_padded <= (1 << 20) &&
                    (a->rows_padded == 0 ||
                                    (kv->num_seqs == 1 && !kv->row_starts && a->rows_padded <= kv->total_rows)),
                "attention_q8: rows_padded needs one sequence without row_starts, at most total_rows");
  Plan pl = make_plan(*kv, *a);
  const size_t room = a->workspace && ((uintptr_t)a->workspace & 15) == 0 ? a->workspace_bytes / part_bytes(*kv, *a) : 0;
  if ((size_t)pl.parts > room && pl.parts > 1) {  // fewer, longer ranges; one needs no workspace
    const int64_t tiles = (int64_t)pl.parts * pl.per;
    pl.parts = room > 1 ? (int)room : 1;
    pl.per = (int)((tiles + pl.parts - 1) / pl.parts);
  }
  AttnQ8Params p{};
  p.kv = *kv;
  p.a = *a;
  p.G = a->num_heads / kv->num_kv_heads;
  p.blocks = pl.blocks;
  p.pairs_wg = 32 * pl.waves;
  p.parts = pl.parts;
  p.per = pl.per;
  p.sink_pages = (a->sink + DTREE_PAGE - 1) / DTREE_PAGE;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.part = static_cast<float*>(a->workspace);
  if (p.parts > 1) p.part_ml = p.part + (size_t)p.parts * kv->total_rows * a->num_heads * D;
  p.tiled = tiled;
  p.h16 = a->out_layout == DTREE_W_TILED_F16;
  if (p.h16) p.a.out_lo = nullptr;
  p.plain = !tiled && !p.a.out_lo && !a->gated && ((uintptr_t)a->out & 15) == 0 && a->ld_out % 8 == 0;
  const int64_t grid = (int64_t)kv->num_seqs * pl.blocks * pl.parts * kv->num_kv_heads;
  // (a launch counts its work items in 32 bits; the join has 256 for up to one (row, head))
  DTREE_REQUIRE(64 * pl.waves * grid < (int64_t)1 << 32 && (int64_t)kv->max_rows * a->num_heads < (int64_t)1 << 31 &&
                    (pl.parts == 1 || (kv->num_seqs <= 65535 && kv->max_rows * (int64_t)a->num_heads < 1 << 24)),
                "attention_q8: num_seqs * max_rows too large for one launch");
  if (D == 64) return launch<64>(p, pl, (unsigned)grid, stream);
  if (D == 128) return launch<128>(p, pl, (unsigned)grid, stream);
  return launch<256>(p, pl, (unsigned)grid, stream);
}
