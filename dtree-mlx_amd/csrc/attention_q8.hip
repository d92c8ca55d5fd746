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
// upper part of fp16's range, and taken back in ks.
// A masked key's t is -inf, whatever its scales and bytes are (u = 0 exactly).
#include <algorithm>

#include "kv_q8.h"

namespace dtree {
namespace {

constexpr float kFloor = -3.4e38f;      // m of a row that has seen no key
constexpr float kMinVs = 0x1p-80f;      // value scales below count as this
constexpr float kTop = 6.f, kSlack = 8.f;  // u <= 2^kTop after a rescale, <= 2^(kTop + kSlack) before the next
constexpr int kWaves = 4;

struct AttnQ8Params {
  DtreeKvQ8 kv;
  DtreeAttnQ8Args a;
  int G, blocks;        // heads per group; row blocks per sequence
  int parts, per;       // key ranges the grid holds; pages of a range
  int sink_pages;
  float scale_log2;
  float* part; float* part_ml;  // [parts][total_rows][Hq] x D, x (m, l)
  int tiled, h16;
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

// 16 int8 -> two fragments of eight fp16, exact: 1024 + 128 + q as fp16 bits,
// less 1152.
__device__ __forceinline__ void q8_to_h16(u32x4_t w, u32x4_t& a, u32x4_t& b) {
  const f16x2_t bias = {(_Float16)1152.f, (_Float16)1152.f};
  auto two = [&](uint32_t x, uint32_t sel) {
    const f16x2_t v = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, sel)) - bias;
    return __builtin_bit_cast(uint32_t, v);
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = w[i] ^ 0x80808080u, lo = two(x, 0x04010400u), hi = two(x, 0x04030402u);
    if (i < 2) {
      a[2 * i] = lo;
      a[2 * i + 1] = hi;
    } else {
      b[2 * i - 4] = lo;
      b[2 * i - 3] = hi;
    }
  }
}

// 16 elements of q at dims 16 c .. of a head.
__device__ __forceinline__ void q8_load16(const AttnQ8Params& p, size_t at, float (&x)[16]) {
  if (p.a.q_type == DTREE_T_BF16) {
    const uint16_t* s = static_cast<const uint16_t*>(p.a.q) + at;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4_t w = ld_u32x4(s + 8 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
        x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  } else {
    const float* s = static_cast<const float*>(p.a.q) + at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4_t w = *reinterpret_cast<const f32x4_t*>(s + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = w[j];
    }
  }
}

// 16 norm weights / 16 table entries, at any address of their type.
__device__ __forceinline__ void q8_weights16(const uint16_t* w, float (&x)[16]) {
  u32x4_t v[2];
  __builtin_memcpy(v, w, sizeof(v));
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t b = v[i >> 3][(i >> 1) & 3];
    x[i] = __uint_as_float((i & 1) ? (b & 0xffff0000u) : (b << 16));
  }
}
__device__ __forceinline__ void q8_table16(const float* t, float (&x)[16]) { __builtin_memcpy(x, t, sizeof(x)); }

// Chunk c (dims 16 c ..) of a row's query head: q_norm, RoPE, the softmax scale
// in log2 units; the row's D / 16 chunks are neighbouring lanes. Every load comes
// before the first use (the rotation's other chunk is loaded rather than
// exchanged).
template <int D>
__device__ __forceinline__ void q8_query16(const AttnQ8Params& p, size_t row, int head, int c, float (&x)[16]) {
  const size_t base = row * p.a.ld_q + (size_t)head * p.a.q_stride;
  const int half = p.a.rope_dims / 2, hc = half / 16;  // the rotation's halves, hc chunks each
  const bool turns = c < 2 * hc, low = c < hc, norm = p.a.q_norm != nullptr;
  const int co = low ? c + hc : c - hc;
  float o[16], w[16], wo[16], cs[16], sn[16];
  q8_load16(p, base + 16 * c, x);
  if (norm) q8_weights16(p.a.q_norm + 16 * c, w);
  if (turns) {
    q8_load16(p, base + 16 * co, o);
    if (norm) q8_weights16(p.a.q_norm + 16 * co, wo);
    const size_t at = row * half + 16 * (low ? c : co);
    q8_table16(p.a.rope_cos + at, cs);
    q8_table16(p.a.rope_sin + at, sn);
  }
  float rs = 1.f;
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int k = 1; k < D / 16; k <<= 1) ss += __shfl_xor(ss, k);
    rs = rsqrtf(ss * (1.0f / D) + p.a.eps);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= rs * w[i];
  }
  if (turns) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float y = norm ? o[i] * (rs * wo[i]) : o[i];
      x[i] = low ? x[i] * cs[i] - y * sn[i] : y * sn[i] + x[i] * cs[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] *= p.scale_log2;
}

// 2^e that takes amax into [2^13, 2^14), and its inverse.
__device__ __forceinline__ void q8_exponent(float amax, float& f, float& inv) {
  const int e = (int)(__float_as_uint(amax) >> 23);
  const int ef = amax > 0.f ? min(max(267 - e, 1), 253) : 127;
  f = __uint_as_float((uint32_t)ef << 23);
  inv = __uint_as_float((uint32_t)(254 - ef) << 23);
}

// The queries of up to PAIRS pairs from pair0 on, in fp16 at qs[pair][D + 8]
// (zeros past `pairs`), moved by one power of two for the workgroup; returns its
// inverse. WAVES waves; the barriers wait for LDS alone.
template <int D, int PAIRS, int WAVES>
__device__ __forceinline__ float q8_queries(const AttnQ8Params& p, const Q8Seq& q, int g, int pair0, int pairs,
                                            uint16_t* qs, float* wmax) {
  constexpr int TPR = D / 16, NT = 64 * WAVES, NR = (PAIRS * TPR + NT - 1) / NT;
  const int tid = threadIdx.x;
  float x[NR][16], amax = 0.f;
#pragma unroll
  for (int k = 0; k < NR; ++k) {
    const int u = tid + NT * k, m = pair0 + u / TPR;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[k][i] = 0.f;
    if (m < pairs && u < PAIRS * TPR) {
      q8_query16<D>(p, (size_t)q.start + m / p.G, g * p.G + m % p.G, u % TPR, x[k]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = fabsf(x[k][i]);
        amax = v < INFINITY ? fmaxf(amax, v) : amax;  // (what is not finite stays in its row)
      }
    }
  }
  amax = fmaxf(amax, dpp<0xB1>(amax));
  amax = fmaxf(amax, dpp<0x4E>(amax));
  amax = fmaxf(amax, dpp<0x141>(amax));
  amax = fmaxf(amax, dpp<0x140>(amax));
  amax = fmaxf(amax, swz_xor16(amax));
  amax = fmaxf(amax, __shfl_xor(amax, 32));
  if ((tid & 63) == 0) wmax[tid >> 6] = amax;
  lds_barrier();
#pragma unroll
  for (int k = 0; k < WAVES; ++k) amax = fmaxf(amax, wmax[k]);
  float f, inv;
  q8_exponent(amax, f, inv);
#pragma unroll
  for (int k = 0; k < NR; ++k) {
    const int u = tid + NT * k;
    if (u < PAIRS * TPR) {
      u32x4_t* o = reinterpret_cast<u32x4_t*>(qs + (u / TPR) * (D + 8) + 16 * (u % TPR));
#pragma unroll
      for (int j = 0; j < 2; ++j)
        o[j] = u32x4_t{pack_h2(x[k][8 * j] * f, x[k][8 * j + 1] * f), pack_h2(x[k][8 * j + 2] * f, x[k][8 * j + 3] * f),
                       pack_h2(x[k][8 * j + 4] * f, x[k][8 * j + 5] * f), pack_h2(x[k][8 * j + 6] * f, x[k][8 * j + 7] * f)};
    }
  }
  lds_barrier();
  return inv;
}

// (ks, log2 vs, 1 / vs) of a key. A NaN reaches a row that sees the key through
// ks and log2 vs; 1 / vs stays finite, since a masked key's u = 0 meets it.
__device__ __forceinline__ void q8_scales(float ks, float vs, float inv, float& k, float& lv, float& iv) {
  const float v = vs < kMinVs ? kMinVs : vs;
  k = ks * inv;
  lv = __builtin_amdgcn_logf(v);
  iv = v == v ? 1.f / v : 1.f;
}

// What a lane's row sees.
struct Q8Mask {
  int pos;             // position; -1: the lane has no pair
  int sink, window;    // window 0: all
  bool tree;
  int past, rows;      // draft tree: the prefix, the sequence's rows,
  const uint32_t* anc;  // and the pair's ancestor words in LDS
  __device__ __forceinline__ bool sees(int key) const {
    if (tree) {
      const int n = key - past;
      return pos >= 0 && (n < 0 || (n < rows && ((anc[(n >> 5) & 3] >> (n & 31)) & 1u)));
    }
    return key <= pos && (window == 0 || key < sink || pos - key < window);
  }
};
__device__ __forceinline__ Q8Mask q8_mask(const AttnQ8Params& p, const Q8Seq& q, bool live, int r, const uint32_t* anc) {
  return Q8Mask{live ? q.past + r : -1, p.a.sink, p.a.window, p.a.ancestors != nullptr, q.past, q.n, anc};
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

// One 32-key block: the logits' statistics and weights of a lane's 16 keys
// (acc_row order), the output rescaled where the maximum has grown. `sc`: the
// page's ks, log2 vs and 1 / vs in LDS.
template <int ND>
__device__ __forceinline__ void q8_softmax(f32x16_t& s, const float* sc, int b, int h, bool masked, const Q8Mask& mask,
                                           int k0, float& m, float& l, f32x16_t (&o)[ND], u32x4_t (&ph)[2]) {
  float mx = kFloor;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4_t ks = *reinterpret_cast<const f32x4_t*>(sc + 32 * b + 8 * q + 4 * h);
    const f32x4_t lv = *reinterpret_cast<const f32x4_t*>(sc + 64 + 32 * b + 8 * q + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[4 * q + e] = fmaf(s[4 * q + e], ks[e], lv[e]);
  }
  if (masked) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (!mask.sees(k0 + 32 * b + acc_row(r, h))) s[r] = -INFINITY;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  if (__any(mx > m + (kTop + kSlack))) {
    const float mn = mx > m + (kTop + kSlack) ? mx - kTop : m, alpha = fast_exp2(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int db = 0; db < ND; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4_t iv = *reinterpret_cast<const f32x4_t*>(sc + 128 + 32 * b + 8 * q + 4 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[4 * q + e] = fast_exp2(s[4 * q + e] - m);
      l = fmaf(s[4 * q + e], iv[e], l);
    }
    ph[q >> 1][2 * (q & 1)] = pack_h2(s[4 * q], s[4 * q + 1]);
    ph[q >> 1][2 * (q & 1) + 1] = pack_h2(s[4 * q + 2], s[4 * q + 3]);
  }
}

// Four values of dims d .. of a pair's output, gated, stored.
__device__ __forceinline__ void q8_store(const AttnQ8Params& p, size_t row, int head, int d, float (&y)[4]) {
  const int D = p.kv.head_dim;
  if (p.a.gated) {
    const size_t at = row * p.a.ld_q + (size_t)head * p.a.q_stride + D + d;
    float gt[4];
    if (p.a.q_type == DTREE_T_BF16) {
      const u32x2_t w = *reinterpret_cast<const u32x2_t*>(static_cast<const uint16_t*>(p.a.q) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) gt[e] = __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
    } else {
      const f32x4_t w = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p.a.q) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) gt[e] = w[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = y[e] / (1.0f + __expf(-gt[e]));
  }
  const int col = head * D + d;
  const size_t oi = p.tiled ? tiled_index((int)row, col, p.a.ld_out) : row * p.a.ld_out + col;
  store_act4(p.a.out, p.a.out_lo, oi, y, p.h16);
}
__device__ __forceinline__ void q8_store_zero(const AttnQ8Params& p, size_t row, int head, int d) {
  float y[4] = {0.f, 0.f, 0.f, 0.f};
  const int col = head * p.kv.head_dim + d;
  const size_t oi = p.tiled ? tiled_index((int)row, col, p.a.ld_out) : row * p.a.ld_out + col;
  store_act4(p.a.out, p.a.out_lo, oi, y, p.h16);
}

// Four values of a pair (softmax sum l) to `out`, or unscaled to the range's
// partials.
__device__ __forceinline__ void q8_emit(const AttnQ8Params& p, bool split, int part, size_t row, int head, int d,
                                        const float (&o)[4], float m, float l) {
  if (split) {
    const size_t u = ((size_t)part * p.kv.total_rows + row) * p.a.num_heads + head;
    *reinterpret_cast<f32x4_t*>(p.part + u * p.kv.head_dim + d) = f32x4_t{o[0], o[1], o[2], o[3]};
    if (d == 0) *reinterpret_cast<f32x2_t*>(p.part_ml + 2 * u) = f32x2_t{m, l};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float y[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  q8_store(p, row, head, d, y);
}

__device__ __forceinline__ f32x4_t mfma16_f16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                0);
}

// A workgroup: all pairs of a sequence and KV head, up to 16 NC, over one key
// range, its pages dealt to the four waves in turn. A wave loads its pages
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
template <int D, int NC>
__global__ __launch_bounds__(256, D == 256 ? 1 : NC == 1 ? 3 : 2) void q8_token_kernel(AttnQ8Params p) {
  constexpr int NJ = D / 64, NK = 4 * NJ, ND = D / 16;  // K loads (block, 64 dims) and V loads (16 dims) per page
  constexpr int RS = D + 4;                             // a pair's row in `red`
  union Lds {
    uint16_t q[16 * NC * (D + 8)];
    float red[kWaves * 16 * NC * RS];
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  __shared__ __attribute__((aligned(16))) float scl[kWaves][192];
  __shared__ float mls[kWaves][2][16 * NC];
  __shared__ float wmax[kWaves];
  __shared__ uint32_t anc[16 * NC][DTREE_MASK_WORDS];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hkv = p.kv.num_kv_heads, g = blockIdx.x % Hkv, b0 = blockIdx.x / Hkv;
  const int part = b0 % p.parts, s = b0 / p.parts;
  const Q8Seq q = q8_seq(p.kv, s);
  if (part == 0 && q.n < p.a.rows_padded) {  // rows past the sequence's
    for (int e = tid; e < (p.a.rows_padded - q.n) * p.G * (D / 4); e += 256)
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
    const int t = t0 + wave + kWaves * (i + lane);
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
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) kb[i * NJ + j] = buf_ld(rk, koff + 128 * i + 2048 * j);
    ksl = page < 0 ? 0.f : p.kv.k_scales[block(page) * DTREE_PAGE + lane];
    vsl = page < 0 ? 0.f : p.kv.v_scales[block(page) * DTREE_PAGE + lane];
  };
  auto load_v = [&](int page) {
    const auto rv = buf_rsrc(p.kv.v_pages + block(page) * (DTREE_PAGE * D), page < 0 ? 0 : DTREE_PAGE * D);
#pragma unroll
    for (int i = 0; i < ND; ++i) vb[i] = buf_ld(rv, voff + 1024 * (i >> 1) + 256 * (i & 1));
  };
  const int steps = max(0, (t1 - t0 - wave + kWaves - 1) / kWaves);  // the wave's pages
  int cur = page_of(0);
  load_k(cur);
  q8_ancestors(p, q, 0, 16 * NC, pairs, anc);
  const float inv = q8_queries<D, 16 * NC, kWaves>(p, q, g, 0, pairs, lds.q, wmax);
  load_v(cur);  // (not earlier: the queries' registers)
  u32x4_t qf[NC][2 * NJ];
  Q8Mask mask[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        qf[n][2 * j + k] = *reinterpret_cast<const u32x4_t*>(lds.q + (16 * n + c) * (D + 8) + 64 * j + 16 * kq + 8 * k);
    const bool live = 16 * n + c < pairs;
    mask[n] = q8_mask(p, q, live, (16 * n + c) / p.G, anc[16 * n + c]);
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
    const int k0 = DTREE_PAGE * rg.page(t0 + wave + kWaves * i);
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
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        u32x4_t a0, a1;
        q8_to_h16(kb[b * NJ + j], a0, a1);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          st[n][b] = mfma16_f16(a0, qf[n][2 * j], st[n][b]);
          st[n][b] = mfma16_f16(a1, qf[n][2 * j + 1], st[n][b]);
        }
      }
    load_k(next);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (cur >= 0) {
      const bool masked = mask[0].tree ? k0 + DTREE_PAGE > q.past
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
          for (int e = 0; e < 4; ++e) st[n][b][e] = fmaf(st[n][b][e], ks[e], lv[e]);
        }
        if (masked) {
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!mask[n].sees(k0 + kkey + 8 * b + e)) st[n][b][e] = -INFINITY;
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

  // the four waves' results
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
    for (int w = 0; w < kWaves; ++w) mt = fmaxf(mt, mls[w][0][pr]);
    const float fac = fast_exp2(m[n] - mt);
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<f32x4_t*>(lds.red + (wave * 16 * NC + pr) * RS + 16 * d + 4 * kq) =
          f32x4_t{o[n][d][0] * fac, o[n][d][1] * fac, o[n][d][2] * fac, o[n][d][3] * fac};
  }
  lds_barrier();
  for (int u = tid; u < pairs * (D / 4); u += 256) {
    const int pr = u / (D / 4), d = 4 * (u % (D / 4));
    float mt = kFloor, lt = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mt = fmaxf(mt, mls[w][0][pr]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      lt += mls[w][1][pr] * fast_exp2(mls[w][0][pr] - mt);
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(lds.red + (w * 16 * NC + pr) * RS + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += v[e];
    }
    q8_emit(p, used > 1, part, (size_t)q.start + pr / p.G, g * p.G + pr % p.G, d, y, mt, lt);
  }
}

// A workgroup: 4 x 32 pairs of one KV head, a wave each, over one key range. A
// page is converted to fp16 once for the four waves, on its way from memory to
// LDS, the next one while the current one is used.
template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void q8_rows_kernel(AttnQ8Params p) {
  constexpr int NB = D / 32, PB = DTREE_PAGE * D;       // bytes of a page's K (or V) as int8
  constexpr int NC = PB / 16 / 256;                     // 16-byte pieces of it per thread
  __shared__ __attribute__((aligned(16))) unsigned char kvb[2][4 * PB];  // fp16 K, then V
  __shared__ __attribute__((aligned(16))) float scl[2][192];
  __shared__ float wmax[kWaves];
  __shared__ uint32_t anc[32 * kWaves][DTREE_MASK_WORDS];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Hkv = p.kv.num_kv_heads, g = blockIdx.x % Hkv;
  int bx = blockIdx.x / Hkv;
  const int part = bx % p.parts;
  bx /= p.parts;
  const int w = p.blocks - 1 - bx % p.blocks, s = bx / p.blocks;  // longest ranges first
  const Q8Seq q = q8_seq(p.kv, s);
  const int pairs = q.n * p.G, pair0 = 32 * kWaves * w, pair = pair0 + 32 * wave + c;
  const int r = pair / p.G, head = g * p.G + pair % p.G;
  if (pair0 >= pairs) {  // rows past the sequence's
    if (part == 0 && r < p.a.rows_padded && h == 0)
      for (int d = 0; d < D; d += 4) q8_store_zero(p, r, head, d);
    return;
  }
  const int from = pair0 / p.G, to = min(q.n - 1, (pair0 + 32 * kWaves - 1) / p.G);  // the workgroup's rows
  const Q8Range rg = q8_range(p, q, from, to);
  const int used = q8_parts(p, rg.tiles), per = (rg.tiles + used - 1) / used;
  const int t0 = part * per, t1 = min(rg.tiles, t0 + per);
  if (part >= used) return;
  const bool live = pair < pairs;
  const size_t row = (size_t)q.start + (live ? r : 0);
  const int wfrom = (pair0 + 32 * wave) / p.G, wto = min(q.n - 1, (pair0 + 32 * wave + 31) / p.G);
  const bool wlive = pair0 + 32 * wave < pairs;

  u32x4_t kr[NC], vr[NC];
  float ksl = 0.f, vsl = 0.f;
  auto load = [&](int t) {  // page t's pieces of this thread; false: the page is absent
    const int page = __builtin_amdgcn_readfirstlane(q8_page(p.kv, s, rg.page(t)));
    const size_t blk = (size_t)max(page, 0) * Hkv + g;
    const u32x4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      kr[i] = page >= 0 ? ld_u32x4(p.kv.k_pages + blk * PB + 16 * (tid + 256 * i)) : zero;
      vr[i] = page >= 0 ? ld_u32x4(p.kv.v_pages + blk * PB + 16 * (tid + 256 * i)) : zero;
    }
    if (tid < DTREE_PAGE) {
      ksl = page >= 0 ? p.kv.k_scales[blk * DTREE_PAGE + tid] : 0.f;
      vsl = page >= 0 ? p.kv.v_scales[blk * DTREE_PAGE + tid] : 0.f;
    }
    return page >= 0;
  };
  bool here = load(t0), next = false;
  static_assert(sizeof(kvb) >= 32 * kWaves * (D + 8) * sizeof(uint16_t), "the queries pass through kvb");
  uint16_t* qs = reinterpret_cast<uint16_t*>(&kvb[0][0]);
  q8_ancestors(p, q, pair0, 32 * kWaves, pairs, anc);
  const float inv = q8_queries<D, 32 * kWaves, kWaves>(p, q, g, pair0, pairs, qs, wmax);
  u32x4_t qf[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    qf[i] = *reinterpret_cast<const u32x4_t*>(qs + (32 * wave + c) * (D + 8) + 32 * (i >> 1) + 16 * h + 8 * (i & 1));
  lds_barrier();
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int u = tid + 256 * i;
      unsigned char* at = &kvb[buf][(u >> 6) * 2048 + (u & 63) * 16];
      u32x4_t a0, a1;
      q8_to_h16(kr[i], a0, a1);
      *reinterpret_cast<u32x4_t*>(at) = a0;
      *reinterpret_cast<u32x4_t*>(at + 1024) = a1;
      q8_to_h16(vr[i], a0, a1);
      *reinterpret_cast<u32x4_t*>(at + 2 * PB) = a0;
      *reinterpret_cast<u32x4_t*>(at + 2 * PB + 1024) = a1;
    }
    if (tid < DTREE_PAGE) {
      float k, lv, iv;
      q8_scales(ksl, vsl, inv, k, lv, iv);
      scl[buf][tid] = k;
      scl[buf][64 + tid] = lv;
      scl[buf][128 + tid] = iv;
    }
  };
  const Q8Mask mask = q8_mask(p, q, live, r, anc[32 * wave + c]);
  f32x16_t o[NB];
#pragma unroll
  for (int db = 0; db < NB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float m = kFloor, l = 0.f;
  stage(0);
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, k0 = DTREE_PAGE * rg.page(t);
    if (t + 1 < t1) next = load(t + 1);
    const int wend = q.past + (mask.tree ? q.n - 1 : wto);  // the wave's last key
    const bool need = here && wlive && k0 <= wend &&
                      (p.a.window == 0 || k0 < p.a.sink || k0 + DTREE_PAGE - 1 > q.past + wfrom - p.a.window);
    if (need) {
      const unsigned char* kp = kvb[buf] + 16 * lane;
      const unsigned char* vp = kp + 2 * PB;
      const bool masked = mask.tree ? k0 + DTREE_PAGE > q.past
                                    : k0 + DTREE_PAGE - 1 > q.past + wfrom ||
                                          (p.a.window > 0 && k0 + DTREE_PAGE - 1 >= p.a.sink &&
                                           q.past + wto - k0 >= p.a.window);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x16_t st;
#pragma unroll
        for (int i = 0; i < 16; ++i) st[i] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
          st = mfma32_f16(*reinterpret_cast<const u32x4_t*>(kp + (b * 2 * NB + i) * 1024), qf[i], st);
        u32x4_t ph[2];
        q8_softmax<NB>(st, scl[buf], b, h, masked, mask, k0, m, l, o, ph);
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            o[db] = mfma32_f16(*reinterpret_cast<const u32x4_t*>(vp + ((b * NB + db) * 2 + i) * 1024), ph[i], o[db]);
      }
    }
    if (t + 1 < t1) stage(buf ^ 1);
    here = next;
    __syncthreads();
  }
  l += __shfl_xor(l, 32);
  if (live) {
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y[4] = {o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
        q8_emit(p, used > 1, part, row, head, 32 * db + 8 * i + 4 * h, y, m, l);
      }
  } else if (part == 0 && r < p.a.rows_padded && h == 0) {
    for (int d = 0; d < D; d += 4) q8_store_zero(p, r, head, d);
  }
}

// Adds the ranges' partial results: D / 4 threads for a pair's dims, NG groups of
// them take its ranges in turn (many ranges of few pairs), and meet in LDS.
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
    const int pair0 = (r * p.G + head % p.G) / (32 * kWaves) * (32 * kWaves);
    from = min(pair0 / p.G, q.n - 1);
    to = min(q.n - 1, (pair0 + 32 * kWaves - 1) / p.G);
  }
  const int tiles = q8_range(p, q, from, to).tiles, used = q8_parts(p, tiles);
  const bool live = r < q.n && used > 1;
  const size_t row = (size_t)q.start + (live ? r : 0), at = row * p.a.num_heads + head;
  const size_t step = (size_t)p.kv.total_rows * p.a.num_heads;
  float m = kFloor, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  if (live) {
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
  if (live) q8_emit(p, false, 0, row, head, d, o, m, l);
}

// The launch for a record: which kernel, its grid and key ranges.
struct Plan {
  bool tokens;
  int blocks, parts, per;
};

size_t part_bytes(const DtreeKvQ8& kv, const DtreeAttnQ8Args& a) {
  return (size_t)kv.total_rows * a.num_heads * (kv.head_dim + 2) * sizeof(float);
}

// Workgroups the key ranges are cut for, and the fewest pages of a range.
constexpr int kFillTokens = 2048, kFillRows = 512;
constexpr int kMinTokens = 16, kMinRows = 4;

Plan make_plan(const DtreeKvQ8& kv, const DtreeAttnQ8Args& a) {
  const int G = a.num_heads / kv.num_kv_heads;
  Plan pl{};
  const int64_t pairs = (int64_t)std::max(kv.max_rows, a.rows_padded) * G;
  pl.tokens = pairs <= (kv.head_dim == 256 ? 16 : 32);  // (registers: 32 columns of 256 dims do not fit)
  pl.blocks = pl.tokens ? 1 : (int)((pairs + 32 * kWaves - 1) / (32 * kWaves));
  // pages that one workgroup's rows can see
  const int64_t end = std::min((int64_t)kv.max_past_length + kv.max_rows, (int64_t)kv.ld_page_table * DTREE_PAGE);
  int64_t tiles = (end + DTREE_PAGE - 1) / DTREE_PAGE;
  if (a.window > 0) {
    const int64_t span = pl.tokens ? kv.max_rows : std::min(kv.max_rows, 32 * kWaves / G + 2);
    tiles = std::min(tiles, ((int64_t)a.sink + DTREE_PAGE - 1) / DTREE_PAGE + (a.window + span) / DTREE_PAGE + 2);
  }
  const int64_t units = (int64_t)kv.num_seqs * kv.num_kv_heads * pl.blocks;
  const int64_t most = std::max<int64_t>(1, (pl.tokens ? kFillTokens : kFillRows) / units);
  pl.per = (int)std::max<int64_t>(pl.tokens ? kMinTokens : kMinRows, (tiles + most - 1) / most);
  pl.parts = (int)((tiles + pl.per - 1) / pl.per);
  return pl;
}

template <int D, bool TOKENS>
int launch_join(const AttnQ8Params& p, hipStream_t stream) {
  constexpr int NG = 1024 / D;  // groups with one pair a workgroup
  const int64_t pairs = (int64_t)p.kv.max_rows * p.a.num_heads;
  // Groups pay where there are ranges for them to share.
  const bool groups = p.parts >= 2 * NG;
  const dim3 grid((unsigned)(groups ? pairs : (pairs + NG - 1) / NG), (unsigned)p.kv.num_seqs);
  if (groups) q8_join_kernel<D, TOKENS, NG><<<grid, 256, 0, stream>>>(p);
  else q8_join_kernel<D, TOKENS, 1><<<grid, 256, 0, stream>>>(p);
  DTREE_LAUNCH_CHECK("attention_q8 join launch");
  return DTREE_OK;
}

template <int D>
int launch(const AttnQ8Params& p, bool tokens, unsigned grid, hipStream_t stream) {
  if (!tokens) q8_rows_kernel<D><<<grid, 256, 0, stream>>>(p);
  else if (D == 256 || std::max(p.kv.max_rows, p.a.rows_padded) * p.G <= 16)
    q8_token_kernel<D, 1><<<grid, 256, 0, stream>>>(p);
  else if constexpr (D != 256) q8_token_kernel<D, 2><<<grid, 256, 0, stream>>>(p);
  DTREE_LAUNCH_CHECK("attention_q8 launch");
  if (p.parts == 1) return DTREE_OK;
  return tokens ? launch_join<D, true>(p, stream) : launch_join<D, false>(p, stream);
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
  p.parts = pl.parts;
  p.per = pl.per;
  p.sink_pages = (a->sink + DTREE_PAGE - 1) / DTREE_PAGE;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.part = static_cast<float*>(a->workspace);
  if (p.parts > 1) p.part_ml = p.part + (size_t)p.parts * kv->total_rows * a->num_heads * D;
  p.tiled = tiled;
  p.h16 = a->out_layout == DTREE_W_TILED_F16;
  if (p.h16) p.a.out_lo = nullptr;
  const int64_t grid = (int64_t)kv->num_seqs * pl.blocks * pl.parts * kv->num_kv_heads;
  DTREE_REQUIRE(grid < (int64_t)1 << 31 && (int64_t)kv->max_rows * a->num_heads < (int64_t)1 << 31 &&
                    (pl.parts == 1 || kv->num_seqs <= 65535),
                "attention_q8: num_seqs * max_rows too large for one launch");
  if (D == 64) return launch<64>(p, pl.tokens, (unsigned)grid, stream);
  if (D == 128) return launch<128>(p, pl.tokens, (unsigned)grid, stream);
  return launch<256>(p, pl.tokens, (unsigned)grid, stream);
}
