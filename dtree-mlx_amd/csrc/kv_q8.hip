// The 8-bit paged KV cache: rows in (the cache append of qwen3_tree.py:146 with
// the k_norm and RoPE before it, :57-62), rows out, and the accepted path's move
// (adapters.py:635-668).
//
// A row is quantised as scale = fp32(max |x| / 127), q = nearest integer of
// x / scale, ties to even. Everything before the rounding to q is fp64: V rows and
// K rows without norm and rotation give the definition's bytes exactly, others x
// within 1e-15 of its value, so that q differs only at borders met by less.
//
// Long runs are bound by the bytes they move, a single row by latency. A
// workgroup owns half a page (32 positions, whole 16-byte pieces of K and of V) of
// one kv head. The rows' side is read and written in runs of their dims, the
// pages' side in runs of their pieces, and LDS, rows of bytes, lies between (without
// it, V's bytes one by one, 4000 rows in and out took 43 us, now 23).
// Measured, 8 heads of 128: 4000 fp32 rows in 13.4 to 15 us (58 MB moved; waves wait
// 61 % of the time, the fp64 arithmetic takes 54 % of the issue), bf16 rows 12.4, and
// back in 9.3 us (4.4 TB/s); 4 x 8192 rows of 256 dims to bf16 28.1 us (120 MB, 4.3
// TB/s, of 4.8 that a copy reaches). Of the 49 MB that the append reads 35 are
// needed: with 8 heads each is on an XCD of its own, and each reads the rows'
// rotations. One row: append 6.0 us, read 3.2, the fp64 chain's latency between them.
#include <cmath>
#include <type_traits>

#include "kv_q8.h"

namespace dtree {
namespace {

constexpr int kHalf = DTREE_PAGE / 2;

// Half pages that max_rows positions from anywhere in one can touch.
int span_halves(const DtreeKvQ8& kv) { return (kv.max_rows + kHalf - 2) / kHalf + 1; }

// This workgroup's half page: its page, the sequence's row in its slot 0, its live
// slots lo .. hi - 1 (none: lo >= hi).
struct Half {
  int page, b, first, lo, hi;
  size_t row0;  // buffer row of the sequence's row 0
};
__device__ __forceinline__ Half q8_half(const DtreeKvQ8& kv, int block, int span) {
  const int s = block / span;
  const Q8Seq q = q8_seq(kv, s);
  const int i = q.past / kHalf + block % span;
  Half w{-1, i & 1, i * kHalf - q.past, 0, 0, (size_t)q.start};
  w.lo = max(0, -w.first);
  w.hi = min(kHalf, q.n - w.first);
  if (w.lo < w.hi) w.page = q8_page(kv, s, i >> 1);
  return w;
}

// Four rows' words of four bytes -> four columns' words.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t t0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), t1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t u0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), u1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(u0, t0, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(u0, t0, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(u1, t1, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(u1, t1, 0x07060302u);
}

struct Q8AppendParams {
  DtreeKvQ8 kv;
  const void* k; const void* v;
  int ld_k, ld_v, span, rope_dims;
  const uint16_t* k_norm;
  const float* cos; const float* sin;
  double eps;
};

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)dpp_i<CTRL>((int)(uint32_t)b), hi = (uint32_t)dpp_i<CTRL>((int)(uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double swz64_xor16(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)swz_xor16_i((int)(uint32_t)b), hi = (uint32_t)swz_xor16_i((int)(uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum or maximum over TPR neighbouring lanes, in each of them.
template <int TPR, class F>
__device__ __forceinline__ double over_row(double v, F f) {
  v = f(v, dpp64<0xB1>(v));
  v = f(v, dpp64<0x4E>(v));
  v = f(v, dpp64<0x141>(v));
  if constexpr (TPR >= 16) v = f(v, dpp64<0x140>(v));
  if constexpr (TPR >= 32) v = f(v, swz64_xor16(v));
  return v;
}
// 1 / sqrt(a) and 1 / a, two Newton steps (2^-52) on the hardware's estimates.
__device__ __forceinline__ double rsqrt64(double a) {
  double r = __builtin_amdgcn_rsq(a);
#pragma unroll
  for (int i = 0; i < 2; ++i) r = fma(r * fma(-a * r, r, 1.0), 0.5, r);
  return r;
}
__device__ __forceinline__ double rcp64(double a) {
  double r = __builtin_amdgcn_rcp(a);
#pragma unroll
  for (int i = 0; i < 2; ++i) r = fma(fma(-a, r, 1.0), r, r);
  return r;
}

// A row's bytes (this lane's two pieces) and scale. Not finite anywhere (or beyond
// what an fp32 scale can stand for): scale NaN, bytes 0. x / scale as x times a
// rounded reciprocal may fall beside a border that it lies on (73.5 / 49); one
// correction by the remainder, which fp64 holds whole for rows of 24 bits, makes
// every quotient that ends in 1 / 2 exact, so that the tie goes to even.
template <int TPR>
__device__ __forceinline__ void quantise(const double (&x)[8], uint32_t (&w)[2], float& scale) {
  constexpr double kMost = 4.3e40;  // fp32's largest times 127, less a little
  double amax = 0.;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double a = fabs(x[i]);
    bad |= !(a <= kMost);
    amax = fmax(amax, a);
  }
  amax = over_row<TPR>(bad ? (double)INFINITY : amax, [](double a, double b) { return fmax(a, b); });
  const bool fine = amax <= kMost;
  scale = fine ? (float)(amax * (1.0 / 127.0)) : NAN;
  const double by = (double)scale, inv = scale > 0.f ? rcp64(by) : 0.;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double t = x[4 * i + e] * inv, r = rint(fma(fma(-t, by, x[4 * i + e]), inv, t));
      // (clamped: a subnormal scale may have been rounded by more than 1 / 254)
      const int q = fine ? min(max((int)r, -127), 127) : 0;
      w[i] |= (uint32_t)(q & 0xff) << (8 * e);
    }
  }
}

template <int D, bool BF16>
__global__ __launch_bounds__(256) void q8_append_kernel(Q8AppendParams p) {
  constexpr int TPR = D / 8, RPP = 256 / TPR;  // lanes a row; rows a pass
  constexpr int LS = D / 4 + 4;                // words of a row in LDS, 16-byte pieces on their own banks
  __shared__ __attribute__((aligned(16))) uint32_t lds[2][kHalf][LS];  // K rows, V rows
  const int g = blockIdx.x % p.kv.num_kv_heads;
  const int tid = threadIdx.x, j = tid % TPR, half = p.rope_dims / 2;
  const Q8Pieces pc = q8_pieces<D>(p.rope_dims, j);
  f32x4_t w0 = {1.f, 1.f, 1.f, 1.f}, w1 = w0;
  if (p.k_norm) {  // (tables and weights at any address of their type)
    u32x2_t a, b;
    __builtin_memcpy(&a, p.k_norm + pc.at[0], 8);
    __builtin_memcpy(&b, p.k_norm + pc.at[1], 8);
    w0 = q8_bf4(a);
    w1 = q8_bf4(b);
  }
  const Half w = q8_half(p.kv, blockIdx.x / p.kv.num_kv_heads, p.span);
  if (w.lo >= w.hi) return;
  const size_t blk = (size_t)w.page * p.kv.num_kv_heads + g;
  const int n = w.hi - w.lo, at0 = g * D + pc.at[0], at1 = g * D + pc.at[1];
  // K rows, then V rows
  for (int i = tid / TPR; i < 2 * n; i += RPP) {
    const bool is_k = i < n;
    const int slot = w.lo + (is_k ? i : i - n);
    const size_t row = w.row0 + w.first + slot;
    const size_t base = row * (is_k ? p.ld_k : p.ld_v);
    // One round of loads: what does not rotate reads its row in the tables' place.
    using T = std::conditional_t<BF16, uint16_t, float>;
    const T* src = static_cast<const T*>(is_k ? p.k : p.v) + base;
    const bool turns = is_k && pc.turns;
    const size_t tab = row * half + 4 * j;
    const void* tc = turns ? static_cast<const void*>(p.cos + tab) : src + g * D;
    const void* ts = turns ? static_cast<const void*>(p.sin + tab) : src + g * D;
    f32x4_t x0, x1, cs, sn;
    if constexpr (BF16) {
      const u32x2_t a = *reinterpret_cast<const u32x2_t*>(src + at0), b = *reinterpret_cast<const u32x2_t*>(src + at1);
      __builtin_memcpy(&cs, tc, 16);
      __builtin_memcpy(&sn, ts, 16);
      x0 = q8_bf4(a);
      x1 = q8_bf4(b);
    } else {
      x0 = *reinterpret_cast<const f32x4_t*>(src + at0);
      x1 = *reinterpret_cast<const f32x4_t*>(src + at1);
      __builtin_memcpy(&cs, tc, 16);
      __builtin_memcpy(&sn, ts, 16);
    }
    double x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = x0[e];
      x[4 + e] = x1[e];
    }
    if (is_k && p.k_norm) {
      double ss = 0.;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fma(x[e], x[e], ss);
      ss = over_row<TPR>(ss, [](double a, double b) { return a + b; });
      const double rs = rsqrt64(ss * (1.0 / D) + p.eps);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] *= rs * w0[e];
        x[4 + e] *= rs * w1[e];
      }
    }
    if (turns) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double a = x[e], b = x[4 + e];
        x[e] = a * cs[e] - b * sn[e];
        x[4 + e] = a * sn[e] + b * cs[e];
      }
    }
    uint32_t q[2];
    float scale;
    quantise<TPR>(x, q, scale);
    uint32_t* o = lds[is_k ? 0 : 1][slot];
    o[pc.at[0] / 4] = q[0];
    o[pc.at[1] / 4] = q[1];
    if (j == 0 && w.page >= 0) (is_k ? p.kv.k_scales : p.kv.v_scales)[blk * DTREE_PAGE + w.b * kHalf + slot] = scale;
  }
  __syncthreads();
  if (w.page < 0) return;  // (not before: the page's number comes behind the rows)
  int8_t* kp = p.kv.k_pages + blk * (DTREE_PAGE * D) + w.b * kHalf * D;
  int8_t* vp = p.kv.v_pages + blk * (DTREE_PAGE * D) + w.b * kHalf * D;
  // K: piece u = (dims 16 (u / 32) .., slot u % 32)
#pragma unroll
  for (int u = tid; u < 2 * D; u += 256) {
    const int slot = u & 31;
    if (slot >= w.lo && slot < w.hi)
      *reinterpret_cast<u32x4_t*>(kp + 16 * u) = ld_u32x4(&lds[0][slot][4 * (u >> 5)]);
  }
  // V: four dims of a 4-slot parity; what other rows own of a piece stays.
  for (int u = tid; u < D / 2; u += 256) {
    const int dq = u % (D / 4), h = u / (D / 4), d = 4 * dq;
    uint32_t v[4][4];  // [slots 8 i + 4 h ..][dims d ..]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = lds[1][8 * i + 4 * h + e][dq];
      transpose4(v[i]);
    }
    int8_t* o = vp + (((d >> 5) * 64 + 32 * h + (d & 31)) << 4);
    if (w.lo <= 4 * h && w.hi >= 28 + 4 * h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<u32x4_t*>(o + 16 * e) = u32x4_t{v[0][e], v[1][e], v[2][e], v[3][e]};
      continue;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int sl = 8 * i + 4 * h;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (sl >= w.lo && sl + 3 < w.hi) {
          *reinterpret_cast<uint32_t*>(o + 16 * e + 4 * i) = v[i][e];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (sl + k >= w.lo && sl + k < w.hi) o[16 * e + 4 * i + k] = (int8_t)(v[i][e] >> (8 * k));
        }
      }
    }
  }
}

struct Q8ReadParams {
  DtreeKvQ8 kv;
  void* k; void* v;
  int ld_k, ld_v, span;
};

template <int D, bool BF16>
__global__ __launch_bounds__(256) void q8_read_kernel(Q8ReadParams p) {
  constexpr int EPT = BF16 ? 8 : 4, TPR = D / EPT, RPP = 256 / TPR;  // 16 bytes out a lane
  constexpr int LS = D / 4 + 4;
  __shared__ __attribute__((aligned(16))) uint32_t lds[2][kHalf][LS];
  __shared__ float sc[2][kHalf];
  const int g = blockIdx.x % p.kv.num_kv_heads;
  const Half w = q8_half(p.kv, blockIdx.x / p.kv.num_kv_heads, p.span);
  if (w.lo >= w.hi) return;
  const bool here = w.page >= 0;
  const size_t blk = (size_t)max(w.page, 0) * p.kv.num_kv_heads + g;
  const int tid = threadIdx.x;
  const int8_t* kb = p.kv.k_pages + blk * (DTREE_PAGE * D) + w.b * kHalf * D;
  const int8_t* vb = p.kv.v_pages + blk * (DTREE_PAGE * D) + w.b * kHalf * D;
  const u32x4_t zero = {0, 0, 0, 0};
  if (tid < 2 * kHalf) {
    const float* s = (tid < kHalf ? p.kv.k_scales : p.kv.v_scales) + blk * DTREE_PAGE + w.b * kHalf;
    sc[tid / kHalf][tid % kHalf] = here ? s[tid % kHalf] : 0.f;
  }
  if (p.k) {
#pragma unroll
    for (int u = tid; u < 2 * D; u += 256)
      *reinterpret_cast<u32x4_t*>(&lds[0][u & 31][4 * (u >> 5)]) = here ? ld_u32x4(kb + 16 * u) : zero;
  }
  if (p.v) {
    for (int u = tid; u < D / 2; u += 256) {
      const int dq = u % (D / 4), h = u / (D / 4), d = 4 * dq;
      const int8_t* o = vb + (((d >> 5) * 64 + 32 * h + (d & 31)) << 4);
      u32x4_t v[4];  // [dim d + e][slots 8 i + 4 h ..]
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = here ? ld_u32x4(o + 16 * e) : zero;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t t[4] = {v[0][i], v[1][i], v[2][i], v[3][i]};
        transpose4(t);
#pragma unroll
        for (int e = 0; e < 4; ++e) lds[1][8 * i + 4 * h + e][dq] = t[e];
      }
    }
  }
  __syncthreads();
  const int n = w.hi - w.lo, j = tid % TPR;
  const int from = p.k ? 0 : n, to = p.v ? 2 * n : n;  // K rows, then V rows
  for (int i = from + tid / TPR; i < to; i += RPP) {
    const bool is_k = i < n;
    const int slot = w.lo + (is_k ? i : i - n), which = is_k ? 0 : 1;
    const size_t at = (w.row0 + w.first + slot) * (is_k ? p.ld_k : p.ld_v) + g * D + EPT * j;
    const float scale = sc[which][slot];
    float y[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const uint32_t x = lds[which][slot][EPT / 4 * j + e / 4];
      y[e] = (float)((int)(x << (24 - 8 * (e & 3))) >> 24) * scale;
    }
    void* out = is_k ? p.k : p.v;
    if constexpr (BF16)
      *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(out) + at) =
          u32x4_t{pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]), pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7])};
    else *reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + at) = f32x4_t{y[0], y[1], y[2], y[3]};
  }
}

constexpr int kHidBlocks = 16;  // workgroups of the hidden rows' select

// The accepted rows of one (layer, kv head), K or V, through LDS: a row's place
// may be another accepted row's source. At most 128 rows: bound by latency, hence
// a workgroup for each, and V's bytes one by one (5 rows of 36 layers of 8 heads of
// 128: 7.5 us).
__global__ __launch_bounds__(256) void q8_compact_kernel(const DtreeStepDesc* desc, int8_t* kp, int8_t* vp, float* ks,
                                                         float* vs, int layers, int num_pages, int Hkv, int D,
                                                         const int32_t* page_table, int table_pages,
                                                         const uint16_t* hid_in, int hid_w, uint16_t* hid_out) {
  __shared__ u32x4_t buf[DTREE_MAX_NODES * 16];  // up to 256 bytes a row
  __shared__ float sc[DTREE_MAX_NODES];
  __shared__ int src[DTREE_MAX_NODES], dst[DTREE_MAX_NODES];  // page * 64 + slot, -1: none
  const int n = min(max(desc->n_accepted, 0), DTREE_MAX_NODES), P = desc->past_length, L = desc->num_nodes;
  const int nkv = layers * Hkv, b = blockIdx.x, t = threadIdx.x;
  if (b >= 2 * nkv) {
    const int nch = hid_w / 8;
    for (int e = (b - 2 * nkv) * 256 + t; e < n * nch; e += kHidBlocks * 256) {
      const int j = e / nch, ch = e % nch, a = min(max(desc->accepted[j], 0), DTREE_MAX_NODES - 1);
      *reinterpret_cast<u32x4_t*>(hid_out + (size_t)j * hid_w + 8 * ch) =
          *reinterpret_cast<const u32x4_t*>(hid_in + (size_t)a * hid_w + 8 * ch);
    }
    return;
  }
  if (n >= L || P < 0) return;  // every tree row kept in place
  auto place = [&](int pos) {
    if (pos < 0 || pos / DTREE_PAGE >= table_pages) return -1;
    const int page = page_table[pos / DTREE_PAGE];
    return page >= 0 && page < num_pages ? page * DTREE_PAGE + pos % DTREE_PAGE : -1;
  };
  if (t < n) {
    src[t] = place(P + desc->accepted[t]);
    dst[t] = place(P + t);
  }
  __syncthreads();
  const int layer = b % nkv / Hkv, g = b % Hkv;
  const size_t pool = (size_t)layer * num_pages * Hkv;
  auto block = [&](int r) { return pool + (size_t)(r / DTREE_PAGE) * Hkv + g; };
  const bool is_k = b < nkv;
  float* scales = is_k ? ks : vs;
  uint8_t* bytes = reinterpret_cast<uint8_t*>(is_k ? kp : vp);
  uint8_t* vb = reinterpret_cast<uint8_t*>(buf);
  const int pieces = is_k ? D / 16 : D;  // a row's 16-byte pieces, or its bytes
  for (int e = t; e < n * pieces; e += 256) {
    const int j = e / pieces, c = e % pieces, r = src[j];
    if (r < 0) continue;
    const uint8_t* at = bytes + block(r) * (DTREE_PAGE * D);
    if (is_k) buf[j * 16 + c] = ld_u32x4(at + q8_k_off(r % DTREE_PAGE, 16 * c, D));
    else vb[j * 256 + c] = at[q8_v_off(r % DTREE_PAGE, c, D)];
    if (c == 0) sc[j] = scales[block(r) * DTREE_PAGE + r % DTREE_PAGE];
  }
  __syncthreads();
  for (int e = t; e < n * pieces; e += 256) {
    const int j = e / pieces, c = e % pieces, r = dst[j];
    if (r < 0 || src[j] < 0) continue;
    uint8_t* at = bytes + block(r) * (DTREE_PAGE * D);
    if (is_k) *reinterpret_cast<u32x4_t*>(at + q8_k_off(r % DTREE_PAGE, 16 * c, D)) = buf[j * 16 + c];
    else at[q8_v_off(r % DTREE_PAGE, c, D)] = vb[j * 256 + c];
    if (c == 0) scales[block(r) * DTREE_PAGE + r % DTREE_PAGE] = sc[j];
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int q8_check(const DtreeKvQ8* kv, const char* what) {
  const std::string w(what);
  DTREE_REQUIRE(kv, w + ": null cache record");
  DTREE_REQUIRE(kv->k_pages && kv->v_pages && kv->k_scales && kv->v_scales && kv->page_tables && kv->past_lengths &&
                    kv->row_counts,
                w + ": null pointer in the cache record");
  DTREE_REQUIRE(aligned16(kv->k_pages) && aligned16(kv->v_pages) && aligned16(kv->k_scales) && aligned16(kv->v_scales),
                w + ": pages and scales must be 16-byte aligned");
  DTREE_REQUIRE(kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256, w + ": head_dim 64, 128 or 256");
  DTREE_REQUIRE(kv->num_kv_heads >= 1 && kv->num_kv_heads <= 256 && kv->num_pages >= 1 && kv->num_pages <= (1 << 25),
                w + ": num_kv_heads in [1, 256], num_pages in [1, 2^25]");
  DTREE_REQUIRE(kv->num_seqs >= 1 && kv->num_seqs <= (1 << 16), w + ": num_seqs in [1, 65536]");
  DTREE_REQUIRE(kv->max_rows >= 1 && kv->max_rows <= (1 << 24) && kv->max_past_length >= 0 &&
                    kv->max_past_length <= (1 << 28),
                w + ": max_rows in [1, 2^24], max_past_length in [0, 2^28]");
  DTREE_REQUIRE(kv->total_rows >= 1 && kv->total_rows <= (1 << 28), w + ": total_rows in [1, 2^28]");
  DTREE_REQUIRE(kv->row_starts || (int64_t)kv->num_seqs * kv->max_rows <= (1 << 28),
                w + ": num_seqs * max_rows beyond 2^28 rows without row_starts");
  DTREE_REQUIRE(kv->ld_page_table >= 1 && kv->ld_page_table <= (1 << 24) &&
                    kv->max_past_length <= (int64_t)kv->ld_page_table * DTREE_PAGE,
                w + ": page tables of 1 to 2^24 pages must cover max_past_length positions");
  return DTREE_OK;
}

}  // namespace dtree

using namespace dtree;

extern "C" size_t dtree_kv_q8_bytes(void) { return sizeof(DtreeKvQ8); }

static int row_buffer_check(const DtreeKvQ8* kv, const void* p, int ld, int type, const std::string& what) {
  const int run = type == DTREE_T_BF16 ? 8 : 4;  // elements of 16 bytes
  DTREE_REQUIRE(((uintptr_t)p & 15) == 0 && ld % run == 0 && ld >= kv->num_kv_heads * kv->head_dim,
                what + ": rows of num_kv_heads * head_dim elements, 16-byte aligned");
  return DTREE_OK;
}

static int grid_of(const DtreeKvQ8* kv, const std::string& what, unsigned* grid) {
  const int64_t n = (int64_t)kv->num_seqs * span_halves(*kv) * kv->num_kv_heads;
  DTREE_REQUIRE(256 * n < (int64_t)1 << 32, what + ": num_seqs * max_rows too large for one launch");  // work items
  *grid = (unsigned)n;
  return DTREE_OK;
}

extern "C" int dtree_kv_q8_append(const DtreeKvQ8* kv, const void* k, const void* v, int32_t type, int32_t ld_k,
                                  int32_t ld_v, const uint16_t* k_norm, float eps, const float* rope_cos,
                                  const float* rope_sin, int32_t rope_dims, hipStream_t stream) {
  if (int rc = q8_check(kv, "kv_q8_append")) return rc;
  DTREE_REQUIRE(k && v, "kv_q8_append: null pointer");
  DTREE_REQUIRE(type == DTREE_T_F32 || type == DTREE_T_BF16, "kv_q8_append: element type");
  if (int rc = row_buffer_check(kv, k, ld_k, type, "kv_q8_append: k")) return rc;
  if (int rc = row_buffer_check(kv, v, ld_v, type, "kv_q8_append: v")) return rc;
  DTREE_REQUIRE(rope_dims >= 0 && rope_dims % 32 == 0 && rope_dims <= kv->head_dim,
                "kv_q8_append: rope_dims must be a multiple of 32, at most head_dim");
  DTREE_REQUIRE(rope_dims == 0 || (rope_cos && rope_sin), "kv_q8_append: null RoPE table");
  DTREE_REQUIRE(eps >= 0.f, "kv_q8_append: eps");
  unsigned grid;
  if (int rc = grid_of(kv, "kv_q8_append", &grid)) return rc;
  const Q8AppendParams p{*kv, k, v, ld_k, ld_v, span_halves(*kv), rope_dims, k_norm, rope_cos, rope_sin, (double)eps};
  const bool bf = type == DTREE_T_BF16;
  if (kv->head_dim == 64) {
    if (bf) q8_append_kernel<64, true><<<grid, 256, 0, stream>>>(p);
    else q8_append_kernel<64, false><<<grid, 256, 0, stream>>>(p);
  } else if (kv->head_dim == 128) {
    if (bf) q8_append_kernel<128, true><<<grid, 256, 0, stream>>>(p);
    else q8_append_kernel<128, false><<<grid, 256, 0, stream>>>(p);
  } else {
    if (bf) q8_append_kernel<256, true><<<grid, 256, 0, stream>>>(p);
    else q8_append_kernel<256, false><<<grid, 256, 0, stream>>>(p);
  }
  DTREE_LAUNCH_CHECK("kv_q8_append launch");
  return DTREE_OK;
}

extern "C" int dtree_kv_q8_read(const DtreeKvQ8* kv, void* k, void* v, int32_t type, int32_t ld_k, int32_t ld_v,
                                hipStream_t stream) {
  if (int rc = q8_check(kv, "kv_q8_read")) return rc;
  DTREE_REQUIRE(k || v, "kv_q8_read: null pointer");
  DTREE_REQUIRE(type == DTREE_T_F32 || type == DTREE_T_BF16, "kv_q8_read: element type");
  if (k)
    if (int rc = row_buffer_check(kv, k, ld_k, type, "kv_q8_read: k")) return rc;
  if (v)
    if (int rc = row_buffer_check(kv, v, ld_v, type, "kv_q8_read: v")) return rc;
  unsigned grid;
  if (int rc = grid_of(kv, "kv_q8_read", &grid)) return rc;
  const Q8ReadParams p{*kv, k, v, ld_k, ld_v, span_halves(*kv)};
  const bool bf = type == DTREE_T_BF16;
  if (kv->head_dim == 64) {
    if (bf) q8_read_kernel<64, true><<<grid, 256, 0, stream>>>(p);
    else q8_read_kernel<64, false><<<grid, 256, 0, stream>>>(p);
  } else if (kv->head_dim == 128) {
    if (bf) q8_read_kernel<128, true><<<grid, 256, 0, stream>>>(p);
    else q8_read_kernel<128, false><<<grid, 256, 0, stream>>>(p);
  } else {
    if (bf) q8_read_kernel<256, true><<<grid, 256, 0, stream>>>(p);
    else q8_read_kernel<256, false><<<grid, 256, 0, stream>>>(p);
  }
  DTREE_LAUNCH_CHECK("kv_q8_read launch");
  return DTREE_OK;
}

extern "C" int dtree_kv_q8_compact(const DtreeStepDesc* desc, int8_t* k_pages, int8_t* v_pages, float* k_scales,
                                   float* v_scales, int32_t layers, int32_t num_pages, int32_t num_kv_heads,
                                   int32_t head_dim, const int32_t* page_table, int32_t table_pages,
                                   const uint16_t* hidden_in, int32_t hidden_width, uint16_t* hidden_out,
                                   hipStream_t stream) {
  DTREE_REQUIRE(desc && k_pages && v_pages && k_scales && v_scales && page_table, "kv_q8_compact: null pointer");
  DTREE_REQUIRE(aligned16(k_pages) && aligned16(v_pages), "kv_q8_compact: the pages must be 16-byte aligned");
  DTREE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "kv_q8_compact: head_dim 64, 128 or 256");
  DTREE_REQUIRE(layers >= 1 && layers <= 1024 && num_kv_heads >= 1 && num_kv_heads <= 256 && num_pages >= 1 &&
                    num_pages <= (1 << 25) && table_pages >= 1,
                "kv_q8_compact: layers, num_kv_heads, num_pages or table_pages");
  DTREE_REQUIRE(!hidden_out || (hidden_in && hidden_width > 0 && hidden_width % 8 == 0 && aligned16(hidden_in) &&
                                aligned16(hidden_out)),
                "kv_q8_compact: hidden rows of a multiple of 8, 16-byte aligned");
  const int grid = 2 * layers * num_kv_heads + (hidden_out ? kHidBlocks : 0);
  q8_compact_kernel<<<grid, 256, 0, stream>>>(desc, k_pages, v_pages, k_scales, v_scales, layers, num_pages,
                                              num_kv_heads, head_dim, page_table, table_pages, hidden_in, hidden_width,
                                              hidden_out);
  DTREE_LAUNCH_CHECK("kv_q8_compact launch");
  return DTREE_OK;
}
