// The 8-bit paged KV cache: rows in (the cache append of qwen3_tree.py:146 with
// the k_norm and RoPE before it, :57-62), rows out, and the accepted path's move
// (adapters.py:635-668).
//
// A row is quantised as scale = fp32(max |x| / 127), q = nearest integer of
// x / scale. Everything before the rounding to q is fp64: x stays within 1e-15
// of its value, so q is the nearest integer but for borders met by less than
// that, and two programs that follow the definition store the same bytes.
//
// All three are bound by the bytes they move (a decode step's by the launch).
// A workgroup owns one page of one kv head. K rows are written by D / 16 threads
// each, 16 dims (one 16-byte store) a thread; V's 16 bytes belong to 16 rows of
// one dim and go through LDS.
#include <cmath>

#include "kv_q8.h"

namespace dtree {
namespace {

struct Q8AppendParams {
  DtreeKvQ8 kv;
  const void* k; const void* v;
  int ld_k, ld_v, span;
  const uint16_t* k_norm; double eps;
  const float* cos; const float* sin; int half;  // rotated pairs
};

// 16 consecutive elements of a row.
template <bool BF16>
__device__ __forceinline__ void load16(const void* base, size_t at, float (&x)[16]) {
  if constexpr (BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4_t w = ld_u32x4(p + 8 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
        x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  } else {
    const float* p = static_cast<const float*>(base) + at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4_t w = *reinterpret_cast<const f32x4_t*>(p + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = w[j];
    }
  }
}

// Quantises a row held by TPR neighbouring lanes, 16 elements each: the bytes,
// and the row's scale in every lane. Not finite anywhere: scale NaN, bytes 0.
template <int TPR>
__device__ __forceinline__ u32x4_t quantise16(const double (&x)[16], float& scale) {
  constexpr double kMost = 4.3e40;  // fp32's largest times 127, less a little
  double amax = 0.;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const double a = fabs(x[i]);
    bad |= !(a <= kMost);
    amax = fmax(amax, a);
  }
  if (bad) amax = INFINITY;
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) amax = fmax(amax, __shfl_xor(amax, o));
  if (amax > kMost) {
    scale = NAN;
    return u32x4_t{0, 0, 0, 0};
  }
  scale = (float)(amax / 127.0);
  const double inv = scale > 0.f ? 1.0 / (double)scale : 0.;
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (a subnormal scale may have been rounded by more than 1 / 254)
      const double q = fmin(fmax(rint(x[4 * i + j] * inv), -127.), 127.);
      b |= (uint32_t)((int)q & 0xff) << (8 * j);
    }
    w[i] = b;
  }
  return w;
}

// Waves 0 and 1 take K rows, waves 2 and 3 V rows, at once.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void q8_append_kernel(Q8AppendParams p) {
  constexpr int TPR = D / 16, RPP = 128 / TPR;  // threads a row; rows a pass
  __shared__ uint32_t vt[D][17];                // V bytes [dim][slot], a word of padding
  const int g = blockIdx.x % p.kv.num_kv_heads, b = blockIdx.x / p.kv.num_kv_heads;
  const int s = b / p.span;
  const Q8Seq q = q8_seq(p.kv, s);
  if (q.n == 0) return;
  const int pg = q.past / DTREE_PAGE + b % p.span;
  const int first = pg * DTREE_PAGE - q.past;  // the sequence's row in slot 0
  const int lo = max(0, -first), hi = min(DTREE_PAGE, q.n - first);  // live slots
  if (lo >= hi) return;
  const int page = q8_page(p.kv, s, pg);
  if (page < 0) return;
  const size_t blk = (size_t)page * p.kv.num_kv_heads + g;
  const int tid = threadIdx.x, t = tid & 127, j = t % TPR;
  for (int slot = lo + t / TPR; slot < hi; slot += RPP) {
    const size_t row = q.start + first + slot;
    double x[16];
    float y[16], scale;
    if (tid < 128) {
      load16<BF16>(p.k, row * p.ld_k + g * D + 16 * j, y);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = y[i];
      double rs = 1.;
      if (p.k_norm) {
        double ss = 0.;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fma(x[i], x[i], ss);
#pragma unroll
        for (int o = 1; o < TPR; o <<= 1) ss += __shfl_xor(ss, o);
        rs = 1. / sqrt(ss * (1.0 / D) + p.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= rs * (double)bf2f(p.k_norm[16 * j + i]);
      }
      const int hc = p.half / 16;  // chunks of 16 dims in a half of the rotated ones
      if (j < 2 * hc) {            // the rotation's other half, loaded once more
        const bool low = j < hc;
        const int jo = low ? j + hc : j - hc;
        load16<BF16>(p.k, row * p.ld_k + g * D + 16 * jo, y);
        const size_t at = row * p.half + 16 * (low ? j : jo);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const double o = p.k_norm ? (double)y[i] * (rs * (double)bf2f(p.k_norm[16 * jo + i])) : (double)y[i];
          const double cs = p.cos[at + i], sn = p.sin[at + i];
          x[i] = low ? x[i] * cs - o * sn : o * sn + x[i] * cs;
        }
      }
      const u32x4_t w = quantise16<TPR>(x, scale);
      *reinterpret_cast<u32x4_t*>(p.kv.k_pages + blk * (DTREE_PAGE * D) + q8_k_off(slot, 16 * j, D)) = w;
      if (j == 0) p.kv.k_scales[blk * DTREE_PAGE + slot] = scale;
    } else {
      load16<BF16>(p.v, row * p.ld_v + g * D + 16 * j, y);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = y[i];
      const u32x4_t w = quantise16<TPR>(x, scale);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        reinterpret_cast<uint8_t*>(&vt[16 * j + i][0])[slot] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
      if (j == 0) p.kv.v_scales[blk * DTREE_PAGE + slot] = scale;
    }
  }
  __syncthreads();
  // V: 16-byte pieces (32-slot half, 32 dims, 4-slot parity, dim); what other
  // rows own of a piece stays.
  int8_t* vp = p.kv.v_pages + blk * (DTREE_PAGE * D);
#pragma unroll
  for (int u = tid; u < 4 * D; u += 256) {
    const int dl = u & 31, h = (u >> 5) & 1, db = (u >> 6) % (D / 32), b2 = (u >> 6) / (D / 32);
    const int s0 = 32 * b2 + 4 * h, d = 32 * db + dl;  // the piece's slots: s0 + 8 i + 0 .. 3
    if (s0 + 27 < lo || s0 >= hi) continue;
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = vt[d][s0 / 4 + 2 * i];
    int8_t* o = vp + (u << 4);
    if (s0 >= lo && s0 + 27 < hi) {
      *reinterpret_cast<u32x4_t*>(o) = w;
      continue;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int sl = s0 + 8 * i;
      if (sl >= lo && sl + 3 < hi) {
        reinterpret_cast<uint32_t*>(o)[i] = w[i];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (sl + e >= lo && sl + e < hi) o[4 * i + e] = (int8_t)(w[i] >> (8 * e));
      }
    }
  }
}

struct Q8ReadParams {
  DtreeKvQ8 kv;
  void* k; void* v;
  int ld_k, ld_v, span;
};

template <bool BF16>
__device__ __forceinline__ void store16(void* base, size_t at, u32x4_t w, float scale) {
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = (float)((int)(w[i >> 2] << (24 - 8 * (i & 3))) >> 24) * scale;
  if constexpr (BF16) {
    uint16_t* o = static_cast<uint16_t*>(base) + at;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<u32x4_t*>(o + 8 * i) = u32x4_t{pack_bf2(y[8 * i], y[8 * i + 1]), pack_bf2(y[8 * i + 2], y[8 * i + 3]),
                                                       pack_bf2(y[8 * i + 4], y[8 * i + 5]), pack_bf2(y[8 * i + 6], y[8 * i + 7])};
  } else {
    float* o = static_cast<float*>(base) + at;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4_t*>(o + 4 * i) = f32x4_t{y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]};
  }
}

template <int D, bool BF16>
__global__ __launch_bounds__(256) void q8_read_kernel(Q8ReadParams p) {
  constexpr int TPR = D / 16;
  __shared__ uint32_t vt[D][17];
  const int g = blockIdx.x % p.kv.num_kv_heads, b = blockIdx.x / p.kv.num_kv_heads;
  const int s = b / p.span;
  const Q8Seq q = q8_seq(p.kv, s);
  if (q.n == 0) return;
  const int pg = q.past / DTREE_PAGE + b % p.span;
  const int first = pg * DTREE_PAGE - q.past;
  const int lo = max(0, -first), hi = min(DTREE_PAGE, q.n - first);
  if (lo >= hi) return;
  const int page = q8_page(p.kv, s, pg), tid = threadIdx.x;
  const size_t blk = (size_t)max(page, 0) * p.kv.num_kv_heads + g;
  const int8_t* kb = p.kv.k_pages + blk * (DTREE_PAGE * D);
  const int8_t* vb = p.kv.v_pages + blk * (DTREE_PAGE * D);
  const u32x4_t zero = {0, 0, 0, 0};
  if (p.v) {
#pragma unroll
    for (int u = tid; u < 4 * D; u += 256) {
      const int dl = u & 31, h = (u >> 5) & 1, db = (u >> 6) % (D / 32), b2 = (u >> 6) / (D / 32);
      const u32x4_t w = page >= 0 ? ld_u32x4(vb + (u << 4)) : zero;
#pragma unroll
      for (int i = 0; i < 4; ++i) vt[32 * db + dl][8 * b2 + h + 2 * i] = w[i];
    }
  }
  __syncthreads();
  for (int slot = lo + tid / TPR; slot < hi; slot += 256 / TPR) {
    const int j = tid % TPR;
    const size_t row = q.start + first + slot;
    if (p.k)
      store16<BF16>(p.k, row * p.ld_k + g * D + 16 * j, page >= 0 ? ld_u32x4(kb + q8_k_off(slot, 16 * j, D)) : zero,
                    page >= 0 ? p.kv.k_scales[blk * DTREE_PAGE + slot] : 0.f);
    if (p.v) {
      u32x4_t w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t x = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x |= (uint32_t) reinterpret_cast<const uint8_t*>(&vt[16 * j + 4 * i + e][0])[slot] << (8 * e);
        w[i] = x;
      }
      store16<BF16>(p.v, row * p.ld_v + g * D + 16 * j, w, page >= 0 ? p.kv.v_scales[blk * DTREE_PAGE + slot] : 0.f);
    }
  }
}

constexpr int kHidBlocks = 16;  // workgroups of the hidden rows' select

// The accepted rows of one (layer, kv head), K or V, through LDS: a row's place
// may be another accepted row's source.
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
  const int64_t n = (int64_t)kv->num_seqs * q8_span_pages(*kv) * kv->num_kv_heads;
  DTREE_REQUIRE(n < (int64_t)1 << 31, what + ": num_seqs * max_rows too large for one launch");
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
  const Q8AppendParams p{*kv, k, v, ld_k, ld_v, q8_span_pages(*kv), k_norm, (double)eps, rope_cos, rope_sin,
                         rope_dims / 2};
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
  const Q8ReadParams p{*kv, k, v, ld_k, ld_v, q8_span_pages(*kv)};
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
