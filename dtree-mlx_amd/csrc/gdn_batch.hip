// One token of each of a batch of sequences through a GatedDeltaNet layer's core
// (qwen35_tree.py:199-322 for a root alone, custom_qwen35_model.py:823-878), each
// from the window and state of the sequence that it continues.
//
// S' = g S + beta (v - g S k) k^T,  y = S' q = g S q + beta (v - g S k) (k . q):
// both products need the old state alone, so it is read once, into registers, and
// written once. A workgroup owns a (sequence, value head): 64 KB of state in 512
// threads, 16 rows of 4 columns each, so a row's products are sums over 32 lanes. The
// state's loads go out first; the convolution, the norms of q and k and the gates are
// computed behind them (a key head's q and k by each of its value heads). The gated
// norm's sum over the head's rows is in the workgroup too: one launch.
//
// Bound by the states' bytes, 2 MB a sequence each way at 32 heads.
#include <cmath>

#include "common.h"

namespace dtree {
namespace {

constexpr int D = 128;
constexpr int kThreads = 512;
constexpr int kRows = D / (kThreads / 32);  // state rows of a thread

struct BatchParams {
  DtreeGdnArgs a;
  const int* sources;
  int seqs, C, key_dim;
};

__device__ __forceinline__ f32x4_t ld4(const float* p) { return *reinterpret_cast<const f32x4_t*>(p); }
__device__ __forceinline__ float dot4(f32x4_t a, f32x4_t b) {
  return fmaf(a[0], b[0], fmaf(a[1], b[1], fmaf(a[2], b[2], a[3] * b[3])));
}

template <int KEEP>
__global__ __launch_bounds__(kThreads) void gdn_batch_kernel(BatchParams p) {
  __shared__ __attribute__((aligned(16))) float qkv[3][D], ys[D];
  const DtreeGdnArgs& a = p.a;
  const int Hv = a.num_v_heads, per = Hv / a.num_k_heads;
  const int b = blockIdx.x / Hv, h = blockIdx.x % Hv, hk = h / per;
  const int tid = threadIdx.x, c4 = 4 * (tid & 31), r0 = tid >> 5;
  const int tiled = a.out_layout != DTREE_W_ROWMAJOR, h16 = a.out_layout == DTREE_W_TILED_F16;
  const size_t oi = tiled ? tiled_index(b, h * D + c4, a.ld_out) : (size_t)b * a.ld_out + h * D + c4;
  if (b >= p.seqs) {  // padding rows of the output
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    if (tid < 32) store_act4(a.out, a.out_lo, oi, zero, h16);
    return;
  }
  int src = p.sources ? p.sources[b] : b;
  src = src >= 0 && src < p.seqs ? src : -1;  // -1: a sequence that begins
  // Everything that does not wait for another load, the gates and the gated norm's
  // operands first, then the state.
  const float* proj = a.proj + (size_t)b * a.ld_proj;
  const float* gates = proj + p.C + (size_t)Hv * D;
  const float gate_a = gates[Hv + h] + a.dt_bias[h], gate_b = gates[h], a_log = a.A_log[h];
  f32x4_t z = {0.f, 0.f, 0.f, 0.f};
  u32x2_t nw = {0, 0};
  if (tid < 32) {
    z = ld4(proj + p.C + h * D + c4);
    __builtin_memcpy(&nw, a.norm_w + c4, 8);
  }
  constexpr int kStep = kThreads / 32;  // rows between a thread's
  const size_t head = (size_t)h * D * D;
  const int part = tid >> 5;  // q, k, v of the first 96 threads
  const int c = (part == 2 ? 2 * p.key_dim + h * D : part * p.key_dim + hk * D) + c4;
  f32x4_t s[kRows], x[KEEP + 1], w[KEEP + 1];
  if (part < 3) {
    x[KEEP] = ld4(proj + c);
#pragma unroll
    for (int r = 0; r <= KEEP; ++r) w[r] = ld4(a.conv_w + (size_t)r * p.C + c);
  }
  if (src >= 0) {
    if (part < 3) {
      const float* win = a.window + (size_t)src * KEEP * p.C + c;
#pragma unroll
      for (int r = 0; r < KEEP; ++r) x[r] = ld4(win + (size_t)r * p.C);
    }
    const float* st = a.state + (size_t)src * Hv * D * D + head + r0 * D + c4;
#pragma unroll
    for (int i = 0; i < kRows; ++i) s[i] = ld4(st + i * kStep * D);
  } else {
#pragma unroll
    for (int r = 0; r < KEEP; ++r) x[r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kRows; ++i) s[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  if (part < 3) {
    f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r <= KEEP; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(x[r][e], w[r][e], y[e]);
    if (part == 2 || h % per == 0) {
      float* wout = a.window_out + (size_t)b * KEEP * p.C + c;
#pragma unroll
      for (int r = 0; r < KEEP; ++r) *reinterpret_cast<f32x4_t*>(wout + (size_t)r * p.C) = x[r + 1];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = silu_f(y[e]);
    const float ss = row_sum32(dot4(y, y));
    const float f = part == 2 ? 1.f : rsqrtf(ss * (1.f / D) + 1e-6f) * (part == 0 ? 1.f / D : 0.08838834764831845f);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= f;
    *reinterpret_cast<f32x4_t*>(&qkv[part][c4]) = y;
  }
  const float g = expf(-expf(a_log) * (gate_a > 20.f ? gate_a : log1pf(expf(gate_a))));
  const float beta = 1.f / (1.f + expf(-gate_b));
  lds_barrier();  // (the state's loads stay in flight)
  const f32x4_t q = ld4(&qkv[0][c4]), k = ld4(&qkv[1][c4]);
  const float kq = row_sum32(dot4(k, q));
  float* st = a.state_out + (size_t)b * Hv * D * D + head + r0 * D + c4;
  // Four rows at a time: their sums over 32 lanes are independent chains.
  constexpr int kTogether = 4;
  static_assert(kRows % kTogether == 0, "whole groups of rows");
#pragma unroll
  for (int i0 = 0; i0 < kRows; i0 += kTogether) {
    float sk[kTogether], sq[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      sk[j] = dot4(s[i0 + j], k);
      sq[j] = dot4(s[i0 + j], q);
    }
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      sk[j] = row_sum32(sk[j]);
      sq[j] = row_sum32(sq[j]);
    }
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      const int r = r0 + (i0 + j) * kStep;
      const float delta = (qkv[2][r] - g * sk[j]) * beta;
      f32x4_t& v = s[i0 + j];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(delta, k[e], g * v[e]);
      __builtin_nontemporal_store(v, reinterpret_cast<f32x4_t*>(st + (i0 + j) * kStep * D));
      if ((tid & 31) == 0) ys[r] = fmaf(delta, kq, g * sq[j]);
    }
  }
  lds_barrier();  // (the new state's stores retire behind it)
  if (tid < 32) {
    const f32x4_t y = ld4(&ys[c4]);
    const float rs = rsqrtf(row_sum32(dot4(y, y)) * (1.f / D) + a.eps);
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = y[e] * rs * __uint_as_float((e & 1) ? nw[e >> 1] & 0xffff0000u : nw[e >> 1] << 16) * silu_f(z[e]);
    store_act4(a.out, a.out_lo, oi, o, h16);
  }
}

bool disjoint(const void* x, size_t nx, const void* y, size_t ny) {
  const char *p = static_cast<const char*>(x), *q = static_cast<const char*>(y);
  return p + nx <= q || q + ny <= p;
}

}  // namespace
}  // namespace dtree

using namespace dtree;

extern "C" int dtree_gdn_layer_batch(const DtreeGdnArgs* a, const int32_t* sources, int32_t num_seqs, hipStream_t stream) {
  DTREE_REQUIRE(a, "gdn_layer_batch: null args");
  DTREE_REQUIRE(num_seqs >= 1 && num_seqs <= a->rows_padded && a->rows_padded <= (1 << 16),
                "gdn_layer_batch: num_seqs in [1, rows_padded]");
  DTREE_REQUIRE(a->num_k_heads > 0 && a->num_v_heads > 0 && a->num_v_heads <= 256 && a->num_v_heads % a->num_k_heads == 0,
                "gdn_layer_batch: num_v_heads % num_k_heads, at most 256");
  DTREE_REQUIRE((int64_t)a->rows_padded * a->num_v_heads < (1 << 23),
                "gdn_layer_batch: rows_padded * num_v_heads below 2^23 (2^32 work items)");
  DTREE_REQUIRE(a->head_k_dim == D && a->head_v_dim == D, "gdn_layer_batch: head dims 128 are compiled");
  DTREE_REQUIRE(a->conv_keep >= 1 && a->conv_keep <= 7, "gdn_layer_batch: conv_keep in [1, 7]");
  DTREE_REQUIRE(a->proj && a->window && a->conv_w && a->A_log && a->dt_bias && a->state && a->norm_w && a->out &&
                    a->window_out && a->state_out,
                "gdn_layer_batch: null pointer");
  const int key_dim = a->num_k_heads * D, value_dim = a->num_v_heads * D, C = 2 * key_dim + value_dim;
  DTREE_REQUIRE(a->ld_proj >= C + value_dim + 2 * a->num_v_heads && a->ld_proj % 4 == 0,
                "gdn_layer_batch: ld_proj >= C + z + b + a, a multiple of 4");
  DTREE_REQUIRE((((uintptr_t)a->proj | (uintptr_t)a->conv_w | (uintptr_t)a->window | (uintptr_t)a->state |
                  (uintptr_t)a->window_out | (uintptr_t)a->state_out) & 15) == 0,
                "gdn_layer_batch: proj, conv_w, windows and states must be 16-byte aligned");
  DTREE_REQUIRE((((uintptr_t)a->out | (uintptr_t)a->out_lo) & 7) == 0 && ((uintptr_t)a->norm_w & 1) == 0,
                "gdn_layer_batch: out and out_lo must be 8-byte aligned");
  DTREE_REQUIRE(a->out_layout == DTREE_W_ROWMAJOR ? (a->ld_out >= value_dim && a->ld_out % 4 == 0)
                                                  : ((a->out_layout == DTREE_W_TILED || a->out_layout == DTREE_W_TILED_F16) &&
                                                     a->ld_out == value_dim && value_dim % 64 == 0 &&
                                                     a->rows_padded % 32 == 0),
                "gdn_layer_batch: out layout (tiled needs ld_out == value dim, rows_padded % 32 == 0)");
  const size_t wb = (size_t)num_seqs * a->conv_keep * C * sizeof(float);
  const size_t sb = (size_t)num_seqs * value_dim * D * sizeof(float);
  DTREE_REQUIRE(disjoint(a->window, wb, a->window_out, wb) && disjoint(a->state, sb, a->state_out, sb),
                "gdn_layer_batch: the new windows and states need buffers of their own");
  BatchParams p{*a, sources, num_seqs, C, key_dim};
  const int grid = a->rows_padded * a->num_v_heads;
  switch (a->conv_keep) {
#define DTREE_BATCH_CASE(K) \
  case K: gdn_batch_kernel<K><<<grid, kThreads, 0, stream>>>(p); break;
    DTREE_BATCH_CASE(1) DTREE_BATCH_CASE(2) DTREE_BATCH_CASE(3) DTREE_BATCH_CASE(4) DTREE_BATCH_CASE(5)
    DTREE_BATCH_CASE(6) DTREE_BATCH_CASE(7)
#undef DTREE_BATCH_CASE
  }
  DTREE_LAUNCH_CHECK("gdn_layer_batch launch");
  return DTREE_OK;
}
