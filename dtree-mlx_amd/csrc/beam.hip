// Beam search's selection: of every group of beams the best (beam, token)
// continuations by summed log-probability (the batched, several-hypotheses
// counterpart of the greedy argmax of adapters.py:114-118).
//
// s(b, t) = score_b + (x_bt - lse_b), rank(b, t) = s / length^penalty, in fp64, but for
// the exponentials and their sums over 4096 logits (lse is within 64 2^-24 = 4e-6: |x - m|
// 2^-23 of a term, log(V) 2^-23 on average, and the additions): two candidates that fp32
// would round together are told apart.
// Ties go to the lower beam, then the lower token.
//
// Two launches.
//
// scan   One pass over the logits, a workgroup per (row, 4096 logits; many of bf16 two
//        in turn) in registers: the chunk's maximum and sum of exp(x - max), and the
//        maximum of each run of 32 logits ("segment"). Bound by the logits' bytes: 244 MB
//        of bf16 in 47 us (5.2 TB/s; a copy on this card reaches 4.7, reads and writes
//        together), 59 MB of fp32 in 11 us, 1.2 MB in 3.5 us (latency). Loads past the
//        caches: the pick kernel's code, partials and segments stay in them (20.0 against
//        21.2 us for the 59 MB).
// pick   A workgroup per group. rank grows with x inside a beam, so a selected token
//        lies in one of the num_select best segments by their maxima, and such a
//        segment in one of the num_select best units (chunks, or parts of them). The
//        quick way: a threshold that num_select to num_select + 32 units reach, its least
//        logit for each beam, the segments and then the logits that reach that, all loads
//        of a step in flight together; the last survivors, a few more than num_select,
//        are ranked by counting. Where ties or a crowd of near ranks leave more than its
//        lists hold (44 us in place of 23 for the selection of 16 groups of 8 beams of
//        normal logits of deviation 0.25; 93 for 4 beams of equal ones), the sure way:
//        the same three levels, each cut to at most twice num_select by bisection on the
//        rank's order-preserving integer and then, among equal ranks, on the position.
//        Bound by latency: three rounds of loads of 1 us and the code's own fetches
//        (little of it is executed twice): 6.5 us for 4 beams, 7.9 for 16 groups of 8,
//        12.2 for 64 groups of 16 (32 selected of each).
//
// Built first with bisection at every level, over each thread's share and with shuffles:
// pick 15 to 45 us. Counting by ballots, one wave a probe, eight probes a round: 3 rounds
// in place of 10 steps of 350 to 600 clocks. fp64 logarithms and powers in full were a
// fifth of the rest, as code more than as arithmetic.
#include <cmath>

#include "common.h"

namespace dtree {
namespace {

constexpr int kChunk = 4096;           // logits of a scan workgroup
constexpr int kSeg = 32;               // logits of a segment
constexpr int kSegs = kChunk / kSeg;   // segments of a chunk
// Chunks of bf16 (of all rows) from which a scan workgroup takes two of a row, the
// second's loads in flight during the first: four times what the card holds at once (2048
// workgroups). us of a selection, one by one and by twos: 4864 chunks 19.3 and 19.4 (21.3 and
// 21.6 for 32 selected of 16 beams), 9728 26.7 and 26.3 (29.0 and 28.5), 16416 41.1 and 39.5,
// 19456 42.3 and 39.9, 38912 73.9 and 67.3 (76.2 and 71.0). A chunk of fp32 has twice the
// loads in flight by itself: 4864 chunks 23.4 and 24.5, 16384 53.0 and 55.5, 38912 114 and
// 117, so it is taken alone (in the same loop: with one chunk a workgroup by construction
// the compiler's order of the loads costs 1 us at 4864).
constexpr int kPairs = 8192;
constexpr int kMaxBeams = 64;
constexpr int kMaxSelect = 64;
constexpr int kMaxVocab = 1 << 20;
constexpr int kPickThreads = 512, kPickWaves = kPickThreads / 64;
constexpr int kKeep = 2 * kMaxSelect;  // survivors of a level
constexpr float kBig = 3.40282347e38f;
// Maxima below which c = max log2 e, rounded, is within 1/16 of it, and 2^(its error) is a
// harmless factor of a sum. (An error grows with the maximum: 440 at 1e10.)
constexpr float kNear = 1048576.f;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
  DtreeBeamArgs a;
  int chunks, run;  // of a row; of a scan workgroup
  float2* part;     // [rows][chunks] maximum, sum of exp(x - maximum)
  float* seg;       // [rows][chunks][kSegs] maxima
};

// A logit as the selection takes it: NaN as -inf, +inf as the largest number.
__device__ __forceinline__ float clean(float x) { return x > -INFINITY ? fminf(x, kBig) : -INFINITY; }

// A beam that is summed over its vocabulary (not finished, with a score).
__device__ __forceinline__ bool beam_over(const DtreeBeamArgs& a, int row) { return a.finished && a.finished[row]; }
__device__ __forceinline__ float beam_score(const DtreeBeamArgs& a, int row) { return a.scores ? a.scores[row] : 0.f; }

// f over the wave's 64 lanes, in each of them: within rows of 16, then the four rows.
template <class F>
__device__ __forceinline__ float wave_all(float v, F f) {
  v = f(v, dpp<0xB1>(v));
  v = f(v, dpp<0x4E>(v));
  v = f(v, dpp<0x141>(v));
  v = f(v, dpp<0x140>(v));
  auto row = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); };
  return f(f(row(0), row(16)), f(row(32), row(48)));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_all(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_all(v, [](float a, float b) { return a + b; });
}

template <bool BF>
__device__ __forceinline__ float logit(const DtreeBeamArgs& a, int row, int t) {
  const size_t at = (size_t)row * a.ld_logits + t;
  if constexpr (BF) return clean(bf2f(static_cast<const uint16_t*>(a.logits)[at]));
  else return clean(static_cast<const float*>(a.logits)[at]);
}

// v_med3_f32 itself: the compiler's median of a constant infinity is a minimum, which
// gives the number for a NaN. Volatile: it stays behind the mode's change below.
__device__ __forceinline__ float median(float x, float low, float high) {
  float y;
  asm volatile("v_med3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(x), "s"(low), "v"(high));
  return y;
}

// (rows at any address of their type)
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));

template <bool BF>
__global__ __launch_bounds__(256) void beam_scan_kernel(BeamParams p) {
  constexpr int E = BF ? 8 : 4, NL = kChunk / 256 / E;  // logits of a load, loads of a thread
  constexpr int LPS = kSeg / E;                         // lanes of a segment
  __shared__ float wm[2][4], ws[2][4];
  const int runs = (p.chunks + p.run - 1) / p.run;
  const int row = blockIdx.x / runs, c0 = blockIdx.x % runs * p.run, c1 = min(c0 + p.run, p.chunks);
  if (beam_over(p.a, row) || !(beam_score(p.a, row) > -INFINITY)) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // The median of x, -inf and the largest number is x, cut to them, or, of a NaN, the
  // least of the two others: -inf. With the mode's IEEE bit (9) cleared that holds for
  // signalling NaNs too, which it otherwise hands on as quiet ones.
  __builtin_amdgcn_s_setreg(1 | 9 << 6, 0);
  const float low = -INFINITY, big = kBig;
  const char* src = static_cast<const char*>(p.a.logits) + (size_t)row * p.a.ld_logits * (BF ? 2 : 4);
  u32x4_t w[NL];
  auto load = [&](int chunk) {
    const int first = chunk * kChunk, left = p.a.vocab - first;
    if (left >= kChunk) {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any_t*>(src + (size_t)(first + (i * 256 + tid) * E) * (BF ? 2 : 4)));
    } else {  // the row's last logits, then -inf
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int at = (i * 256 + tid) * E;
        if constexpr (BF) w[i] = u32x4_t{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
        else w[i] = u32x4_t{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
        if (at + E <= left) {
          w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any_t*>(src + (size_t)(first + at) * (BF ? 2 : 4)));
        } else {
          for (int e = 0; at + e < left; ++e) {
            if constexpr (BF) {
              const uint32_t v = reinterpret_cast<const uint16_t*>(src)[first + at + e];
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (k == e) w[i][k >> 1] = (k & 1) ? (w[i][k >> 1] & 0xffffu) | v << 16 : (w[i][k >> 1] & 0xffff0000u) | v;
            } else {
              const uint32_t v = reinterpret_cast<const uint32_t*>(src)[first + at + e];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k == e) w[i][k] = v;
            }
          }
        }
      }
    }
  };
  load(c0);
#pragma unroll 1
  for (int chunk = c0; chunk < c1; ++chunk) {
    const int turn = chunk & 1;
    const size_t block = (size_t)row * p.chunks + chunk;
    float x[NL][E], mx = -INFINITY, keep = 0.f;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      float m = -INFINITY;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float v;
        if constexpr (BF) v = __uint_as_float((e & 1) ? (w[i][e >> 1] & 0xffff0000u) : (w[i][e >> 1] << 16));
        else v = __uint_as_float(w[i][e]);
        x[i][e] = median(v, low, big);
        m = fmaxf(m, x[i][e]);
      }
      m = fmaxf(m, dpp<0xB1>(m));
      m = fmaxf(m, dpp<0x4E>(m));
      if constexpr (LPS == 8) m = fmaxf(m, dpp<0x141>(m));
      if ((tid & (LPS - 1)) == i) keep = m;
      mx = fmaxf(mx, m);
    }
    if (chunk + 1 < c1) load(chunk + 1);  // (in flight across the barriers, which wait for LDS alone)
    // lane i of a segment's lanes has load i's
    const int sl = tid & (LPS - 1);
    if (sl < NL) p.seg[block * kSegs + sl * (256 / LPS) + tid / LPS] = keep;
    mx = wave_max(mx);
    if (lane == 0) wm[turn][wave] = mx;
    lds_barrier();
    mx = fmaxf(fmaxf(wm[turn][0], wm[turn][1]), fmaxf(wm[turn][2], wm[turn][3]));
    const float base = fmaxf(mx, -kBig);
    float sum = 0.f;
    if (fabsf(base) < kNear) {
      // one operation an exponent: x log2 e - c, c = base log2 e rounded, whose rounding
      // is a factor of the whole sum
      const float c = base * kLog2e;
#pragma unroll
      for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) sum += fast_exp2(fmaf(x[i][e], kLog2e, -c));
      sum *= fast_exp2(-fmaf(base, kLog2e, -c));
    } else {  // (the difference first, which no magnitude spoils)
#pragma unroll
      for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) sum += fast_exp2((x[i][e] - base) * kLog2e);
    }
    sum = wave_sum(sum);
    if (lane == 0) ws[turn][wave] = sum;
    lds_barrier();
    if (tid == 0) p.part[block] = make_float2(mx, ws[turn][0] + ws[turn][1] + ws[turn][2] + ws[turn][3]);
  }
}

// Order-preserving integer of a rank; 0 for what is no candidate.
__device__ __forceinline__ uint64_t order_of(double v) {
  if (!(v > -INFINITY)) return 0;
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double rank_of(uint64_t key) {
  return __builtin_bit_cast(double, (key >> 63) ? key & 0x7fffffffffffffffull : ~key);
}

template <int CTRL>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  return (uint64_t)(uint32_t)dpp_i<CTRL>((int)(uint32_t)(v >> 32)) << 32 | (uint32_t)dpp_i<CTRL>((int)(uint32_t)v);
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  return __builtin_bit_cast(double, dpp64<CTRL>(__builtin_bit_cast(uint64_t, v)));
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
template <class F>
__device__ __forceinline__ uint64_t wave_all64(uint64_t v, F f) {
  v = f(v, dpp64<0xB1>(v));
  v = f(v, dpp64<0x4E>(v));
  v = f(v, dpp64<0x141>(v));
  v = f(v, dpp64<0x140>(v));
  return f(f(lane64(v, 0), lane64(v, 16)), f(lane64(v, 32), lane64(v, 48)));
}

// Lists of the quick way. A level of it keeps more than it must; where ties or a
// crowd of near ranks overflow one, the group goes the sure way.
constexpr int kSlack = 32;                  // more than the selected ones that a threshold may leave
constexpr int kUnits1 = kMaxSelect + kSlack;  // units kept
constexpr int kSegs1 = 512, kBest1 = 256;   // segments, logits
constexpr int kStaged = 4096;               // (beam, chunk) pairs and units it takes, in LDS

__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t o) {
  return __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}

// ln s for s >= 1/2, within 1e-9 (the sums are good to 4e-6): s = 2^e m, m in [0.7,
// 1.4], ln m = 2 atanh((m - 1) / (m + 1)). Little code: the kernel's own instructions
// are part of its latency.
__device__ __forceinline__ double ln_of(double s) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, s);
  const uint64_t shift = (bits & 0x000fffffffffffffull) > 0x0006a09e667f3bcdull ? 1 : 0;
  const int e = (int)(bits >> 52) - 1023 + (int)shift;
  const double m = __builtin_bit_cast(double, (bits & 0x000fffffffffffffull) | (1023 - shift) << 52);
  const double d = m + 1.;
  double r = __builtin_amdgcn_rcp(d);
  r = fma(r, fma(-d, r, 1.), r);
  const double t = (m - 1.) * r, u = t * t;
  double y = 1. / 11;
  y = fma(y, u, 1. / 9);
  y = fma(y, u, 1. / 7);
  y = fma(y, u, 1. / 5);
  y = fma(y, u, 1. / 3);
  y = fma(y, u, 1.);
  return fma((double)e, 0.69314718055994531, 2. * t * y);
}

struct Item {
  uint64_t key;
  uint32_t id;  // position: the lower one wins a tie
};

struct PickLds {
  double score[kMaxBeams], lse[kMaxBeams];        // lse: less the maximum
  double weight[kMaxBeams], back[kMaxBeams];      // length^-penalty, length^penalty
  float m[kMaxBeams], least[kMaxBeams];                        // least: the logits that reach the threshold
  int kind[kMaxBeams], length[kMaxBeams];                      // kind 1: summed over its vocabulary, 2: finished
  int count[2][kPickWaves];
  uint64_t lo[kPickWaves], hi[kPickWaves];
  int n, n2, n3;
  uint32_t list[2][kKeep];
  uint32_t units[kUnits1], segs[kSegs1];  // beam << 16 | first segment, segment of the row
  struct {
    uint64_t key;
    uint32_t id;
    float x;
  } cand[kBest1];
  float top[kStaged];  // the chunks' maxima, of live beams
  __attribute__((aligned(16))) float unit[kStaged];
};

// The sum over the waves of a count that is uniform in each. Two buffers, so that one
// barrier a call is enough.
__device__ __forceinline__ int block_count(PickLds& l, int& turn, int c) {
  if ((threadIdx.x & 63) == 0) l.count[turn][threadIdx.x >> 6] = c;
  lds_barrier();
  int n = 0;
#pragma unroll
  for (int w = 0; w < kPickWaves; ++w) n += l.count[turn][w];
  turn ^= 1;
  return n;
}

// A place in a list for each lane of `take`.
__device__ __forceinline__ int place(int* n, bool take) {
  const uint64_t mask = __ballot(take);
  if (!mask) return 0;
  int at = 0;
  if ((threadIdx.x & 63) == 0) at = atomicAdd(n, (int)__popcll(mask));
  return __builtin_amdgcn_readfirstlane(at) + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Keeps n >= want of a level's N items, at most 2 want, that hold the best `want`
// (all, if there are fewer): put(n, item) for each, in any order. `from`: a key that
// `want` items are known to reach (1: nothing is known); returns one for the next
// level. Bisection on the key, then, where keys tie, on the position: it ends whatever
// the items are.
template <class Get, class Put>
__device__ __forceinline__ uint64_t level(PickLds& l, int& turn, int N, int want, uint64_t from, Get get, Put put) {
  const int tid = threadIdx.x;
  const int most = 2 * want;
  auto each = [&](auto f) {
    for (int i0 = 0; i0 < N; i0 += kPickThreads) f(i0 + tid < N ? get(i0 + tid) : Item{0, 0});
  };
  auto count = [&](auto pred) {
    int c = 0;
    each([&](const Item& it) { c += __popcll(__ballot(it.key && pred(it))); });
    return block_count(l, turn, c);
  };
  uint64_t key = from;
  uint32_t id = ~0u;
  int n = count([&](const Item& it) { return it.key >= key; });
  if (n > most) {
    // more than `most` reach lo, fewer than `want` reach hi
    uint64_t lo = ~0ull, hi = 0;
    each([&](const Item& it) {
      if (it.key >= key && it.key) {
        lo = it.key < lo ? it.key : lo;
        hi = it.key > hi ? it.key : hi;
      }
    });
    lo = wave_all64(lo, [](uint64_t a, uint64_t b) { return a < b ? a : b; });
    hi = wave_all64(hi, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    if ((tid & 63) == 0) {
      l.lo[tid >> 6] = lo;
      l.hi[tid >> 6] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w) {
      lo = l.lo[w] < lo ? l.lo[w] : lo;
      hi = l.hi[w] > hi ? l.hi[w] : hi;
    }
    hi += 1;  // (no rank is NaN: there is room)
    bool done = false;
    int above = 0;  // items that reach hi
    while (hi - lo > 1 && !done) {
      const uint64_t mid = lo + (hi - lo) / 2;
      n = count([&](const Item& it) { return it.key >= mid; });
      if (n > most) lo = mid;
      else if (n < want) hi = mid, above = n;
      else key = mid, done = true;
    }
    if (!done) {  // ties at lo: by position
      key = lo;
      uint32_t a = 0, b = ~0u;  // positions <= b are too many, those < a too few
      while (!done) {
        const uint32_t mid = a + (b - a) / 2;
        n = above + count([&](const Item& it) { return it.key == lo && it.id <= mid; });
        if (n > most) b = mid;
        else if (n < want) a = mid + 1;
        else id = mid, done = true;
      }
    }
  }
  if (tid == 0) l.n = 0;
  __syncthreads();
  each([&](const Item& it) {
    const bool take = it.key && (it.key > key || (it.key == key && it.id <= id));
    const int at = place(&l.n, take);
    if (take) put(at, it);
  });
  __syncthreads();
  return key;
}

template <bool BF>
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamParams p) {
  __shared__ PickLds l;
  const DtreeBeamArgs& a = p.a;
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int K = a.beams, M = a.num_select, NC = p.chunks, row0 = g * K, V = a.vocab;
  const int N1 = K * NC;
  const float2* part = p.part + (size_t)row0 * NC;
  const bool staged = N1 <= kStaged;
  if (wave == kPickWaves - 1) {  // the beams' words
    const int row = row0 + min(lane, K - 1);
    const float score = beam_score(a, row);
    const bool over = beam_over(a, row);
    const int length = (a.lengths ? a.lengths[row] : 0) + (over ? 0 : 1);
    double w = 1., back = 1.;
    if (a.length_penalty != 0.f) {
      back = exp((double)a.length_penalty * log((double)max(length, 1)));
      w = 1. / back;
    }
    if (lane < K) {
      l.kind[lane] = over ? 2 : score > -INFINITY ? 1 : 0;
      l.score[lane] = score == score ? (double)score : -(double)INFINITY;
      l.length[lane] = length;
      l.weight[lane] = w;
      l.back[lane] = back;
    }
    if (lane == 0) l.n = l.n2 = l.n3 = 0;
  } else {  // their log sum exp over the chunks, 16 lanes each
    for (int b = 4 * wave + (lane >> 4); b < K; b += 4 * (kPickWaves - 1)) {
      const bool live = !beam_over(a, row0 + b) && beam_score(a, row0 + b) > -INFINITY;
      float m = -INFINITY;
      constexpr int kHeld = 3;  // pairs of a lane that stay in registers
      float2 held[kHeld];
#pragma unroll
      for (int r = 0; r < kHeld; ++r) {
        const int c = (lane & 15) + 16 * r;
        held[r] = c < NC ? part[b * NC + c] : make_float2(-INFINITY, 0.f);
      }
      // (a finished beam's are whatever the workspace holds)
      auto each = [&](auto f) {
#pragma unroll
        for (int r = 0; r < kHeld; ++r)
          if ((lane & 15) + 16 * r < NC) f((lane & 15) + 16 * r, held[r]);
#pragma unroll 1
        for (int c = (lane & 15) + 16 * kHeld; c < NC; c += 16) f(c, part[b * NC + c]);
      };
      each([&](int c, float2 v) {
        const float x = live ? v.x : -INFINITY;
        if (staged) l.top[b * NC + c] = x;
        m = fmaxf(m, x);
      });
      m = fmaxf(m, dpp<0xB1>(m));
      m = fmaxf(m, dpp<0x4E>(m));
      m = fmaxf(m, dpp<0x141>(m));
      m = fmaxf(m, dpp<0x140>(m));
      const float base = fmaxf(m, -kBig);
      double s = 0.;
      each([&](int, float2 v) { s += (double)(v.y * fast_exp2((v.x - base) * kLog2e)); });
      s += dpp_f64<0xB1>(s);
      s += dpp_f64<0x4E>(s);
      s += dpp_f64<0x141>(s);
      s += dpp_f64<0x140>(s);
      if ((lane & 15) == 0) {
        l.m[b] = m;  // (-inf: a row without a token to choose, which no rank below stands for)
        l.lse[b] = m > -INFINITY ? ln_of(s) : 0.;
      }
    }
  }
  __syncthreads();
  int turn = 0;
  auto total = [&](int b, float x) { return l.score[b] + (((double)x - (double)l.m[b]) - l.lse[b]); };
  auto key_of = [&](int b, float x) {
    return l.kind[b] == 1 && x > -INFINITY ? order_of(total(b, x) * l.weight[b]) : 0ull;
  };
  // the nearest fp32: in the same order, ranks below its range at its end
  auto rank32 = [&](int b, float x) { return fmaxf((float)(total(b, x) * l.weight[b]), -kBig); };
  auto ended = [&](int b) { return l.kind[b] == 2 ? order_of(l.score[b] * l.weight[b]) : 0ull; };

  int n = -1;  // the candidates left, in l.cand; -1: none yet
  if (staged) {
    // The quick way. Units by their maxima: chunks, or, where there are few, parts of
    // them, so that the threshold is one among many.
    int shift = 7;  // segments of a unit: 1 << shift, at least four
    if (N1 < 8 * M)
      while (shift > 2 && (N1 << (8 - shift)) <= kPickThreads) --shift;  // (a unit a thread)
    const int NU = N1 << (7 - shift), ends = (NU + 255) & ~255;  // (padded with -inf)
    const float inv = 1.f / NC;
    // (i / NC for i < 4096: the half is far above the product's error)
    auto beam_of = [&](int u) { return (int)(((u >> (7 - shift)) + 0.5f) * inv); };
    const f32x4_t* seg4 = reinterpret_cast<const f32x4_t*>(p.seg + (size_t)row0 * NC * kSegs);
#pragma unroll 1
    for (int i = tid; i < ends; i += kPickThreads) {
      const int b = min(beam_of(i), K - 1);
      float x = -INFINITY;
      if (i < NU && l.kind[b] == 1) {
        if (shift == 7) {
          x = l.top[i];
        } else {
          const f32x4_t* v = seg4 + ((size_t)i << (shift - 2));
#pragma unroll 4
          for (int j = 0; j < 1 << (shift - 2); ++j) x = fmaxf(fmaxf(fmaxf(x, v[j][0]), fmaxf(v[j][1], v[j][2])), v[j][3]);
        }
      }
      l.unit[i] = x > -INFINITY ? rank32(b, x) : -INFINITY;
    }
    __syncthreads();
    // A threshold that M to M + kSlack of them reach, if there is one: below the best
    // rank by growing steps, then between two; eight thresholds at a time, one a wave.
    const f32x4_t* unit4 = reinterpret_cast<const f32x4_t*>(l.unit);
    float best = -INFINITY;
    if (lane < K && l.kind[lane] == 1 && l.m[lane] > -INFINITY) best = rank32(lane, l.m[lane]);
    best = wave_max(best);
    const uint32_t all32 = order_of(-kBig);
    uint32_t lo = all32, hi = order_of(best) + 1;  // more than M + kSlack reach lo, fewer than M hi
    float t = -kBig;
    bool ok = false;
    for (int round = 0; !ok && (round == 0 || hi - lo > 1); ++round) {
      const int w = lane & (kPickWaves - 1);  // the probe of lane w, from the highest down
      uint32_t at;
      if (round == 0) at = w == kPickWaves - 1 ? all32 : order_of(fmaxf(best - ldexpf((float)l.weight[0], w - 1), -kBig));
      else at = hi - max((uint32_t)((uint64_t)(hi - lo) * (w + 1) / (kPickWaves + 1)), min((uint32_t)w + 1, hi - lo));
      const float mine = from_order((uint32_t)__builtin_amdgcn_readlane((int)at, wave));
      int c = 0;
#pragma unroll 1
      for (int i = lane; i < ends / 4; i += 64) {
        const f32x4_t v = unit4[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) c += (int)__popcll(__ballot(v[e] >= mine));
      }
      if (lane == 0) l.count[turn][wave] = c;
      lds_barrier();
      const int n = l.count[turn][w];
      turn ^= 1;
      if (round == 0 && __builtin_amdgcn_readlane(n, kPickWaves - 1) <= M) {  // all there are
        ok = true;
        break;
      }
      const int first = __ffsll((unsigned long long)(__ballot(n >= M) & ((1 << kPickWaves) - 1))) - 1;
      if (first >= 0) {
        const uint32_t reached = (uint32_t)__builtin_amdgcn_readlane((int)at, first);
        if (__builtin_amdgcn_readlane(n, first) <= M + kSlack && !(round == 0 && first == kPickWaves - 1)) {
          ok = true;
          t = from_order(reached);
          break;
        }
        lo = max(lo, reached);
      }
      if (first) hi = min(hi, (uint32_t)__builtin_amdgcn_readlane((int)at, first > 0 ? first - 1 : kPickWaves - 1));
    }
    if (ok) {
#pragma unroll 1
      for (int i = tid; i - lane < NU; i += kPickThreads) {
        const bool take = l.unit[i] >= t;
        const int at = place(&l.n, take);
        if (take) {
          const int b = beam_of(i);
          l.units[at] = (uint32_t)(b << 16 | ((i << shift) - b * NC * kSegs));
        }
      }
      // The least logit of a beam that reaches the number below t (and so every rank that
      // rounds to t), or one just below.
      const double low_rank = t > -kBig ? (double)from_order(order_of(t) - 1) : -INFINITY;
      if (wave == kPickWaves - 1 && lane < K) {
        float least = INFINITY;
        if (l.kind[lane] == 1) {
          const double by = low_rank * l.back[lane], m = (double)l.m[lane];
          const double x = ((by - l.score[lane]) + l.lse[lane]) + m;
          const double low = x - 1e-13 * (fabs(by) + fabs(l.score[lane]) + l.lse[lane] + fabs(m));
          least = low > -(double)kBig ? (float)low : -kBig;
          if ((double)least > low && least > -kBig) least = from_order(order_of(least) - 1);
        }
        l.least[lane] = least;
      }
      __syncthreads();
      // their segments, four a lane
      const int all = l.n << (shift - 2);
      constexpr int kAhead = 4;
      for (int i0 = tid; i0 - tid < all; i0 += kAhead * kPickThreads) {
        f32x4_t x[kAhead];
        uint32_t e[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = min(i0 + u * kPickThreads, all - 1);
          e[u] = l.units[i >> (shift - 2)] + 4 * (i & ((1 << (shift - 2)) - 1));
          x[u] = seg4[(e[u] >> 16) * (NC * kSegs / 4) + (e[u] & 0xffff) / 4];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const float least = i0 + u * kPickThreads < all ? l.least[e[u] >> 16] : INFINITY;
          const int c = (x[u][0] >= least) + (x[u][1] >= least) + (x[u][2] >= least) + (x[u][3] >= least);
          if (c) {
            int at = atomicAdd(&l.n2, c);
            for (int k = 0; k < 4; ++k)
              if (x[u][k] >= least) {
                if (at < kSegs1) l.segs[at] = e[u] + k;
                ++at;
              }
          }
        }
      }
      __syncthreads();
      // their logits: half a wave per segment
      const int ns = min(l.n2, kSegs1);
      const bool fits = l.n2 <= kSegs1;
      if (wave == kPickWaves - 1) {  // and the beams that have ended
        const uint64_t key = lane < K ? ended(lane) : 0;
        const bool take = key && rank_of(key) >= low_rank;
        const int at = take ? atomicAdd(&l.n3, 1) : 0;
        if (take && at < kBest1) {
          l.cand[at].id = (uint32_t)(lane * V + a.pad_token);
          l.cand[at].key = key;
        }
      }
      for (int j0 = 2 * wave; j0 < ns && fits; j0 += 2 * kAhead * kPickWaves) {
        float x[kAhead];
        uint32_t e[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int j = j0 + 2 * u * kPickWaves + (lane >> 5);
          e[u] = l.segs[min(j, ns - 1)];
          const int at = (e[u] & 0xffff) * kSeg + (lane & 31);
          x[u] = j < ns && at < V ? logit<BF>(a, row0 + (e[u] >> 16), at) : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int b = e[u] >> 16;
          if (x[u] >= l.least[b]) {
            const int at = atomicAdd(&l.n3, 1);
            if (at < kBest1) {
              l.cand[at].id = (uint32_t)(b * V) + (e[u] & 0xffff) * kSeg + (lane & 31);
              l.cand[at].x = x[u];
              l.cand[at].key = key_of(b, x[u]);
            }
          }
        }
      }
      __syncthreads();
      if (fits && l.n3 <= kBest1) n = l.n3;
    }
  }
  if (n < 0) {
    // The sure way, level by level.
    uint64_t from = 1;
    auto item = [&](int b, float x, uint32_t id) { return Item{key_of(b, x), id}; };
    from = level(l, turn, N1, M, from, [&](int i) { return item(i / NC, part[i].x, (uint32_t)i); },
                 [&](int at, const Item& it) { l.list[0][at] = it.id; });
    const int nc = l.n;
    from = level(l, turn, nc * kSegs, M, from,
                 [&](int i) {
                   const uint32_t c = l.list[0][i / kSegs];
                   const uint32_t id = c * kSegs + i % kSegs;
                   return item(c / NC, p.seg[(size_t)row0 * NC * kSegs + id], id);
                 },
                 [&](int at, const Item& it) { l.list[1][at] = it.id; });
    const int ns = l.n;
    level(l, turn, ns * kSeg + K, M, from,
          [&](int i) {
            if (i >= ns * kSeg) return Item{ended(i - ns * kSeg), (uint32_t)((i - ns * kSeg) * V + a.pad_token)};
            const uint32_t s = l.list[1][i / kSeg];
            const int b = s / (NC * kSegs), t = (s % (NC * kSegs)) * kSeg + i % kSeg;
            return t < V ? item(b, logit<BF>(a, row0 + b, t), (uint32_t)(b * V + t)) : Item{0, 0};
          },
          [&](int at, const Item& it) {
            l.cand[at].key = it.key;
            l.cand[at].id = it.id;
            const int b = it.id / V;
            l.cand[at].x = l.kind[b] == 1 ? logit<BF>(a, row0 + b, it.id % V) : 0.f;
          });
    n = l.n;
  }
  // Ranked by counting, eight threads a candidate (as many as there are for them all).
  const int q = n <= kPickThreads / 8 ? 8 : n <= kPickThreads / 4 ? 4 : 2;
  const int i = tid / q;
  int rank = 0;
  if (i < n) {
    const uint64_t key = l.cand[i].key;
    const uint32_t id = l.cand[i].id;
#pragma unroll 4
    for (int j = tid % q; j < n; j += q) rank += l.cand[j].key > key || (l.cand[j].key == key && l.cand[j].id < id);
  }
  rank += dpp_i<0xB1>(rank);
  if (q >= 4) rank += dpp_i<0x4E>(rank);
  if (q == 8) rank += dpp_i<0x141>(rank);
  // (what the outputs may replace has been read)
  const size_t o = (size_t)g * M;
  if (i < n && rank < M && tid % q == 0) {
    const uint32_t id = l.cand[i].id;
    const int b = id / V, t = id % V, over = l.kind[b] == 2, end = over || t == a.eos_token;
    a.scores_out[o + rank] = (float)(over ? l.score[b] : total(b, l.cand[i].x));
    a.tokens_out[o + rank] = t;
    a.parents_out[o + rank] = row0 + b;
    if (a.lengths_out) a.lengths_out[o + rank] = l.length[b];
    if (a.finished_out) a.finished_out[o + rank] = end;
    if (a.sources_out) a.sources_out[o + rank] = end ? -1 : row0 + b;
  }
  if (tid >= n && tid < M) {
    a.scores_out[o + tid] = -INFINITY;
    a.tokens_out[o + tid] = -1;
    a.parents_out[o + tid] = -1;
    if (a.lengths_out) a.lengths_out[o + tid] = 0;
    if (a.finished_out) a.finished_out[o + tid] = 0;
    if (a.sources_out) a.sources_out[o + tid] = -1;
  }
}

int beam_chunks(const DtreeBeamArgs* a) { return (a->vocab + kChunk - 1) / kChunk; }

int beam_check(const DtreeBeamArgs* a) {
  DTREE_REQUIRE(a, "beam_select: null args");
  DTREE_REQUIRE(a->type == DTREE_T_F32 || a->type == DTREE_T_BF16, "beam_select: type");
  DTREE_REQUIRE(a->vocab >= 1 && a->vocab <= kMaxVocab, "beam_select: vocab in [1, 2^20]");
  DTREE_REQUIRE(a->beams >= 1 && a->beams <= kMaxBeams, "beam_select: beams in [1, 64]");
  DTREE_REQUIRE(a->num_select >= 1 && a->num_select <= kMaxSelect, "beam_select: num_select in [1, 64]");
  DTREE_REQUIRE(a->groups >= 1 && (int64_t)a->groups * a->beams * beam_chunks(a) < (1 << 24),
                "beam_select: groups >= 1, and fewer than 2^24 blocks of 4096 logits in all rows");
  return DTREE_OK;
}

}  // namespace
}  // namespace dtree

using namespace dtree;

extern "C" size_t dtree_beam_args_bytes(void) { return sizeof(DtreeBeamArgs); }

extern "C" size_t dtree_beam_select_workspace_bytes(const DtreeBeamArgs* a) {
  if (beam_check(a)) return 0;
  const size_t bytes = (size_t)a->groups * a->beams * beam_chunks(a) * (kSegs * sizeof(float) + sizeof(float2));
  return (bytes + 15) & ~(size_t)15;
}

extern "C" int dtree_beam_select(const DtreeBeamArgs* a, hipStream_t stream) {
  if (int rc = beam_check(a)) return rc;
  DTREE_REQUIRE(a->logits && a->scores_out && a->tokens_out && a->parents_out, "beam_select: null pointer");
  DTREE_REQUIRE(((uintptr_t)a->logits & (a->type == DTREE_T_BF16 ? 1 : 3)) == 0, "beam_select: logits not aligned to their type");
  DTREE_REQUIRE(a->ld_logits >= a->vocab, "beam_select: ld_logits below vocab");
  DTREE_REQUIRE(a->eos_token >= -1 && a->eos_token < a->vocab, "beam_select: eos_token in [-1, vocab)");
  DTREE_REQUIRE(a->pad_token >= 0 && a->pad_token < a->vocab, "beam_select: pad_token in [0, vocab)");
  DTREE_REQUIRE(std::fabs(a->length_penalty) <= 16.f, "beam_select: length_penalty in [-16, 16]");
  auto replaces = [](const void* out, const void* in) { return in && out == in; };
  DTREE_REQUIRE(a->num_select == a->beams || !(replaces(a->scores_out, a->scores) || replaces(a->lengths_out, a->lengths) ||
                                              replaces(a->finished_out, a->finished)),
                "beam_select: outputs replace inputs with num_select == beams alone");
  DTREE_REQUIRE(((uintptr_t)a->workspace & 15) == 0 && a->workspace, "beam_select: workspace (16-byte aligned)");
  if (a->workspace_bytes < dtree_beam_select_workspace_bytes(a))
    return fail(DTREE_E_WORKSPACE, "beam_select: workspace below dtree_beam_select_workspace_bytes");
  BeamParams p{};
  p.a = *a;
  p.chunks = beam_chunks(a);
  const size_t blocks = (size_t)a->groups * a->beams * p.chunks;
  p.run = a->type == DTREE_T_BF16 && blocks >= kPairs ? 2 : 1;
  const unsigned scans = (unsigned)((size_t)a->groups * a->beams * ((p.chunks + p.run - 1) / p.run));
  p.seg = static_cast<float*>(a->workspace);  // (first: it is read 16 bytes at a time)
  p.part = reinterpret_cast<float2*>(p.seg + blocks * kSegs);
  if (a->type == DTREE_T_BF16) {
    beam_scan_kernel<true><<<scans, 256, 0, stream>>>(p);
    DTREE_LAUNCH_CHECK("beam_select scan launch");
    beam_pick_kernel<true><<<a->groups, kPickThreads, 0, stream>>>(p);
  } else {
    beam_scan_kernel<false><<<scans, 256, 0, stream>>>(p);
    DTREE_LAUNCH_CHECK("beam_select scan launch");
    beam_pick_kernel<false><<<a->groups, kPickThreads, 0, stream>>>(p);
  }
  DTREE_LAUNCH_CHECK("beam_select launch");
  return DTREE_OK;
}
