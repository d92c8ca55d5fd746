// Beam search's selection: of every group of beams the best (beam, token)
// continuations by summed log-probability (the batched, several-hypotheses
// counterpart of the greedy argmax of adapters.py:114-118).
//
// s(b, t) = score_b + (x_bt - lse_b), rank(b, t) = s / length^penalty, all in fp64:
// two candidates of different beams that fp32 would round together are told apart.
// Ties go to the lower beam, then the lower token.
//
// Two launches.
//
// scan   One pass over the logits, a workgroup per (row, 4096 logits) in registers:
//        the chunk's maximum and sum of exp(x - max), and the maximum of each run of
//        32 logits ("segment"). Bound by the logits' bytes.
// pick   A workgroup per group. rank grows with x inside a beam, so a selected token
//        lies in one of the num_select best segments by their maxima, and such a
//        segment in one of the num_select best chunks. Three levels, each over the
//        survivors of the one before: chunks, segments, logits. A level keeps what is
//        not below a threshold, found by bisection on the order-preserving integer of
//        the rank (then, where ranks tie, on the position) and loose: any that leaves
//        num_select to twice as many does, and the level before hands its own down,
//        which usually does. The last survivors are ranked by counting. Bound by
//        latency.
#include <cmath>

#include "common.h"

namespace dtree {
namespace {

constexpr int kChunk = 4096;           // logits of a scan workgroup
constexpr int kSeg = 32;               // logits of a segment
constexpr int kSegs = kChunk / kSeg;   // segments of a chunk
constexpr int kMaxBeams = 64;
constexpr int kMaxSelect = 64;
constexpr int kMaxVocab = 1 << 20;
constexpr int kPickThreads = 512, kPickWaves = kPickThreads / 64;
constexpr int kKeep = 2 * kMaxSelect;  // survivors of a level
constexpr int kInReg = 8;              // a level's items of a thread that stay in registers
constexpr float kBig = 3.40282347e38f;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
  DtreeBeamArgs a;
  int chunks;
  float2* part;     // [rows][chunks] maximum, sum of exp(x - maximum)
  float* seg;       // [rows][chunks][kSegs] maxima
};

// A logit as the selection takes it: NaN as -inf, +inf as the largest number.
__device__ __forceinline__ float clean(float x) { return x > -INFINITY ? fminf(x, kBig) : -INFINITY; }

// A beam that is summed over its vocabulary (not finished, with a score).
__device__ __forceinline__ bool beam_over(const DtreeBeamArgs& a, int row) { return a.finished && a.finished[row]; }
__device__ __forceinline__ float beam_score(const DtreeBeamArgs& a, int row) { return a.scores ? a.scores[row] : 0.f; }

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  v = fmaxf(v, dpp<0x141>(v));
  v = fmaxf(v, dpp<0x140>(v));
  v = fmaxf(v, swz_xor16(v));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = row_sum32(v);
  return v + __shfl_xor(v, 32);
}

template <bool BF>
__device__ __forceinline__ float logit(const DtreeBeamArgs& a, int row, int t) {
  const size_t at = (size_t)row * a.ld_logits + t;
  if constexpr (BF) return clean(bf2f(static_cast<const uint16_t*>(a.logits)[at]));
  else return clean(static_cast<const float*>(a.logits)[at]);
}

template <bool BF>
__global__ __launch_bounds__(256) void beam_scan_kernel(BeamParams p) {
  constexpr int E = BF ? 8 : 4, NL = kChunk / 256 / E;  // logits of a load, loads of a thread
  constexpr int LPS = kSeg / E;                         // lanes of a segment
  __shared__ float wm[4], ws[4];
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  if (beam_over(p.a, row) || !(beam_score(p.a, row) > -INFINITY)) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int left = p.a.vocab - chunk * kChunk;
  float x[NL][E];
  const char* src = static_cast<const char*>(p.a.logits) + ((size_t)row * p.a.ld_logits + chunk * kChunk) * (BF ? 2 : 4);
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int at = (i * 256 + tid) * E;
    if (at + E <= left) {
      u32x4_t w;
      __builtin_memcpy(&w, src + (size_t)at * (BF ? 2 : 4), 16);  // (rows at any address of their type)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (BF) x[i][e] = __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
        else x[i][e] = __uint_as_float(w[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[i][e] = -INFINITY;
        if (at + e < left) {
          if constexpr (BF) x[i][e] = bf2f(reinterpret_cast<const uint16_t*>(src)[at + e]);
          else x[i][e] = reinterpret_cast<const float*>(src)[at + e];
        }
      }
    }
  }
  float mx = -INFINITY, keep = 0.f;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[i][e] = clean(x[i][e]);
      m = fmaxf(m, x[i][e]);
    }
    m = fmaxf(m, dpp<0xB1>(m));
    m = fmaxf(m, dpp<0x4E>(m));
    if constexpr (LPS == 8) m = fmaxf(m, dpp<0x141>(m));
    if ((tid & (LPS - 1)) == i) keep = m;
    mx = fmaxf(mx, m);
  }
  // lane i of a segment's lanes has load i's
  const int sl = tid & (LPS - 1);
  if (sl < NL) p.seg[(size_t)blockIdx.x * kSegs + sl * (256 / LPS) + tid / LPS] = keep;
  mx = wave_max(mx);
  if (lane == 0) wm[wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
  const float base = fmaxf(mx, -kBig);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NL; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) sum += fast_exp2((x[i][e] - base) * kLog2e);
  sum = wave_sum(sum);
  if (lane == 0) ws[wave] = sum;
  __syncthreads();
  if (tid == 0) p.part[blockIdx.x] = make_float2(mx, ws[0] + ws[1] + ws[2] + ws[3]);
}

// Order-preserving integer of a rank; 0 for what is no candidate.
__device__ __forceinline__ uint64_t order_of(double v) {
  if (!(v > -INFINITY)) return 0;
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

struct Item {
  uint64_t key;
  uint32_t id;  // position: the lower one wins a tie
};

struct PickLds {
  double score[kMaxBeams], lse[kMaxBeams], weight[kMaxBeams];  // lse: less the maximum
  int live[kMaxBeams];  // 1: summed over its vocabulary, 2: finished
  float m[kMaxBeams];
  int count[2][kPickWaves];
  uint64_t lo[kPickWaves], hi[kPickWaves];
  int n;
  uint32_t list[2][kKeep];
  uint64_t key[kKeep];
  double total[kKeep];
};

// How many of the workgroup's threads' counts there are, in every thread.
__device__ __forceinline__ int block_count(PickLds& l, int& turn, int c) {
  // (sums over lanes; two buffers, so that one barrier a call is enough)
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o);
  if ((threadIdx.x & 63) == 0) l.count[turn][threadIdx.x >> 6] = c;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int w = 0; w < kPickWaves; ++w) n += l.count[turn][w];
  turn ^= 1;
  return n;
}

// Keeps n >= want of a level's N items, at most 2 want, that hold the best `want`
// (all, if there are fewer): put(item) for each, in any order. `from`: a key that
// `want` items are known to reach (1: nothing is known); returns one for the next level.
template <class Get, class Put>
__device__ __forceinline__ uint64_t level(PickLds& l, int& turn, int N, int want, uint64_t from, Get get, Put put) {
  const int tid = threadIdx.x;
  const int most = 2 * want;
  Item mine[kInReg];
#pragma unroll
  for (int r = 0; r < kInReg; ++r) {
    const int i = tid + r * kPickThreads;
    mine[r] = i < N ? get(i) : Item{0, 0};
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int r = 0; r < kInReg; ++r) f(mine[r]);
    for (int i = tid + kInReg * kPickThreads; i < N; i += kPickThreads) f(get(i));
  };
  auto count = [&](auto pred) {
    int c = 0;
    each([&](const Item& it) { c += it.key && pred(it) ? 1 : 0; });
    return block_count(l, turn, c);
  };
  uint64_t key = from;
  uint32_t id = ~0u;
  int n = count([&](const Item& it) { return it.key >= key; });
  if (n > most) {
    // bisection: more than `most` reach lo, fewer than `want` reach hi
    uint64_t lo = ~0ull, hi = 0;
    each([&](const Item& it) {
      if (it.key >= key && it.key) {
        lo = it.key < lo ? it.key : lo;
        hi = it.key > hi ? it.key : hi;
      }
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t a = __shfl_xor(lo, o), b = __shfl_xor(hi, o);
      lo = a < lo ? a : lo;
      hi = b > hi ? b : hi;
    }
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
    hi += 1;  // (below the largest key's end: no rank is NaN)
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
    if (it.key && (it.key > key || (it.key == key && it.id <= id))) put(atomicAdd(&l.n, 1), it);
  });
  __syncthreads();
  return key;
}

template <bool BF>
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamParams p) {
  __shared__ PickLds l;
  const DtreeBeamArgs& a = p.a;
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int K = a.beams, M = a.num_select, NC = p.chunks, row0 = g * K;
  // the beams' sums: log sum exp over the chunks
  for (int b = wave; b < K; b += kPickWaves) {
    const float2* part = p.part + (size_t)(row0 + b) * NC;
    const bool over = beam_over(a, row0 + b);
    const bool live = !over && beam_score(a, row0 + b) > -INFINITY;
    float m = -INFINITY;
    double s = 0.;
    if (live) {
      for (int c = lane; c < NC; c += 64) m = fmaxf(m, part[c].x);
      m = wave_max(m);
      const float base = fmaxf(m, -kBig);
      for (int c = lane; c < NC; c += 64) s += (double)(part[c].y * fast_exp2((part[c].x - base) * kLog2e));
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    }
    if (lane == 0) {
      l.live[b] = over ? 2 : live && m > -INFINITY ? 1 : 0;
      l.m[b] = m;
      l.lse[b] = s;
    }
  }
  __syncthreads();
  if (tid < K) {
    const float score = beam_score(a, row0 + tid);
    const int kind = l.live[tid];
    const int len = max((a.lengths ? a.lengths[row0 + tid] : 0) + (kind == 2 ? 0 : 1), 1);
    l.score[tid] = score == score ? (double)score : -(double)INFINITY;
    l.lse[tid] = kind == 1 ? log(l.lse[tid]) : 0.;
    l.weight[tid] = a.length_penalty != 0.f ? pow((double)len, -(double)a.length_penalty) : 1.;
  }
  __syncthreads();
  int turn = 0;
  auto total = [&](int b, float x) { return l.score[b] + (((double)x - (double)l.m[b]) - l.lse[b]); };
  auto item = [&](int b, float x, uint32_t id) {
    return Item{x > -INFINITY && l.live[b] == 1 ? order_of(total(b, x) * l.weight[b]) : 0ull, id};
  };
  uint64_t from = 1;
  from = level(l, turn, K * NC, M, from,
               [&](int i) {
                 const int b = i / NC;
                 return l.live[b] == 1 ? item(b, p.part[(size_t)row0 * NC + i].x, (uint32_t)i) : Item{0, 0};
               },
               [&](int n, const Item& it) { l.list[0][n] = it.id; });
  const int nc = l.n;
  from = level(l, turn, nc * kSegs, M, from,
               [&](int i) {
                 const uint32_t c = l.list[0][i / kSegs];
                 const uint32_t id = c * kSegs + i % kSegs;
                 return item(c / NC, p.seg[(size_t)row0 * NC * kSegs + id], id);
               },
               [&](int n, const Item& it) { l.list[1][n] = it.id; });
  const int ns = l.n;
  level(l, turn, ns * kSeg + K, M, from,
        [&](int i) {
          if (i >= ns * kSeg) {
            const int b = i - ns * kSeg;
            return Item{l.live[b] == 2 ? order_of(l.score[b] * l.weight[b]) : 0ull, (uint32_t)(b * a.vocab + a.pad_token)};
          }
          const uint32_t s = l.list[1][i / kSeg];
          const int b = s / (NC * kSegs), t = (s % (NC * kSegs)) * kSeg + i % kSeg;
          return t < a.vocab ? item(b, logit<BF>(a, row0 + b, t), (uint32_t)(b * a.vocab + t)) : Item{0, 0};
        },
        [&](int n, const Item& it) {
          l.key[n] = it.key;
          l.list[0][n] = it.id;
        });
  const int n = l.n;
  // (inputs that the outputs may replace are read before this barrier)
  int rank = 0, b = 0, t = 0, len = 0, over = 0;
  if (tid < n) {
    const uint64_t key = l.key[tid];
    const uint32_t id = l.list[0][tid];
    for (int i = 0; i < n; ++i) rank += l.key[i] > key || (l.key[i] == key && l.list[0][i] < id);
    b = id / a.vocab;
    t = id % a.vocab;
    over = l.live[b] == 2;
    len = (a.lengths ? a.lengths[row0 + b] : 0) + (over ? 0 : 1);
  }
  __syncthreads();
  const size_t o = (size_t)g * M;
  if (tid < n && rank < M) {
    const double s = over ? l.score[b] : total(b, logit<BF>(a, row0 + b, t));
    const int end = over || t == a.eos_token;
    a.scores_out[o + rank] = (float)s;
    a.tokens_out[o + rank] = t;
    a.parents_out[o + rank] = row0 + b;
    if (a.lengths_out) a.lengths_out[o + rank] = len;
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
  return (size_t)a->groups * a->beams * beam_chunks(a) * (sizeof(float2) + kSegs * sizeof(float));
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
  p.part = static_cast<float2*>(a->workspace);
  p.seg = reinterpret_cast<float*>(p.part + blocks);
  if (a->type == DTREE_T_BF16) {
    beam_scan_kernel<true><<<(unsigned)blocks, 256, 0, stream>>>(p);
    DTREE_LAUNCH_CHECK("beam_select scan launch");
    beam_pick_kernel<true><<<a->groups, kPickThreads, 0, stream>>>(p);
  } else {
    beam_scan_kernel<false><<<(unsigned)blocks, 256, 0, stream>>>(p);
    DTREE_LAUNCH_CHECK("beam_select scan launch");
    beam_pick_kernel<false><<<a->groups, kPickThreads, 0, stream>>>(p);
  }
  DTREE_LAUNCH_CHECK("beam_select launch");
  return DTREE_OK;
}
