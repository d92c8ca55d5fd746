// Forking, sharing and freeing the pages of a pool of sequences (the caches of
// adapters.py:478-484 for several hypotheses of one prompt), and the copies that a
// fork asks for.
//
// A page's count is the number of sequences whose table holds it; 0 is free. There is
// no other state (no list of free pages), so a fork's result follows from its inputs
// alone: the counts change by integer atomics, whose order does not matter, and the
// pages taken are the lowest free ones, by ascending sequence.
//
// share  A workgroup per (sequence, 1024 table entries): the entry of its parent into
//        its new table, and its old table's pages' counts by (children - 1), or down by
//        one past its length. Sequences with one child touch no count.
// take   One workgroup, a thread per sequence: which page must be copied (held by others
//        and about to be written), how many are needed, a prefix sum over the
//        sequences; then one pass over the counts in page order, in which the free page
//        of rank r goes to the sequence whose range holds r (a search of the sums in LDS).
// copy   Persistent workgroups over (copy, layer, head): the half pages in use of every
//        pool. Bound by the bytes, the tables' two launches by latency.
#include "common.h"

namespace dtree {
namespace {

constexpr int kMaxSeqs = 1024;
constexpr int kShare = 1024;          // table entries of a share workgroup
constexpr int kTake = 1024, kTakeWaves = kTake / 64;
constexpr int kScan = 16 * 4;         // counts a thread looks at in one round
constexpr int kRound = kTake * kScan;
constexpr int kHalfPage = DTREE_PAGE / 2;

__device__ __forceinline__ int fork_parent(const DtreePagesFork& a, int i) {
  const int p = a.parents ? a.parents[i] : i;
  return p >= 0 && p < a.num_seqs ? p : -1;
}
__device__ __forceinline__ int fork_length(const DtreePagesFork& a, int p) {
  const int64_t n = (int64_t)a.lengths[p] + a.advance;
  return (int)min(max(n, (int64_t)0), (int64_t)a.ld_tables * DTREE_PAGE);
}
__device__ __forceinline__ bool is_page(const DtreePagesFork& a, int page) {
  return page >= 0 && page < a.num_pages && page != a.absent;
}

__global__ __launch_bounds__(256) void pages_share_kernel(DtreePagesFork a) {
  __shared__ int kids;
  const int s = blockIdx.x, tid = threadIdx.x;
  int children = 1;
  if (a.parents) {
    if (tid == 0) kids = 0;
    __syncthreads();
    int c = 0;
    for (int i = tid; i < a.num_seqs; i += 256) c += a.parents[i] == s;
    if (c) atomicAdd(&kids, c);
    __syncthreads();
    children = kids;
  }
  const int par = fork_parent(a, s);
  const int have = (fork_length(a, s) + DTREE_PAGE - 1) / DTREE_PAGE;
  const int take = par >= 0 ? (fork_length(a, par) + DTREE_PAGE - 1) / DTREE_PAGE : 0;
  const int end = min(a.ld_tables, (int)(blockIdx.y + 1) * kShare);
  for (int e = blockIdx.y * kShare + tid; e < end; e += 256) {
    const int mine = a.tables[(size_t)s * a.ld_tables + e];
    int out = a.absent;
    if (e < take) {
      const int page = par == s ? mine : a.tables[(size_t)par * a.ld_tables + e];
      if (is_page(a, page)) out = page;
    }
    a.tables_out[(size_t)s * a.ld_tables + e] = out;
    const int by = e < have ? children - 1 : -1;
    if (by && is_page(a, mine)) atomicAdd(a.refs + mine, by);
  }
}

// Exclusive prefix sum over the workgroup's threads; `all`: the total.
__device__ __forceinline__ int block_scan(int v, int* waves, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();  // (the last call's sums are read)
  if (lane == 63) waves[wave] = inc;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kTakeWaves; ++w) {
    before += w < wave ? waves[w] : 0;
    sum += waves[w];
  }
  all = sum;
  return before + inc - v;
}

__global__ __launch_bounds__(kTake) void pages_take_kernel(DtreePagesFork a) {
  __shared__ int waves[kTakeWaves];
  __shared__ int writes[kMaxSeqs];       // the shared page that a sequence is about to write, -1
  __shared__ int start[kMaxSeqs + 1];    // pages wanted before a sequence's
  __shared__ int first[kMaxSeqs];        // its table entry of the first page past its length; copies: complemented
  __shared__ int shared_any;
  const int i = threadIdx.x, n = a.num_seqs;
  const bool in = i < n;
  const int par = in ? fork_parent(a, i) : -1;
  const int L = par >= 0 ? fork_length(a, par) : 0;
  const int covered = (L + DTREE_PAGE - 1) / DTREE_PAGE, at = L / DTREE_PAGE;
  const int64_t wanted = in ? ((int64_t)L + a.rows + DTREE_PAGE - 1) / DTREE_PAGE : 0;
  const int last = (int)min(wanted, (int64_t)a.ld_tables);
  int* row = a.tables_out + (size_t)i * a.ld_tables;
  if (i == 0) shared_any = 0;
  __syncthreads();  // (every length is read: lengths_out may be lengths)
  if (in) a.lengths_out[i] = L;
  int page = -1, holders = 0;
  if (in && a.rows > 0 && L % DTREE_PAGE) {
    page = row[at];
    if (is_page(a, page)) holders = a.refs[page];
    else page = -1;
  }
  writes[i] = holders > 1 ? page : -1;
  if (holders > 1) shared_any = 1;
  __syncthreads();
  // Writers of one page, in ascending order: the k-th copies where others are left.
  bool copy = false;
  if (shared_any) {
    if (holders > 1) {
      int k = 0;
      for (int j = 0; j < i; ++j) k += writes[j] == page;
      copy = holders - k > 1;
    }
  }
  if (copy) atomicAdd(a.refs + page, -1);
  int total, copies;
  const int grow = in ? max(last - covered, 0) : 0;
  const int before = block_scan((copy ? 1 : 0) + grow, waves, total);
  start[i] = before;
  first[i] = copy ? ~covered : covered;
  if (i == 0) start[n] = total;
  // (no page: the entries past the length, and a copy's own, stay without one)
  if (copy) row[at] = a.absent;
  __syncthreads();
  // The free pages in ascending order: wave w looks at 64 kScan counts of a round, 256 a load.
  const int lane = i & 63, wave = i >> 6;
  int taken = 0;
  for (int64_t base = 0; base < a.num_pages && taken < total; base += kRound) {
    const int64_t w0 = base + (int64_t)wave * 64 * kScan;
    int found = 0;
    uint64_t mask = 0;  // bit 4 k + e: count 256 k + 4 lane + e of the wave's is 0
#pragma unroll
    for (int k = 0; k < kScan / 4; ++k) {
      const int64_t p0 = w0 + 256 * k + 4 * lane;
      int c[4] = {1, 1, 1, 1};
      if (p0 + 3 < a.num_pages) {
        __builtin_memcpy(c, a.refs + p0, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (p0 + e < a.num_pages) c[e] = a.refs[p0 + e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c[e] == 0 && (int)(p0 + e) != a.absent) mask |= 1ull << (4 * k + e);
    }
    found = __popcll(mask);
    int sum = found;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    __syncthreads();
    if (lane == 0) waves[wave] = sum;
    __syncthreads();
    int rank = taken, all = 0;
#pragma unroll
    for (int w = 0; w < kTakeWaves; ++w) {
      rank += w < wave ? waves[w] : 0;
      all += waves[w];
    }
#pragma unroll 1
    for (int k = 0; k < kScan / 4; ++k) {
      if (rank >= total) break;  // (a wave's rank is the same in its lanes)
      const int bits = (int)(mask >> (4 * k)) & 15, c = __popc(bits);
      int inc = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o);
        if (lane >= o) inc += u;
      }
      int r = rank + inc - c;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!(bits >> e & 1)) continue;
        if (r < total) {
          const int pg = (int)(w0 + 256 * k + 4 * lane + e);
          int lo = 0, hi = n;  // the last sequence whose range starts at r or before, of those with one
          while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (start[mid] <= r) lo = mid;
            else hi = mid;
          }
          const int f = first[lo], j = r - start[lo];
          int* out = a.tables_out + (size_t)lo * a.ld_tables;
          // a copy takes the sequence's first page, for the entry before its new ones
          out[f < 0 ? ~f + j - 1 : f + j] = pg;
          a.refs[pg] = 1;
        }
        ++r;
      }
      rank += __shfl(inc, 63);
    }
    taken += all;
  }
  __syncthreads();
  const int to = copy ? row[at] : a.absent;
  const bool made = copy && is_page(a, to);
  const int spot = block_scan(made ? 1 : 0, waves, copies);
  if (a.copies) {
    if (made) {
      a.copies[3 * spot] = page;
      a.copies[3 * spot + 1] = to;
      a.copies[3 * spot + 2] = L % DTREE_PAGE;
    }
    if (in && i >= copies) {
      a.copies[3 * i] = -1;
      a.copies[3 * i + 1] = -1;
      a.copies[3 * i + 2] = -1;
    }
  }
  if (a.status) {
    const int beyond = in ? (int)min(wanted - last, (int64_t)1 << 20) : 0;
    int past;
    block_scan(beyond, waves, past);
    if (i == 0) {
      a.status[0] += max(total - taken, 0) + past;
      a.status[1] = copies;
    }
  }
}

__global__ __launch_bounds__(256) void pages_copy_kernel(DtreePagesCopy a) {
  __shared__ int ends;  // the list's first negative source
  const int tid = threadIdx.x, per = a.layers * a.num_heads;
  if (tid == 0) ends = a.max_copies;
  __syncthreads();
  for (int c = tid; c < a.max_copies; c += 256)
    if (a.copies[3 * c] < 0) {
      atomicMin(&ends, c);
      break;
    }
  __syncthreads();
  const int units = ends * per;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = u / per, lh = u % per, layer = lh / a.num_heads, head = lh % a.num_heads;
    const int src = a.copies[3 * c], dst = a.copies[3 * c + 1], used = a.copies[3 * c + 2];
    if (src >= a.num_pages || dst < 0 || dst >= a.num_pages || used <= 0) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!a.pools[i]) continue;
      const int bytes = a.block_bytes[i], n = (used > kHalfPage ? bytes : bytes / 2) / 16;
      char* pool = static_cast<char*>(a.pools[i]);
      const size_t layer0 = (size_t)layer * a.num_pages;
      const u32x4_t* from = reinterpret_cast<const u32x4_t*>(pool + ((layer0 + src) * a.num_heads + head) * bytes);
      u32x4_t* to = reinterpret_cast<u32x4_t*>(pool + ((layer0 + dst) * a.num_heads + head) * bytes);
      for (int v = tid; v < n; v += 256) to[v] = from[v];
    }
  }
}

}  // namespace
}  // namespace dtree

using namespace dtree;

extern "C" size_t dtree_pages_fork_bytes(void) { return sizeof(DtreePagesFork); }
extern "C" size_t dtree_pages_copy_bytes(void) { return sizeof(DtreePagesCopy); }

extern "C" int dtree_pages_fork(const DtreePagesFork* a, hipStream_t stream) {
  DTREE_REQUIRE(a, "pages_fork: null args");
  DTREE_REQUIRE(a->refs && a->tables && a->tables_out && a->lengths && a->lengths_out, "pages_fork: null pointer");
  DTREE_REQUIRE(a->num_seqs >= 1 && a->num_seqs <= kMaxSeqs, "pages_fork: num_seqs in [1, 1024]");
  DTREE_REQUIRE(a->num_pages >= 1, "pages_fork: num_pages");
  DTREE_REQUIRE(a->ld_tables >= 1 && a->ld_tables <= (1 << 22), "pages_fork: ld_tables in [1, 2^22]");
  DTREE_REQUIRE(a->rows >= 0 && a->advance >= 0, "pages_fork: rows and advance not negative");
  DTREE_REQUIRE(a->absent >= -1 && a->absent < a->num_pages, "pages_fork: absent is -1 or a page");
  DTREE_REQUIRE(a->tables != a->tables_out || !a->parents, "pages_fork: in place without parents alone");
  const int64_t rows = a->num_seqs;
  const int64_t size = rows * a->ld_tables;
  DTREE_REQUIRE(size < (1 << 30), "pages_fork: fewer than 2^30 table entries");
  DTREE_REQUIRE(a->tables == a->tables_out || a->tables + size <= a->tables_out || a->tables_out + size <= a->tables,
                "pages_fork: tables and tables_out overlap");
  DTREE_REQUIRE(a->lengths == a->lengths_out || a->lengths + rows <= a->lengths_out || a->lengths_out + rows <= a->lengths,
                "pages_fork: lengths and lengths_out partly overlap");
  const dim3 grid(a->num_seqs, (a->ld_tables + kShare - 1) / kShare);
  pages_share_kernel<<<grid, 256, 0, stream>>>(*a);
  DTREE_LAUNCH_CHECK("pages_fork share launch");
  pages_take_kernel<<<1, kTake, 0, stream>>>(*a);
  DTREE_LAUNCH_CHECK("pages_fork take launch");
  return DTREE_OK;
}

extern "C" int dtree_pages_copy(const DtreePagesCopy* a, hipStream_t stream) {
  DTREE_REQUIRE(a && a->copies, "pages_copy: null pointer");
  DTREE_REQUIRE(a->max_copies >= 1 && a->max_copies <= kMaxSeqs, "pages_copy: max_copies in [1, 1024]");
  DTREE_REQUIRE(a->num_pages >= 1 && a->layers >= 1 && a->num_heads >= 1 && (int64_t)a->layers * a->num_heads <= (1 << 20),
                "pages_copy: num_pages, layers and num_heads positive, layers * num_heads <= 2^20");
  bool any = false;
  for (int i = 0; i < 4; ++i) {
    if (!a->pools[i]) continue;
    any = true;
    DTREE_REQUIRE(((uintptr_t)a->pools[i] & 15) == 0 && a->block_bytes[i] >= 32 && a->block_bytes[i] % 32 == 0,
                  "pages_copy: pools 16-byte aligned, block_bytes a multiple of 32");
  }
  DTREE_REQUIRE(any, "pages_copy: no pool");
  const int units = a->max_copies * a->layers * a->num_heads;
  pages_copy_kernel<<<units < 2048 ? units : 2048, 256, 0, stream>>>(*a);
  DTREE_LAUNCH_CHECK("pages_copy launch");
  return DTREE_OK;
}
