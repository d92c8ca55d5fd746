// Forking, sharing and freeing the pages of a pool of sequences (the caches of
// adapters.py:478-484 for several hypotheses of one prompt), and the copies that a
// fork asks for.
//
// A page's count is the number of sequences whose table holds it; 0 is free. There is
// no other state (no list of free pages), so a fork's result follows from its inputs
// alone: the counts change by integer atomics, whose order does not matter, and the
// pages taken are the lowest free ones, by ascending sequence.
//
// share  The entry of a sequence's parent into its new table, and its old table's pages'
//        counts by (children - 1), or down by one past its length. Sequences with one
//        child touch no count, and neighbours that hold a page change it together. A
//        workgroup per 256 entries of a few sequences.
// take   One workgroup, a thread per sequence: which page must be copied (held by others
//        and about to be written), how many are needed, a prefix sum over the
//        sequences. The free pages come from one pass over the counts in page order,
//        whose loads go out first; they are listed in LDS, and the page of rank r goes
//        to the sequence whose range holds r (a search of the sums).
//        Small forks (kOneLaunch entries) are shared by this workgroup too.
// copy   Persistent workgroups over (copy, layer, head): the half pages in use of every
//        pool.
//
// The copies are bound by their bytes, the tables by latency (four loads in a row: the
// parent, its length, its page, the page's count). Measured: 8 sequences of 1020
// positions, 36 layers of 8 heads of 128 in 8 bits: take 6.0 us, copy 6.5 (29 MB moved,
// 4.5 TB/s), 12.8 together; 128 sequences of 4100, 8 layers of 4 heads of 256: share 4,
// take 6.0, copy 12.9 (78 MB, 6 TB/s); 512 sequences of 32808 (264 000 entries): share 6,
// take 9.0, copy 6.3. The share step within the take workgroup (one launch fewer) pays up
// to 4096 entries, us of a fork in one launch and in two: 8 sequences of 64 entries 5.6
// and 7.9, of 129 5.7 and 7.7; 32 of 64 6.8 and 8.3; 24 of 129 7.1 to 7.5 and 8.4; 32 of
// 129 8.3 to 8.7 and 8.4; 64 of 96 9.2 and 8.6; 128 of 64 11.7 and 8.7; 512 of 16 15.1 and 9.5.
#include "common.h"

namespace dtree {
namespace {

constexpr int kMaxSeqs = 1024;
// Neighbouring sequences of a share workgroup: 512 sequences of 32808 positions take 21.1
// us (24.4 with one, each by its own atomics), 20.6 with 8, 128 of 4100 25.5 and 26.5.
constexpr int kSide = 4;
constexpr int kTake = 1024, kTakeWaves = kTake / 64;
constexpr int kOneLaunch = 4096;      // table entries that the take workgroup shares by itself (figures above)
constexpr int kRun = 32;              // neighbouring counts of a thread in one round
constexpr int kRound = kTake * kRun;
constexpr int kList = 4096;           // free pages listed at a time
constexpr int kHash = 2 * kMaxSeqs;
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

// Entry e of sequence s: the new table's, and the old one's page's count, by a lone
// workgroup, whose atomics are done in its own cache (an agent's behind the XCDs').
__device__ __forceinline__ void share_entry(const DtreePagesFork& a, int s, int e, int par, int take, int have, int children) {
  const int mine = a.tables[(size_t)s * a.ld_tables + e];
  int out = a.absent;
  if (e < take) {
    const int page = par == s ? mine : a.tables[(size_t)par * a.ld_tables + e];
    if (is_page(a, page)) out = page;
  }
  a.tables_out[(size_t)s * a.ld_tables + e] = out;
  const int by = e < have ? children - 1 : -1;
  if (by && is_page(a, mine)) __hip_atomic_fetch_add(a.refs + mine, by, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// A workgroup: 256 entries of kSide neighbouring sequences, a thread an entry of all of
// them. Neighbours that hold one page there, as a prompt's hypotheses do, change its
// count once, by the sum, which is often 0.
__global__ __launch_bounds__(256) void pages_share_kernel(DtreePagesFork a) {
  __shared__ int kids[kSide], from[kSide], have[kSide], take[kSide];
  const int s0 = blockIdx.x * kSide, tid = threadIdx.x, e = blockIdx.y * 256 + tid;
  if (tid < kSide) {
    const int s = min(s0 + tid, a.num_seqs - 1), p = fork_parent(a, s);
    kids[tid] = a.parents ? 0 : 1;
    from[tid] = p;
    have[tid] = (fork_length(a, s) + DTREE_PAGE - 1) / DTREE_PAGE;
    take[tid] = p >= 0 ? (fork_length(a, p) + DTREE_PAGE - 1) / DTREE_PAGE : 0;
  }
  __syncthreads();
  if (a.parents) {
    for (int i = tid; i < a.num_seqs; i += 256) {
      const uint32_t k = (uint32_t)a.parents[i] - (uint32_t)s0;  // (no sequence: 2^31 or more)
      if (k < kSide) atomicAdd(&kids[k], 1);
    }
    __syncthreads();
  }
  if (e >= a.ld_tables) return;
  int mine[kSide], out[kSide];
#pragma unroll
  for (int j = 0; j < kSide; ++j) {  // (loads without branches go out together)
    mine[j] = a.tables[(size_t)min(s0 + j, a.num_seqs - 1) * a.ld_tables + e];
    out[j] = a.tables[(size_t)max(from[j], 0) * a.ld_tables + e];
  }
  int page = -1, by = 0;
#pragma unroll
  for (int j = 0; j < kSide; ++j) {
    if (s0 + j >= a.num_seqs) break;
    a.tables_out[(size_t)(s0 + j) * a.ld_tables + e] = e < take[j] && is_page(a, out[j]) ? out[j] : a.absent;
    if (!is_page(a, mine[j])) continue;
    if (mine[j] != page) {
      if (by) atomicAdd(a.refs + page, by);
      page = mine[j];
      by = 0;
    }
    by += e < have[j] ? kids[j] - 1 : -1;
  }
  if (by) atomicAdd(a.refs + page, by);
}

// Inclusive prefix sum over a wave: within rows of 16, then from row to row.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2, 3
  return v;
}
// Exclusive prefix sum over the workgroup's threads; `all`: the total. `waves`: a
// buffer that no call shares with the one before it.
__device__ __forceinline__ int block_scan(int v, int* waves, int& all) {
  const int wave = threadIdx.x >> 6, inc = wave_scan(v);
  if ((threadIdx.x & 63) == 63) waves[wave] = inc;
  lds_barrier();
  const int w = wave_scan((threadIdx.x & 63) < kTakeWaves ? waves[threadIdx.x & 63] : 0);
  all = __builtin_amdgcn_readlane(w, kTakeWaves - 1);
  return inc - v + (wave ? __builtin_amdgcn_readlane(w, wave - 1) : 0);
}

// The kRun counts from `first` on (past the last page, the last one's), and the free
// pages among them, a bit each.
struct Counts {
  int c[kRun];
};
// ONE: this launch changed counts by atomics, which the loads have to see: past this
// CU's cache, where a line may lie that other arrays share with the counts.
template <bool ONE>
__device__ __forceinline__ Counts load_counts(const DtreePagesFork& a, int64_t first) {
  Counts r;
  if constexpr (ONE) {
    if (first < a.num_pages) {
      const int most = (int)min((int64_t)kRun, a.num_pages - first) - 1;
#pragma unroll
      for (int e = 0; e < kRun; ++e)
        r.c[e] = __hip_atomic_load(a.refs + first + min(e, most), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  } else if (first + kRun <= a.num_pages) {
    __builtin_memcpy(r.c, a.refs + first, sizeof(r.c));
  } else if (first < a.num_pages) {
#pragma unroll
    for (int e = 0; e < kRun; ++e) r.c[e] = a.refs[min(first + e, (int64_t)a.num_pages - 1)];
  }
  return r;
}
__device__ __forceinline__ uint32_t free_pages(const DtreePagesFork& a, int64_t first, const Counts& r) {
  const int64_t left = a.num_pages - first, keep = a.absent - first;
  if (left <= 0) return 0;
  uint32_t mask = 0;
#pragma unroll
  for (int e = 0; e < kRun; ++e) mask |= r.c[e] == 0 ? 1u << e : 0u;
  if (left < kRun) mask &= (1u << left) - 1;
  return keep >= 0 && keep < kRun ? mask & ~(1u << keep) : mask;
}

template <bool ONE>
__global__ __launch_bounds__(kTake) void pages_take_kernel(DtreePagesFork a) {
  __shared__ int waves[2][kTakeWaves];
  __shared__ int got[kMaxSeqs];          // the page that a copying sequence took
  __shared__ int pages[kHash], writers[kHash], latest[kHash];  // shared pages about to be written
  __shared__ int start[kMaxSeqs];        // pages wanted before a sequence's
  __shared__ int first[kMaxSeqs];        // its table entry of the first page past its length; copies: complemented
  __shared__ int list[kList];            // free pages, ascending
  __shared__ int kids[ONE ? kMaxSeqs : 1], from[ONE ? kMaxSeqs : 1], size[ONE ? kMaxSeqs : 1];
  __shared__ int past, fewer;
  const int i = threadIdx.x, n = a.num_seqs, wave = i >> 6;
  const bool in = i < n;
  const int64_t mine = (int64_t)i * kRun;
  // (no count becomes or stops being 0 before the pages are taken: a copied page has
  // another holder)
  Counts counts;
  if constexpr (!ONE) counts = load_counts<ONE>(a, mine);
  const int par = in ? fork_parent(a, i) : -1;
  const int L = par >= 0 ? fork_length(a, par) : 0;
  if (i == 0) past = fewer = 0;
#pragma unroll
  for (int h = i; h < kHash; h += kTake) {
    pages[h] = -1;
    writers[h] = 0;
    latest[h] = -1;
  }
  if constexpr (ONE) {
    const int own = in ? fork_length(a, i) : 0;
    kids[i] = a.parents ? 0 : 1;
    from[i] = par;
    size[i] = own;
    __syncthreads();
    if (a.parents && par >= 0) atomicAdd(&kids[par], 1);
    __syncthreads();
    const int all = n * a.ld_tables;
    const float inv = 1.f / a.ld_tables;
    for (int j = i; j < all; j += kTake) {
      const int s = (int)((j + 0.5f) * inv);  // (j < 4096: the half is far above the product's error)
      const int p = from[s];
      share_entry(a, s, j - s * a.ld_tables, p, p >= 0 ? (size[p] + DTREE_PAGE - 1) / DTREE_PAGE : 0,
                                                (size[s] + DTREE_PAGE - 1) / DTREE_PAGE, kids[s]);
    }
    wait_stores_done();  // (the counts' changes too)
  }
  __syncthreads();  // (every length is read: lengths_out may be lengths)
  if constexpr (ONE) counts = load_counts<ONE>(a, mine);
  const int covered = (L + DTREE_PAGE - 1) / DTREE_PAGE, at = L / DTREE_PAGE;
  const int64_t wanted = in ? ((int64_t)L + a.rows + DTREE_PAGE - 1) / DTREE_PAGE : 0;
  const int last = (int)min(wanted, (int64_t)a.ld_tables);
  int* row = a.tables_out + (size_t)i * a.ld_tables;
  if (in) a.lengths_out[i] = L;
  if (wanted > last) atomicAdd(&past, (int)min(wanted - last, (int64_t)1 << 20));
  int page = -1, holders = 0;
  if (in && a.rows > 0 && L % DTREE_PAGE) {
    page = row[at];
    if (is_page(a, page)) holders = ONE ? __hip_atomic_load(a.refs + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) : a.refs[page];
  }
  // Writers of one page: all copy if others hold it too, else all but the latest.
  uint32_t h = (uint32_t)page * 2654435761u >> 21;
  static_assert(kHash == 1 << 11, "the hash keeps 11 bits");
  if (holders > 1) {
    for (;; h = (h + 1) % kHash) {
      const int old = atomicCAS(&pages[h], -1, page);
      if (old == -1 || old == page) break;
    }
    atomicAdd(&writers[h], 1);
    atomicMax(&latest[h], i);
  }
  uint32_t mask = free_pages(a, mine, counts);
  __syncthreads();
  bool copy = false;
  if (holders > 1) {
    const int leave = min(writers[h], holders - 1);
    copy = leave == writers[h] || latest[h] != i;
    if (latest[h] == i) a.refs[page] = holders - leave;
  }
  int total, copies;
  const int grow = in ? max(last - covered, 0) : 0;
  const int before = block_scan((copy ? 1 : 0) + grow, waves[0], total);
  int spot = block_scan(copy ? 1 : 0, waves[1], copies);
  start[i] = before;
  first[i] = copy ? ~covered : covered;
  // The free pages in ascending order, kList at a time.
  int seen = 0;  // free pages of the rounds before
  for (int64_t base = 0; base < a.num_pages && seen < total; base += kRound) {
    if (base) mask = free_pages(a, base + mine, load_counts<ONE>(a, base + mine));
    int all;
    lds_barrier();
    int rank = seen + block_scan(__popc(mask), waves[0], all);
    const int end = min(total, seen + all);
    for (int r0 = seen; r0 < end; r0 += kList) {
      const int upto = min(end, r0 + kList);
      while (mask && rank < upto) {
        list[rank - r0] = (int)(base + mine) + __ffs((int)mask) - 1;
        mask &= mask - 1;
        ++rank;
      }
      lds_barrier();
      for (int r = r0 + i; r < upto; r += kTake) {
        int lo = 0, hi = n;  // the last sequence whose range starts at r or before: the one that holds r
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (start[mid] <= r) lo = mid;
          else hi = mid;
        }
        const int f = first[lo], j = r - start[lo], pg = list[r - r0];
        // a copy takes the sequence's first page, for the entry before its new ones
        a.tables_out[(size_t)lo * a.ld_tables + (f < 0 ? ~f + j - 1 : f + j)] = pg;
        if (f < 0 && j == 0) got[lo] = pg;
        a.refs[pg] = 1;
      }
      lds_barrier();
    }
    seen += all;
  }
  // the copies, by sequence; without pages for all of them, those before some sequence
  const bool made = copy && before < seen;
  if (seen < total) {
    if (copy && !made) {
      atomicAdd(&fewer, 1);
      row[at] = a.absent;
    }
    __syncthreads();
    copies -= fewer;
  }
  if (a.copies) {
    if (made) {
      a.copies[3 * spot] = page;
      a.copies[3 * spot + 1] = got[i];
      a.copies[3 * spot + 2] = L % DTREE_PAGE;
    }
    if (in && i >= copies) {
      a.copies[3 * i] = -1;
      a.copies[3 * i + 1] = -1;
      a.copies[3 * i + 2] = -1;
    }
  }
  if (a.status && i == 0) {
    a.status[0] += max(total - seen, 0) + past;
    a.status[1] = copies;
  }
}

// 16-byte pieces of a unit's blocks in all pools, one after the other; a thread's loads
// of kFlight pieces go out before their first store.
__global__ __launch_bounds__(256) void pages_copy_kernel(DtreePagesCopy a) {
  constexpr int kFlight = 4;
  __shared__ int ends;  // the list's first negative source
  const int tid = threadIdx.x, per = a.layers * a.num_heads;
  int u = blockIdx.x;
  int src = a.copies[3 * (u / per)], dst = a.copies[3 * (u / per) + 1], used = a.copies[3 * (u / per) + 2];
  if (tid == 0) ends = a.max_copies;
  __syncthreads();
  for (int c = tid; c < a.max_copies; c += 256)
    if (a.copies[3 * c] < 0) {
      atomicMin(&ends, c);
      break;
    }
  __syncthreads();
  const int units = ends * per;
  while (u < units) {
    const int lh = u % per, layer = lh / a.num_heads, head = lh % a.num_heads;
    if (src < a.num_pages && dst >= 0 && dst < a.num_pages && used > 0) {
      int upto[4], all = 0;  // pieces up to the end of pool i's
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        all += a.pools[i] ? (used > kHalfPage ? a.block_bytes[i] : a.block_bytes[i] / 2) / 16 : 0;
        upto[i] = all;
      }
      const size_t layer0 = (size_t)layer * a.num_pages;
      const size_t from = (layer0 + src) * a.num_heads + head, to = (layer0 + dst) * a.num_heads + head;
      for (int v0 = tid; v0 < all; v0 += 256 * kFlight) {
        u32x4_t piece[kFlight];
        u32x4_t* at[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
          const int v = min(v0 + 256 * k, all - 1);
          const int i = (v >= upto[0]) + (v >= upto[1]) + (v >= upto[2]);
          const int w = v - (i == 0 ? 0 : i == 1 ? upto[0] : i == 2 ? upto[1] : upto[2]);
          char* pool = static_cast<char*>(i == 0 ? a.pools[0] : i == 1 ? a.pools[1] : i == 2 ? a.pools[2] : a.pools[3]);
          const size_t bytes = (size_t)(i == 0 ? a.block_bytes[0] : i == 1 ? a.block_bytes[1] : i == 2 ? a.block_bytes[2] : a.block_bytes[3]);
          piece[k] = reinterpret_cast<const u32x4_t*>(pool + from * bytes)[w];
          at[k] = reinterpret_cast<u32x4_t*>(pool + to * bytes) + w;
        }
#pragma unroll
        for (int k = 0; k < kFlight; ++k)
          if (v0 + 256 * k < all) *at[k] = piece[k];
      }
    }
    u += gridDim.x;
    if (u >= units) break;
    const int c = 3 * (u / per);
    src = a.copies[c];
    dst = a.copies[c + 1];
    used = a.copies[c + 2];
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
  DTREE_REQUIRE(a->copies || a->rows == 0, "pages_fork: copies are needed where rows > 0");
  DTREE_REQUIRE(a->absent >= -1 && a->absent < a->num_pages, "pages_fork: absent is -1 or a page");
  DTREE_REQUIRE(a->tables != a->tables_out || !a->parents, "pages_fork: in place without parents alone");
  const int64_t rows = a->num_seqs;
  const int64_t size = rows * a->ld_tables;
  DTREE_REQUIRE(size < (1 << 30), "pages_fork: fewer than 2^30 table entries");
  DTREE_REQUIRE(a->tables == a->tables_out || a->tables + size <= a->tables_out || a->tables_out + size <= a->tables,
                "pages_fork: tables and tables_out overlap");
  DTREE_REQUIRE(a->lengths == a->lengths_out || a->lengths + rows <= a->lengths_out || a->lengths_out + rows <= a->lengths,
                "pages_fork: lengths and lengths_out partly overlap");
  if (size <= kOneLaunch) {
    pages_take_kernel<true><<<1, kTake, 0, stream>>>(*a);
  } else {
    const dim3 grid((a->num_seqs + kSide - 1) / kSide, (a->ld_tables + 255) / 256);
    pages_share_kernel<<<grid, 256, 0, stream>>>(*a);
    DTREE_LAUNCH_CHECK("pages_fork share launch");
    pages_take_kernel<false><<<1, kTake, 0, stream>>>(*a);
  }
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
