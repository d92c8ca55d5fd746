// The 8-bit KV cache's page order and batch bounds, shared by its kernels.
#pragma once
#include "common.h"

namespace dtree {

// One (page, kv head) block: DTREE_PAGE positions x D dims of int8. A lane's 16
// bytes are its operands of two 32x32x16 MFMA steps:
// * K: lane 32 h + s % 32 of piece (s / 32, d / 32) holds dims 32 (d / 32) +
//   16 h .. + 15 of one key, the first 8 for one step of S^T = K Q^T, the next
//   8 for the other (a step's contraction index (h, e) stands for dim 32 J +
//   16 h + 8 step + e, in q alike).
// * V: lane 32 h + d % 32 holds one dim at the 16 positions 32 (s / 32) + 8 q +
//   4 h + e, byte 4 q + e: the keys of the 16 accumulator registers that S^T
//   leaves in the lanes of half h, in register order (acc_row), so P needs no
//   exchange between lanes on its way into O^T = V^T P^T.
__host__ __device__ __forceinline__ int q8_k_off(int slot, int d, int D) {
  return ((((slot >> 5) * (D >> 5) + (d >> 5)) * 64 + ((d >> 4) & 1) * 32 + (slot & 31)) << 4) + (d & 15);
}
__host__ __device__ __forceinline__ int q8_v_off(int slot, int d, int D) {
  return ((((slot >> 5) * (D >> 5) + (d >> 5)) * 64 + ((slot >> 2) & 1) * 32 + (d & 31)) << 4) +
         (((slot >> 3) & 3) << 2) + (slot & 3);
}

// A sequence's rows, clipped to the bounds the host gave (DtreeKvQ8).
struct Q8Seq {
  int past, n, start;
};
__device__ __forceinline__ Q8Seq q8_seq(const DtreeKvQ8& kv, int s) {
  const int past = kv.past_lengths[s], start = kv.row_starts ? kv.row_starts[s] : s * kv.max_rows;
  const bool ok = past >= 0 && past <= kv.max_past_length && start >= 0 && start < kv.total_rows;
  const int room = min(kv.total_rows - start, kv.ld_page_table * DTREE_PAGE - past);
  const int n = ok ? max(0, min(min(kv.row_counts[s], kv.max_rows), room)) : 0;
  return Q8Seq{n ? past : 0, n, n ? start : 0};
}

// Physical page i of sequence s, -1 if absent. i < ld_page_table.
__device__ __forceinline__ int q8_page(const DtreeKvQ8& kv, int s, int i) {
  const int page = kv.page_tables[(size_t)s * kv.ld_page_table + i];
  return page >= 0 && page < kv.num_pages ? page : -1;
}

// A projection row's head as D / 8 neighbouring lanes with two pieces of 4 dims
// each: lane j of the first R / 8 has the halves 4 j .. and R / 2 + 4 j .. of a
// rotation of R dims, the others 8 dims that do not rotate. A wave's loads are then
// whole runs of the rows.
struct Q8Pieces {
  int at[2];   // first dim of each
  bool turns;  // the two rotate
};
template <int D>
__device__ __forceinline__ Q8Pieces q8_pieces(int rope_dims, int j) {
  const int hp = rope_dims / 8;  // pieces of a rotation's half
  const bool turns = j < hp;
  return Q8Pieces{{4 * (turns ? j : 2 * j), 4 * (turns ? j + hp : 2 * j + 1)}, turns};
}
__device__ __forceinline__ f32x4_t q8_bf4(u32x2_t w) {
  return f32x4_t{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                 __uint_as_float(w[1] & 0xffff0000u)};
}

// Host check of the record, common to the entries (`what`: the entry's name).
int q8_check(const DtreeKvQ8* kv, const char* what);

}  // namespace dtree
