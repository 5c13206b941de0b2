// Ragged batches over a paged KV cache: what the kernels of paged*.hip are given, and how they read
// a sequence's bounds and pages. All of it lives in device memory, where a step that was captured
// once finds the lengths of the step that it replays, so none of it can be checked on the host:
// every value is held to its range here, and one outside it is latched in the status word.
#pragma once

#include "tl_internal.hpp"

namespace tl {

// bits of the context's status word
enum : int32_t { kBadSequence = 4, kBadPage = 8, kBadPosition = 16, kBadShare = 32 };

struct PagedBatch {
  const int32_t* table;  // [n_seqs, cols], rows ld_table apart
  const int32_t* q_start;
  const int32_t* kv_len;
  int64_t ld_table;
  int cols, n_seqs, n_rows, n_pages;
  int page_shift;  // log2 of the positions in a page
  int Hq, Hkv;
  int32_t* status;
};

__device__ __forceinline__ void latch(int32_t* status, int32_t bit) { atomicOr(status, bit); }

// One sequence: its rows [row0, row0 + n) of the batch, and its length with them.
struct PagedSeq {
  int row0, n, len;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int s, bool report) {
  const int a = b.q_start[s], e = b.q_start[s + 1], l = b.kv_len[s];
  PagedSeq q;
  q.row0 = min(max(a, 0), b.n_rows);
  q.n = min(max(e, q.row0), b.n_rows) - q.row0;
  q.len = min(max(l, 0), b.cols << b.page_shift);
  if (report && (a < 0 || e < a || e > b.n_rows || l != q.len)) latch(b.status, kBadSequence);
  return q;
}

// Reports, by a whole wave, a sequence that does not begin with the batch's `shared` first positions:
// other pages than sequence 0's, or a row inside them.
__device__ __forceinline__ void check_shared(const PagedBatch& b, int s, const PagedSeq& q, int shared, int lane) {
  bool bad = q.n > 0 && q.len - q.n < shared;
  for (int j = lane; j < (shared >> b.page_shift); j += 64) bad |= b.table[s * b.ld_table + j] != b.table[j];
  if (__any(bad) && lane == 0) latch(b.status, kBadShare);
}

// The sequence that row t belongs to, by a whole wave: the last s with q_start[s] <= t, found by
// 64 probes a round (one round up to 64 sequences, two up to 4096). n_seqs for a row of none.
__device__ __forceinline__ int seq_of_row(const PagedBatch& b, int t, int lane) {
  int lo = 0, n = b.n_seqs;  // q_start[lo] <= t as far as probed; the answer is in [lo, lo + n)
  int hits = 0;
  while (true) {
    const int step = (n + 63) >> 6;
    const int at = lo + (lane + 1) * step;
    const bool hit = at <= lo + n && at <= b.n_seqs && b.q_start[at] <= t;
    hits = __popcll(__ballot(hit));
    if (step == 1) break;
    lo += hits * step;
    n = min(step, b.n_seqs - lo);
    if (n <= 0) break;
  }
  return min(lo + (n > 0 ? hits : 0), b.n_seqs);
}

// Checks a descriptor and turns it into the kernels' form.
int paged_batch(tl_ctx* ctx, const tl_paged_desc* d, PagedBatch* b);
// Checks a tensor of the batch's rows: 16-byte aligned rows that do not overlap.
int paged_rows(const tl_paged_desc* d, const void* p, int64_t ld, int64_t cols, const char* what);

// Calls f with a D of the descriptor's head_dim as a type.
template <int D>
struct HeadDim {
  static constexpr int value = D;
};
template <typename F>
static void for_head_dim(int64_t d, F f) {
  switch (d) {
    case 32: f(HeadDim<32>{}); break;
    case 64: f(HeadDim<64>{}); break;
    case 128: f(HeadDim<128>{}); break;
    default: f(HeadDim<256>{}); break;
  }
}

}  // namespace tl
