// The paged key/value cache as the kernels see it, and the lookups they share.
//
// Pools k_pages [num_pages, page, H_kv, D], v_pages [num_pages, page, H_kv, D_v].
// Sequence n owns the tokens q_start[n] .. q_start[n+1]-1 of the call (its new
// ones) and holds kv_len[n] cached tokens, those included; key j of it lies at
// row j % page of page_table[n][j / page].  All three arrays are int32 on the
// device and are read by the kernels, never by the host, so a captured graph
// follows them.  Entries outside their ranges never reach memory: a page id
// outside the pool reads as zeros and is not written, lengths are clamped to
// the table's capacity, starts to the call's tokens, and each raises
// kStatusBadIndex.  So does a q_start that descends: a sequence between two
// descending starts is empty, and where others then share tokens (the work that
// the host launched for (tokens, seqs) would not cover theirs) the attention
// does nothing at all.  The cache write, which goes by token, leaves out those
// that its search finds no sequence for.
#pragma once
#include <cstdint>

#include "ptx.cuh"

namespace sdpa_b200 {

constexpr unsigned int kStatusBadIndex = 2u;  // a page id, length or position outside its range

struct PagedView {
  const int* page_table;  // [seqs, width]
  const int* kv_len;      // [seqs]
  const int* q_start;     // [seqs + 1]
  int seqs, width, num_pages;
  int page_shift;         // log2 of the page size
  int tokens;             // new tokens of the call
};

// New tokens [begin, begin + count) and cached length of sequence n, clamped
// so that no index built from them leaves its array.
struct SeqLens {
  int begin, count, held;
  bool ascends;  // q_start[n] <= q_start[n + 1]
};
__device__ __forceinline__ SeqLens seq_lens(const PagedView& v, int n) {
  const int q0 = v.q_start[n], q1 = v.q_start[n + 1];
  const int a = max(0, min(q0, v.tokens)), e = max(0, min(q1, v.tokens));
  const long long cap = static_cast<long long>(v.width) << v.page_shift;
  const int held = v.kv_len[n];
  SeqLens s;
  s.begin = a;
  s.ascends = a <= e;
  s.count = s.ascends ? e - a : 0;
  s.held = held < 0 ? 0 : (held > cap ? static_cast<int>(cap) : held);
  if (s.held != held || a != q0 || e != q1 || !s.ascends) atomicOr(&g_status_word, kStatusBadIndex);
  return s;
}

// Whether two sequences share tokens, which takes starts that descend somewhere
// (callers ask then alone).
__device__ __forceinline__ bool seqs_overlap(const PagedView& v) {
  int last = 0;
  for (int n = 0; n < v.seqs; ++n) {
    const SeqLens s = seq_lens(v, n);
    if (s.count == 0) continue;
    if (s.begin < last) return true;
    last = s.begin + s.count;
  }
  return false;
}

// Pool page of entry i of sequence n, or -1 (status raised) for an id outside
// the pool.  i must be below width.
__device__ __forceinline__ int page_of(const PagedView& v, int n, int i) {
  const int p = __ldg(v.page_table + static_cast<int64_t>(n) * v.width + i);
  if (static_cast<unsigned>(p) < static_cast<unsigned>(v.num_pages)) return p;
  atomicOr(&g_status_word, kStatusBadIndex);
  return -1;
}

// Raises the status for starts that descend or lie outside the call's tokens (the
// first `threads` of one block; where the work goes by token, not by sequence).
__device__ __forceinline__ void starts_check(const PagedView& v, int threads) {
  bool bad = false;
  for (int n = threadIdx.x; n <= v.seqs; n += threads) {
    const int a = __ldg(v.q_start + n);
    bad |= a < 0 || a > v.tokens || (n < v.seqs && __ldg(v.q_start + n + 1) < a);
  }
  if (bad) atomicOr(&g_status_word, kStatusBadIndex);
}

// The sequence that owns token t, or -1 (before the first or behind the last).
// LANES neighbouring lanes (mask: their warp mask) search together: LANES
// probes a round, so 256 sequences take two rounds of 16 lanes.
template <int LANES>
__device__ __forceinline__ int seq_of_token(const PagedView& v, int t, unsigned mask, int lane) {
  int lo = 0, hi = v.seqs + 1;  // the number of entries <= t lies in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + LANES - 1) / LANES;
    const int i = lo + (lane + 1) * step - 1;
    const bool le = i < hi && __ldg(v.q_start + i) <= t;
    const int c = __popc(__ballot_sync(mask, le) & mask);
    lo = min(hi, lo + c * step);
    hi = min(hi, lo + step - 1);
  }
  return lo > v.seqs ? -1 : lo - 1;
}

}  // namespace sdpa_b200
