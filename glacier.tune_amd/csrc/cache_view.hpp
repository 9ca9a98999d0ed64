// cache_view.hpp -- device-side reading of the paged cache's index arrays,
// shared by cache_append.hip and cache_attn.hip.  cu, kv_lens and the page
// table are device data that no host check sees, so every use of them is
// bounded here: a token row lies in [0, T), a position in [0, max_pages
// page_size), a page in [0, n_pages).
#pragma once

#include "attn_common.hpp"
#include "cache_launch.hpp"

namespace glacier {

// A sequence of the batch: its rows [tok0, tok0 + n) of the new tokens, and
// the position of the first.  Position pos0 + n is its length with them.
struct CacheSeq {
  int b, tok0, n, pos0;
};

// How many of 0 .. n_seqs - 1 satisfy the test (b), which holds for a prefix
// of them: 64 at a time, one a lane, so that a search is one load deep.
template <typename F>
__device__ inline int count_prefix(int n_seqs, int lane, F test) {
  int count = 0;
  for (int b0 = 0; b0 < n_seqs; b0 += 64) {
    const int b = b0 + lane;
    const unsigned long long m = __ballot(b < n_seqs && test(b));
    count += __popcll(m);
    if (m != ~0ull) break;
  }
  return count;
}

__device__ inline int clamp_row(int r, int T) { return r < 0 ? 0 : r > T ? T : r; }

__device__ inline CacheSeq cache_seq(const CacheView& c, int b) {
  CacheSeq s;
  s.b = b;
  s.tok0 = clamp_row(c.cu[b], c.T);
  const int end = clamp_row(c.cu[b + 1], c.T);
  s.n = end > s.tok0 ? end - s.tok0 : 0;
  s.pos0 = c.kv_lens[b] - s.n;
  return s;
}

// The page of positions p .. (same page) of sequence b, or -1.
__device__ inline int cache_page(const CacheView& c, int b, int p) {
  const int i = p >> c.page_shift;
  if (p < 0 || i >= c.max_pages) return -1;
  const int page = c.table[(long)b * c.table_stride + i];
  return static_cast<unsigned>(page) < static_cast<unsigned>(c.n_pages) ? page : -1;
}

}  // namespace glacier
