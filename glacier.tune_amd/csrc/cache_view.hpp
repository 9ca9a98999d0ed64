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

__device__ inline int clamp_row(int r, int T) { return r < 0 ? 0 : r > T ? T : r; }

// The sequence b with start(b, cu[b]) <= x < start(b + 1, cu[b + 1]), start
// growing with b; b = n_seqs if there is none.  Every lane reads one sequence's
// entries, 64 sequences at a time, and the lane that holds the sequence hands
// them out: the search and the sequence's lengths are one load deep together.
template <typename F>
__device__ inline CacheSeq find_seq(const CacheView& c, int lane, int x, F start) {
  CacheSeq s{c.n_seqs, 0, 0, 0};
  for (int b0 = 0; b0 < c.n_seqs; b0 += 64) {
    const int b = b0 + lane, i = b < c.n_seqs ? b : c.n_seqs - 1;
    const int from = clamp_row(c.cu[i], c.T), to = clamp_row(c.cu[i + 1], c.T), len = c.kv_lens[i];
    const int before = __popcll(__ballot(b < c.n_seqs && start(i + 1, to) <= x));
    if (before == 64) continue;
    if (b0 + before >= c.n_seqs) break;
    s.b = b0 + before;
    s.tok0 = __builtin_amdgcn_readlane(from, before);
    const int end = __builtin_amdgcn_readlane(to, before);
    s.n = end > s.tok0 ? end - s.tok0 : 0;
    s.pos0 = __builtin_amdgcn_readlane(len, before) - s.n;
    break;
  }
  return s;
}
// The sequence that token row t belongs to.
__device__ inline CacheSeq seq_of_token(const CacheView& c, int lane, int t) {
  return find_seq(c, lane, t, [](int, int to) { return to; });
}

// The page of positions p .. (same page) of sequence b, or -1.
__device__ inline int cache_page(const CacheView& c, int b, int p) {
  const int i = p >> c.page_shift;
  if (p < 0 || i >= c.max_pages) return -1;
  const int page = c.table[(long)b * c.table_stride + i];
  return static_cast<unsigned>(page) < static_cast<unsigned>(c.n_pages) ? page : -1;
}

}  // namespace glacier
