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
// growing with b; b = n_seqs if there is none.  Up to 64 sequences every lane reads
// one's entries, and the lane that holds the sequence hands them out: the search
// and the sequence's lengths are one load deep together.  More are narrowed down to
// 64 first, 64 parts at a time.
template <typename F>
__device__ inline CacheSeq find_seq(const CacheView& c, int lane, int x, F start) {
  CacheSeq s{c.n_seqs, 0, 0, 0};
  int b0 = 0, end = c.n_seqs;  // the sequence is in here, if anywhere
  while (end - b0 > 64) {
    const int part = (end - b0 + 63) / 64, last = min(end, b0 + (lane + 1) * part) - 1;
    const int before = __popcll(__ballot(b0 + lane * part < end && start(last + 1, clamp_row(c.cu[last + 1], c.T)) <= x));
    b0 += before * part;
    if (b0 >= end) return s;
    end = min(end, b0 + part);
  }
  const int b = b0 + lane, i = b < end ? b : end - 1;
  const int from = clamp_row(c.cu[i], c.T), to = clamp_row(c.cu[i + 1], c.T), len = c.kv_lens[i];
  const int before = __popcll(__ballot(b < end && start(i + 1, to) <= x));
  if (b0 + before >= end) return s;
  s.b = b0 + before;
  s.tok0 = __builtin_amdgcn_readlane(from, before);
  const int to_row = __builtin_amdgcn_readlane(to, before);
  s.n = to_row > s.tok0 ? to_row - s.tok0 : 0;
  s.pos0 = __builtin_amdgcn_readlane(len, before) - s.n;
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
