// cache_tiles.hpp -- the tiles of an attention call over the paged cache and
// their keys, by formulas that every kernel of the call shares: which tiles
// exist and how their keys are split follows from device data.
#pragma once

#include "cache_view.hpp"
#include "lds_mfma.hpp"

namespace glacier {

constexpr int kMaxSplits = 64;   // one lane each in the join
constexpr int kSplitUnit = 128;  // splits begin at multiples of it

// Tiles are numbered through all sequences: sequence b's first one is
// first_tile(a, b, cu[b]), which leaves room for every tile it can have.
__device__ inline int first_tile(const CacheAttn& a, int b, int cu) { return cu * a.group / a.rows + b; }
// The sequence of tile `number`.
__device__ inline CacheSeq seq_of_tile(const CacheAttn& a, int lane, int number) {
  return find_seq(a.c, lane, number, [&](int b, int to) { return first_tile(a, b, to); });
}

// How many tile numbers a batch of the call's size can use at most.
inline unsigned tile_numbers(const CacheAttn& a) {
  return static_cast<unsigned>((long)a.c.T * a.group / a.rows + a.c.n_seqs);
}

// The keys of a tile whose last row is token `last`, and how they are split.
struct TileKeys {
  int kend;  // keys 0 .. kend - 1
  int per, active;  // keys of a split, and how many splits have any
};
__device__ inline TileKeys tile_keys(const CacheAttn& a, const CacheSeq& s, int tile) {
  TileKeys k;
  const int last = min(s.n - 1, (tile * a.rows + a.rows - 1) / a.group);
  const long cap = (long)a.c.max_pages << a.c.page_shift;
  const long end = (long)s.pos0 + last + 1;
  k.kend = static_cast<int>(end < 0 ? 0 : end < cap ? end : cap);
  const int even = (k.kend + a.n_splits - 1) / a.n_splits;
  k.per = max(a.split_keys, (even + kSplitUnit - 1) / kSplitUnit * kSplitUnit);
  k.active = max(1, (k.kend + k.per - 1) / k.per);
  // as many splits as that, evenly
  k.per = ((k.kend + k.active - 1) / k.active + kSplitUnit - 1) / kSplitUnit * kSplitUnit;
  k.active = max(1, (k.kend + k.per - 1) / k.per);
  return k;
}

// exp2 of the weights: the instruction itself, whose results below 2^-126 are
// zero (exp2f spends four more instructions to keep them).
__device__ inline float weight(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes at `off` of the wave's [base, base + bytes); zeros past its end.
__device__ inline i32x4 load_within(const void* base, int bytes, int off) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_raw_buffer_load_b128(wave_rsrc(base, bytes), off, 0, 0);
#else
  return i32x4{0, 0, 0, 0};
#endif
}

}  // namespace glacier
