// cache_tiles.hpp -- the tiles of an attention call over the paged cache and
// their keys, by formulas that every kernel of the call shares: which tiles
// exist and how their keys are split follows from device data.
#pragma once

#include "cache_split.hpp"
#include "cache_view.hpp"
#include "lds_mfma.hpp"

namespace glacier {

constexpr float kLeast = -3.402823466e38f;  // where running maxima begin: below every score

// Tiles are numbered through all sequences: sequence b's first one is
// first_tile(a, b, cu[b]), which leaves room for every tile it can have.
__device__ inline int first_tile(const CacheAttn& a, int b, int cu) { return cu * a.group / a.rows + b; }
// The sequence of tile `number`.
__device__ inline CacheSeq seq_of_tile(const CacheAttn& a, int lane, int number) {
  return find_seq(a.c, lane, number, [&](int b, int to) { return first_tile(a, b, to); });
}

// The sequence of tile `number` and the tile's place in it when tiles are numbered
// from the longest sequence to the shortest and from a sequence's last tile to
// its first (batches of at most 64 sequences; others from the last to the first),
// so that long tiles start first and short ones fill in beside them.  tile: -1 if
// there is no such tile.
__device__ inline CacheSeq seq_of_long_tile(const CacheAttn& a, int lane, int number, int numbers, int& tile) {
  const CacheView& c = a.c;
  tile = -1;
  if (c.n_seqs > 64) {
    number = numbers - 1 - number;
    const CacheSeq s = seq_of_tile(a, lane, number);
    if (s.b < c.n_seqs) tile = number - first_tile(a, s.b, s.tok0);
    return s;
  }
  const int i = lane < c.n_seqs ? lane : c.n_seqs - 1;
  const int from = clamp_row(c.cu[i], c.T), len = c.kv_lens[i];
  const int n = lane < c.n_seqs ? max(0, clamp_row(c.cu[i + 1], c.T) - from) : 0;
  const int tiles = (n * a.group + a.rows - 1) / a.rows;
  int before = 0;  // tiles of the sequences that go first
  for (int u = 0; u < c.n_seqs; ++u) {
    const int other = __builtin_amdgcn_readlane(len, u);
    if (other > len || (other == len && u < lane)) before += __builtin_amdgcn_readlane(tiles, u);
  }
  const unsigned long long mine = __ballot(number >= before && number < before + tiles);
  CacheSeq s{c.n_seqs, 0, 0, 0};
  if (mine == 0) return s;
  s.b = __ffsll(mine) - 1;
  s.tok0 = __builtin_amdgcn_readlane(from, s.b);
  s.n = __builtin_amdgcn_readlane(n, s.b);
  s.pos0 = __builtin_amdgcn_readlane(len, s.b) - s.n;
  tile = __builtin_amdgcn_readlane(before + tiles, s.b) - 1 - number;
  return s;
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
// a / b rounded up (0 <= a < 2^24, b >= 1): the reciprocal's product is off by at most
// two downwards and one upwards, which the remainder tells; an integer division is 30
// instructions.
__device__ inline int div_up(int a, int b) {
  const int q = static_cast<int>(static_cast<float>(a) * __builtin_amdgcn_rcpf(static_cast<float>(b)));
  const int rest = a - q * b;
  return q + (rest > 0 ? 1 : 0) + (rest > b ? 1 : 0) + (rest > 2 * b ? 1 : 0) - (rest <= -b ? 1 : 0);
}
__device__ inline TileKeys keys_up_to(const CacheAttn& a, const CacheSeq& s, int last) {
  TileKeys k;
  const long cap = (long)a.c.max_pages << a.c.page_shift;
  const long end = (long)s.pos0 + last + 1;
  k.kend = static_cast<int>(end < 0 ? 0 : end < cap ? end : cap);
  KeySplit split{(k.kend + kSplitUnit - 1) / kSplitUnit * kSplitUnit, 1};  // (n_splits 1: what split_with gives)
  if (split.per == 0) split.per = kSplitUnit;
  if (a.n_splits > 1) split = split_with(k.kend, a.n_splits, a.split_keys, div_up);
  k.per = __builtin_amdgcn_readfirstlane(split.per);
  k.active = __builtin_amdgcn_readfirstlane(split.active);
  return k;
}
__device__ inline TileKeys tile_keys(const CacheAttn& a, const CacheSeq& s, int tile) {
  return keys_up_to(a, s, min(s.n - 1, (tile * a.rows + a.rows - 1) / a.group));
}

// A masked weight is zero, but zero times an infinity or a NaN is not.  The
// kernels find out at the end: where a sum is not finite they walk the keys once
// more, clear what is not finite in V before the products, note which key blocks
// had any, and give those values to the rows that see their keys afterwards.
constexpr int kNotedBlocks = 1024;  // blocks share a note past so many
// All ones where an element of the word (one fp32 or two bf16) is not finite: an
// exponent of all ones carries into the sign's place when one is added.  (No
// comparisons: their results would crowd the scalar registers of the main loop.)
template <typename T>
__device__ inline unsigned not_finite_mask(unsigned u) {
  if constexpr (sizeof(T) == 2)
    return ((((u & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
  else
    return static_cast<unsigned>(static_cast<int>((u & 0x7f800000u) + 0x00800000u) >> 31);
}
// Clears the elements of a 16-byte word that are not finite; their places.
template <typename T>
__device__ inline unsigned clear_not_finite(i32x4& w) {
  unsigned found = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const unsigned m = not_finite_mask<T>(static_cast<unsigned>(w[x]));
    w[x] &= static_cast<int>(~m);
    found |= m;
  }
  return found;
}
// x if it is not finite and the lane's row sees its key (all ones), else zero
__device__ inline float given_back(float x, unsigned sees) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  return __builtin_bit_cast(float, u & not_finite_mask<float>(u) & sees);
}
// Accumulates whether any of the values is not finite (nonzero then).
__device__ inline unsigned not_finite(float x) { return not_finite_mask<float>(__builtin_bit_cast(unsigned, x)); }

// exp2 of the weights: the instruction itself, whose results below 2^-126 are
// zero (exp2f spends four more instructions to keep them).
__device__ inline float weight(float x) { return __builtin_amdgcn_exp2f(x); }

// 8 bytes at `off` of the wave's [base, base + bytes); zeros past its end.
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ inline i32x2 load8_within(const void* base, int bytes, int off) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_raw_buffer_load_b64(wave_rsrc(base, bytes), off, 0, 0);
#else
  return i32x2{0, 0};
#endif
}

// 16 bytes at `off` of the wave's [base, base + bytes); zeros past its end.
__device__ inline i32x4 load_within(const void* base, int bytes, int off) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_raw_buffer_load_b128(wave_rsrc(base, bytes), off, 0, 0);
#else
  return i32x4{0, 0, 0, 0};
#endif
}

}  // namespace glacier
