// cache_split.hpp -- how the keys of an attention tile over the paged cache are
// split, one formula for every kernel of a call (cache_tiles.hpp) and for the host.
#pragma once

namespace glacier {

constexpr int kMaxSplits = 64;   // one lane each in the join
constexpr int kSplitUnit = 128;  // splits begin at multiples of it

struct KeySplit {
  int per, active;  // keys of a split, at least one unit; splits that have keys, at least one
};
// Of keys 0 .. kend - 1 (none where kend is 0): split_keys of them a split, more
// where that would take more than n_splits, and as many splits as that evenly, all
// counted in units.  up(a, b): a / b rounded up, a below 2^24, b at least 1.
template <typename F>
constexpr KeySplit split_with(int kend, int n_splits, int split_keys, F up) {
  auto one = [](int n) { return n < 1 ? 1 : n; };
  const int keys = (kend + kSplitUnit - 1) / kSplitUnit, given = (split_keys + kSplitUnit - 1) / kSplitUnit;
  const int least = one(up(keys, n_splits));
  const int active = one(up(keys, given > least ? given : least));
  const int per = one(up(keys, active));
  return {per * kSplitUnit, one(up(keys, per))};
}
constexpr KeySplit split_of(int kend, int n_splits, int split_keys) {
  return split_with(kend, n_splits, split_keys, [](int a, int b) { return (a + b - 1) / b; });
}

// Work numbered by the sequences' lengths: how many splits each tile of a sequence of `tiles`
// tiles and kend keys stands for; `last`: those that its last tile has.  An earlier tile,
// which sees fewer keys, may have more than the last: a split has split_keys keys as long as
// n_splits of them reach, and grows by whole units then, so that one key more can leave fewer
// (4 of 256: 1024 keys take 4, 1025 take 3).  Splits of split_keys that the keys would take,
// n_splits at most, are the most that a tile of so many keys or fewer has; while n_splits
// reach they are the last one's.  (n_splits for each tile would do, but leaves workgroups
// without work: 8 sequences of 4 tokens over 300 keys beside 24 single ones over up to 8192,
// 28/4 heads of 128, 28.7 us so and 33 with n_splits.)
template <typename F>
constexpr int splits_a_tile(int tiles, int last, int kend, int n_splits, int split_keys, F up) {
  if (tiles <= 1 || n_splits == 1) return last;
  const int keys = (kend + kSplitUnit - 1) / kSplitUnit, given = (split_keys + kSplitUnit - 1) / kSplitUnit;
  const int most = up(keys, given < 1 ? 1 : given);
  return most < 1 ? 1 : most < n_splits ? most : n_splits;
}

}  // namespace glacier
