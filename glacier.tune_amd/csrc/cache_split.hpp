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

// Work numbered by the sequences' lengths: how many (tile, split) pairs a sequence of
// `tiles` tiles stands for, `last` the splits of its last one.  An earlier tile may have
// more splits than the last: past n_splits splits of split_keys a split grows by whole
// units, so that one key more can leave fewer (4 of 256: 1024 keys take 4, 1025 take 3).
// Sequences of several tiles therefore stand for all that a tile may have.
constexpr int items_of(int tiles, int last, int n_splits) { return tiles > 1 ? tiles * n_splits : tiles * last; }
struct TileItem {
  int tile, split;
};
// The x-th of them.  down(a): a / n_splits.
template <typename F>
constexpr TileItem item_at(int x, int tiles, int n_splits, F down) {
  const int tile = tiles > 1 ? down(x) : 0;
  return {tile, x - tile * n_splits};
}

}  // namespace glacier
