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
// where that would take more than n_splits, and as many splits as that evenly.
constexpr KeySplit split_of(int kend, int n_splits, int split_keys) {
  auto units = [](int keys) { return keys <= kSplitUnit ? kSplitUnit : (keys + kSplitUnit - 1) / kSplitUnit * kSplitUnit; };
  auto splits = [](int keys, int per) { return keys <= per ? 1 : (keys + per - 1) / per; };
  const int least = units((kend + n_splits - 1) / n_splits);
  const int active = splits(kend, split_keys > least ? split_keys : least);
  const int per = units((kend + active - 1) / active);
  return {per, splits(kend, per)};
}

}  // namespace glacier
