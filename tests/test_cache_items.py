"""Which workgroup takes which split of which tile where the work of a 4-bit cache's attention
is numbered by the sequences' lengths (glacier.tune_amd/csrc/cache_split.hpp), compiled for
the CPU: every split that the join counts is taken once, whatever max_kv said, a launch by
number of tiles has room for all of them, and where max_kv holds none is taken in vain but
those that only a sequence's last tile has."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = """
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
#include "cache_split.hpp"
using namespace glacier;

// Keys of the tile of 16 rows from row 16 tile on: its last row's token sees up to its own.
static int keys_of(int tile, int n, int kv, int group) {
  return std::max(0, kv - n + std::min(n - 1, (16 * tile + 15) / group) + 1);
}

struct Seq {
  int n, kv;
};
static bool check(const std::vector<Seq>& seqs, int group, int n_splits, int split_keys) {
  long tokens = 0, room, used = 0;
  for (const Seq& s : seqs) tokens += s.n;
  room = (tokens * group / 16 + (long)seqs.size()) * n_splits;
  for (const Seq& s : seqs) {
    const int tiles = (s.n * group + 15) / 16;
    const int last = split_of(std::max(0, s.kv), n_splits, split_keys).active;
    std::vector<int> taken(tiles * n_splits, 0);
    const int each = splits_a_tile(tiles, last, std::max(0, s.kv), n_splits, split_keys,
                                   [](int a, int b) { return (a + b - 1) / b; });
    const int items = tiles * each;
    if (each < 1 || each > n_splits || (s.kv <= n_splits * split_keys && each != last)) {
      std::printf("%d keys: %d splits a tile, %d of the last (%d of %d)\\n", s.kv, each, last, n_splits, split_keys);
      return false;
    }
    for (int x = 0; x < items; ++x) ++taken[x / each * n_splits + x % each];
    for (int t = 0; t < tiles; ++t) {
      const int active = split_of(keys_of(t, s.n, s.kv, group), n_splits, split_keys).active;
      for (int u = 0; u < n_splits; ++u)
        if (taken[t * n_splits + u] > 1 || (u < active && taken[t * n_splits + u] != 1)) {
          std::printf("tile %d of %d new, %d keys, group %d: split %d of %d (%d of %d) taken %d times\\n", t, s.n, s.kv,
                      group, u, active, n_splits, split_keys, taken[t * n_splits + u]);
          return false;
        }
    }
    used += items;
  }
  return used <= room;
}

int main() {
  // longer than the hint of 1024, and of 2048
  if (!check({{3, 1025}, {1, 1000}}, 8, 4, 256)) return 1;
  if (!check({{4, 2049}, {1, 1900}, {1, 1900}, {1, 1900}}, 7, 8, 256)) return 1;
  std::mt19937 rng(5);
  auto upto = [&](int n) { return 1 + static_cast<int>(rng() % n); };
  long seen = 0;
  for (int i = 0; i < 200000; ++i) {
    const int hint = 256 * upto(40), n_splits = std::min(upto(kMaxSplits), std::max(1, hint / 256));
    const int split_keys = ((hint + n_splits - 1) / n_splits + kSplitUnit - 1) / kSplitUnit * kSplitUnit;
    std::vector<Seq> seqs(upto(6));
    for (Seq& s : seqs) s = {static_cast<int>(rng() % 12), static_cast<int>(rng() % (2 * hint + 2)) - 1};
    if (!check(seqs, upto(20), n_splits, split_keys)) return 1;
    ++seen;
  }
  std::printf("OK %ld\\n", seen);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_every_split_is_taken_once(tmp_path):
    src, exe = tmp_path / "items.cpp", str(tmp_path / "items")
    src.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(ROOT, "glacier.tune_amd", "csrc"),
                    str(src), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout.startswith("OK"), (res.returncode, res.stdout)
