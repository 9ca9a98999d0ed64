"""How the keys of an attention tile are split (glacier.tune_amd/csrc/cache_split.hpp),
compiled for the CPU: every split has keys and is counted once, also where the
tile sees none."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = """
#include <cstdio>
#include <initializer_list>
#include "cache_split.hpp"
using namespace glacier;
int main() {
  long seen = 0;
  const int ends[] = {0, 1, 2, 127, 128, 129, 255, 256, 257, 1000, 1024, 4097, 65536, 1 << 20, (1 << 30) - 1};
  for (int kend : ends)
    for (int n = 1; n <= kMaxSplits; ++n)
      for (int given : {0, 128, 256, 512, 1024, 65536, 1 << 23}) {
        const KeySplit s = split_of(kend, n, given);
        const bool units = s.per > 0 && s.per % kSplitUnit == 0;
        const bool count = s.active >= 1 && s.active <= n;
        const bool whole = (long)s.active * s.per >= kend;
        const bool none_empty = kend == 0 ? s.active == 1 : (long)(s.active - 1) * s.per < kend;
        if (!units || !count || !whole || !none_empty) {
          std::printf("kend %d splits %d given %d: per %d active %d\\n", kend, n, given, s.per, s.active);
          return 1;
        }
        ++seen;
      }
  std::printf("OK %ld\\n", seen);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_every_split_has_keys(tmp_path):
    # (a division by zero ends the program: x86 traps it)
    src, exe = tmp_path / "split.cpp", str(tmp_path / "split")
    src.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I" + os.path.join(ROOT, "glacier.tune_amd", "csrc"), str(src),
                    "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout.startswith("OK"), (res.returncode, res.stdout)
