"""Which workgroup of a product with 4-bit weights takes what (glacier.tune_amd/csrc/
quant_grid.hpp), compiled for the CPU: every set of outputs meets every block of tokens in one
workgroup, none is without work, and a set's blocks lie eight apart, on one XCD, but for the
last few sets."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = """
#include <cstdio>
#include <vector>
#include "quant_grid.hpp"
using namespace glacier;
int main() {
  long seen = 0;
  for (int sets = 1; sets <= 200; ++sets)
    for (int blocks = 1; blocks <= 40; ++blocks) {
      std::vector<int> at(sets * blocks, -1);
      const int grid = quant_grid(sets, blocks);
      for (int i = 0; i < grid; ++i) {
        const QuantPlace p = quant_place(i, sets, blocks);
        const bool inside = p.set >= 0 && p.set < sets && p.block >= 0 && p.block < blocks;
        if (!inside || at[p.set * blocks + p.block] != -1) {
          std::printf("sets %d blocks %d: workgroup %d has no work of its own\\n", sets, blocks, i);
          return 1;
        }
        at[p.set * blocks + p.block] = i;
        ++seen;
      }
      for (int s = 0; s < sets; ++s)
        for (int b = 0; b < blocks; ++b)
          if (at[s * blocks + b] < 0 || (s < sets / 8 * 8 && at[s * blocks + b] % 8 != at[s * blocks] % 8)) {
            std::printf("sets %d blocks %d: set %d block %d at %d\\n", sets, blocks, s, b, at[s * blocks + b]);
            return 1;
          }
    }
  std::printf("OK %ld\\n", seen);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_every_workgroup_has_work(tmp_path):
    src, exe = tmp_path / "grid.cpp", str(tmp_path / "grid")
    src.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I" + os.path.join(ROOT, "glacier.tune_amd", "csrc"),
                    str(src), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout.startswith("OK"), (res.returncode, res.stdout)
