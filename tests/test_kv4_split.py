"""CPU test of where the 4-bit cache's split attention keeps its partial sums
(csrc/si_kv4_split.hpp): every output on a boundary of 16 bytes, every (maximum,
sum) on one of 8, no two over one another, and all within the scratch, at odd and
even numbers of tokens, heads and splits."""
import os
import subprocess

from common import PKG

DRIVER = r"""
#include <cstdio>
#include <vector>
#include "si_kv4_split.hpp"
using namespace si;
int main() {
  for (int D : {64, 128})
    for (size_t T : {1, 2, 3, 7})
      for (size_t heads : {1, 5, 7, 8, 28})
        for (size_t splits : {1, 2, 5, 8, 9, 17, 49, 55, 63, 65, 157}) {
          const size_t slots = T * heads * splits;
          std::vector<char> used(kv4_part_size(slots, D), 0);
          auto take = [&](size_t at, size_t n, size_t align) {
            if (4 * at % align || at + n > used.size()) return false;
            for (size_t i = at; i < at + n; ++i) {
              if (used[i]) return false;
              used[i] = 1;
            }
            return true;
          };
          for (size_t s = 0; s < slots; ++s)
            if (!take(kv4_part_out(s, D), D, 16) || !take(kv4_part_ml(slots, s, D), 2, 8)) {
              printf("D %d, %zu x %zu x %zu, slot %zu\n", D, T, heads, splits, s);
              return 1;
            }
        }
  return 0;
}
"""


def test_partial_sums_are_aligned_and_apart(tmp_path):
    (tmp_path / "t.cpp").write_text(DRIVER)
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover=all", "-I", os.path.join(PKG, "csrc"),
                    str(tmp_path / "t.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
