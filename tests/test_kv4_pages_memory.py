"""CPU tests of the 4-bit cache's page bookkeeping (csrc/si_kv4_pages.hpp) when the host
runs out of memory, and after a change that did not reach the device: a call that
throws has changed nothing, and lost pages refuse every call."""
import os
import subprocess

import pytest

from common import PKG

HEAD = r"""
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <new>
#include "si_kv4_pages.hpp"
using namespace si;
"""

MEMORY = HEAD + r"""
static long left = -1;  // allocations until one fails; -1: none does
void *operator new(size_t n) {
  if (left == 0) throw std::bad_alloc();
  if (left > 0) --left;
  if (void *p = malloc(n ? n : 1)) return p;
  throw std::bad_alloc();
}
void operator delete(void *p) noexcept { free(p); }
void operator delete(void *p, size_t) noexcept { free(p); }

static bool same(const Kv4Pages &a, const Kv4Pages &b) {
  if (a.free_pages() != b.free_pages()) return false;
  for (int p = 0; p < a.n_pages(); ++p)
    if (a.refs(p) != b.refs(p)) return false;
  for (int s = 0; s < a.n_seqs(); ++s) {
    if (a.count(s) != b.count(s)) return false;
    for (int i = 0; i < a.max_pages(); ++i)
      if (a.page(s, i) != b.page(s, i)) return false;
  }
  return true;
}

int main() {
  // Sequences 0 to 3 share a prompt's pages; 4 has its own; 5 to 7 are empty.
  Kv4Pages start(8, 40, 300, 16);
  Kv4Edits e;
  const Kv4Run prompt[2] = {{0, 0, 200}, {4, 0, 77}};
  const int src[3] = {0, 0, 0}, dst[3] = {1, 2, 3}, lens[3] = {200, 199, 64};
  const int gone[1] = {2}, zero[1] = {0};
  if (!start.reserve(prompt, 2, &e) || !start.fork(src, dst, lens, 3, &e) ||
      !start.release(gone, zero, 1, &e))
    return 2;
  const Kv4Run runs[5] = {{0, 100, 60}, {1, 0, 210}, {3, 10, 300}, {4, 500, 40}, {5, 0, 400}};
  const int to[3] = {5, 6, 7}, from[3] = {1, 4, 3}, keep[3] = {199, 65, 64};
  const int seqs[3] = {5, 6, 7}, counts[3] = {2, 0, 3}, pages[5] = {9, 250, 0, 251, 251};
  const int rel[3] = {0, 3, 4}, stay[3] = {33, 0, 16};
  const std::function<bool(Kv4Pages &, Kv4Edits *)> calls[] = {
      [&](Kv4Pages &k, Kv4Edits *x) { return k.reserve(runs, 5, x); },
      [&](Kv4Pages &k, Kv4Edits *x) { return k.fork(from, to, keep, 3, x); },
      [&](Kv4Pages &k, Kv4Edits *x) { return k.assign(seqs, counts, 3, pages, x); },
      [&](Kv4Pages &k, Kv4Edits *x) { return k.release(rel, stay, 3, x); },
      [&](Kv4Pages &k, Kv4Edits *x) { return k.compact(x) >= 0; },
  };
  int op = 0;
  for (const auto &call : calls) {
    Kv4Pages want(start);
    Kv4Edits x;
    if (!call(want, &x)) return 3;
    int failed = 0;
    for (long n = 0;; ++n) {
      Kv4Pages k(start);
      Kv4Edits y;
      bool threw = false;
      left = n;
      try {
        if (!call(k, &y)) return 4;
      } catch (const std::bad_alloc &) {
        threw = true;
      }
      left = -1;
      if (threw) {
        ++failed;
        if (!same(k, start)) {
          printf("call %d changed the pages when allocation %ld failed\n", op, n);
          return 1;
        }
        y.clear();
        if (!call(k, &y)) return 5;
      }
      if (!same(k, want) || y.copies != x.copies || y.table != x.table) {
        printf("call %d gives other pages after allocation %ld failed\n", op, n);
        return 1;
      }
      if (!threw) break;
    }
    if (!failed) return 6;
    ++op;
  }
  return 0;
}
"""

LOST = HEAD + r"""
int main() {
  Kv4Pages k(3, 4, 8, 16);
  Kv4Edits e;
  const Kv4Run run[1] = {{0, 0, 20}};
  const int a[1] = {0}, b[1] = {1}, c[1] = {1}, d[1] = {7};
  if (!k.reserve(run, 1, &e) || k.lost()) return 1;
  k.lose();
  if (!k.lost()) return 2;
  e.clear();
  if (k.runs_ok(run, 1) || k.seq_ok(0) || k.writable(run, 1)) return 3;
  if (k.reserve(run, 1, &e) || k.assign(b, c, 1, d, &e) || k.fork(a, b, c, 1, &e) ||
      k.release(a, nullptr, 1, &e) || k.compact(&e) >= 0)
    return 4;
  if (!e.spans.empty() || !e.table.empty() || !e.copies.empty() || k.why().empty()) return 5;
  if (k.count(0) != 2 || k.free_pages() != 6) return 6;
  return 0;
}
"""


@pytest.mark.parametrize("name", ["MEMORY", "LOST"])
def test_pages(name, tmp_path):
    (tmp_path / "t.cpp").write_text(globals()[name])
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=undefined",
                    "-fno-sanitize-recover=all", "-D_GLIBCXX_ASSERTIONS", "-I",
                    os.path.join(PKG, "csrc"), str(tmp_path / "t.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)
