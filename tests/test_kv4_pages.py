"""CPU tests of the 4-bit cache's page bookkeeping (csrc/si_kv4_pages.hpp): the
C++ class behind the C ABI is compiled here with the host compiler and driven
with seeded random sequences of calls against a plain model that holds, for
every sequence, the contents of its positions.  Contents travel as the class
says (copies, table entries), so a page shared too long or freed too early shows
as a wrong content; refused calls must change nothing."""
import os
import random
import subprocess

import pytest

from common import PKG, ROOT  # noqa: F401

DRIVER = r"""
#include <cstdio>
#include <iostream>
#include "si_kv4_pages.hpp"
using namespace si;
int main() {
  int S, P, N, L;
  std::cin >> S >> P >> N >> L;
  Kv4Pages k(S, P, N, L);
  std::string op;
  while (std::cin >> op) {
    Kv4Edits e;
    bool ok = true;
    int used = -1, n = 0;
    if (op != "compact") std::cin >> n;
    if (op == "reserve") {
      std::vector<Kv4Run> r(n);
      for (auto &x : r) std::cin >> x.seq >> x.pos >> x.count;
      ok = k.reserve(r.data(), n, &e);
      if (ok && !k.writable(r.data(), n)) { printf("NOT WRITABLE\n"); return 1; }
    } else if (op == "assign") {
      std::vector<int> s(n), c(n), p;
      for (int i = 0; i < n; ++i) std::cin >> s[i] >> c[i];
      int m;
      std::cin >> m;
      p.resize(m);
      for (int &x : p) std::cin >> x;
      ok = k.assign(s.data(), c.data(), n, p.data(), &e);
    } else if (op == "fork") {
      std::vector<int> a(n), b(n), c(n);
      for (int i = 0; i < n; ++i) std::cin >> a[i] >> b[i] >> c[i];
      ok = k.fork(a.data(), b.data(), c.data(), n, &e);
    } else if (op == "release") {
      std::vector<int> a(n), b(n);
      for (int i = 0; i < n; ++i) std::cin >> a[i] >> b[i];
      ok = k.release(a.data(), b.data(), n, &e);
    } else {
      used = k.compact(&e);
    }
    printf("%d %d %d", ok, used, k.free_pages());
    printf(" C %zu", e.copies.size());
    for (auto &c : e.copies) printf(" %d %d", c.first, c.second);
    printf(" S %zu", e.spans.size());
    for (auto &c : e.spans) printf(" %d %d %d", c.to, c.n, c.from);
    printf(" T %zu", e.table.size());
    for (auto &c : e.table) printf(" %d %d", c.first, c.second);
    printf(" L %zu", e.literal.size());
    for (int p : e.literal) printf(" %d", p);
    printf("\n");
    fflush(stdout);
  }
}
"""


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4")
    (d / "t.cpp").write_text(DRIVER)
    exe = str(d / "t")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover=all", "-D_GLIBCXX_ASSERTIONS", "-I",
                    os.path.join(PKG, "csrc"), str(d / "t.cpp"), "-o", exe], check=True)
    return exe


LITERAL = 1 << 30  # Kv4Span::kLiteral


class Model:
    """Contents by position, and a pool that only the class's edits move."""

    def __init__(self, exe, S, P, N, L):
        self.S, self.P, self.N, self.L = S, P, N, L
        self.want = [dict() for _ in range(S)]      # seq -> {position: content}
        self.pool = [[None] * L for _ in range(N)]
        self.table = [-1] * (S * P)
        self.refs = [0] * N
        self.p = subprocess.Popen([exe], stdin=subprocess.PIPE, stdout=subprocess.PIPE, text=True)
        self._send(f"{S} {P} {N} {L}")

    def _send(self, line):
        self.p.stdin.write(line + "\n")
        self.p.stdin.flush()

    def call(self, op, *nums):
        self._send(" ".join([op] + [str(n) for n in nums]))
        out = self.p.stdout.readline().split()
        assert out and out[0] in "01", out
        ok, used, free = int(out[0]), int(out[1]), int(out[2])
        at, parts = 3, {}
        while at < len(out):
            key, n = out[at], int(out[at + 1])
            k = {"S": 3, "L": 1}.get(key, 2)
            v = list(map(int, out[at + 2:at + 2 + k * n]))
            parts[key] = [tuple(v[i:i + k]) for i in range(0, k * n, k)]
            at += 2 + k * n
        if not ok:
            assert not any(parts.values()), "a refused call asked for changes"
            assert free == sum(r == 0 for r in self.refs)
            return ok, used, free
        froms, tos = {a for a, _ in parts["C"]}, [b for _, b in parts["C"]]
        assert not froms & set(tos) and len(tos) == len(set(tos)), "copies chain or collide"
        written = [t + i for t, n, _ in parts["S"] for i in range(n)] + [t for t, _ in parts["T"]]
        sources = {f + i for _, n, f in parts["S"] if 0 <= f < LITERAL for i in range(n)}
        assert len(written) == len(set(written)) and not sources & set(written), "entries collide"
        for a, b in parts["C"]:
            assert self.refs[b] == 0, "copied over a page that was in use"
            self.pool[b] = list(self.pool[a])
        lit = [p for p, in parts["L"]]
        for t, n, f in parts["S"]:
            self.table[t:t + n] = ([-1] * n if f < 0 else lit[f - LITERAL:f - LITERAL + n]
                                   if f >= LITERAL else self.table[f:f + n])
        for t, pg in parts["T"]:
            self.table[t] = pg
        self.refs = [0] * self.N
        for t in self.table:
            if t >= 0:
                self.refs[t] += 1
        return ok, used, free

    def check(self, free):
        assert free == self.refs.count(0)
        for s in range(self.S):
            row = self.table[s * self.P:(s + 1) * self.P]
            n = sum(t >= 0 for t in row)
            assert all(t >= 0 for t in row[:n]), "a hole in a table"
            for pos, what in self.want[s].items():
                assert pos < n * self.L and self.pool[row[pos // self.L]][pos % self.L] == what

    def count(self, s):
        return sum(t >= 0 for t in self.table[s * self.P:(s + 1) * self.P])

    def write(self, s, pos, what):
        pg = self.table[s * self.P + pos // self.L]
        assert self.refs[pg] == 1, "a write into a shared page"
        self.pool[pg][pos % self.L] = what
        self.want[s][pos] = what

    def close(self):
        self.p.stdin.close()
        assert self.p.wait(timeout=20) == 0


@pytest.mark.parametrize("seed", range(8))
def test_random_calls_keep_every_sequence(driver, seed):
    rng = random.Random(seed)
    S, P, L = rng.randint(2, 9), rng.randint(1, 7), 16
    N = rng.randint(1, S * P)
    m = Model(driver, S, P, N, L)
    tick = 0
    refused = 0
    for _ in range(400):
        op = rng.choice(["write", "write", "write", "fork", "release", "compact", "assign"])
        if op == "write":
            runs = []
            for _ in range(rng.randint(1, 3)):
                s = rng.randrange(S)
                pos = rng.randrange(P * L)
                runs.append((s, pos, rng.randint(0, min(40, P * L - pos))))
            ok, _, free = m.call("reserve", len(runs), *[x for r in runs for x in r])
            if ok:
                for s, pos, c in runs:
                    for q in range(pos, pos + c):
                        tick += 1
                        m.write(s, q, tick)
        elif op == "fork":
            n = rng.randint(1, 3)
            a = [(rng.randrange(S), rng.randrange(S), rng.randint(0, P * L)) for _ in range(n)]
            ok, _, free = m.call("fork", n, *[x for r in a for x in r])
            if ok:
                for s, d, ln in a:
                    m.want[d] = {p: v for p, v in m.want[s].items() if p < ln}
        elif op == "release":
            n = rng.randint(1, 3)
            a = [(rng.randrange(S), rng.choice([0, 0, rng.randint(0, P * L)])) for _ in range(n)]
            ok, _, free = m.call("release", n, *[x for r in a for x in r])
            assert ok
            for s, keep in a:
                m.want[s] = {p: v for p, v in m.want[s].items() if p < m.count(s) * L}
        elif op == "assign":
            s, c = rng.randrange(S), rng.randint(0, P)
            pages = [rng.randrange(N) for _ in range(c)]
            ok, _, free = m.call("assign", 1, s, c, c, *pages)
            if ok:
                m.want[s] = {i * L + j: m.pool[pg][j] for i, pg in enumerate(pages)
                             for j in range(L)}
        else:
            ok, used, free = m.call("compact")
            assert ok and used == N - free
            assert all(t < used for t in m.table)
        refused += not ok
        m.check(free)
    assert refused < 400
    m.close()


def test_reserve_copies_once_less_than_holders(driver):
    """Three sequences share a page and all write: two copies, the last holder keeps it."""
    m = Model(driver, 3, 2, 3, 16)
    assert m.call("reserve", 1, 0, 0, 16)[0]
    assert m.call("fork", 2, 0, 1, 16, 0, 2, 16)[0]
    assert m.refs[0] == 3
    ok, _, free = m.call("reserve", 3, 0, 3, 1, 1, 3, 1, 2, 3, 1)
    assert ok and free == 0 and sorted(m.refs) == [1, 1, 1]
    m.close()


@pytest.mark.parametrize("call", [
    ("reserve", 1, 3, 0, 1), ("reserve", 1, -1, 0, 1), ("reserve", 1, 0, -1, 1),
    ("reserve", 1, 0, 0, -1), ("reserve", 1, 0, 32, 1), ("reserve", 1, 0, 2147483647, 2147483647),
    ("reserve", 3, 0, 0, 32, 1, 0, 32, 2, 0, 32),          # six pages of four
    ("assign", 1, 0, 1, 1, 4), ("assign", 1, 0, 1, 1, -1), ("assign", 1, 0, 3, 3, 0, 1, 2),
    ("assign", 2, 0, 1, 0, 1, 2, 0, 1), ("assign", 1, 7, 1, 1, 0),
    ("fork", 1, 0, 0, 0), ("fork", 1, 0, 1, 1), ("fork", 1, 0, 9, 0), ("fork", 1, 0, 1, -1),
    ("fork", 2, 0, 1, 0, 2, 1, 0), ("release", 1, 5, 0), ("release", 1, 0, -1)])
def test_refusals_change_nothing(driver, call):
    m = Model(driver, 3, 2, 4, 16)
    ok, _, free = m.call(*call)
    assert not ok and free == 4
    m.check(free)
    m.close()
