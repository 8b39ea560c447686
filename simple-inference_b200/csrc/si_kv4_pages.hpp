// si_kv4_pages.hpp -- host bookkeeping of the paged KV cache: which page holds
// which positions of which sequence, how many sequences hold a page, and which
// pages are free.  Plain C++ without CUDA; the C ABI (si_api.cu) queues what
// each change asks of the device (table entries, reference counts, page
// copies) on the context's stream.
//
// Every change is checked in full, and the room for what it asks of the device is
// taken, before anything is touched: a call that is refused or throws (host memory
// has run out) leaves the tables as they were.  Free pages are handed out lowest first.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

namespace si {

struct Kv4Run {  // `count` consecutive tokens of sequence seq from position pos on
  int seq, pos, count;
};

// Table entries [to, to + n) become entries [from, from + n); -1 where from is
// kNone; or, where from is kLiteral + i, the pages literal[i .. i + n).
struct Kv4Span {
  static constexpr int kNone = -1, kLiteral = 1 << 30;  // (tables have fewer entries)
  int to, n, from;
};

// What a change asks of the device, where the reference counts follow the table:
// an entry that changes lets its old page go and holds its new one.  Copies never
// chain: no destination of a change is a source of the same change, and no
// destination occurs twice; the same holds of the table's entries and spans.
struct Kv4Edits {
  std::vector<Kv4Span> spans;
  std::vector<int> literal;
  std::vector<std::pair<int, int>> table;  // (entry, page)
  std::vector<std::pair<int, int>> copies; // (from page, to page)
  // Room for as many more of each, so that adding them does not throw.
  void room(size_t n_spans, size_t n_literal, size_t n_table, size_t n_copies) {
    spans.reserve(spans.size() + n_spans);
    literal.reserve(literal.size() + n_literal);
    table.reserve(table.size() + n_table);
    copies.reserve(copies.size() + n_copies);
  }
  void clear() {
    spans.clear();
    literal.clear();
    table.clear();
    copies.clear();
  }
};

class Kv4Pages {
 public:
  Kv4Pages(int n_seqs, int max_pages, int n_pages, int page_len)
      : n_seqs_(n_seqs), max_pages_(max_pages), page_len_(page_len), n_free_(n_pages),
        count_(n_seqs, 0), refs_(n_pages, 0),
        table_((size_t)n_seqs * max_pages, -1) {}

  int n_pages() const { return (int)refs_.size(); }
  int n_seqs() const { return n_seqs_; }
  int max_pages() const { return max_pages_; }
  int page_len() const { return page_len_; }
  int free_pages() const { return n_free_; }
  int count(int seq) const { return count_[seq]; }
  int refs(int page) const { return refs_[page]; }
  int page(int seq, int i) const { return table_[at(seq, i)]; }
  const std::string &why() const { return why_; }
  // Positions of seq that its pages cover.
  int64_t covered(int seq) const { return (int64_t)count_[seq] * page_len_; }

  // A change did not reach the device in full, whose tables are no longer these:
  // from now on every call is refused.
  void lose() { lost_ = true; }
  bool lost() const { return lost_; }

  // Runs within the cache's sequences and positions.
  bool runs_ok(const Kv4Run *runs, int n) {
    if (!usable()) return false;
    for (int i = 0; i < n; ++i) {
      if (!seq_ok(runs[i].seq)) return false;
      if (runs[i].pos < 0 || runs[i].count < 0 ||
          (int64_t)runs[i].pos + runs[i].count > (int64_t)max_pages_ * page_len_)
        return no("positions outside the cache's max_ctx");
    }
    return true;
  }

  // Every page that the runs write to is there and held by their sequence alone.
  bool writable(const Kv4Run *runs, int n) const {
    if (lost_) return false;
    for (int i = 0; i < n; ++i) {
      const Kv4Run &x = runs[i];
      if (x.count <= 0) continue;
      const int p1 = last_page(x);
      if (p1 >= count_[x.seq]) return false;
      for (int p = x.pos / page_len_; p <= p1; ++p)
        if (refs_[table_[at(x.seq, p)]] > 1) return false;
    }
    return true;
  }

  bool seq_ok(int seq) {
    return usable() && ((seq >= 0 && seq < n_seqs_) || no("sequence out of range"));
  }

  // Positions [pos, pos + count) of every run get pages that no other
  // sequence holds: missing pages (from the sequence's first missing one) are
  // taken, a shared page is replaced by a copy of it.
  bool reserve(const Kv4Run *runs, int n, Kv4Edits *e) {
    if (!runs_ok(runs, n)) return false;
    if (writable(runs, n)) return true;  // the common decode step
    std::vector<Kv4Run> r;
    for (int i = 0; i < n; ++i)
      if (runs[i].count > 0) r.push_back(runs[i]);
    // A dry run that counts the pages taken.  Of a page's holders the ones that
    // write get copies, except that the last holder left keeps the page.
    std::vector<int> have(count_);
    int64_t grown = 0, copied = 0;
    std::vector<std::pair<int, int>> shared;  // (page, table entry), each pair once
    for (const Kv4Run &x : r) {
      const int p0 = x.pos / page_len_, p1 = last_page(x);
      for (int p = p0; p < std::min(p1 + 1, count_[x.seq]); ++p) {
        const int pg = table_[at(x.seq, p)];
        if (refs_[pg] > 1) shared.push_back({pg, (int)at(x.seq, p)});
      }
      if (p1 + 1 > have[x.seq]) {
        grown += p1 + 1 - have[x.seq];
        have[x.seq] = p1 + 1;
      }
    }
    std::sort(shared.begin(), shared.end());
    shared.erase(std::unique(shared.begin(), shared.end()), shared.end());
    for (size_t i = 0; i < shared.size();) {
      size_t j = i;
      while (j < shared.size() && shared[j].first == shared[i].first) ++j;
      copied += std::min((int64_t)(j - i), (int64_t)refs_[shared[i].first] - 1);
      i = j;
    }
    if (grown + copied > n_free_) return no("not enough free pages");
    e->room(r.size(), grown, copied, copied);
    for (const Kv4Run &x : r) {
      const int p0 = x.pos / page_len_, p1 = last_page(x);
      for (int p = p0; p < std::min(p1 + 1, count_[x.seq]); ++p) {
        const int old = table_[at(x.seq, p)];
        if (refs_[old] <= 1) continue;
        const int pg = take();
        e->copies.push_back({old, pg});
        drop(old);
        put(x.seq, p, pg, e);
      }
      if (p1 >= count_[x.seq]) {
        const int n = p1 + 1 - count_[x.seq];
        int *row = literal(x.seq, count_[x.seq], n, e);
        for (int p = 0; p < n; ++p) row[p] = take();
        copy_literal(x.seq, count_[x.seq], row, n);
        count_[x.seq] = p1 + 1;
      }
    }
    return true;
  }

  // Sequence seqs[i] (empty until now) holds the next counts[i] pages of the
  // list, each of which may be held by others already.
  bool assign(const int *seqs, const int *counts, int n, const int *pages, Kv4Edits *e) {
    if (!usable()) return false;
    std::vector<char> seen(n_seqs_, 0);
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
      if (!seq_ok(seqs[i])) return false;
      if (count_[seqs[i]] || seen[seqs[i]]) return no("sequence already holds pages");
      if (counts[i] < 0 || counts[i] > max_pages_) return no("page count out of range");
      seen[seqs[i]] = 1;
      total += counts[i];
    }
    const unsigned limit = n_pages();
    bool bad = false;
    for (int64_t i = 0; i < total; ++i) bad |= (unsigned)pages[i] >= limit;
    if (bad) return no("page out of range");
    e->room(n, total, 0, 0);
    int *__restrict refs = refs_.data();
    int taken = 0;
    for (int64_t i = 0; i < total; ++i) taken += refs[pages[i]]++ == 0;
    n_free_ -= taken;
    for (int i = 0; i < n; pages += counts[i++]) {
      if (counts[i] == 0) continue;
      const int at0 = (int)at(seqs[i], 0);
      e->spans.push_back({at0, counts[i], Kv4Span::kLiteral + (int)e->literal.size()});
      e->literal.insert(e->literal.end(), pages, pages + counts[i]);
      std::copy(pages, pages + counts[i], table_.data() + at0);
      count_[seqs[i]] = counts[i];
    }
    return true;
  }

  // dst[i] (empty until now) begins with the first lens[i] positions of
  // src[i]: whole pages are shared, the page that lens[i] ends in is copied.
  bool fork(const int *src, const int *dst, const int *lens, int n, Kv4Edits *e) {
    if (!usable()) return false;
    std::vector<char> seen(n_seqs_, 0);
    int64_t need = 0;
    for (int i = 0; i < n; ++i) {
      if (!seq_ok(src[i]) || !seq_ok(dst[i])) return false;
      if (count_[dst[i]] || seen[dst[i]]) return no("destination sequence already holds pages");
      if (src[i] == dst[i]) return no("a sequence cannot be forked into itself");
      if (lens[i] < 0 || lens[i] > covered(src[i])) return no("length beyond the source's pages");
      seen[dst[i]] = 1;
      need += lens[i] % page_len_ != 0;
    }
    if (need > n_free_) return no("not enough free pages");
    e->room(n, 0, need, need);
    for (int i = 0; i < n; ++i) {
      const int whole = lens[i] / page_len_;
      const int *from = table_.data() + at(src[i], 0);
      int *to = table_.data() + at(dst[i], 0);
      for (int p = 0; p < whole; ++p) ++refs_[to[p] = from[p]];
      if (whole) e->spans.push_back({(int)at(dst[i], 0), whole, (int)at(src[i], 0)});
      count_[dst[i]] = whole;
      if (lens[i] % page_len_) {
        const int pg = take();
        e->copies.push_back({table_[at(src[i], whole)], pg});
        put(dst[i], whole, pg, e);
        count_[dst[i]] = whole + 1;
      }
    }
    return true;
  }

  // seqs[i] keeps the pages of its first keep[i] positions (keep null: none).
  bool release(const int *seqs, const int *keep, int n, Kv4Edits *e) {
    if (!usable()) return false;
    for (int i = 0; i < n; ++i) {
      if (!seq_ok(seqs[i])) return false;
      if (keep && keep[i] < 0) return no("negative length");
    }
    e->room(n, 0, 0, 0);
    for (int i = 0; i < n; ++i) {
      const int64_t len = keep ? keep[i] : 0;
      const int64_t stay = (len + page_len_ - 1) / page_len_;
      const int n = count_[seqs[i]] - (int)std::min<int64_t>(count_[seqs[i]], stay);
      if (n == 0) continue;
      int *row = table_.data() + at(seqs[i], count_[seqs[i]] - n);
      int *__restrict refs = refs_.data();
      int freed = 0, lowest = first_free_;
      for (int p = 0; p < n; ++p) {  // (the page lists are in any order: no branches)
        const int pg = row[p], left = --refs[pg];
        freed += left == 0;
        lowest = std::min(lowest, left == 0 ? pg : lowest);
      }
      std::fill(row, row + n, -1);
      n_free_ += freed;
      first_free_ = lowest;
      e->spans.push_back({(int)(row - table_.data()), n, Kv4Span::kNone});
      count_[seqs[i]] -= n;
    }
    return true;
  }

  // The used pages become pages [0, used): the used pages from `used` on move,
  // in ascending order, to the free ones below.  Returns used, -1 where refused.
  int compact(Kv4Edits *e) {
    if (!usable()) return -1;
    const int used = n_pages() - n_free_;
    // Which pages are used follows no pattern: lists without branches.  The i-th hole
    // takes the i-th mover; to[] is where a page ends up.
    std::vector<int> to(refs_.size()), hole(used + 1);
    int holes = 0, moves = 0;
    for (int pg = 0; pg < used; ++pg) {
      to[pg] = pg;
      hole[holes] = pg;
      holes += refs_[pg] == 0;
    }
    e->copies.resize(holes + 1);
    for (int pg = used; pg < n_pages(); ++pg) {
      to[pg] = hole[moves];
      e->copies[moves] = {pg, hole[moves]};
      moves += refs_[pg] != 0;
    }
    e->copies.resize(moves);
    if (!moves) return finish_compact(used);
    size_t entries = 0;
    for (int s = 0; s < n_seqs_; ++s) entries += count_[s];
    e->table.resize(entries + 1);
    for (const auto &c : e->copies) {
      refs_[c.second] = refs_[c.first];
      refs_[c.first] = 0;
    }
    size_t edits = 0;
    for (int s = 0; s < n_seqs_; ++s) {
      int *row = table_.data() + at(s, 0);
      for (int p = 0; p < count_[s]; ++p) {
        const int pg = row[p];
        row[p] = to[pg];
        e->table[edits] = {(int)at(s, p), to[pg]};
        edits += to[pg] != pg;
      }
    }
    e->table.resize(edits);
    return finish_compact(used);
  }

 private:
  int finish_compact(int used) {
    first_free_ = used;
    return used;
  }
  size_t at(int seq, int p) const { return (size_t)seq * max_pages_ + p; }
  int last_page(const Kv4Run &x) const {
    return (int)(((int64_t)x.pos + x.count - 1) / page_len_);
  }
  bool usable() {
    return !lost_ || no("an earlier change of the pages did not reach the device");
  }
  bool no(const char *why) {
    why_ = why;
    return false;
  }
  int take() {  // the lowest free page; the caller has checked that there is one
    while (refs_[first_free_]) ++first_free_;
    const int pg = first_free_++;
    --n_free_;
    refs_[pg] = 1;
    return pg;
  }
  void drop(int pg) {
    if (--refs_[pg] == 0) {
      ++n_free_;
      first_free_ = std::min(first_free_, pg);
    }
  }
  // Room for n pages of seq from its p-th on, and the same into the table.
  int *literal(int seq, int p, int n, Kv4Edits *e) {
    const int i = (int)e->literal.size();
    e->literal.resize(i + n);
    e->spans.push_back({(int)at(seq, p), n, Kv4Span::kLiteral + i});
    return e->literal.data() + i;
  }
  void copy_literal(int seq, int p, const int *row, int n) {
    std::copy(row, row + n, table_.data() + at(seq, p));
  }
  void put(int seq, int p, int pg, Kv4Edits *e) {
    table_[at(seq, p)] = pg;
    e->table.push_back({(int)at(seq, p), pg});
  }

  int n_seqs_, max_pages_, page_len_, n_free_;
  int first_free_ = 0;  // no free page lies below
  bool lost_ = false;
  std::vector<int> count_, refs_, table_;
  std::string why_;
};

}  // namespace si
