// Host side of the batch operators (kernels/batch.hip): the checks of their push words against
// the buffers they are bound to, and the launch a dispatch of theirs becomes.  Plain C++, no HIP.
#pragma once

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

namespace batch {

enum Op { kNone, kAppend, kAttend, kMerge, kLogits };

inline Op op_of(const char *name) {
  if (std::strcmp(name, "kv_append") == 0) return kAppend;
  if (std::strcmp(name, "attention_paged") == 0) return kAttend;
  if (std::strcmp(name, "attention_paged_merge") == 0) return kMerge;
  if (std::strcmp(name, "logits_adjust") == 0) return kLogits;
  return kNone;
}

constexpr uint32_t kHead = 128, kPart = kHead + 2;
constexpr uint32_t kMaxSlots = 1024;      // partials of a row and head
constexpr uint32_t kMaxGrid = 65535;      // rows of a dispatch
// Workgroups of 16 heads from which kv_append takes 64 heads each (48 heads a row, f16 keys and 8-bit
// values, us, 16 / 64: 2048 rows 36 / 33.5, 1000 rows 24 / 26.5, 300 rows 15.4 / 16, 64 rows 10.4 / 10.4).
constexpr uint32_t kAppendMany = 4096;
// Partials above which eight waves merge a head, where rows times heads make two such workgroups a
// compute unit at most (32 heads, us, one wave / eight: 1 row of 12 parts 3.9 / 4.0, of 32 5.3 / 4.0, of 64
// 6.8 / 4.1; 16 rows of 17 4.8 / 5.0, of 32 5.4 / 5.0, of 64 7.1 / 5.0; 24 rows of 32 5.6 / 6.8; 128 of 17
// 11.8 / 25.1).
constexpr uint32_t kMergeParts = 16, kMergeHeads = 512;
// Room for a history from which a logits workgroup takes 16384 tokens for 4096, so that a quarter of
// them read it (us, 4096 / 16384: 128 rows of 32768 50 / 45, of 8192 33.7 / 33.3, of 1000 28 / 29; 12
// rows of 30000 12.2 / 9.9, of 4096 7.4 / 8.0; 1 row of 30000 9.7 / 8.6, of 1000 5.7 / 6.4).
constexpr uint32_t kLogitsHistory = 8192;
constexpr uint32_t kMaxWork = 1u << 23;   // workgroups of an attention launch

// A buffer bound to a dispatch: where it lies and how large it is.
struct Binding {
  uint64_t at, bytes;
};
// [off, off + stride (rows - 1) + width) of a binding, in elements of `size` bytes
struct Region {
  const char *what;
  Binding in;
  uint64_t size, off, stride, width, rows;
  uint64_t end() const { return rows ? off + stride * (rows - 1) + width : off; }
  bool meets(const Region &o) const {
    return rows && o.rows && in.at + off * size < o.in.at + o.end() * o.size &&
           o.in.at + o.off * o.size < in.at + end() * size;
  }
  bool same(const Region &o) const {  // row by row
    return in.at + off * size == o.in.at + o.off * o.size && (stride == o.stride || rows == 1);
  }
};

class Check {
 public:
  std::string error;
  void fail(const char *fmt, ...) {
    if (!error.empty()) return;
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    error = buf;
  }
  void need(bool ok, const char *what) {
    if (!ok) fail("%s", what);
  }
  // r lies in its binding, its rows apart from each other, offset and stride multiples of `align`
  void holds(const Region &r, uint32_t align) {
    if (!r.rows) return;
    const uint64_t elements = r.in.bytes / r.size;
    if (r.off % align || (r.rows > 1 && r.stride % align)) fail("%s: offset or stride not a multiple of %u", r.what, align);
    if (r.rows > 1 && r.stride < r.width) fail("%s: stride %llu below the row's %llu", r.what,
                                               (unsigned long long)r.stride, (unsigned long long)r.width);
    if (r.end() > elements)
      fail("%s ends at %llu, past the binding's %llu", r.what, (unsigned long long)r.end(), (unsigned long long)elements);
  }
  void apart(const Region &a, const Region &b) {
    if (a.meets(b)) fail("%s and %s overlap", a.what, b.what);
  }
  // what a dispatch writes: apart from each other and from what it reads
  void writes(const std::vector<Region> &written, const std::vector<Region> &read) {
    for (size_t i = 0; i < written.size(); i++) {
      for (size_t j = 0; j < i; j++) apart(written[j], written[i]);
      for (const Region &r : read) apart(written[i], r);
    }
  }
};

// the page table's words and the words of the rows
inline void check_pages(Check &c, const Region &rows, const Region &table, uint32_t page_log2, uint32_t n_pages) {
  c.need(page_log2 >= 4 && page_log2 <= 12, "pages hold 16 to 4096 positions");
  c.need(n_pages >= 1, "the pool has no pages");
  c.holds(rows, 4);
  c.holds(table, 1);
}

// a pool's keys and values and the scales of its 8-bit halves: in their bindings, apart from each other
inline std::vector<Region> check_pool(Check &c, bool k8, bool v8, const uint32_t off[4], uint64_t slots, uint64_t kv_dim,
                                      Binding kv, Binding kv8) {
  std::vector<Region> pool;
  for (int i = 0; i < 2; i++) {
    const bool q8 = i ? v8 : k8;
    pool.push_back({i ? "the pool's values" : "the pool's keys", q8 ? kv8 : kv, q8 ? 1u : 2u, off[i], 0, slots * kv_dim, 1});
    c.holds(pool.back(), 8);
    if (q8) {
      pool.push_back({i ? "the values' scales" : "the keys' scales", kv, 2, off[2 + i], 0, slots * (kv_dim / 32), 1});
      c.holds(pool.back(), 4);
    }
  }
  c.writes(pool, {});
  return pool;
}

// "" or why a dispatch of `op` (spec, push words, grid, the bound buffers' sizes and places) is
// refused.  Without places (at) the buffers are the engine's: arena and control words one, the
// pool's bindings another, the tables a third.
inline std::string refusal(Op op, const uint32_t *spec, const uint32_t *w, const uint32_t *groups, const uint64_t *bytes,
                           const uint64_t *at = nullptr) {
  Check c;
  const uint64_t rows = groups[1];
  c.need(groups[0] == 1 && groups[2] == 1, "the grid is [1, rows, 1]");
  if (rows > kMaxGrid) c.fail("%llu rows: at most %u", (unsigned long long)rows, kMaxGrid);
  if (!c.error.empty() || rows == 0 || op == kNone) return c.error;
  auto bound = [&](int i) {
    static const uint64_t place[2][5] = {{2, 0, 0, 1, 1}, {0, 0, 1, 1, 1}};
    return Binding{at ? at[i] : place[op != kAppend][i] << 40, bytes[i]};
  };
  const Binding A = bound(op == kAppend), C = bound(op == kAppend ? 2 : 1);  // arena, control words
  const Region ctl{"the control words", C, 4, 0, 0, 5, 1};
  c.holds(ctl, 1);
  if (op == kAppend) {
    const uint64_t n_head = w[9], n_kv = w[10], kv_dim = n_kv * kHead;
    c.need(n_head >= 1 && n_head <= 1024 && n_kv >= 1 && n_kv <= 1024, "1 to 1024 heads");
    if (!c.error.empty()) return c.error;
    const Binding W = bound(0);
    const Region q{"q", A, 4, w[0], w[11], n_head * kHead, rows}, k{"k", A, 4, w[1], w[12], kv_dim, rows},
        v{"v", A, 4, w[2], w[12], kv_dim, rows}, o{"the rotated q", A, 4, w[3], w[13], n_head * kHead, rows};
    const Region words{"the rows' words", C, 4, w[18], 4, 4, rows},
        table{"the page table", C, 4, w[19], 0, (uint64_t)w[21] * w[20], 1};
    const Region qn{"q's norm weights", W, 4, w[4], 0, kHead, 1}, kn{"k's norm weights", W, 4, w[5], 0, kHead, 1},
        rope{"the rotation's frequencies", W, 4, w[6], 0, kHead / 2, 1};
    check_pages(c, words, table, w[23], w[22]);
    c.need(w[20] >= 1 && w[21] >= 1, "the page table is empty");
    if (!c.error.empty()) return c.error;
    for (const Region *r : {&q, &k, &v, &o}) c.holds(*r, 4);
    for (const Region *r : {&qn, &kn, &rope}) c.holds(*r, 1);
    std::vector<Region> written = check_pool(c, spec[0], spec[1], w + 14, (uint64_t)w[22] << w[23], kv_dim, bound(3), bound(4));
    if (!c.error.empty()) return c.error;
    for (const Region &r : written) c.apart(r, q);
    // in place, or apart: another wave may still read what this one writes
    if (!o.same(q)) c.apart(o, q);
    written.push_back(o);
    c.writes(written, {k, v, qn, kn, rope, words, table, ctl});
  } else if (op == kAttend) {
    const uint64_t n_kv = w[9], kv_dim = n_kv * kHead, n_head = n_kv * spec[0];
    const uint64_t parts = (uint64_t)w[11] + w[12];
    c.need(w[19] <= 1, "the shared run takes 16 query rows a workgroup (0) or 128 (1)");
    c.need(n_kv >= 1 && n_kv <= 1024, "1 to 1024 key heads");
    c.need(w[12] >= 1 && parts <= kMaxSlots, "a row's own positions take 1 part or more, all of them at most 1024");
    if (!c.error.empty()) return c.error;
    const Region q{"q", A, 4, w[0], w[1], n_head * kHead, rows}, o{"the output", A, 4, w[2], w[3], n_head * kHead, rows};
    const Region part{"the partials", A, 4, w[4], 0, rows * n_head * parts * kPart, 1};
    const Region words{"the rows' words", C, 4, w[13], 4, 4, rows},
        table{"the page table", C, 4, w[14], 0, (uint64_t)w[16] * w[15], 1};
    check_pages(c, words, table, w[18], w[17]);
    c.need(w[15] >= 1 && w[16] >= 1, "the page table is empty");
    c.need(w[15] <= w[17], "a sequence has more pages than the pool");  // bounds every length, and so every loop
    if (!c.error.empty()) return c.error;
    c.holds(q, 4);
    c.holds(o, 2);
    c.holds(part, 2);
    std::vector<Region> read = check_pool(c, spec[1], spec[2], w + 5, (uint64_t)w[17] << w[18], kv_dim, bound(2), bound(3));
    if (!c.error.empty()) return c.error;
    read.insert(read.end(), {words, table, ctl});
    if (!o.same(q)) c.apart(o, q);
    c.apart(part, q);
    c.writes({o, part}, read);
    if (n_kv * ((rows * spec[0] + 15) / 16 * w[11] + rows * w[12]) > kMaxWork)
      c.fail("%llu rows in %llu parts: too many workgroups", (unsigned long long)rows, (unsigned long long)parts);
  } else if (op == kMerge) {
    const uint64_t n_head = w[3], parts = (uint64_t)w[4] + w[5];
    c.need(n_head >= 1 && n_head <= 8192, "1 to 8192 heads");
    c.need(w[5] >= 1 && parts <= kMaxSlots, "a row's own positions take 1 part or more, all of them at most 1024");
    c.need(parts > 1, "one part in all is the attention's result already");
    c.need(w[9] >= 4 && w[9] <= 12, "pages hold 16 to 4096 positions");
    if (!c.error.empty()) return c.error;
    const Region part{"the partials", A, 4, w[0], 0, rows * n_head * parts * kPart, 1},
        o{"the output", A, 4, w[1], w[2], n_head * kHead, rows}, words{"the rows' words", C, 4, w[6], 4, 4, rows};
    c.holds(part, 2);
    c.holds(o, 2);
    c.holds(words, 4);
    c.writes({o}, {part, words, ctl});
  } else if (op == kLogits) {
    const uint64_t v = w[4];
    c.need(v >= 1, "an empty vocabulary");
    const Region x{"the logits", A, 4, w[0], w[2], v, rows}, y{"the adjusted logits", A, 4, w[1], w[3], v, rows};
    const Region ctrl{"the rows' words", C, 4, w[5], 8, 8, rows}, hist{"the histories", C, 4, w[6], w[7], w[7], w[7] ? rows : 0},
        bias{"the biases", C, 4, w[8], w[9], w[9], w[9] ? rows : 0}, mask{"the masks", C, 4, w[10], w[11], w[11], w[11] ? rows : 0};
    c.holds(x, 4);
    c.holds(y, 4);
    c.holds(ctrl, 4);
    c.holds(hist, 4);
    c.holds(bias, 2);
    c.holds(mask, 1);
    if (w[11] && w[11] < (v + 31) / 32) c.fail("a mask of %u words for %llu tokens", w[11], (unsigned long long)v);
    if (!y.same(x)) c.apart(y, x);
    c.writes({y}, {ctrl, hist, bias, mask, ctl});
  }
  return c.error;
}

// The launch of a dispatch: its grid, threads, form (0: the pipeline's own kernel, 1: the other
// one, other_form) and trailing by-value words.
struct Shape {
  uint32_t groups[3] = {1, 1, 1}, threads = 256, form = 0;
  std::vector<uint32_t> extra;
};
inline std::string other_form(Op op, const std::string &symbol) {
  if (op == kLogits) return "logits_adjust_1024";
  if (op == kMerge) return "attention_paged_merge_8__128";
  if (op == kAppend) return "kv_append_4" + symbol.substr(std::strlen("kv_append"));
  return symbol;
}
inline Shape shape(Op op, const uint32_t *spec, const uint32_t *w, uint32_t rows) {
  Shape s;
  s.groups[1] = rows;
  if (op == kAppend) {
    const uint32_t heads = (w[9] + 2 * w[10] + 15) / 16;  // 16 heads a pass
    s.form = (uint64_t)rows * heads >= kAppendMany;
    s.groups[0] = s.form ? (heads + 3) / 4 : heads;
  } else if (op == kAttend) {
    const uint32_t q = rows * spec[0], groups = w[9] * w[11], own = rows * w[9] * w[12];
    if (w[19] && w[11])
      s.groups[0] = (groups + 7) / 8 * 8 * ((q + 127) / 128) + own;
    else
      s.groups[0] = groups * ((q + 15) / 16) + own;
    s.groups[1] = 1;
    s.extra = {rows};
  } else if (op == kMerge) {
    s.form = w[4] + w[5] > kMergeParts && rows * w[3] <= kMergeHeads;
    s.groups[0] = s.form ? w[3] : (w[3] + 3) / 4;
    s.threads = s.form ? 512 : 256;
  } else {
    s.form = w[7] >= kLogitsHistory;
    s.threads = s.form ? 1024 : 256;
    s.groups[0] = (w[4] + 16 * s.threads - 1) / (16 * s.threads);
  }
  return s;
}

}  // namespace batch
