// The operators of a served batch, gfx950: rows of many sequences over a paged KV cache, and
// what is done to their logits before a token is chosen.
//
// Contract (bindings, push words; every grid is [1, rows, 1], and the runtime chooses the launch):
//   kv_append              [W, A, C, KV, KV8]   24 words  spec [K_Q8, V_Q8, head_dim]
//   kv_append_axes         [W, A, C, KV, KV8]   26 words  spec [K_Q8, V_Q8, head_dim]
//   attention_paged        [A, C, KV, KV8, KVS] 20 words  spec [N_REP, K_Q8, V_Q8, head_dim]
//   attention_paged_merge  [A, C]               10 words  spec [head_dim]
//   attention_paged_shaped       [A, C, KV, KV8, KVS] 25 words  spec [N_REP, K_Q8, V_Q8, head_dim]
//   attention_paged_shaped_merge [A, C]         14 words  spec [head_dim]
//   logits_adjust          [A, C]               12 words
// Bindings as in attention.hip.  Heads are 128 wide.
//
// Rows: ctl[2] of them are live (the others are left as they were).  Row r has four words at
// rows_off + 4 r: {seq, len, share, 0}.  Its token is at position len - 1 of sequence seq and
// attends to the positions below len; a row of len 0 has no token: it appends nothing and
// attends to nothing (its output is zeros).  Position p of sequence s lies in slot
// table[s * table_stride + p / page] * page + p % page of the pool, whose rows are laid out as a
// contiguous cache's (attention.hip: slot for pos).
// Shared positions: ctl[3] = P of them, in the pages of sequence ctl[4].  A row with share != 0
// and len >= P takes the positions below P from there; its own pages serve those from P on (all
// of them otherwise).
// Words that name no page or sequence reach no memory outside the pool: a row of such a sequence
// counts as one of len 0, a length past the table's ends there, keys and values of such a page
// are not stored, and a read of it goes to the pool's last page.
// Keys and values are finite (kv_append stores no others but NaN, in 8 bits as a block's scale): a row
// that attends to a NaN or an infinity is not finite where that reaches, and what a row does not attend
// to reaches nothing.
#include <type_traits>

#include "matmul_common.h"

namespace {

constexpr uint32_t HD = 128;         // head width
constexpr uint32_t PART = HD + 2;    // one partial: m, l, acc[128]
constexpr uint32_t TILE = 64;        // the parts of a run are whole multiples of it
constexpr float F16_MAX = 65504.0f;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct AppendPush {
  uint32_t q_off, k_off, v_off, o_off, qn_off, kn_off, rope_off;
  float eps, mscale;
  uint32_t n_head, n_kv, q_stride, kv_stride, o_stride, kc_off, vc_off, ks_off, vs_off, rows_off, table_off,
      table_stride, n_seq, n_pages, page_log2;
};
struct AppendAxesPush {
  AppendPush append;
  uint32_t axes_off, n_axes;
};
struct PagedPush {
  uint32_t q_off, q_stride, o_off, o_stride, part_off, kc_off, vc_off, ks_off, vs_off, n_kv;
  float scale;
  uint32_t n_shared, n_own, rows_off, table_off, table_stride, n_seq, n_pages, page_log2, wide;
};
struct PagedMergePush {
  uint32_t part_off, o_off, o_stride, n_head, n_shared, n_own, rows_off, table_stride, n_seq, page_log2;
};
struct ShapedPush : PagedPush {
  uint32_t spans_off, slopes_off, window, n_lead;
  float cap;
};
struct CappedPush : ShapedPush {};  // of the kernels for a cap above 0
struct ShapedMergePush : PagedMergePush {
  uint32_t spans_off, window, n_lead, rep;
};
template <typename P>
constexpr bool SHAPED = std::is_base_of<ShapedPush, P>::value || std::is_base_of<ShapedMergePush, P>::value;
template <typename P>
constexpr bool CAPPED = std::is_base_of<CappedPush, P>::value;
struct LogitsPush {
  uint32_t x_off, y_off, x_stride, y_stride, n_vocab, ctrl_off, hist_off, hist_stride, bias_off, bias_stride, mask_off,
      mask_stride;
};

SK_DEV float max3(float a, float b, float c) { return __builtin_fmaxf(__builtin_fmaxf(a, b), c); }
SK_DEV float wave_max(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}

// What a row attends to: [0, shared) from the shared pass and [start, len) of its own pages.
struct Range {
  uint32_t seq, len, start;
  bool member;
};
// Shared positions, as the kernels take them: none without slots for their partials or a
// sequence that holds them.
SK_DEV uint32_t shared_positions(const uint32_t *ctl, uint32_t n_shared, uint32_t n_seq, uint32_t table_stride,
                                 uint32_t page_log2) {
  if (n_shared == 0 || ctl[4] >= n_seq) return 0;
  const uint64_t cap = (uint64_t)table_stride << page_log2;
  return ctl[3] < cap ? ctl[3] : (uint32_t)cap;
}
SK_DEV Range row_range(const uint32_t *ctl, uint32_t rows_off, uint32_t row, uint32_t shared, uint32_t n_seq,
                       uint32_t table_stride, uint32_t page_log2) {
  const uint4 w = *(const uint4 *)(ctl + rows_off + 4 * row);
  const uint64_t cap = (uint64_t)table_stride << page_log2;
  Range r;
  r.seq = w.x < n_seq ? w.x : 0;
  r.len = w.x < n_seq ? (w.y < cap ? w.y : (uint32_t)cap) : 0;
  r.member = shared != 0 && w.z != 0 && r.len >= shared;
  r.start = r.member ? shared : 0;
  return r;
}

// attention_paged_shaped: row r's token, at position i = len - 1, attends to the positions j of [lo, hi): from
// `from`, and with a window from len - window on, up to len, or to `until` where that is more ({from, until} at
// spans_off + 2 r; their positions are in the cache when the kernel runs).  A row of len 0, or whose mask leaves
// nothing, gives zeros.  With s = scale q k a score is cap tanh(s / cap) (cap 0: s), less slope_h |i - j| (the
// heads' slopes at slopes_off, of 2^16 at most; ~0: none).  A row that attends to a NaN or an infinity may be not finite
// in all of a head's dims.
// The shared run is [S, P), S the tile's end at or above ctl[5], and with a window at or above ctl[6] - window, ctl[6]
// the longest of the rows (0: ctl[5] alone; layers of one step may have windows of their own).  No row attends to a
// part of it: a row takes it with share != 0 and len >= P if it attends to all of it, lo <= S.  Its own pages serve
// [lo, S), its lead, in n_lead parts (without lead parts lo must be S), and those from P on.
// The bodies are attention_paged's, with these masks, scores and runs, so that what bounds them is the same.  Own runs of
// rows that are one prompt's go together (16 query rows a workgroup for 2 to 8 as elsewhere): a chunk's 128 rows would
// else read their common positions once each (73 -> 57 us a chunk behind a window of 4096 of 12000 positions).  A window
// leaves out tiles before they are read: a pass of that chunk takes, with windows of 64 / 512 / 4096 / none, 32 / 41 / 61 /
// 106 us one by one (57 of 4096 among others).
// Measured (MI355X, + merge): 8 rows of up to 100 own positions, capped, 8.0 us; 32 rows with a window of 1024, f16 keys
// and 8-bit values, 27.8, no merge (97 MB, 3.5 TB/s); 128 rows of 32 heads over 16384 shared and 300 own positions of 8 key
// heads, capped, f16, 105 to 111 + 12 (products 0.68 to 0.72 PFLOP/s in two f16 parts); the chunk above 41.8 + 9.6; 100 rows of
// documents to 4000 positions of 4 key heads, sloped, 8 bits, 34.5 + 7.6 (partials of 20 MB written and read).
// What shaping costs a pass of those 128 rows (f16 / f16 keys, 8-bit values / 8 bits): scores as they are 122 / 148 / 156
// us, sloped 125 / 152 / 163, capped 134 / 152 / 174, both 150 / 171 / 191, one by one: vector instructions beside the
// products.
struct ShapedRange : Range {  // tail: [start, len), len the end hi
  uint32_t lo, at;            // lead: [lo, S) of a member; the position i
};
template <typename P>
SK_DEV uint32_t shared_first(const uint32_t *ctl, const P &p, uint32_t shared) {
  const uint32_t longest = ctl[6], window = p.window && longest > p.window ? longest - p.window : 0;
  const uint32_t first = min(max(ctl[5], window), shared);
  return (first + TILE - 1) / TILE * TILE;
}
template <typename P>
SK_DEV uint32_t shared_end(const uint32_t *ctl, const P &p) {  // 0: none
  const uint32_t shared = shared_positions(ctl, p.n_shared, p.n_seq, p.table_stride, p.page_log2);
  if constexpr (SHAPED<P>) return shared_first(ctl, p, shared) < shared ? shared : 0;
  return shared;
}
template <typename P>
SK_DEV ShapedRange shaped_range(const uint32_t *ctl, const P &p, uint32_t row, uint32_t shared) {
  ShapedRange r;
  (Range &)r = row_range(ctl, p.rows_off, row, shared, p.n_seq, p.table_stride, p.page_log2);
  const uint2 span = *(const uint2 *)(ctl + p.spans_off + 2 * row);
  const uint64_t cap = (uint64_t)p.table_stride << p.page_log2;
  const uint32_t len = r.len;
  r.at = len - 1;
  r.lo = p.window && len > p.window ? max(span.x, len - p.window) : span.x;
  if (len && span.y > len) r.len = span.y < cap ? span.y : (uint32_t)cap;
  if (r.lo >= r.len) {
    r.lo = r.start = r.len = 0, r.member = false;
    return r;
  }
  const uint32_t first = shared_first(ctl, p, shared);
  r.member = r.member && (p.n_lead ? r.lo <= first : r.lo == first);
  r.start = r.member ? shared : r.lo;
  return r;
}
// Whether the T rows from row / T * T on go together: those with a token are of one sequence that there is, and at most
// 256 positions apart, as a prompt's are.  Their own runs (tails, and leads) are then one, cut into parts as one, with each
// row's mask.  (The words through the scalar cache: nothing writes them while the kernel runs.)
typedef const __attribute__((address_space(4))) uint32_t ConstWord;
template <uint32_t T>
SK_DEV bool rows_together(const uint32_t *ctl, uint32_t rows_off, uint32_t row, uint32_t n_rows, uint32_t n_grid,
                          uint32_t n_seq) {
  ConstWord *w = (ConstWord *)(uintptr_t)(ctl + rows_off);
  uint32_t seq = ~0u, least = ~0u, most = 0;
  bool one = true;
#pragma unroll
  for (uint32_t i = 0; i < T; i++) {
    // (the grid's rows, so that the loads wait for no control word)
    const uint32_t r = row / T * T + i, of = w[4 * min(r, n_grid - 1)], len = w[4 * min(r, n_grid - 1) + 1];
    const bool live = r < n_rows && len != 0 && of < n_seq;  // (so that no live one is of ~0)
    one = one && (!live || seq == ~0u || of == seq);
    seq = live ? of : seq, least = live ? min(least, len) : least, most = live ? max(most, len) : most;
  }
  return one && most != 0 && most - least <= 256;
}
// The same for a T that is known when the kernel runs, by whole waves, lane l with row l % T (the merge's: with each T
// unrolled as above a launch of 100 rows took 8.8 us for 8.4).
SK_DEV bool rows_together(const uint32_t *ctl, uint32_t rows_off, uint32_t row, uint32_t n_rows, uint32_t n_grid,
                          uint32_t n_seq, uint32_t T) {
  const uint32_t r = row / T * T + (threadIdx.x & (T - 1));
  const uint2 w = *(const uint2 *)(ctl + rows_off + 4 * min(r, n_grid - 1));
  const bool live = r < n_rows && w.y != 0 && w.x < n_seq;
  const uint64_t m = __ballot(live);
  const uint32_t seq = __builtin_amdgcn_readlane(w.x, m ? (uint32_t)__builtin_ctzll(m) : 0);
  const bool one = m && !__ballot(live && w.x != seq);
  uint32_t least = live ? w.y : ~0u, most = live ? w.y : 0;
  for (uint32_t d = T / 2; d >= 1; d >>= 1)
    least = min(least, (uint32_t)__shfl_xor(least, d, 64)), most = max(most, (uint32_t)__shfl_xor(most, d, 64));
  return __builtin_amdgcn_readfirstlane(one && most - least <= 256);
}
// The positions of row row's own run, its tail or its lead, and of the run that it is part of.  (Whole waves: lane l
// looks at row l % T of the rows that may go together.)
struct OwnRun {
  uint32_t lo, hi, all_lo, all_hi;  // the row's, and the run's; [0, 0): nothing
  uint32_t seq, lane_lo, lane_hi, lane_at;  // row l % T's, in lane l
};
template <typename P>
SK_DEV OwnRun own_run(const uint32_t *ctl, const P &p, uint32_t row, uint32_t n_rows, uint32_t T, bool together,
                      uint32_t shared, bool lead) {
  uint32_t lo = 0, hi = 0, seq = 0, at = 0;
  auto look = [&](uint32_t i) {
    const ShapedRange r = shaped_range(ctl, p, i, shared);
    at = r.at, lo = lead ? r.lo : r.start, hi = lead ? shared_first(ctl, p, shared) : r.len, seq = r.seq;
    if (lo >= hi || (lead && !r.member)) lo = hi = 0;
  };
  if (!together) {  // (the same words in every lane: scalar loads, and nothing to be passed between lanes)
    look(row);
    return {lo, hi, lo, hi, seq, lo, hi, at};
  }
  const uint32_t lane = threadIdx.x & 63, row0 = row / T * T, mine = row0 + (lane & (T - 1));
  if (mine < n_rows) look(mine);
  OwnRun x;
  x.lane_lo = lo, x.lane_hi = hi, x.lane_at = at;
  x.lo = __shfl(lo, row - row0, 64), x.hi = __shfl(hi, row - row0, 64);
  uint32_t from = hi ? lo : ~0u, to = hi, of = hi ? seq : 0;
  for (uint32_t d = T / 2; d >= 1; d >>= 1) {
    from = min(from, (uint32_t)__shfl_xor(from, d, 64)), to = max(to, (uint32_t)__shfl_xor(to, d, 64));
    of = max(of, (uint32_t)__shfl_xor(of, d, 64));
  }
  x.seq = of;
  x.all_lo = to ? from : 0, x.all_hi = to;
  return x;
}
// A head's slope in powers of two, so that no bias reaches what masked scores are set to.
template <typename P>
SK_DEV float slope_of(const uint32_t *ctl, const P &p, uint32_t head) {
  if (p.slopes_off == ~0u) return 0.0f;
  const float slope = __builtin_bit_cast(float, ctl[p.slopes_off + head]);
  return __builtin_amdgcn_fmed3f(slope, -0x1p16f, 0x1p16f) * 1.44269504088896340736f;
}
// a row's range, whichever kernel's
template <typename P>
SK_DEV auto range_of(const uint32_t *ctl, const P &p, uint32_t row, uint32_t shared) {
  if constexpr (SHAPED<P>)
    return shaped_range(ctl, p, row, shared);
  else
    return row_range(ctl, p.rows_off, row, shared, p.n_seq, p.table_stride, p.page_log2);
}

// A run of positions [lo, hi) in tiles of TILE from a multiple of 16 at or below lo, cut into at
// most n parts of whole tiles.
struct Split {
  uint32_t base, tiles, per;
};
SK_DEV Split split_of(uint32_t lo, uint32_t hi, uint32_t n) {
  Split s;
  s.base = lo & ~15u;
  s.tiles = hi > lo ? (hi - s.base + TILE - 1) / TILE : 0;
  s.per = max((s.tiles + n - 1) / n, 1u);
  return s;
}
SK_DEV uint32_t live_parts(const Split &s) { return (s.tiles + s.per - 1) / s.per; }

// Elements 4 t + [0, 4) and 64 + 4 t + [0, 4) (t = lane % 16) of one head's cache row, held as
// attention.hip holds them but for two things: an f16 past the type's largest value is stored as
// that value, and a block's scale too, its values as at most 127 of it, so that the cache has no
// infinity (its products with the f16 parts of a query or a weight would be NaN); and a block that
// holds a NaN has one for its scale.
template <int Q8>
SK_DEV void store_row(f16 *kv, int8_t *kv8, uint32_t cache, uint32_t scales, uint32_t kv_dim, uint32_t slot,
                      uint32_t head, uint32_t t, const float4 (&y)[2]) {
  auto fit = [](float v) { return v > F16_MAX ? F16_MAX : v < -F16_MAX ? -F16_MAX : v; };  // keeps NaN
  const uint32_t dst = cache + slot * kv_dim + head * HD + 4 * t;
#pragma unroll
  for (uint32_t n = 0; n < 2; n++) {
    const float v[4] = {y[n].x, y[n].y, y[n].z, y[n].w};
    if constexpr (!Q8) {
      *(f16x4 *)(kv + dst + 64 * n) = f16x4{(f16)fit(v[0]), (f16)fit(v[1]), (f16)fit(v[2]), (f16)fit(v[3])};
    } else {  // a block: eight lanes' values
      auto bits = [](float x) { return __builtin_bit_cast(uint32_t, fabsf(x)); };  // in the values' order, NaN above all
      uint32_t m = max(max(bits(v[0]), bits(v[1])), max(bits(v[2]), bits(v[3])));
      m = max(m, bits(dpp_f<0xb1>(__builtin_bit_cast(float, m))));
      m = max(m, bits(dpp_f<0x4e>(__builtin_bit_cast(float, m))));
      m = max(m, bits(dpp_f<0x141>(__builtin_bit_cast(float, m))));
      const float s = fit(__builtin_bit_cast(float, m) / 127.0f);
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float x = s > 0.0f ? __builtin_amdgcn_fmed3f(__builtin_rintf(v[e] / s), -127.0f, 127.0f) : 0.0f;
        w |= ((uint32_t)(int)x & 255u) << (8 * e);
      }
      *(uint32_t *)(kv8 + dst + 64 * n) = w;
      if ((t & 7) == 0) kv[scales + slot * (kv_dim / 32) + head * 4 + 2 * n + t / 8] = (f16)s;
    }
  }
}

// A wave holds four heads of a row, 16 lanes each: lane t = lane % 16 has the pairs (d, d + 64), d
// in 4 t + [0, 4), that the rotation turns.  A workgroup's four waves take 16 PASSES heads of one
// row, every load in flight before the first product.  The angle (len - 1) f_d is formed in 64
// bits as revolutions and reduced there: an f32 product is off by 2^-24 of an angle of 1e5, 3e-3
// of a radian.  Each wave turns its row's 64 angles once, one a lane, for all its heads.
// Measured (MI355X): 2048 rows of 48 heads, f16 keys and 8-bit values, 23 us where the caches hold other
// data (90 MB, 3.9 TB/s; f16 25, 8 bits 23), 32 to 38 where a launch before left them written, 18 from
// the caches (f16 15, 8 bits 19); 79 for 34 with a wave a head and 4 bytes a lane and load.  A pass loads
// its norm weights behind the stores of the pass before and so waits for these; the row's words are two
// dependent loads before all others; and 65 registers with 8-bit values leave seven workgroups a
// compute unit for eight.  PASSES = 4 where 16 heads a workgroup would make 4096 of them or more (2048
// rows 33.5 us against 36), below it more workgroups are better (1000 rows 24 against 26.5).  1 row 2.5
// us: the launch and the dependent round trips.
//
// kv_append_axes turns by positions of several axes (time, height, width of images and video): row r has four words
// at axes_off + 4 r, and pair d's angle is the sum over the axes a < n_axes <= 4 of word a times the frequency
// at rope_off + 64 a + d, formed in 64 bits.  A pair that one axis turns has its frequency at that axis and 0 at
// the others, so any layout of sections is the table's.  A row's four words come with a load beside its others, and the
// sum is four f64 products a lane: 1 row 2.8 us, 37 rows in 8 bits 4.4, 2048 rows of 48 heads, f16 keys and 8-bit values,
// 42 (where a launch before left the caches written; the smallest 23), bound as kv_append is.
template <int K8, int V8, int PASSES, int AXES>
SK_DEV void append_body(const float *w, float *a, const uint32_t *ctl, f16 *kv, int8_t *kv8, const AppendPush &p,
                        uint32_t axes_off = 0, uint32_t n_axes = 0) {
#pragma clang fp contract(off)
  __shared__ float2 turn[4][64];
  const uint32_t row = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = lane & 15;
  if (row >= ctl[2]) return;
  const Range r = row_range(ctl, p.rows_off, row, 0, p.n_seq, p.table_stride, p.page_log2);
  if (r.len == 0) return;
  const uint32_t pos = r.len - 1, n_heads = p.n_head + 2 * p.n_kv;
  const uint32_t h0 = (blockIdx.x * PASSES * 4 + wave) * 4 + (lane >> 4);
  float4 x[PASSES][2];
#pragma unroll
  for (uint32_t n = 0; n < PASSES; n++) {
    const uint32_t h = h0 + 16 * n;
    if (h < n_heads) {
      const uint32_t at = h < p.n_head            ? p.q_off + row * p.q_stride + h * HD
                          : h < p.n_head + p.n_kv ? p.k_off + row * p.kv_stride + (h - p.n_head) * HD
                                                  : p.v_off + row * p.kv_stride + (h - p.n_head - p.n_kv) * HD;
      x[n][0] = *(const float4 *)(a + at + 4 * t);
      x[n][1] = *(const float4 *)(a + at + 64 + 4 * t);
    }
  }
  const uint32_t page = ctl[p.table_off + r.seq * p.table_stride + (pos >> p.page_log2)];
  const uint32_t slot = (page << p.page_log2) + (pos & ((1u << p.page_log2) - 1));
  const uint32_t kv_dim = p.n_kv * HD;
  {
    double angle;
    if constexpr (AXES) {
      const uint4 at = *(const uint4 *)(ctl + axes_off + 4 * row);
      const float *f = w + p.rope_off + lane;
      angle = (double)at.x * (double)f[0];
      if (n_axes > 1) angle += (double)at.y * (double)f[64];
      if (n_axes > 2) angle += (double)at.z * (double)f[128];
      if (n_axes > 3) angle += (double)at.w * (double)f[192];
    } else {
      angle = (double)pos * (double)w[p.rope_off + lane];
    }
    const double turns = angle * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turns - __builtin_rint(turns))), &s, &c);
    turn[wave][lane] = make_float2(c * p.mscale, s * p.mscale);
  }
  __syncthreads();
  const float4 cs0 = *(const float4 *)&turn[wave][4 * t], cs1 = *(const float4 *)&turn[wave][4 * t + 2];
  const float c[4] = {cs0.x, cs0.z, cs1.x, cs1.z}, s[4] = {cs0.y, cs0.w, cs1.y, cs1.w};
#pragma unroll
  for (uint32_t n = 0; n < PASSES; n++) {
    const uint32_t h = h0 + 16 * n;
    if (h >= n_heads) break;
    if (h >= p.n_head + p.n_kv) {  // a value head: kept as it is
      if (page < p.n_pages) store_row<V8>(kv, kv8, p.vc_off, p.vs_off, kv_dim, slot, h - p.n_head - p.n_kv, t, x[n]);
      continue;
    }
    const bool is_q = h < p.n_head;
    const float *nw = w + (is_q ? p.qn_off : p.kn_off) + 4 * t;
    const float u[8] = {x[n][0].x, x[n][0].y, x[n][0].z, x[n][0].w, x[n][1].x, x[n][1].y, x[n][1].z, x[n][1].w};
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) ss += u[e] * u[e];
    const float rms = 1.0f / sqrtf(lane_sum<16>(ss) / (float)HD + p.eps);
    float y[8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float n0 = u[e] * rms * nw[e], n1 = u[e + 4] * rms * nw[e + 64];
      y[e] = n0 * c[e] - n1 * s[e];
      y[e + 4] = n0 * s[e] + n1 * c[e];
    }
    const float4 out[2] = {make_float4(y[0], y[1], y[2], y[3]), make_float4(y[4], y[5], y[6], y[7])};
    if (is_q) {
      float *o = a + p.o_off + row * p.o_stride + h * HD + 4 * t;
      *(float4 *)o = out[0];
      *(float4 *)(o + 64) = out[1];
    } else if (page < p.n_pages) {
      store_row<K8>(kv, kv8, p.kc_off, p.ks_off, kv_dim, slot, h - p.n_head, t, out);
    }
  }
}

// What both forms of the attention share.  A query row is held as two f16 parts of q scale log2(e)
// 2^sh, each rounded to nearest (2^-23 of a value, 2^-36 of the row's largest at least; a product with
// a key is exact), scores are in powers of two.  The largest score is followed loosely: the sums are
// scaled down only where a score passes the reference m by LOOSE.  e = 2^(score - m) is held times
// 2^E_SHIFT = 2^(15 - LOOSE), so that it stays in f16's range, as two f16 parts, each rounded to nearest:
// what they leave is 2^-23 of it at most, as often above as below (cut off, it is 6e-8 below on average
// while l sums all of e), or 2^-32 of the row's largest e.  Products are f16 by f16 with f32 sums, each
// value by both parts; of an 8-bit value's two parts the product of the last ones, 2^-24, is left out.
// Measured over positive values, mean / rms of the relative error: 1 position 0 / 2e-8, 5 -3e-8 / 1.0e-7 (f32
// products and sums 0 / 9e-8), 100 -6e-8 / 1.3e-7 (0 / 1.1e-7), 1000 -6e-8 / 1.3e-7, with 128 rows a workgroup
// -1.1e-7 / 3.6e-7 (0 / 1.8e-7); with the parts cut off the mean was twice that.  The rest of it is the
// matrix cores' sums, of which one is rounded for each product.
// One part of q or e would halve the products and cost 2^-12 of a result, 50 times what f32 loses; a third
// of e would make 2^-32 2^-40 and five products four.  LOOSE = 2 would make it 2^-38 and scale the sums
// often: 128 rows over 4000 positions 41.8 -> 43.5 us, over 32768 163 -> 170.
constexpr float LOOSE = 8.0f;
constexpr int E_SHIFT = 7;
SK_DEV int query_shift(float big) { return big > 0.0f && big < INFINITY ? 11 - __builtin_amdgcn_frexp_expf(big) : 0; }
// scores a and b, in units of ua and ub, as weights: x + y into l, the parts at elements e and e + 1
SK_DEV void weigh(float a, float b, float ua, float ub, float c, float &l, f16x8 &ph, f16x8 &pl, int e) {
  const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(a, ua, c));
  const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(b, ub, c));
  l += x;
  l += y;
  uint32_t both = as_u32(pack_f16x2(x, y));
  asm("" : "+v"(both));  // known as a word alone: the compiler would round x and y again for the next line
  const f16x2 hi = as_f16x2(both);
  const f16x2 lo = pack_f16x2(__builtin_fmaf((float)hi.x, -1.0f, x), __builtin_fmaf((float)hi.y, -1.0f, y));
  ph[e] = hi.x, ph[e + 1] = hi.y;
  pl[e] = lo.x, pl[e + 1] = lo.y;
}
// A block's scale s 2^up as the f16 that 8-bit values are multiplied by: 0 outside [2^-14, 2^TOP), where
// it would lose bits or has been taken; infinities and NaN stay.  Scales below this window are
// taken by a further run over the positions with up WINDOW more.
template <int TOP>
constexpr int WINDOW = TOP + 14;
template <int TOP>
SK_DEV f16 scale_in(f16 s, int up) {
  const f16 x = __builtin_ldexpf16(s, up), y = __builtin_fabsf16(x);
  const bool out = y < (f16)0x1p-14f || (y >= (f16)(float)(1 << TOP) && __builtin_fabsf16(s) < (f16)INFINITY);
  return out ? (f16)0.0f : x;
}
// two bytes picked by sel as an f16 pair: 1024 + (byte ^ 0x80), minus 1152
SK_DEV f16x2 widen(uint32_t x1, uint32_t x0, uint32_t sel) {
  const f16x2 off = {(f16)1152.0f, (f16)1152.0f};
  return as_f16x2((__builtin_amdgcn_perm(x1, x0, sel) ^ 0x00800080u) | 0x64006400u) - off;
}
SK_DEV f16x8 widen8(uint2 x) {
  return __builtin_bit_cast(f16x8, make_uint4(as_u32(widen(x.x, x.x, 0x0c010c00u)), as_u32(widen(x.x, x.x, 0x0c030c02u)),
                                              as_u32(widen(x.y, x.y, 0x0c010c00u)), as_u32(widen(x.y, x.y, 0x0c030c02u))));
}
// Scores in powers of two to what they are capped at: c tanh(s / c) = s P((s / c)^2), P the polynomial of degree 4
// nearest to tanh(x) / x for |x| <= 1/2 (1.3e-8 of it at most); where a wave has a larger score, c (1 - e) / (1 + e),
// e = exp(-2 |s| / c), for those (within 4e-7).
struct Cap {
  float c, inv, edge, p[5];
};
SK_DEV float to_scalar(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
SK_DEV Cap cap_of(float cap) {
  const float c = cap * 1.44269504088896340736f, inv = 1.0f / c, k = inv * inv;
  Cap x{c, inv, 0.5f * c, {0.9999999869f, -0.3333306939f * k, 0.1332477932f * k * k, -0.0529860752f * k * k * k,
                           0.0171350065f * k * k * k * k}};
  x.c = to_scalar(x.c), x.inv = to_scalar(x.inv), x.edge = to_scalar(x.edge);
#pragma unroll
  for (int i = 0; i < 5; i++) x.p[i] = to_scalar(x.p[i]);
  return x;
}
template <int N, typename S>
SK_DEV void cap_scores(S &s, const Cap &x) {
  float big = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2) big = max3(big, fabsf(s[i]), fabsf(s[i + 1]));
  const bool any = __any(!(big <= x.edge));
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float v = s[i], u = v * v;
    float y = __builtin_fmaf(x.p[4], u, x.p[3]);
    y = __builtin_fmaf(y, u, x.p[2]);
    y = __builtin_fmaf(y, u, x.p[1]);
    y = __builtin_fmaf(y, u, x.p[0]) * v;
    if (any) {
      const float e = __builtin_amdgcn_exp2f(fabsf(v) * x.inv * -2.88539008177792681472f);
      const float far = __builtin_copysignf(x.c * (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), v);
      y = fabsf(v) > x.edge ? far : y;
    }
    s[i] = y;
  }
}

// The page table through the scalar cache: nothing writes it while the kernel runs, and a vector
// load's wait would be one for the cache rows in flight, too.
struct Pages {
  ConstWord *table;
  uint32_t n_pages, log2;
  __device__ __forceinline__ uint32_t slot(uint32_t pos) const {
    const uint32_t page = min(table[pos >> log2], n_pages - 1);
    return (page << log2) + (pos & ((1u << log2) - 1));
  }
};
SK_DEV Pages pages_of(const uint32_t *ctl, const PagedPush &p, uint32_t seq) {
  return {(ConstWord *)(uintptr_t)(ctl + p.table_off + seq * p.table_stride), p.n_pages, p.page_log2};
}

// A run of positions [begin, end) through one wave, for 16 query rows (this lane's, row c = lane %
// 16, at q); row c's partial goes to out[c].  Of the positions those in [lo, hi) count.  A step
// takes HALF = 32 positions, two groups of 16; the next step's rows are in flight while one is
// computed.  No row of the cache passes through LDS:
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16, A = key rows as loaded (row: position 16 t + c, dims 8 g +
//                 32 k, g = lane / 16), B = query rows; a lane then has row c's scores at 16 t + 4 g + r
//   O^T = V^T P^T B = those weights: element e of group g is position 16 (e / 4) + 4 g + e % 4; A =
//                 value rows of these positions, lane c holding dims 8 c + [0, 8): tile d takes dim
//                 8 c + d as row c, so the transposition is 8 x 8 inside a lane
// Loads of positions outside [lo, hi) go to ones inside, and their scores are -inf, so what lies
// there reaches nothing.  8-bit values are two f16 parts, exact, of q s 2^(4 - ve), ve the exponent of
// the largest scale of the 32 dims, followed as loosely.  Scales 2^18 below it, whose positions may be
// those that a row attends to, would lose bits: a run that meets one is run again with the m and ve that
// it found, once for each window of scales.
// Measured (MI355X, with the waves' join; from the 256 MB cache / where it holds other data): one row of
// 16384 positions of 8 key heads, f16 keys and 8-bit values, 15.9 / 25 us (50 MB), f16 14.9 / 24, 8 bits
// 17 / 27; 128 rows of up to 512 own positions in f16 27 / 55 us (135 MB), f16 keys and 8-bit values 31 /
// 57, 8 bits 37 / 58; 8 rows of up to 100 positions 5.9 us.  Bound by memory's latency: a workgroup's
// dependent round trips (arguments, control words, row words, page numbers one after another, rows) and
// one step in flight behind the one that is waited for.  Without that step the first ran 24 us for 15.5.
constexpr uint32_t HALF = 32;
template <int K8, int V8>
struct HalfRows {
  typename std::conditional<K8, uint2, uint4>::type k[2][4];
  f16x4 ks[K8 ? 2 : 1][4];
  typename std::conditional<V8, uint2, uint4>::type v[8];
  f16 vs[V8 ? 8 : 1];
};
template <int K8, int V8, typename P>
SK_DEV void wave_run(float *a, const uint32_t *ctl, const f16 *kv, const int8_t *kv8, const P &p, uint32_t kvh,
                     const float *q, float (*out)[PART], uint32_t seq, uint32_t lo, uint32_t hi, uint32_t begin,
                     uint32_t end, float slope = 0.0f, uint32_t row_at = 0, uint32_t my_lo = 0, uint32_t my_hi = 0) {
  const uint32_t lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, kv_dim = p.n_kv * HD;
  // wave-uniform, and known to be
  lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
  begin = __builtin_amdgcn_readfirstlane(begin), end = __builtin_amdgcn_readfirstlane(end);
  kvh = __builtin_amdgcn_readfirstlane(kvh);
  const Pages pages = pages_of(ctl, p, __builtin_amdgcn_readfirstlane(seq));
  struct Groups {
    uint32_t pos[2], slot[2];  // a step's groups of 16, moved to ones with live positions
  };
  auto look = [&](uint32_t at) {
    Groups x;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      x.pos[t] = min(max(at + 16 * t, lo & ~15u), (hi - 1) & ~15u);
      x.slot[t] = pages.slot(x.pos[t]);
    }
    return x;
  };
  auto load = [&](HalfRows<K8, V8> &r, const Groups &x) {
    auto row = [&](uint32_t t, uint32_t i) { return x.slot[t] + min(max(x.pos[t] + i, lo), hi - 1) - x.pos[t]; };
#pragma unroll
    for (uint32_t t = 0; t < 2; t++) {
      const uint32_t src = p.kc_off + row(t, c) * kv_dim + kvh * HD + 8 * g;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (K8)
          r.k[t][k] = *(const uint2 *)(kv8 + src + 32 * k);
        else
          r.k[t][k] = *(const uint4 *)(kv + src + 32 * k);
      }
      if constexpr (K8)
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
          r.ks[t][i] = *(const f16x4 *)(kv + p.ks_off + row(t, 4 * g + i) * (kv_dim / 32) + kvh * 4);
    }
#pragma unroll
    for (uint32_t e = 0; e < 8; e++) {
      const uint32_t n = row(e >> 2, 4 * g + (e & 3)), src = p.vc_off + n * kv_dim + kvh * HD + 8 * c;
      if constexpr (V8) {
        r.v[e] = *(const uint2 *)(kv8 + src);
        r.vs[e] = kv[p.vs_off + n * (kv_dim / 32) + kvh * 4 + (c >> 2)];
      } else {
        r.v[e] = *(const uint4 *)(kv + src);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // in flight before what is computed next
  };

  Groups soon;
  HalfRows<K8, V8> ra, rb;
  auto start = [&] {  // (not from a known position: its addresses would be kept in registers for the next run)
    const uint32_t at = begin + (V8 ? opaque_mask(0) : 0);
    const Groups now = look(at);
    soon = look(at + HALF);
    load(ra, now);
  };
  start();
  uint64_t more;  // lanes of a step with scales below the window
  int run = 0, window = 0;
  f16x8 qh[4], ql[4];
  float inv;
  {
    float u[4][8], big = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float4 x = *(const float4 *)(q + 8 * g + 32 * k), y = *(const float4 *)(q + 8 * g + 32 * k + 4);
      const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        u[k][e] = w[e] * (p.scale * 1.44269504088896340736f);
        big = fmaxf(big, fabsf(u[k][e]));
      }
    }
    big = fmaxf(big, __shfl_xor(big, 16, 64));
    big = fmaxf(big, __shfl_xor(big, 32, 64));
    const int sh = query_shift(big);
    inv = ldexpf(1.0f, -sh);
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float x = ldexpf(u[k][e], sh);
        qh[k][e] = (f16)x;
        ql[k][e] = (f16)(x - (float)qh[k][e]);
      }
  }
  [[maybe_unused]] Cap cap;
  [[maybe_unused]] uint32_t all_lo = 0, all_hi = 0;  // what every row sees
  if constexpr (CAPPED<P>) cap = cap_of(p.cap);
  if constexpr (SHAPED<P>) {
    all_lo = my_lo, all_hi = my_hi;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) {
      all_lo = max(all_lo, (uint32_t)__shfl_xor(all_lo, d, 64));
      all_hi = min(all_hi, (uint32_t)__shfl_xor(all_hi, d, 64));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  }
  const float unit = SHAPED<P> ? 1.0f : inv;  // of the scores as they are weighed
  float m = -INFINITY, l;
  int ve = -200, vo = -200;  // of the dims that this lane's values and sums hold (blocks c / 4 and g)
  f32x4 o[8];
  auto word = [](const auto &u, int i) {
    if constexpr (sizeof(u) == 8)
      return i == 0 ? u.x : u.y;
    else
      return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
  };
  auto compute = [&](HalfRows<K8, V8> &r, uint32_t at) {
    float sc[2][4];
#pragma unroll
    for (uint32_t t = 0; t < 2; t++) {
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if constexpr (K8) {
          const f16x8 b = widen8(r.k[t][k]);
          f32x4 part = {0.0f, 0.0f, 0.0f, 0.0f};
          part = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ql[k], part, 0, 0, 0);
          part = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, qh[k], part, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; i++) acc[i] = __builtin_fmaf((float)r.ks[t][i][k], part[i], acc[i]);
        } else {
          const f16x8 b = __builtin_bit_cast(f16x8, r.k[t][k]);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ql[k], acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, qh[k], acc, 0, 0, 0);
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < 4; i++) sc[t][i] = acc[i];
    }
    if constexpr (SHAPED<P>) {
      float s[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) s[i] = sc[i >> 2][i & 3] * inv;
      if constexpr (CAPPED<P>) cap_scores<8>(s, cap);
      const int away = (int)(at + 4 * g - row_at);
#pragma unroll
      for (uint32_t i = 0; i < 8; i++)
        sc[i >> 2][i & 3] = __builtin_fmaf(-slope, fabsf((float)(away + (int)(16 * (i >> 2) + (i & 3)))), s[i]);
    }
    if (SHAPED<P> ? at < all_lo || at + HALF > all_hi : at < lo || at + HALF > hi) {
#pragma unroll
      for (uint32_t t = 0; t < 2; t++)
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
          const uint32_t pos = at + 16 * t + 4 * g + i;
          if (SHAPED<P> ? pos < my_lo || pos >= my_hi : pos < lo || pos >= hi) sc[t][i] = -INFINITY;
        }
      if constexpr (SHAPED<P>) {
        // A weight of 0 would not keep a value that is not finite out of a row that does not see it: such a value is
        // taken for 0, and of the rows that see it the weight for NaN.
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) {
          bool odd;
          if constexpr (V8) {
            odd = !(__builtin_fabsf16(r.vs[e]) < (f16)INFINITY);
            if (odd) r.vs[e] = (f16)0.0f;
          } else {
            uint32_t any = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) any |= (word(r.v[e], k) & 0x7c007c00u) + 0x04000400u;
            odd = any & 0x80008000u;
            if (odd) r.v[e] = make_uint4(0, 0, 0, 0);
          }
          const uint64_t which = __ballot(odd);
          if (which && (which >> (16 * g) & 0xffff) && sc[e >> 2][e & 3] > -INFINITY) sc[e >> 2][e & 3] = NAN;
        }
      }
    }
    float mt = max3(sc[0][0], sc[0][1], sc[0][2]);
    mt = max3(mt, sc[0][3], sc[1][0]);
    mt = max3(mt, sc[1][1], sc[1][2]);
    mt = fmaxf(mt, sc[1][3]);
    mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * unit;
    int top = -200;      // the scales' largest exponent
    float least = 0.0f;  // and the smallest of this lane's that is not 0
    if constexpr (V8) {
      u16x2 big = {0, 0}, low = {0, 0};  // by their bits w: the largest w and the largest -w (0: none above 0)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const u16x2 w = __builtin_bit_cast(u16x2, as_u32(f16x2{r.vs[2 * e], r.vs[2 * e + 1]}) & 0x7fff7fffu);
        big = __builtin_elementwise_max(big, w);
        low = __builtin_elementwise_max(low, (u16x2){0, 0} - w);
      }
      float f = f16_bits_to_f32(max(big.x, big.y));
      least = f16_bits_to_f32((uint16_t)-max(low.x, low.y));
      f = fmaxf(f, __shfl_xor(f, 16, 64));
      f = fmaxf(f, __shfl_xor(f, 32, 64));
      top = f > 0.0f && f < INFINITY ? __builtin_amdgcn_frexp_expf(f) : -200;
    }
    if (__any(mt > m + LOOSE || top > ve + 5)) {
      const float mn = mt > m + LOOSE ? mt : m;
      float down = mn > -INFINITY ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
      m = mn;
      l *= down;
      if constexpr (V8) {
        if (top > ve + 5) ve = top;
        const int vn = __shfl(ve, (int)(4 * g), 64);
        down = ldexpf(down, vo - vn);
        vo = vn;
      }
#pragma unroll
      for (int d = 0; d < 8; d++) o[d] *= down;
    }
    const float cm = (float)E_SHIFT - (m > -INFINITY ? m : 0.0f);
    f16x8 ph, pl;
#pragma unroll
    for (int n = 0; n < 4; n++)
      weigh(sc[n >> 1][2 * (n & 1)], sc[n >> 1][2 * (n & 1) + 1], unit, unit, cm, l, ph, pl, 2 * n);
    f16x2 sv[V8 ? 4 : 1];
    if constexpr (V8) {
      const int up = 4 - ve + WINDOW<9> * window;
      more |= __ballot(least > 0.0f && ldexpf(least, up) < 0x1p-14f);
      if (run) {
#pragma unroll
        for (int e = 0; e < 8; e++) sv[e >> 1][e & 1] = scale_in<9>(r.vs[e], up);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) sv[e >> 1][e & 1] = __builtin_ldexpf16(r.vs[e], up);
      }
    }
#pragma unroll
    for (int d = 0; d < 8; d++) {
      uint32_t x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (V8) {
          const f16x2 v = widen(word(r.v[2 * e + 1], d >> 2), word(r.v[2 * e], d >> 2), 0x0c040c00u + (d & 3) * 0x00010001u);
          const f16x2 hi_ = v * sv[e];
          x[e] = as_u32(hi_);
          y[e] = as_u32(__builtin_elementwise_fma(v, sv[e], -hi_));
        } else {
          x[e] = __builtin_amdgcn_perm(word(r.v[2 * e + 1], d >> 1), word(r.v[2 * e], d >> 1), d & 1 ? 0x07060302u : 0x05040100u);
        }
      }
      const f16x8 vh = __builtin_bit_cast(f16x8, make_uint4(x[0], x[1], x[2], x[3]));
      if constexpr (V8)
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, make_uint4(y[0], y[1], y[2], y[3])), ph,
                                                      o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl, o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph, o[d], 0, 0, 0);
    }
  };
  for (;; run++) {
    more = 0, l = 0.0f;
#pragma unroll
    for (int d = 0; d < 8; d++) o[d] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t at = begin;; at += 2 * HALF) {
      if (at + HALF < end) {
        load(rb, soon);
        soon = look(at + 2 * HALF);
      }
      compute(ra, at);
      if (at + HALF >= end) break;
      if (at + 2 * HALF < end) {
        load(ra, soon);
        soon = look(at + 3 * HALF);
      }
      compute(rb, at + HALF);
      if (at + 2 * HALF >= end) break;
    }
    // the first run is the result, or its m and ve are where the second starts; a window a run from there
    if (!V8 || run || !more) {
      const int back = V8 ? vo - WINDOW<9> * window - 4 - E_SHIFT : -E_SHIFT;
#pragma unroll
      for (int d = 0; d < 8; d++)
#pragma unroll
        for (int r = 0; r < 4; r++) o[d][r] = ldexpf(o[d][r], back);
      float *to = &out[c][2 + 8 * (4 * g)];
      if (V8 && window) {
#pragma unroll
        for (int d = 0; d < 8; d++)
#pragma unroll
          for (int r = 0; r < 4; r++) o[d][r] += to[8 * r + d];
      }
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int d = 0; d < 8; d += 2) *(float2 *)(to + 8 * r + d) = make_float2(o[d][r], o[d + 1][r]);
    }
    if (!V8 || !more) break;
    window = run;
    start();
    __builtin_amdgcn_s_waitcnt(0);  // as behind the first run's queries: the loop waits for none of them
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) *(float2 *)out[c] = make_float2(m, ldexpf(l, -E_SHIFT));
}

// The shared run for WIDE = 128 query rows a workgroup, 32 a wave: what 16 rows a wave read from
// L2 again and again passes through LDS once for all four waves, STEP = 32 positions at a time:
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16, A = keys (row: position lane % 32, dims 16 k + 8 h +
//                 [0, 8), h = lane / 32), B = the query rows' two f16 parts, held in registers
//   O^T = V^T P^T B = this lane's own e: element e of k-step s is position 16 s + 8 (e / 4) + 4 h +
//                 e % 4, as S^T leaves them; A = values of those positions, row: dim 32 d + lane % 32
// The cache's rows are loaded straight into LDS, into rings of DEPTH steps, each wave loading
// positions 8 w to 8 w + 7 of a step with four loads (so a wait for all but 4 (DEPTH - 2) loads
// leaves that many steps in flight).  f16 rows: 16 pieces of 16 bytes at places piece ^ (position %
// 16) for keys, so that 16 rows' like pieces lie in 16 bank groups, and piece ^ 4 (position % 4)
// for values, which are read transposed (ds_read_b64_tr_b16: of 16 lanes, lanes 4 j to 4 j + 3 read
// 16 dims of position j, and lane i receives dim i of the four).  8-bit rows are converted to f16
// in LDS a step before they are read: keys as they are, values into fragments of 64 pieces, lane
// l's at place l ^ (d | (l / 16 % 2) 4), so that a row's dims go to 16 bank groups.
// With f16 keys a step multiplies the next step's scores while it makes this one's e, so that the
// matrix pipe and the vector ALU work side by side in one wave; reads from LDS run two products
// ahead.  (8-bit keys' block sums leave no registers for a second step's scores.)
// 8-bit values are held as two f16 parts, exact, of q s 2^(7 - ve), ve the exponent of the part's
// largest scale of the 32 dims, found first.  A part with scales 2^21 below it is run again for each
// window of them, with the largest score that the first run found.
// Measured (MI355X): 128 rows of 32 heads over 32768 positions of 8 key heads, f16: 138 us, 137 GFLOP
// of f16 products, 1.0 PFLOP/s, where an 8192-cube f16 library product reaches 1.31 (keys and
// values through registers into LDS 147 for 134); 8-bit values 189 (five products for four); 8-bit keys
// too 208.  With up to 512 own positions a row beside the run 151 to 160, 492 with 16 rows a wave.  The
// matrix pipe is busy 52% of the cycles (at the 1.87 GHz that such work is clocked down to) and a wave
// waits 26% of its own (each step's barrier, loads): the products share each wave's issue with the
// vector instructions that make the weights, and neither alone binds it.  Under 1000 positions a part,
// bound by what a workgroup does once: 15 us of round trips, the pass over the scales, the query rows'
// parts and the partials' writes.
constexpr uint32_t WIDE = 128, STEP = 32;
template <typename P>
SK_DEV uint32_t slots_of(const P &p) {  // partials of a row and head
  if constexpr (SHAPED<P>) return p.n_shared + p.n_own + p.n_lead;
  return p.n_shared + p.n_own;
}
template <int Q8>
struct RawRows {
  uint4 x[STEP][Q8 ? 8 : 16];
  uint2 s[Q8 ? STEP : 1];  // the four blocks' scales
};
template <int K8, int V8>
struct WideStage {  // at most half of the 160 KB: two workgroups a compute unit
  static constexpr int DEPTH = V8 ? 3 : 4;
  RawRows<K8> k[DEPTH];
  RawRows<V8> v[DEPTH];
  uint4 kh[K8 ? 2 : 1][K8 ? STEP : 1][16];        // converted keys,
  float ks[K8 ? 2 : 1][4][K8 ? STEP : 4];         // their scales: [step][dims / 32][position]
  uint4 vh[V8 ? 2 : 1][V8 ? 2 : 1][2][4][V8 ? 64 : 1];  // and values: [step][part][k-step][dims / 32]
  u16x2 ends[4][4];
};
template <int K8, int V8, typename P>
SK_DEV void wide_run(float *a, const uint32_t *ctl, const f16 *kv, const int8_t *kv8, const P &p, uint32_t rep,
                     uint32_t kvh, uint32_t tile, uint32_t part, uint32_t shared, uint32_t n_rows,
                     WideStage<K8, V8> &st) {
  const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, col = lane & 31,
                 h = lane >> 5;
  const uint32_t kv_dim = p.n_kv * HD;
  uint32_t first_at = 0;
  if constexpr (SHAPED<P>) first_at = shared_first(ctl, p, shared);
  const Split sp = split_of(first_at, shared, p.n_shared);
  const uint32_t begin = first_at + part * sp.per * TILE, end = min(begin + sp.per * TILE, shared);
  if (begin >= end) return;
  const uint32_t i = tile * WIDE + wave * 32 + col;
  uint32_t row = i / rep;
  const uint32_t head = i % rep;
  const Pages pages = pages_of(ctl, p, __builtin_amdgcn_readfirstlane(ctl[4]));

  // Staging.  Positions past the end are read as the last one.
  constexpr int DEPTH = WideStage<K8, V8>::DEPTH;
  const uint32_t n_at = 8 * wave;  // the wave's first position of a step
  struct Rows {
    uint32_t first, room;  // that position's pool row, and how many live positions follow it
  };
  auto look = [&](uint32_t step) {
    const uint32_t pos = min(begin + step * STEP + n_at, end - 1);
    return Rows{pages.slot(pos), end - 1 - pos};
  };
  const uint64_t pool = (uint64_t)(p.n_pages << p.page_log2) * kv_dim;
  const u32x4 kres = K8 ? dl_res(kv8 + p.kc_off, pool) : dl_res(kv + p.kc_off, 2 * pool);
  const u32x4 vres = V8 ? dl_res(kv8 + p.vc_off, pool) : dl_res(kv + p.vc_off, 2 * pool);
  const u32x4 ksres = dl_res(kv + p.ks_off, pool / 16), vsres = dl_res(kv + p.vs_off, pool / 16);
  // two loads: the wave's rows in 16 bits, or in 8 and their scales
  auto load_f16 = [&](RawRows<0> &to, const u32x4 &res, const Rows &at, bool is_v) {
#pragma unroll
    for (uint32_t j = 0; j < 2; j++) {
      const uint32_t n = 4 * j + (lane >> 4), piece = (lane & 15) ^ (is_v ? (n & 3) << 2 : (n_at + n) & 15);
      dl_load16(res, lds_addr(&to.x[n_at + 4 * j][0]), (__umul24(min(n, at.room), kv_dim) + 8 * piece) * 2,
                (at.first * kv_dim + kvh * HD) * 2);
    }
  };
  auto load_q8 = [&](RawRows<1> &to, const u32x4 &res, const u32x4 &sres, const Rows &at) {
    dl_load16(res, lds_addr(&to.x[n_at][0]), __umul24(min(lane >> 3, at.room), kv_dim) + 16 * (lane & 7),
              at.first * kv_dim + kvh * HD);
    const uint32_t base = __builtin_amdgcn_readfirstlane(at.first * (kv_dim / 16) + kvh * 8);
    if (lane < 16)
      dl_load4(sres, lds_addr(&to.s[n_at]), __umul24(min(lane >> 1, at.room), kv_dim / 16) + 4 * (lane & 1), base);
  };
  auto load_keys = [&](uint32_t step, const Rows &at) {
    if constexpr (K8)
      load_q8(st.k[step % DEPTH], kres, ksres, at);
    else
      load_f16(st.k[step % DEPTH], kres, at, false);
  };
  auto load_values = [&](uint32_t step, const Rows &at) {
    if constexpr (V8)
      load_q8(st.v[step % DEPTH], vres, vsres, at);
    else
      load_f16(st.v[step % DEPTH], vres, at, true);
  };

  // The first steps' rows are on their way before anything else is waited for.
  // Step s's values are loaded with step s + VK's keys: keys (scores come a step ahead) and 8-bit
  // rows (converted a step ahead) are free for the next load a step before f16 values.
  constexpr uint32_t VK = !V8, LEAD = DEPTH - 1 + V8;  // ... at the top of step s - LEAD
  // (not from a constant: the addresses would be kept in registers from run to run)
  auto prime = [&] {
    const uint32_t first = V8 ? opaque_mask(0) : 0;
    for (uint32_t s = 0; s < DEPTH; s++) {
      load_keys(first + s, look(first + s));
      if (s < LEAD) load_values(first + s, look(first + s));
    }
  };
  prime();

  const bool live = row < n_rows && range_of(ctl, p, row, shared).member;
  row = min(row, n_rows - 1);
  [[maybe_unused]] Cap cap;
  [[maybe_unused]] float slope = 0.0f;
  [[maybe_unused]] uint32_t row_at = 0;
  if constexpr (SHAPED<P>) {
    if constexpr (CAPPED<P>) cap = cap_of(p.cap);
    slope = slope_of(ctl, p, kvh * rep + head);
    row_at = range_of(ctl, p, row, shared).at;
  }
  // this wave's query rows
  f16x8 qh[8], ql[8];
  float inv;
  {
    const float *q = a + p.q_off + row * p.q_stride + (kvh * rep + head) * HD + 8 * h;
    float u[8][8], big = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float4 x = *(const float4 *)(q + 16 * k), y = *(const float4 *)(q + 16 * k + 4);
      const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        u[k][e] = w[e] * (p.scale * 1.44269504088896340736f);
        big = fmaxf(big, fabsf(u[k][e]));
      }
    }
    big = fmaxf(big, __shfl_xor(big, 32, 64));
    if (!__syncthreads_or(live)) {
      dl_wait_vm<0>();
      return;
    }
    const int sh = query_shift(big);
    inv = ldexpf(1.0f, -sh);
#pragma unroll
    for (int k = 0; k < 8; k++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float x = ldexpf(u[k][e], sh);
        qh[k][e] = (f16)x;
        ql[k][e] = (f16)(x - (float)qh[k][e]);
      }
  }

  int ve[4] = {0, 0, 0, 0};
  int runs = 1;  // of the part: a window of scales each
  if constexpr (V8) {
    u16x2 ends[4] = {};  // a block's scales by their bits w: the largest w and the largest -w (0: none above 0)
    for (uint32_t pos = begin + t; pos < end; pos += 256) {
      const f16x4 s = *(const f16x4 *)(kv + p.vs_off + pages.slot(pos) * (kv_dim / 32) + kvh * 4);
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const f16 x = s[b];  // (a bit cast of an element itself takes element 0)
        const uint16_t w = __builtin_bit_cast(uint16_t, x) & 0x7fff;
        ends[b] = __builtin_elementwise_max(ends[b], u16x2{w, (uint16_t)-w});
      }
    }
#pragma unroll
    for (int b = 0; b < 4; b++) {
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1)
        ends[b] = __builtin_elementwise_max(
            ends[b], __builtin_bit_cast(u16x2, __shfl_xor(__builtin_bit_cast(uint32_t, ends[b]), d, 64)));
      if (lane == 0) st.ends[wave][b] = ends[b];
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const u16x2 e = __builtin_elementwise_max(__builtin_elementwise_max(st.ends[0][b], st.ends[1][b]),
                                                __builtin_elementwise_max(st.ends[2][b], st.ends[3][b]));
      const float m = f16_bits_to_f32(e.x), n = f16_bits_to_f32((uint16_t)-e.y);
      ve[b] = __builtin_amdgcn_readfirstlane(m > 0.0f && m < INFINITY ? __builtin_amdgcn_frexp_expf(m) : 0);
      for (int k = 1; n > 0.0f && ldexpf(n, 7 - ve[b] + WINDOW<7> * (k - 1)) < 0x1p-14f; k++) runs = max(runs, k + 1);
    }
    runs = __builtin_amdgcn_readfirstlane(runs);
  }

  // 8-bit rows to f16: dims 8 dg + [0, 8) of positions 2 pr and 2 pr + 1
  const uint32_t dg = t & 15, pr = t >> 4;
  int vmine = ve[0];
  if constexpr (V8) vmine = dg >> 2 == 0 ? ve[0] : dg >> 2 == 1 ? ve[1] : dg >> 2 == 2 ? ve[2] : ve[3];
  constexpr bool AHEAD = !K8;
  auto convert_keys = [&](uint32_t step) {
    if constexpr (K8) {
#pragma unroll
      for (uint32_t j = 0; j < 2; j++) {
        const uint32_t pos = 2 * pr + j;
        const uint2 x = ((const uint2 *)st.k[step % DEPTH].x[pos])[dg];
        st.kh[step & 1][pos][dg ^ (pos & 15)] = __builtin_bit_cast(uint4, widen8(x));
      }
      if (t < 4 * STEP) st.ks[step & 1][t & 3][t >> 2] = (float)((const f16 *)st.k[step % DEPTH].s)[t];
    }
  };
  auto convert_values = [&](uint32_t step) {
    if constexpr (V8) {
      const RawRows<1> &from = st.v[step % DEPTH];
      const uint32_t dt = dg >> 2, hh = pr >> 1 & 1, w = 2 * (pr >> 2 & 1) + (pr & 1);
      const uint32_t sw = dt | ((dg >> 1 & 1) << 2);
      const uint2 x0 = ((const uint2 *)from.x[2 * pr])[dg], x1 = ((const uint2 *)from.x[2 * pr + 1])[dg];
      const f16 s0 = ((const f16 *)&from.s[2 * pr])[dt], s1 = ((const f16 *)&from.s[2 * pr + 1])[dt];
      const f16x2 sv = {scale_in<7>(s0, 7 - vmine), scale_in<7>(s1, 7 - vmine)};
#pragma unroll
      for (uint32_t e = 0; e < 8; e++) {
        const uint32_t at = (hh * 32 + 8 * (dg & 3) + e) ^ sw;
        const f16x2 v = widen(e < 4 ? x1.x : x1.y, e < 4 ? x0.x : x0.y, 0x0c040c00u + (e & 3) * 0x00010001u);
        const f16x2 hi = v * sv;
        ((uint32_t *)&st.vh[step & 1][0][pr >> 3][dt][at])[w] = as_u32(hi);
        ((uint32_t *)&st.vh[step & 1][1][pr >> 3][dt][at])[w] = as_u32(__builtin_elementwise_fma(v, sv, -hi));
      }
    }
  };

  // keys of a staged step: dims 16 k + [0, 16)
  uint32_t kbase = col * 16 + (h ^ (col & 15));
  auto key = [&](uint32_t step, uint32_t k) {
    if constexpr (K8)
      return __builtin_bit_cast(f16x8, (&st.kh[step & 1][0][0])[kbase ^ (2 * k)]);
    else
      return __builtin_bit_cast(f16x8, (&st.k[step % DEPTH].x[0][0])[kbase ^ (2 * k)]);
  };
  auto zero = [](f32x16 &x) {
#pragma unroll
    for (int r = 0; r < 16; r++) x[r] = 0.0f;
  };
  // scores of a staged step; 8-bit keys: blocks of 32 dims times their scales
  auto scores = [&](uint32_t step) {
    f32x16 sc;
    zero(sc);
    if constexpr (K8) {
#pragma unroll
      for (uint32_t b = 0; b < 4; b++) {
        f32x16 x;
        zero(x);
#pragma unroll
        for (uint32_t k = 2 * b; k < 2 * b + 2; k++) {
          const f16x8 w = key(step, k);
          x = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, ql[k], x, 0, 0, 0);
          x = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, qh[k], x, 0, 0, 0);
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
          const float4 f = *(const float4 *)&st.ks[step & 1][b][8 * j + 4 * h];
          sc[4 * j] = __builtin_fmaf(f.x, x[4 * j], sc[4 * j]);
          sc[4 * j + 1] = __builtin_fmaf(f.y, x[4 * j + 1], sc[4 * j + 1]);
          sc[4 * j + 2] = __builtin_fmaf(f.z, x[4 * j + 2], sc[4 * j + 2]);
          sc[4 * j + 3] = __builtin_fmaf(f.w, x[4 * j + 3], sc[4 * j + 3]);
        }
      }
    } else {
#pragma unroll
      for (uint32_t k = 0; k < 8; k++) {
        const f16x8 w = key(step, k);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, ql[k], sc, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, qh[k], sc, 0, 0, 0);
      }
    }
    return sc;
  };
  // values of a staged step: k-step k, dims 32 d + [0, 32)
  typedef __fp16 half4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) half4 LdsHalf4;
  const uint32_t lr = lane >> 2 & 3;
  const uint32_t vbase = (4 * h + lr) * 256 + 32 * (lane >> 4 & 1) + 8 * (lane & 3);
  auto value = [&](uint32_t step, int part_, uint32_t k, uint32_t d) {
    if constexpr (V8) {
      return __builtin_bit_cast(f16x8, st.vh[step & 1][part_][k][d][lane ^ (d | ((lane >> 4 & 1) << 2))]);
    } else {
      const uint32_t at = lds_addr(&st.v[step % DEPTH].x[16 * k][0]) + vbase + ((d ^ lr) << 6);
      const half4 x = __builtin_amdgcn_ds_read_tr16_b64_v4f16((LdsHalf4 *)(uintptr_t)at);
      const half4 y = __builtin_amdgcn_ds_read_tr16_b64_v4f16((LdsHalf4 *)(uintptr_t)(at + 8 * 256));
      const f16x4 u = __builtin_bit_cast(f16x4, x), v = __builtin_bit_cast(f16x4, y);
      return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };

  f32x16 o[4];
  float m = -INFINITY, l;
  // What the scores are weighed in: as they are times `unit`, or, capped, times c P(x^2) of x = s / c, P the polynomial
  // of degree 3 nearest to tanh(x) / x for |x| <= 0.35 (3.5e-8 of it at most; the largest of a step's scores is past that
  // in few steps: those, like biased ones, are capped before)
  float unit = inv;
  if constexpr (SHAPED<P>) unit = p.slopes_off != ~0u ? 1.0f : inv;
  [[maybe_unused]] float over = 0.0f;
  if constexpr (CAPPED<P>) over = inv * cap.inv;
  const uint32_t n_steps = (end - begin + STEP - 1) / STEP;
  Rows vat, kat;
  // `sc`: this step's scores; into `next` the next step's
  auto do_step = [&](uint32_t step, f32x16 &sc, f32x16 &next) {
    // here: this step's scores (AHEAD), and what is multiplied below lies in LDS, converted; what the
    // loads write is read
    load_values(step + LEAD, vat);
    load_keys(step + LEAD + VK, kat);
    vat = look(step + 1 + LEAD);
    kat = look(step + 1 + LEAD + VK);
    const uint32_t at = begin + step * STEP;
    f16x8 kf[3];
    if constexpr (AHEAD) {
      kf[0] = key(step + 1, 0);
      kf[1] = key(step + 1, 1);
    } else {
      sc = scores(step);
    }
    [[maybe_unused]] float p0 = 1.0f, p1 = 0.0f, p2 = 0.0f, p3 = 0.0f;
    [[maybe_unused]] auto lifted = [&](float x) {
      const float u = x * x;
      float y = __builtin_fmaf(p3, u, p2);
      y = __builtin_fmaf(y, u, p1);
      return __builtin_fmaf(y, u, p0);
    };
    const bool tail = at + STEP > end;  // the run's last positions
    [[maybe_unused]] auto bias = [&] {  // (every position is below the row's)
      const float away = (float)(int)(at + 4 * h - row_at) * slope;
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) sc[r] += __builtin_fmaf(slope, (float)(8 * (r >> 2) + (r & 3)), away);
    };
    if constexpr (CAPPED<P>) {
      float big = 0.0f;
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) sc[r] *= over;
#pragma unroll
      for (uint32_t r = 0; r < 16; r += 2) big = max3(big, fabsf(sc[r]), fabsf(sc[r + 1]));
      if (p.slopes_off == ~0u && !tail && !__any(!(big <= 0.35f))) {
        p0 = 0.9999999653f * cap.c, p1 = -0.3333242243f * cap.c, p2 = 0.1329579931f * cap.c, p3 = -0.0489582307f * cap.c;
      } else {
#pragma unroll
        for (uint32_t r = 0; r < 16; r++) sc[r] *= cap.c;
        cap_scores<16>(sc, cap);
        if (p.slopes_off != ~0u) bias();
        if (tail) {  // (not infinite: it is squared)
#pragma unroll
          for (uint32_t r = 0; r < 16; r++)
            if (at + 8 * (r >> 2) + 4 * h + (r & 3) >= end) sc[r] = -0x1p50f;
        }
      }
    } else {
      if constexpr (SHAPED<P>) {
        if (p.slopes_off != ~0u) {
#pragma unroll
          for (uint32_t r = 0; r < 16; r++) sc[r] *= inv;
          bias();
        }
      }
      if (tail) {
#pragma unroll
        for (uint32_t r = 0; r < 16; r++)
          if (at + 8 * (r >> 2) + 4 * h + (r & 3) >= end) sc[r] = -INFINITY;
      }
    }
    float mt = max3(sc[0], sc[1], sc[2]);
#pragma unroll
    for (int r = 3; r < 15; r += 2) mt = max3(mt, sc[r], sc[r + 1]);
    mt = fmaxf(mt, sc[15]);
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    if constexpr (CAPPED<P>) {
      mt *= lifted(mt);
    } else {
      mt *= unit;
    }
    if (__any(mt > m + LOOSE)) {  // rare after the first steps
      const float mn = mt > m + LOOSE ? mt : m;
      const float down = mn > -INFINITY ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
      m = mn;
      l *= down;
#pragma unroll
      for (int d = 0; d < 4; d++) o[d] *= down;
    }
    const float c = (float)E_SHIFT - (m > -INFINITY ? m : 0.0f);
    f16x8 ph[2], pl[2];
    auto weigh2 = [&](uint32_t n) {
      const float x = sc[2 * n], y = sc[2 * n + 1];
      if constexpr (CAPPED<P>)
        weigh(x, y, lifted(x), lifted(y), c, l, ph[n >> 2], pl[n >> 2], 2 * (n & 3));
      else
        weigh(x, y, unit, unit, c, l, ph[n >> 2], pl[n >> 2], 2 * (n & 3));
    };
    f16x8 vf[V8 ? 2 : 1][3];
    auto read_values = [&](uint32_t n) {  // of product n: k-step n / 4, dims 32 (n % 4) + [0, 32)
      vf[0][n % 3] = value(step, 0, n >> 2, n & 3);
      if constexpr (V8) vf[V8 ? 1 : 0][n % 3] = value(step, 1, n >> 2, n & 3);
    };
    if constexpr (AHEAD) {
      zero(next);
#pragma unroll
      for (uint32_t k = 0; k < 8; k++) {
        if (k < 6)
          kf[(k + 2) % 3] = key(step + 1, k + 2);
        else
          read_values(k - 6);
        next = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k % 3], ql[k], next, 0, 0, 0);
        weigh2(k);
        next = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k % 3], qh[k], next, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      read_values(0);
      read_values(1);
#pragma unroll
      for (uint32_t k = 0; k < 4; k++) weigh2(k);
    }
#pragma unroll
    for (uint32_t n = 0; n < 8; n++) {
      const uint32_t k = n >> 2, d = n & 3;
      if (n < 6) read_values(n + 2);
      if constexpr (V8) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[V8 ? 1 : 0][n % 3], ph[k], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[0][n % 3], pl[k], o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[0][n % 3], ph[k], o[d], 0, 0, 0);
      if constexpr (!AHEAD)
        if (n < 4) weigh2(n + 4);
      if (n == (AHEAD ? 1 : 4)) convert_values(step + 1);
      if (n == 5) convert_keys(step + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    dl_wait_vm<4 * (DEPTH - 2)>();
    __syncthreads();
  };
  for (int run = 0;; run++) {
#pragma unroll
    for (int d = 0; d < 4; d++) zero(o[d]);
    l = 0.0f;
    dl_wait_vm<0>();
    __syncthreads();
    const uint32_t first = V8 ? opaque_mask(0) : 0;
    if constexpr (V8) asm volatile("" : "+v"(kbase));  // (as prime's: nothing of it is kept from run to run)
    convert_keys(first);
    convert_values(first);
    __syncthreads();
    f32x16 sc, other;
    if constexpr (AHEAD) {
      sc = scores(first);
      __syncthreads();  // before the loop's first loads write its keys
    }
    vat = look(LEAD), kat = look(LEAD + VK);
    if constexpr (V8) {  // two steps a round would need more registers than two waves a SIMD have
      for (uint32_t step = 0; step < n_steps; step++) {
        do_step(step, sc, other);
        if constexpr (AHEAD) sc = other;
      }
    } else {
      uint32_t step = 0;
      for (; step + 2 <= n_steps; step += 2) {
        do_step(step, sc, other);
        do_step(step + 1, other, sc);
      }
      if (step < n_steps) do_step(step, sc, other);
    }
    dl_wait_vm<0>();  // nothing is left to write this workgroup's LDS
    uint32_t me;  // the lane again: no register held it through the loop
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(me));
    const uint32_t mine = me >> 5, to = tile * WIDE + wave * 32 + (me & 31);
    l += __shfl_xor(l, 32, 64);
    if (live) {
      float *out = a + p.part_off +
                   ((to / rep * p.n_kv * rep + kvh * rep + to % rep) * slots_of(p) + part) * PART;
      float *dims = out + 2 + 4 * mine;
#pragma unroll
      for (int d = 0; d < 4; d++) o[d] *= ldexpf(1.0f, V8 ? ve[d] - WINDOW<7> * run - 7 - E_SHIFT : -E_SHIFT);
      if (V8 && run) {
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[d][r] += dims[32 * d + 8 * (r >> 2) + (r & 3)];
      }
#pragma unroll
      for (int d = 0; d < 4; d++)
#pragma unroll
        for (int r = 0; r < 16; r += 2)
          *(float2 *)(dims + 32 * d + 8 * (r >> 2) + (r & 3)) = make_float2(o[d][r], o[d][r + 1]);
      if (mine == 0) *(float2 *)out = make_float2(m, ldexpf(l, -E_SHIFT));
    }
    if (!V8 || run + 1 == runs) return;
    // (every wave is past the last step's reads)
    prime();
    vmine -= WINDOW<7>;
  }
}

// Workgroups of four waves: first those of the shared run, `wide` (wide_run; the row tiles of a key
// head's part lie 8 workgroups apart, so on one XCD and its L2) or for 16 query rows each; then one
// for each (row, part of its own run, key head).  The latter two cut their part into the waves'
// runs and join these in LDS.  Where a row has one part in all (slots == 1) the joined run is the
// result.
template <int K8, int V8>
union PagedShared {
  WideStage<K8, V8> wide;
  float run[4][16][PART];
};
template <int N_REP, int K8, int V8, typename P>
SK_DEV void paged_body(float *a, const uint32_t *ctl, const f16 *kv, const int8_t *kv8, const P &p, uint32_t n_grid) {
  const bool wide = p.wide && p.n_shared;
  __shared__ __attribute__((aligned(1024))) PagedShared<K8, V8> st;
  const uint32_t t = threadIdx.x, wave = t >> 6, c = t & 15;
  const uint32_t n_rows = min(ctl[2], n_grid), slots = slots_of(p), groups = p.n_kv * p.n_shared;
  const uint32_t shared = shared_end(ctl, p);
  uint32_t w = blockIdx.x, kvh, part, seq, lo, hi;
  if constexpr (!SHAPED<P>)
    if (n_rows == 0) return;
  const uint32_t tiles = wide ? (n_grid * N_REP + WIDE - 1) / WIDE : (n_grid * N_REP + 15) / 16;
  const uint32_t n_first = wide ? (groups + 7) / 8 * 8 * tiles : groups * tiles;
  const bool own = w >= n_first;
  uint32_t i0;  // query rows i0 + [0, n_live) of the key head: row i / N_REP, head i % N_REP
  Split sp;
  // of an own run: its partial, the first of the rows that may go together, the query rows that do
  [[maybe_unused]] uint32_t slot = 0, tile0 = 0, n_own_rows = N_REP;
  [[maybe_unused]] OwnRun run;
  if (!own) {
    if (shared == 0 || (SHAPED<P> && n_rows == 0)) return;
    if (wide) {
      const uint32_t g = w / (8 * tiles) * 8 + w % 8;
      if (g < groups)
        wide_run<K8, V8>(a, ctl, kv, kv8, p, N_REP, g % p.n_kv, w / 8 % tiles, g / p.n_kv, shared, n_rows, st.wide);
      return;
    }
    kvh = w % p.n_kv, part = w / p.n_kv % p.n_shared, i0 = w / groups * 16;
    lo = 0, hi = shared, seq = ctl[4];
    if constexpr (SHAPED<P>) lo = shared_first(ctl, p, shared);
    sp = split_of(lo, hi, p.n_shared);
  } else {
    w -= n_first;
    const uint32_t n_own = slots - p.n_shared;
    kvh = w % p.n_kv, part = w / p.n_kv % n_own;
    uint32_t row = w / (p.n_kv * n_own);
    if constexpr (SHAPED<P>) {
      // (the first rows of every T come first: the others of those that go together end at once, and would else hold
      // places up)
      constexpr uint32_t T = 16 / N_REP;
      const uint32_t tiles = (n_grid + T - 1) / T;
      row = row % tiles * T + row / tiles;
      const bool together = rows_together<T>(ctl, p.rows_off, row, n_rows, n_grid, p.n_seq), lead = part >= p.n_own;
      tile0 = row / T * T;
      if (row >= n_rows || (together && row != tile0)) return;
      run = own_run(ctl, p, row, n_rows, T, together, shared, lead);
      slot = p.n_shared + part;
      if (together) n_own_rows = min(T, n_rows - tile0) * N_REP;
      if (lead) part -= p.n_own;
      i0 = row * N_REP, lo = run.all_lo, hi = run.all_hi, seq = run.seq;
      sp = split_of(lo, hi, lead ? p.n_lead : p.n_own);
    } else {
      if (row >= n_rows) return;
      const auto r = range_of(ctl, p, row, shared);
      i0 = row * N_REP, lo = r.start, hi = r.len, seq = r.seq;
      sp = split_of(lo, hi, p.n_own);
    }
  }
  const uint32_t n_live = own ? SHAPED<P> ? n_own_rows : N_REP : 16;
  const uint32_t begin = sp.base + part * sp.per * TILE, end = min(begin + sp.per * TILE, hi);
  auto result = [&](uint32_t i, uint32_t j) -> float * {  // query row i's dims 2 j and 2 j + 1
    return a + p.o_off + i / N_REP * p.o_stride + (kvh * N_REP + i % N_REP) * HD + 2 * j;
  };
  if (part * sp.per >= sp.tiles) {
    if (slots == 1 && hi == 0)  // a row without positions, or all that go together
      for (uint32_t j = t; j < n_live * 64; j += 256) *(float2 *)result(i0 + j / 64, j % 64) = make_float2(0.0f, 0.0f);
    return;
  }
  // Each row's [lo, hi) of the run (shaped): rows that go together may see parts of it.
  [[maybe_unused]] __shared__ uint4 sees[SHAPED<P> ? 16 : 1];  // and its position
  if constexpr (SHAPED<P>) {
    if (t < 16) {
      if (own) {
        const uint32_t at = (i0 + c % n_live) / N_REP - tile0;
        sees[t] = make_uint4(__shfl(run.lane_lo, at, 64), __shfl(run.lane_hi, at, 64), __shfl(run.lane_at, at, 64), 0);
      } else {
        sees[t] = make_uint4(lo, hi, range_of(ctl, p, min((i0 + t) / N_REP, n_rows - 1), shared).at, 0);
      }
    }
    __syncthreads();
  }
  // whether query row i takes part in this run
  auto live = [&](uint32_t i) {
    if constexpr (SHAPED<P>)
      if (own) return max(sees[i - i0].x, begin) < min(sees[i - i0].y, end);
    return own || (i / N_REP < n_rows && range_of(ctl, p, i / N_REP, shared).member);
  };
  if (!own && !__syncthreads_or(live(i0 + c))) return;
  const uint32_t steps = (end - begin + HALF - 1) / HALF, per = (steps + 3) / 4 * HALF;
  if (begin + wave * per < end) {
    const uint32_t i = i0 + c % n_live, row = min(i / N_REP, n_rows - 1);
    [[maybe_unused]] float slope = 0.0f;
    [[maybe_unused]] uint32_t row_at = 0;
    [[maybe_unused]] uint4 mine = {};
    if constexpr (SHAPED<P>) {
      slope = slope_of(ctl, p, kvh * N_REP + i % N_REP);
      mine = sees[c % n_live];
      row_at = mine.z;
    }
    wave_run<K8, V8>(a, ctl, kv, kv8, p, kvh, a + p.q_off + row * p.q_stride + (kvh * N_REP + i % N_REP) * HD,
                     st.run[wave], seq, lo, hi, begin + wave * per, min(begin + (wave + 1) * per, end), slope, row_at, mine.x,
                     mine.y);
  }
  const uint32_t used = (steps * HALF + per - 1) / per;  // waves with a run
  __syncthreads();
  for (uint32_t j = t; j < n_live * 64; j += 256) {
    const uint32_t r = j / 64, d = j % 64, i = i0 + r;
    if (!live(i)) {
      if constexpr (SHAPED<P>)  // a row without positions among others
        if (slots == 1 && sees[r].y == 0) *(float2 *)result(i, d) = make_float2(0.0f, 0.0f);
      continue;
    }
    float m = st.run[0][r][0];
#pragma unroll
    for (uint32_t n = 1; n < 4; n++)
      if (n < used) m = fmaxf(m, st.run[n][r][0]);
    const float mu = m > -INFINITY ? m : 0.0f;
    float l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
    for (uint32_t n = 0; n < 4; n++)
      if (n < used) {
        const float f = __builtin_amdgcn_exp2f(st.run[n][r][0] - mu);
        const float2 v = *(const float2 *)&st.run[n][r][2 + 2 * d];
        l = __builtin_fmaf(f, st.run[n][r][1], l);
        x = __builtin_fmaf(f, v.x, x);
        y = __builtin_fmaf(f, v.y, y);
      }
    if (slots == 1) {
      *(float2 *)result(i, d) = make_float2(x / l, y / l);
    } else {
      float *out = a + p.part_off +
                   ((i / N_REP * p.n_kv * N_REP + kvh * N_REP + i % N_REP) * slots +
                    (SHAPED<P> && own ? slot : (own ? p.n_shared : 0) + part)) * PART;
      *(float2 *)(out + 2 + 2 * d) = make_float2(x, y);
      if (d == 0) *(float2 *)out = make_float2(m, l);
    }
  }
}

}  // namespace

#define APPEND(K8, V8)                                                                                 \
  extern "C" __global__ __launch_bounds__(256) void kv_append__##K8##_##V8##_128(                      \
      const float *w, float *a, const uint32_t *ctl, f16 *kv, int8_t *kv8, AppendPush p) {              \
    append_body<K8, V8, 1, 0>(w, a, ctl, kv, kv8, p);                                                   \
  }                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void kv_append_4__##K8##_##V8##_128(                    \
      const float *w, float *a, const uint32_t *ctl, f16 *kv, int8_t *kv8, AppendPush p) {              \
    append_body<K8, V8, 4, 0>(w, a, ctl, kv, kv8, p);                                                   \
  }                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void kv_append_axes__##K8##_##V8##_128(                 \
      const float *w, float *a, const uint32_t *ctl, f16 *kv, int8_t *kv8, AppendAxesPush p) {          \
    append_body<K8, V8, 1, 1>(w, a, ctl, kv, kv8, p.append, p.axes_off, p.n_axes);                      \
  }                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void kv_append_axes_4__##K8##_##V8##_128(               \
      const float *w, float *a, const uint32_t *ctl, f16 *kv, int8_t *kv8, AppendAxesPush p) {          \
    append_body<K8, V8, 4, 1>(w, a, ctl, kv, kv8, p.append, p.axes_off, p.n_axes);                      \
  }
APPEND(0, 0)
APPEND(0, 1)
APPEND(1, 1)

#define PAGED(R, K8, V8)                                                                               \
  extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))                  \
  void attention_paged__##R##_##K8##_##V8##_128(float *a, const uint32_t *ctl, const f16 *kv,           \
                                                const int8_t *kv8, const f16 *kvs, PagedPush p,         \
                                                uint32_t n_grid) {                                      \
    (void)kvs;                                                                                         \
    paged_body<R, K8, V8>(a, ctl, kv, kv8, p, n_grid);                                                 \
  }                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))                  \
  void attention_paged_shaped__##R##_##K8##_##V8##_128(float *a, const uint32_t *ctl, const f16 *kv,    \
                                                       const int8_t *kv8, const f16 *kvs, ShapedPush p, \
                                                       uint32_t n_grid) {                               \
    (void)kvs;                                                                                         \
    paged_body<R, K8, V8>(a, ctl, kv, kv8, p, n_grid);                                                 \
  }                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))                  \
  void attention_paged_shaped_cap__##R##_##K8##_##V8##_128(float *a, const uint32_t *ctl, const f16 *kv, \
                                                           const int8_t *kv8, const f16 *kvs, CappedPush p, \
                                                           uint32_t n_grid) {                           \
    (void)kvs;                                                                                         \
    paged_body<R, K8, V8>(a, ctl, kv, kv8, p, n_grid);                                                 \
  }
#define PAGED_REP(K8, V8) PAGED(1, K8, V8) PAGED(2, K8, V8) PAGED(4, K8, V8) PAGED(8, K8, V8)
PAGED_REP(0, 0)
PAGED_REP(0, 1)
PAGED_REP(1, 1)

// o = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s over a row's live partials, W waves of a
// (head, row), lane t dims 2 t and 2 t + 1, wave w the partials w + W i, the waves' sums added in
// order.  Eight partials of a wave are in flight together.  Measured (MI355X): 128 rows of 32 heads
// and 17 partials 10 us (36 MB, 3.5 TB/s), one row's 32 heads of 64 partials 4.1 us with eight waves a
// head; one row of 256 partials took 79 us with one wave and a load at a time.  Bound by the launch
// and three round trips.
template <uint32_t W, typename P>
SK_DEV void paged_merge(float *a, const uint32_t *ctl, const P &p, uint32_t h, uint32_t row, uint32_t wave,
                        uint32_t lane) {
  uint32_t ns, no, nl = 0;  // live partials: the shared run's, the row's own, its lead's
  uint32_t o0 = p.n_shared, l0 = 0;  // the first of the latter two
  if constexpr (SHAPED<P>) {
    // by the first wave for all of the workgroup's heads (500 vector instructions: by each wave a launch of 100 rows and 12
    // partials took 8.4 us for 7.6, of 128 rows and 10 10.4 for 9.6)
    __shared__ uint32_t of_row[5];
    if (threadIdx.x < 64) {
      const uint32_t shared = shared_end(ctl, p);
      const auto r = range_of(ctl, p, row, shared);
      const uint32_t n_rows = min(ctl[2], gridDim.y);  // the attention's
      const bool together = rows_together(ctl, p.rows_off, row, n_rows, gridDim.y, p.n_seq, 16 / p.rep);
      // the parts of [x.all_lo, x.all_hi) with some of [x.lo, x.hi)
      auto parts_of = [&](bool lead, uint32_t n_parts, uint32_t &at) {
        const OwnRun x = own_run(ctl, p, row, n_rows, 16 / p.rep, together, shared, lead);
        if (x.lo >= x.hi) return 0u;
        const Split sp = split_of(x.all_lo, x.all_hi, n_parts);
        const uint32_t k = min((x.lo - sp.base) / TILE / sp.per, n_parts - 1);
        at += k;
        return min((x.hi - 1 - sp.base) / TILE / sp.per, n_parts - 1) - k + 1;
      };
      ns = r.member ? live_parts(split_of(shared_first(ctl, p, shared), shared, p.n_shared)) : 0;
      no = parts_of(false, p.n_own, o0);
      l0 = p.n_shared + p.n_own;
      if (p.n_lead) nl = parts_of(true, p.n_lead, l0);
      if (lane == 0) of_row[0] = ns, of_row[1] = no, of_row[2] = nl, of_row[3] = o0, of_row[4] = l0;
    }
    __syncthreads();
    ns = of_row[0], no = of_row[1], nl = of_row[2], o0 = of_row[3], l0 = of_row[4];
    if (h >= p.n_head) return;
  } else {
    const uint32_t shared = shared_end(ctl, p);
    const auto r = range_of(ctl, p, row, shared);
    ns = r.member ? live_parts(split_of(0, shared, p.n_shared)) : 0;
    no = live_parts(split_of(r.start, r.len, p.n_own));
  }
  const uint32_t n = ns + no + nl;
  const float *part = a + p.part_off + (row * p.n_head + h) * slots_of(p) * PART;
  // live partial i
  auto at = [&](uint32_t i) {
    if (SHAPED<P> && i >= ns + no) return part + (l0 + i - ns - no) * PART;
    return part + (i < ns ? i : o0 + i - ns) * PART;
  };
  float big = -INFINITY;
  for (uint32_t i = lane; i < n; i += 64) big = fmaxf(big, at(i)[0]);
  big = wave_max(big);
  big = big > -INFINITY ? big : 0.0f;
  float l = 0.0f, ox = 0.0f, oy = 0.0f;
  constexpr uint32_t U = 8;  // partials in flight
  for (uint32_t i0 = wave; i0 < n; i0 += U * W) {
    float2 ml[U], v[U];
#pragma unroll
    for (uint32_t k = 0; k < U; k++) {
      const float *s = at(min(i0 + k * W, n - 1));
      ml[k] = *(const float2 *)s;
      v[k] = *(const float2 *)(s + 2 + 2 * lane);
    }
#pragma unroll
    for (uint32_t k = 0; k < U; k++) {
      const float w = i0 + k * W < n ? __builtin_amdgcn_exp2f(ml[k].x - big) : 0.0f;
      l = __builtin_fmaf(w, ml[k].y, l);
      ox = __builtin_fmaf(w, v[k].x, ox);
      oy = __builtin_fmaf(w, v[k].y, oy);
    }
  }
  if constexpr (W > 1) {
    __shared__ float3 sum[W][64];
    sum[wave][lane] = make_float3(l, ox, oy);
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (uint32_t w = 1; w < W; w++) {
      l += sum[w][lane].x;
      ox += sum[w][lane].y;
      oy += sum[w][lane].z;
    }
  }
  *(float2 *)(a + p.o_off + row * p.o_stride + h * HD + 2 * lane) =
      n ? make_float2(ox / l, oy / l) : make_float2(0.0f, 0.0f);
}
// a wave a head, four heads a workgroup
extern "C" __global__ __launch_bounds__(256) void attention_paged_merge__128(float *a, const uint32_t *ctl,
                                                                             PagedMergePush p) {
  const uint32_t h = blockIdx.x * 4 + (threadIdx.x >> 6), row = blockIdx.y;
  if (row < ctl[2] && h < p.n_head) paged_merge<1>(a, ctl, p, h, row, 0, threadIdx.x & 63);
}
// eight waves a head
extern "C" __global__ __launch_bounds__(512) void attention_paged_merge_8__128(float *a, const uint32_t *ctl,
                                                                               PagedMergePush p) {
  const uint32_t h = blockIdx.x, row = blockIdx.y;
  if (row < ctl[2]) paged_merge<8>(a, ctl, p, h, row, threadIdx.x >> 6, threadIdx.x & 63);
}
// and of attention_paged_shaped's partials
extern "C" __global__ __launch_bounds__(256) void attention_paged_shaped_merge__128(float *a, const uint32_t *ctl,
                                                                                    ShapedMergePush p) {
  const uint32_t h = blockIdx.x * 4 + (threadIdx.x >> 6), row = blockIdx.y;
  if (row < ctl[2]) paged_merge<1>(a, ctl, p, h, row, 0, threadIdx.x & 63);
}
extern "C" __global__ __launch_bounds__(512) void attention_paged_shaped_merge_8__128(float *a, const uint32_t *ctl,
                                                                                      ShapedMergePush p) {
  const uint32_t h = blockIdx.x, row = blockIdx.y;
  if (row < ctl[2]) paged_merge<8>(a, ctl, p, h, row, threadIdx.x >> 6, threadIdx.x & 63);
}

// logits_adjust: y = adjust(x) for every token of a row's vocabulary.  Row r has eight words at
// ctrl_off + 8 r: {history length, prompt length, biases, mask (0: none), repetition, frequency,
// presence, 0} (the last three floats); its history is token ids, the prompt's first, its biases
// pairs (id, f32), its mask one bit a token (1: allowed).  With c the token's count past the prompt:
//   in the history   x / repetition where x > 0, x repetition elsewhere
//   c > 0            - (frequency c + presence)
//   biased           + the last bias of its id
//   not allowed      -inf
// Ids past the vocabulary count for nothing.  Lengths are cut to the strides.
//
// A workgroup of T threads takes 16 T tokens of a row: it loads its logits and mask words, counts the
// history's tokens among them in LDS (integer counts, so any order gives the same), and writes the
// row's part once.  Its biases come last, each by the thread whose entry is the last of its id.
// Measured (MI355X), a vocabulary of 151936, half of the rows masked, from the 256 MB cache, where an
// output head leaves logits / where it holds other data: 128 rows of histories to 32768 44 / 75 us (169
// MB; 50 with T = 256, whose 38 workgroups a row each read the history, and 215 with a load of it at a
// time and two counts a token), of 100 27 / 46, 48 rows of 4096 14.5 / 28, 1 row of 1000 5.2 / 9.5.  Long
// histories are bound by their counting; short ones by round trips: the branches for a row's end put
// a wait behind the first of a thread's four logits loads and, in masked rows, behind each mask word.
// Non-temporal stores save 1 to 2 us of a launch of many rows.
template <uint32_t T>
SK_DEV void logits_body(float *a, const uint32_t *ctl, const LogitsPush &p) {
#pragma clang fp contract(off)
  constexpr uint32_t VT = 16 * T;
  __shared__ uint32_t count[VT];  // uses past the prompt; bit 31: in the prompt
  const uint32_t row = blockIdx.y, t = threadIdx.x, base = blockIdx.x * VT, n = min(VT, p.n_vocab - base);
  if (row >= ctl[2]) return;
  const uint32_t *c = ctl + p.ctrl_off + 8 * row;
  const float rho = __builtin_bit_cast(float, c[4]), freq = __builtin_bit_cast(float, c[5]),
              pres = __builtin_bit_cast(float, c[6]);
  const uint32_t n_hist = rho != 1.0f || freq != 0.0f || pres != 0.0f ? min(c[0], p.hist_stride) : 0;
  const uint32_t n_prompt = c[1], n_bias = min(c[2], p.bias_stride / 2);
  const uint32_t *hist = ctl + p.hist_off + row * p.hist_stride, *bias = ctl + p.bias_off + row * p.bias_stride;
  const uint32_t *mask = ctl + p.mask_off + row * p.mask_stride;
  const bool masked = c[3] != 0 && p.mask_stride != 0;
  const float *x = a + p.x_off + row * p.x_stride + base;
  float *y = a + p.y_off + row * p.y_stride + base;
  // tokens 4 (t + T k) + [0, 4): offset and stride are multiples of 4, so a last float4 that
  // passes n stays in its row's stride or is read one by one
  float4 v[4];
  uint32_t bits[4];
#pragma unroll
  for (uint32_t k = 0; k < 4; k++) {
    const uint32_t i = 4 * (t + T * k);
    v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    bits[k] = 15;
    if (i + 4 <= n) {
      v[k] = *(const float4 *)(x + i);
    } else if (i < n) {
      v[k].x = x[i];
      if (i + 1 < n) v[k].y = x[i + 1];
      if (i + 2 < n) v[k].z = x[i + 2];
    }
    if (masked && i < n) bits[k] = (mask[(base + i) / 32] >> ((base + i) & 31)) & 15;
  }
  if (n_hist) {
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) *(uint4 *)&count[4 * (t + T * k)] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto use = [&](uint32_t i, uint32_t id) {
      id -= base;
      if (id < n) {
        if (i < n_prompt)
          atomicOr(&count[id], 0x80000000u);
        else
          atomicAdd(&count[id], 1u);
      }
    };
    const uint32_t whole = n_hist & ~3u;
    constexpr uint32_t U = 4;  // loads in flight
    for (uint32_t i0 = 4 * t; i0 < whole; i0 += 4 * T * U) {
      uint4 h[U];
#pragma unroll
      for (uint32_t k = 0; k < U; k++) h[k] = *(const uint4 *)(hist + min(i0 + 4 * T * k, whole - 4));
#pragma unroll
      for (uint32_t k = 0; k < U; k++) {
        const uint32_t i = i0 + 4 * T * k;
        if (i < whole) {
          use(i, h[k].x);
          use(i + 1, h[k].y);
          use(i + 2, h[k].z);
          use(i + 3, h[k].w);
        }
      }
    }
    if (whole + t < n_hist) use(whole + t, hist[whole + t]);
    __syncthreads();
  }
#pragma unroll
  for (uint32_t k = 0; k < 4; k++) {
    const uint32_t i = 4 * (t + T * k);
    const uint4 u = n_hist ? *(const uint4 *)&count[i] : make_uint4(0, 0, 0, 0);
    float w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
    const uint32_t uses[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t made = uses[j] & 0x7fffffffu;
      if (uses[j]) w[j] = w[j] > 0.0f ? w[j] / rho : w[j] * rho;
      if (made) w[j] -= freq * (float)made + pres;
      if (!((bits[k] >> j) & 1)) w[j] = -INFINITY;
    }
    if (i + 4 <= n) {
      __builtin_nontemporal_store(f32x4{w[0], w[1], w[2], w[3]}, (f32x4 *)(y + i));
    } else if (i < n) {
      y[i] = w[0];
      if (i + 1 < n) y[i + 1] = w[1];
      if (i + 2 < n) y[i + 2] = w[2];
    }
  }
  if (n_bias == 0) return;
  // the counts are read: their words now hold 1 + the place of a token's last bias
  __syncthreads();
  for (uint32_t i = t; i < n_bias; i += T) {
    const uint32_t id = bias[2 * i] - base;
    if (id < n) count[id] = 0;
  }
  __syncthreads();
  for (uint32_t i = t; i < n_bias; i += T) {
    const uint32_t id = bias[2 * i] - base;
    if (id < n) atomicMax(&count[id], i + 1);
  }
  __syncthreads();  // and this workgroup's y is written
  for (uint32_t i = t; i < n_bias; i += T) {
    const uint32_t at = bias[2 * i], id = at - base;
    if (id < n && count[id] == i + 1 && (!masked || ((mask[at / 32] >> (at & 31)) & 1)))
      y[id] += __builtin_bit_cast(float, bias[2 * i + 1]);
  }
}
#define LOGITS(T)                                                                                        \
  extern "C" __global__ __launch_bounds__(T) void logits_adjust_##T(float *a, const uint32_t *ctl, LogitsPush p) { \
    logits_body<T>(a, ctl, p);                                                                           \
  }
LOGITS(256)
LOGITS(1024)
