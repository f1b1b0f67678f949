// A token of each row of logits, gfx950: temperature, top-k, min-p and top-p, from a given random number.
//
// Contract (bindings, push words; both grids are [1, rows, 1], and the runtime chooses the launch):
//   logits_sample       [A, C]  5 words   the rows' histograms
//   logits_sample_draw  [A, C]  6 words   their tokens, behind a barrier
// Row r < ctl[2] (the others are left as they were) has eight words at ctrl_off + 8 r: {temperature T,
// top_p, min_p (floats), top_k, draw, 0, 0, 0}, and gets four at out_off + 4 r: {token, kept, logprob, 0}.
// Its tokens are ordered by their logits, the largest first, equal ones by their ids.  With weights
// w = exp((x - max) / T) and C(n) the sum of the first n:
//   n1  the tokens whose w >= min_p (0: all), at most top_k of them (0: all), at least one
//   n2  the first n with C(n) >= top_p C(n1) (n1 where top_p is 1 or more)
//   the token is the first with C(n) > (draw + 1/2) 2^-32 C(n2); kept = n2, logprob = ln(w / C(n2))
// T = 0 (or below 0, or no number) takes the first of the order.  Logits of -inf or NaN have no weight and
// no place; +inf counts as the type's largest value.  A row without tokens gets {~0, 0, -inf, 0}.
//
// Sums decide which token it is, so they are held to more than 32 bits: a row's tokens fall into bins of
// t = x 8 log2(e) / T, one rint(t) each, in which a weight is 2^((t - rint(t)) / 8) of its bin's middle's.
// A bin's count and sum of weights are integers (36 bits after the point: a weight is off by 8e-12 of itself at
// most), the same in any order, and only the tokens of the bins in which a border lies (min_p's or top_k's,
// top_p's, the draw's) are looked at one by one.  The last bin holds whatever is 44 temperatures or more below the
// largest: there a weight is off by 2^-37 of the bin's middle's, and again where a chunk's bin is taken into the row's,
// and is nothing from 26 temperatures further down.  All of them are less than 2^-43 of a row, which no top_p below 1
// (2^-24) and no draw (2^-33) tells from the whole; min_p's border goes by t and top_k's by the count.
// No order of a whole row is ever made: a row is read once, by many workgroups, and a draw reads an eighth of that (of
// 152k tokens 78 KB of bins) and what lies around the borders: up to 8192 tokens, which it takes into LDS, of more the
// sums of 1024 buckets and the tokens of the buckets with a border.  Only borders in the last bin, or in a bucket of
// more than 512 tokens (equal logits), cost passes over the row, five for each border.
//
// Measured (MI355X, 151936 tokens, both kernels): 1 row 6.0 + 10.6 us, 16 rows at their temperature alone 9.5 to 11 +
// 15, 48 masked rows 15.7 + 10.6, 128 rows of wide nuclei 30.4 + 23.  A replay of two empty launches takes 14.7.
// Logits of N(0, 2.5^2) at temperature 0.7 / 2 / 5 with top_p 0.95, 1 row 34 / 38 / 39 us on the device, 128 rows 60 /
// 95 / 114; top_k 50000 and top_p 0.9 at 5 80 and 143.
// Low temperatures cost more.  Tokens 44 to 70 temperatures below their chunk's largest are weighed one by one into one
// bin: at 0.3 / 0.2 / 0.1 / 0.05 / 0.02 logits_sample takes 25 / 41 / 27 / 17 / 14 us for 1 row, 74 / 195 / 112 / 70 / 57
// for 128.  And where a top_k's last token lies 44 temperatures down, the search for it takes the draw from 17 to 380
// us (top_k 50: 1 row at 0.05, the slowest of 128 at 0.1).
#include "common.h"

namespace {

struct SamplePush {
  uint32_t x_off, x_stride, n_vocab, ctrl_off, part_off;
};
struct DrawPush {
  uint32_t x_off, x_stride, n_vocab, ctrl_off, part_off, out_off;
};

constexpr uint32_t THREADS = 512, EACH = 16, CHUNK = THREADS * EACH;  // tokens of a workgroup of logits_sample
constexpr uint32_t BINS = 512;  // from a chunk's (a row's) largest value down; the last holds all below it, too
// a chunk's part: {rint(t) of its largest value (f64), that value, how many there are, 0, 0, 0, 0}, its bins, and
// its tokens in the bins' order (16 bits each, from the chunk's first)
constexpr uint32_t HEAD = 8, PART = HEAD + 2 * BINS + CHUNK / 2;
// a bin's word: its weights' sum times 2^36, and from this bit on how many tokens end with it
constexpr int COUNT_AT = 50;
constexpr uint64_t SUM = (1ull << COUNT_AT) - 1;

// What both kernels take a logit for, to the same bits.
SK_DEV bool has_weight(float x) { return x > -INFINITY; }  // (not NaN)
SK_DEV double scale_of(float T) { return 11.541560327111707 / (T > 0.0f ? (double)T : 1.0); }  // 8 log2(e) / T
SK_DEV float finite(float x) { return fminf(x, 3.402823466e38f); }  // of one with a weight
SK_DEV double scaled(float x, double c) { return (double)finite(x) * c; }
SK_DEV uint32_t saturated(double x) {  // (as the instruction converts: past the largest the largest, NaN 0)
  uint32_t y;
  asm("v_cvt_i32_f64 %0, %1" : "=v"(y) : "v"(x));
  return y;
}
// 2^(f / 8) for |f| <= 1/2 in units of 2^-36, as the low bits of the double behind 2^52: 1 + the polynomial of degree 5
// nearest to the rest (4e-13 of it at most).  The constants are scalar registers: known as constants they would be moved
// into vector ones for each use.
struct Series {
  double a, b, c, d, e, one;
};
SK_DEV Series series() {
  Series k{4.0687475846311098e-8 * 0x1p36, 2.3483805669065314e-6 * 0x1p36, 1.0840646378828406e-4 * 0x1p36,
           3.7535391554191859e-3 * 0x1p36, 8.6643397569895267e-2 * 0x1p36, 0x1p36 + 0x1p52};
  asm("" : "+s"(k.a), "+s"(k.b), "+s"(k.c), "+s"(k.d), "+s"(k.e), "+s"(k.one));
  return k;
}
SK_DEV uint64_t fixed_weight(const Series &k, double f) {
  double y = __builtin_fma(k.a, f, k.b);
  y = __builtin_fma(y, f, k.c);
  y = __builtin_fma(y, f, k.d);
  y = __builtin_fma(y, f, k.e);
  y = __builtin_fma(y, f, k.one);
  return __builtin_bit_cast(uint64_t, y) - 0x4330000000000000ull;
}
// what a token adds to the last bin from d bins below the first, below that one's lower edge
SK_DEV uint64_t far_weight(const Series &k, double f, double d) {
  return (uint64_t)__builtin_rint((double)fixed_weight(k, f) * exp2(((double)(BINS - 1) - d) * 0.125));
}
SK_DEV uint64_t fixed_weight_at(const Series &k, double t, double d) {
#pragma clang fp contract(off)
  const double f = t - __builtin_rint(t);
  return d < BINS ? fixed_weight(k, f) : far_weight(k, f, d);
}
// a place in the order: the smaller, the earlier (-0 and 0 are equal)
SK_DEV uint64_t place(float x, uint32_t id) {
  const uint32_t u = __builtin_bit_cast(uint32_t, fminf(x, 3.402823466e38f) + 0.0f);
  return (uint64_t)(u & 0x80000000u ? u : ~u & 0x7fffffffu) << 32 | id;
}
SK_DEV float value_at(uint64_t place) {
  const uint32_t u = (uint32_t)(place >> 32);
  return __builtin_bit_cast(float, u & 0x80000000u ? u : ~u & 0x7fffffffu);
}

// Sums over the lanes up to each (inclusive) and the largest of all, by moves between lanes: 1, 2, 4 and 8 lanes up
// within a row of 16, then a row's last lane into the rows above it.
template <int CTRL, int ROWS>
SK_DEV uint32_t moved(uint32_t v, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf, typename T>
SK_DEV T moved_or_0(T v) {
  if constexpr (sizeof(T) == 8) {
    const uint2 u = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(T, make_uint2(moved<CTRL, ROWS>(u.x, 0), moved<CTRL, ROWS>(u.y, 0)));
  } else {
    return __builtin_bit_cast(T, moved<CTRL, ROWS>(__builtin_bit_cast(uint32_t, v), 0));
  }
}
template <typename T>
SK_DEV T wave_scan(T v) {
  v += moved_or_0<0x111>(v);
  v += moved_or_0<0x112>(v);
  v += moved_or_0<0x114>(v);
  v += moved_or_0<0x118>(v);
  v += moved_or_0<0x142, 0xa>(v);
  v += moved_or_0<0x143, 0xc>(v);
  return v;
}
template <int CTRL, int ROWS = 0xf>
SK_DEV float larger(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  return fmaxf(v, __builtin_bit_cast(float, moved<CTRL, ROWS>(u, u)));
}
SK_DEV float wave_max(float v) {
  v = larger<0x118>(larger<0x114>(larger<0x112>(larger<0x111>(v))));
  v = larger<0x143, 0xc>(larger<0x142, 0xa>(v));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

}  // namespace

// A workgroup's CHUNK tokens of a row: their bins below its own largest value, and the tokens in the bins' order.
// 128 rows of 151936 tokens (78 MB read, 47 written) take 30.4 us: 38 vector instructions a token, half the cycles'
// issue (41, with clamps of every logit, took 32; with moves of the series' constants 42), and the atomics' and lists'
// LDS banks (8 us) beside them; 2 fewer, the far tokens told by wave, changed nothing.  Chunks of 16384 (1024 threads, 61
// registers) took 85 us for 78 then, 8 or 16 tokens on their way at once 83 and 79, a workgroup that goes on to a second
// chunk with its loads ahead 101 (171 registers).
extern "C" __global__ __launch_bounds__(THREADS) void logits_sample(float *a, const uint32_t *ctl, SamplePush p) {
#pragma clang fp contract(off)
  constexpr uint32_t WAVES = THREADS / 64;
  __shared__ unsigned long long bin[BINS + 64];  // and a lane's own for what is in none
  __shared__ uint32_t start[BINS];
  __shared__ __attribute__((aligned(16))) uint16_t ids[CHUNK];
  __shared__ float big[WAVES];
  __shared__ uint32_t counts[WAVES];
  const uint32_t row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const uint32_t base = blockIdx.x * CHUNK, n = min(CHUNK, p.n_vocab - base);
  const float *x = a + p.x_off + (size_t)row * p.x_stride + base;
  float *part = a + p.part_off + ((size_t)row * gridDim.x + blockIdx.x) * PART;
  f32x4 v[EACH / 4];
#pragma unroll
  for (uint32_t k = 0; k < EACH / 4; k++) {  // tokens 4 (t + THREADS k) + [0, 4); on their way before anything is known
    const uint32_t i = 4 * (t + THREADS * k);
    v[k] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (i + 4 <= n) {
      v[k] = *(const f32x4 *)(x + i);
    } else if (i < n) {
      v[k][0] = x[i];
      if (i + 1 < n) v[k][1] = x[i + 1];
      if (i + 2 < n) v[k][2] = x[i + 2];
    }
  }
  if (row >= ctl[2]) return;
  const double c = scale_of(__builtin_bit_cast(float, ctl[p.ctrl_off + 8 * row]));
  float top = -INFINITY;
#pragma unroll
  for (uint32_t k = 0; k < EACH / 4; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) top = fmaxf(top, v[k][e]);  // (leaves NaN aside)
  top = wave_max(top);
  if (lane == 0) big[wave] = top;
  if (t < BINS) bin[t] = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < WAVES; w++) top = fmaxf(top, big[w]);
  const double first = __builtin_rint(scaled(top, c));
  if (!has_weight(top)) {  // nothing here, and nothing more is read
    if (t == 0) {
      *(double *)part = -INFINITY;
      part[2] = top;
      ((uint32_t *)part)[3] = 0;
    }
    return;
  }
  if (top == INFINITY) {  // (+inf alone: a minimum would make a number of NaN)
#pragma unroll
    for (uint32_t i = 0; i < EACH; i++)
      if (v[i / 4][i % 4] == INFINITY) v[i / 4][i % 4] = 3.402823466e38f;
  }
  const Series series_ = series();
  uint32_t at[EACH];  // a token's bin (BINS and above: none), and its place among those of the bin
  uint32_t far = 0;   // one bit each: below the last bin, as most of a row are where T is low
  constexpr uint32_t U = 4;
#pragma unroll
  for (uint32_t i0 = 0; i0 < EACH; i0 += U) {  // (without branches, so that U are under way at once)
    uint64_t word[U];
    uint32_t b[U];
#pragma unroll
    for (uint32_t j = 0; j < U; j++) {
      const float y = v[(i0 + j) / 4][(i0 + j) % 4];
      const double s = (double)y * c, g = __builtin_rint(s);
      word[j] = fixed_weight(series_, s - g) + (1ull << COUNT_AT);
      b[j] = saturated(first - g);
      far |= has_weight(y) && b[j] >= BINS ? 1u << (i0 + j) : 0;
      b[j] = has_weight(y) && b[j] < BINS ? b[j] : BINS + lane;
    }
#pragma unroll
    for (uint32_t j = 0; j < U; j++) word[j] = atomicAdd(&bin[b[j]], (unsigned long long)word[j]);
#pragma unroll
    for (uint32_t j = 0; j < U; j++) at[i0 + j] = b[j] | (uint32_t)(word[j] >> COUNT_AT) << 16;
  }
  if (__any(far != 0)) {
#pragma unroll
    for (uint32_t i = 0; i < EACH; i++) {
      const uint64_t m = __ballot(far >> i & 1);
      if (!m) continue;
      uint64_t before = 0;
      if (lane == 0) before = atomicAdd(&bin[BINS - 1], (unsigned long long)__builtin_popcountll(m) << COUNT_AT);
      const uint32_t rank = __builtin_amdgcn_readfirstlane((uint32_t)(before >> COUNT_AT)) +
                            __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
      if (far >> i & 1) at[i] = (BINS - 1) | rank << 16;
    }
    for (; far; far &= far - 1) {  // (read again: the registers are used)
      const uint32_t i = (uint32_t)__builtin_ctz(far);
      const double s = scaled(x[4 * (t + THREADS * (i / 4)) + i % 4], c), g = __builtin_rint(s);
      // what is 2^-37 of the last bin's middle's or less adds nothing
      if (first - g < BINS + 8 * 37)
        atomicAdd(&bin[BINS - 1], (unsigned long long)far_weight(series_, s - g, first - g));
    }
  }
  __syncthreads();
  const uint64_t mine = t < BINS ? bin[t] : 0;
  const uint32_t count = (uint32_t)(mine >> COUNT_AT);
  uint32_t end = wave_scan(count);
  if (lane == 63) counts[wave] = end;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (uint32_t w = 0; w < WAVES; w++) {
    if (w < wave) end += counts[w];
    all += counts[w];
  }
  if (t < BINS) {
    start[t] = end - count;
    ((uint64_t *)(part + HEAD))[t] = (mine & SUM) | (uint64_t)end << COUNT_AT;
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < EACH; i++)
    if ((at[i] & 0xffff) < BINS) ids[start[at[i] & 0xffff] + (at[i] >> 16)] = 4 * (t + THREADS * (i / 4)) + i % 4;
  __syncthreads();
  uint4 *list = (uint4 *)(part + HEAD + 2 * BINS);
  for (uint32_t i = t; 8 * i < all; i += THREADS) list[i] = ((const uint4 *)ids)[i];
  if (t == 0) {
    *(double *)part = first;
    part[2] = top;
    ((uint32_t *)part)[3] = all;
  }
}

namespace {

constexpr uint32_t DRAW = 1024, DRAW_WAVES = DRAW / 64;
constexpr uint32_t MOST = 8192;    // values of the bins with borders that are taken into LDS
constexpr uint32_t RANKED = 512;   // and of one bucket of these that are put in order
constexpr uint32_t SPANS = 64;     // such bins
constexpr uint32_t CHUNKS = 128;   // of a row
constexpr uint32_t RUNS = 512;     // 3 * CHUNKS and more, a power of two
constexpr uint32_t ID_BITS = 20;   // of a token's id
constexpr uint32_t DIGITS = 2048;  // buckets of the search that takes any number of them

// Where a row's borders lie: of bin b1 some tokens stay (BINS: all of all bins), as min_p has it if that is bm, as
// top_k if bk; n2 ends in bins [p_lo, p_hi] and the draw falls into [d_lo, d_hi].
struct Borders {
  double least;  // min_p's t
  uint32_t k, bm, bk, b1, p_lo, p_hi, d_lo, d_hi;
};
// The tokens of up to three runs of bins, as the chunks list them: run w of chunk i is run w n_chunks + i of all.  Bin f
// of them, f0 and on, f1 and on (~0: none) and f2, is span 0 and on, span1 and on, span2, each of `per` buckets.
struct Lists {
  uint32_t f0, f1, f2, span1, span2, per, n_chunks, half, n;
};
struct DrawShared {
  union {
    // few: as they came, then those of one bucket in order and behind them C there; by buckets.  More: those of one
    // bucket in order, C there; as they came, and how many end with a bucket.
    uint64_t place[2][MOST];
    struct {
      unsigned long long sum[DIGITS];
      uint32_t count[DIGITS];
    } digit;
    uint16_t ends[CHUNKS][BINS];  // of a chunk's tokens, those that end with a bin
  };
  union {
    uint64_t half_sum[BINS];
    uint32_t next[DRAW];  // a bucket's next free place, or how many it has
  };
  uint32_t half_n[BINS];
  float largest[CHUNKS];
  uint32_t down[CHUNKS];  // how many bins below the row's a chunk's lie (BINS: that or more; ~0: it has none)
  double c[BINS + 1];     // C before a bin, in weights of the first bin's middle
  uint32_t n[BINS + 1];   // tokens before it
  double edge[BINS];      // its middle's weight
  unsigned long long bucket[DRAW];  // a word like a bin's
  double first[CHUNKS];   // the chunks' rint(t) of their largest values
  double sums[DRAW_WAVES];
  uint64_t words[DRAW_WAVES];
  uint32_t counts[DRAW_WAVES];
  unsigned long long below;
  Borders at;
  uint2 runs[RUNS];       // of a chunk's list the tokens in a run of bins: where from, less their place here; their end
  Lists lists;
  uint32_t fits, fill, found[2];
};

// What lies `bytes` past an address that is the same for all lanes: an offset of 32 bits a lane is one register and no
// sum (a draw is bound by what one compute unit issues).
template <typename T>
SK_DEV T past(const void *base, uint32_t bytes) {
  return *(const T *)((const char *)base + bytes);
}
template <uint32_t U>
struct Count {
  static constexpr uint32_t value = U;
};
// A row as its kernel sees it.
struct Row {
  const float *x;
  uint32_t n_vocab;
  double c, edge;  // t = x c; rint(t) of the largest value
};
SK_DEV uint32_t bin_of(const Row &r, double t) {
  const double d = r.edge - __builtin_rint(t);
  return d < BINS - 1 ? (uint32_t)(int)d : BINS - 1;
}
SK_DEV uint64_t fixed_weight(const Series &k, const Row &r, double t) {
  return fixed_weight_at(k, t, r.edge - __builtin_rint(t));
}
// a sum of a bin's weights
SK_DEV double sum_of(uint64_t fixed, double edge) { return (double)fixed * 0x1p-36 * edge; }
// 2^(1/16), 2^(-1/16): a weight's bounds in its bin's middle's
constexpr double UP = 1.0442737824274138, DOWN = 0.9576032806985737;

// Every value of the row that may lie in [least, most) by its t, among them all that do: f(place, t).
template <typename F>
SK_DEV void each_value(const Row &r, double least, double most, F f) {
  // in f32, with room for both roundings (without a scale everything is taken)
  const float low = (float)(least / r.c), high = (float)(most / r.c);
  const float from = low - fabsf(low) * 1e-6f, to = high + fabsf(high) * 1e-6f;
  constexpr uint32_t U = 4;
  for (uint32_t i0 = 4 * threadIdx.x; i0 < r.n_vocab; i0 += 4 * DRAW * U) {
    f32x4 v[U];
#pragma unroll
    for (uint32_t k = 0; k < U; k++) {
      const uint32_t i = i0 + 4 * DRAW * k;
      v[k] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (i + 4 <= r.n_vocab) {
        v[k] = *(const f32x4 *)(r.x + i);
      } else if (i < r.n_vocab) {
        v[k][0] = r.x[i];
        if (i + 1 < r.n_vocab) v[k][1] = r.x[i + 1];
        if (i + 2 < r.n_vocab) v[k][2] = r.x[i + 2];
      }
    }
#pragma unroll
    for (uint32_t k = 0; k < U; k++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (has_weight(v[k][e]) && !(v[k][e] < from) && !(v[k][e] > to))
          f(place(v[k][e], i0 + 4 * DRAW * k + e), scaled(v[k][e], r.c));
  }
}
// those of bin b
template <typename F>
SK_DEV void each_value_of(const Row &r, uint32_t b, F f) {
  each_value(r, b < BINS - 1 ? r.edge - (double)b - 0.5 : -INFINITY, b ? r.edge - (double)b + 0.5 : INFINITY,
             [&](uint64_t place, double t) {
    if (bin_of(r, t) == b) f(place, t);
  });
}

// The first bin b whose end satisfies ok(end), BINS if none does; ok is false, then true.  The same in every wave.
template <typename A, typename F>
SK_DEV uint32_t first_bin(const A *before, F ok) {  // (without branches: two of them go on side by side)
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t m = __ballot(ok(before[8 * lane + 8]));
  const uint32_t b = 8 * (uint32_t)__builtin_ctzll(m | 1ull << 63);
  const uint32_t e = b + (uint32_t)__builtin_ctzll(__ballot(lane >= 7 || ok(before[b + lane % 8 + 1])));
  return m ? e : BINS;
}

template <typename T>
SK_DEV T block_scan(T v, T *waves, T &total) {  // inclusive, over DRAW threads; a barrier at its start and one inside
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (uint32_t w = 0; w < DRAW_WAVES; w++) {
    if (w < wave) before += waves[w];
    total += waves[w];
  }
  return before + v;
}

// A token of weight w and value `value` into word b of sums and counts; of a wave that has one value and one word, all
// its tokens at once (equal logits would else wait for one another: 1 row of them 2500 -> 740 us).
SK_DEV void count_in(unsigned long long *sums, uint32_t *counts, uint32_t b, uint32_t value, uint64_t w) {
  const bool other = b != __builtin_amdgcn_readfirstlane(b) || value != __builtin_amdgcn_readfirstlane(value);
  uint32_t n = 1;
  if (!__ballot(other)) {
    const uint64_t all = __ballot(true);
    if ((threadIdx.x & 63) != (uint32_t)__builtin_ctzll(all)) return;
    n = (uint32_t)__builtin_popcountll(all);
  }
  atomicAdd(&sums[b], (unsigned long long)(w * n));
  atomicAdd(&counts[b], n);
}

// A token of the order: its place, how many tokens end with it and their sum.
struct Found {
  uint64_t place;
  uint32_t n;
  double sum;
};
enum Want { kCount, kReach, kPass };  // n >= goal, C >= goal, C > goal
SK_DEV bool meets(Want want, double goal, uint32_t n, double sum) {
  return want == kCount ? (double)n >= goal : want == kReach ? sum >= goal : sum > goal;
}

// The first token that meets `want` (the last of all if rounding leaves none) where the bins hold too many to order
// them, or tokens of any weight (the last bin): the bin, then its places' digits, each by a pass over the row.
__device__ __attribute__((noinline)) Found search(DrawShared &s, const Row r, Want want, double goal) {
  const uint32_t t = threadIdx.x;
  uint32_t b = want == kCount  ? first_bin(s.n, [&](uint32_t n) { return (double)n >= goal; })
               : want == kReach ? first_bin(s.c, [&](double c) { return c >= goal; })
                                : first_bin(s.c, [&](double c) { return c > goal; });
  const uint32_t last = first_bin(s.n, [&](uint32_t n) { return n >= s.n[BINS]; });
  b = min(b, last);
  const double edge = s.edge[b];
  const Series series_ = series();
  Found f{0, s.n[b], s.c[b]};
  constexpr int at[5] = {53, 42, 32, 10, 0}, bits[5] = {11, 11, 10, 22, 10};
  // (ids are below 2^20: 10 bits from bit 10 on, all 22 of them compared as a prefix)
  for (int k = 0; k < 5; k++) {
    __syncthreads();
    for (uint32_t i = t; i < DIGITS; i += DRAW) s.digit.sum[i] = 0, s.digit.count[i] = 0;
    __syncthreads();
    const int above = at[k] + bits[k];
    each_value_of(r, b, [&](uint64_t place, double v) {
      if (above < 64 && place >> above != f.place >> above) return;
      const uint32_t d = (uint32_t)(place >> at[k]) & (DIGITS - 1);
      count_in(s.digit.sum, s.digit.count, d, (uint32_t)(place >> 32), fixed_weight(series_, r, v));
    });
    __syncthreads();
    // two digits a thread
    const uint64_t w0 = s.digit.sum[2 * t], w1 = s.digit.sum[2 * t + 1];
    const uint32_t c0 = s.digit.count[2 * t], c1 = s.digit.count[2 * t + 1];
    uint64_t w_all;
    uint32_t c_all;
    const uint64_t w_end = block_scan(w0 + w1, s.words, w_all);
    const uint32_t c_end = block_scan(c0 + c1, s.counts, c_all);
    if (t == 0) s.found[0] = ~0u, s.found[1] = 0;
    __syncthreads();
    auto sum = [&](uint64_t w) { return f.sum + sum_of(w, edge); };
    if (c0 && meets(want, goal, f.n + c_end - c1, sum(w_end - w1))) atomicMin(&s.found[0], 2 * t);
    if (c1 && meets(want, goal, f.n + c_end, sum(w_end))) atomicMin(&s.found[0], 2 * t + 1);
    if (c0 || c1) atomicMax(&s.found[1], 2 * t + (c1 ? 1 : 0));  // the last digit there is
    __syncthreads();
    const uint32_t d = s.found[0] < DIGITS ? s.found[0] : s.found[1];
    if (2 * t == (d & ~1u)) {
      s.words[0] = w_end - w1 - (d & 1 ? 0 : w0);
      s.counts[0] = c_end - c1 - (d & 1 ? 0 : c0);
      s.words[1] = d & 1 ? w1 : w0;
    }
    __syncthreads();
    f.sum = sum(s.words[0]);
    f.n += s.counts[0];
    f.place |= (uint64_t)d << at[k];
    if (k == 4) f.sum += sum_of(s.words[1], edge), f.n++;
  }
  __syncthreads();
  return f;
}

// The tokens with t >= least, all of them and their sum, least in bin b.
__device__ __attribute__((noinline)) Found search_above(DrawShared &s, const Row r, double least, uint32_t b) {
  uint64_t sum = 0;
  uint32_t n = 0;
  const Series series_ = series();
  each_value_of(r, b, [&](uint64_t, double v) {
    if (v >= least) sum += fixed_weight(series_, r, v), n++;
  });
  uint64_t all;
  uint32_t count;
  block_scan(sum, s.words, all);
  block_scan(n, s.counts, count);
  return {0, s.n[b] + count, s.c[b] + sum_of(all, s.edge[b])};
}

// The first of [0, n) that satisfies ok, n if none does; ok is false, then true.  The same in every wave.
template <typename F>
SK_DEV uint32_t first_of(uint32_t n, F ok) {
  uint32_t lo = 0, hi = n;  // none before lo does, hi does
  while (lo < hi) {
    const uint32_t step = (hi - lo - 1) / 64 + 1, i = lo + (threadIdx.x & 63) * step + step - 1;
    const uint64_t m = __ballot(i >= hi || ok(i));
    if (!m) return hi;
    const uint32_t k = (uint32_t)__builtin_ctzll(m);
    hi = min(hi, lo + k * step + step - 1);
    lo += k * step;
  }
  return hi;
}

SK_DEV uint32_t bucket_of(const Row &r, const Lists &l, double v) {
  const double g = __builtin_rint(v), f = 0.5 - (v - g);
  const uint32_t b = (uint32_t)(int)(r.edge - g);
  const uint32_t i = b >= l.f2 ? l.span2 + b - l.f2 : b >= l.f1 ? l.span1 + b - l.f1 : b - l.f0;
  return min(i * l.per + min((uint32_t)(int)(f * (double)l.per), l.per - 1), DRAW - 1);
}
// The lists' tokens base + t + DRAW u of thread t, all of them on their way at once: f(number, logit, id).
template <uint32_t U, typename F>
SK_DEV void each_listed(const DrawShared &s, const Row &r, const float *parts, const Lists &l, uint32_t base, F f) {
  uint32_t id[U], j[U];
  float x[U];
  auto number = [&](uint32_t u) { return base + threadIdx.x + DRAW * u; };
#pragma unroll
  for (uint32_t u = 0; u < U; u++) j[u] = 0;
  for (uint32_t h = l.half; h; h /= 2)  // the first run that ends behind it
#pragma unroll
    for (uint32_t u = 0; u < U; u++) j[u] += s.runs[j[u] + h - 1].y <= min(number(u), l.n - 1) ? h : 0;
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    const uint32_t i = j[u] < l.n_chunks ? j[u] : j[u] < 2 * l.n_chunks ? j[u] - l.n_chunks : j[u] - 2 * l.n_chunks;
    const uint32_t at = min(s.runs[j[u]].x + min(number(u), l.n - 1), CHUNK - 1);
    id[u] = past<uint16_t>(parts + HEAD + 2 * BINS, min(i, l.n_chunks - 1) * (PART * 4) + 2 * at) + i * CHUNK;
  }
#pragma unroll
  for (uint32_t u = 0; u < U; u++) id[u] = min(id[u], r.n_vocab - 1), x[u] = past<float>(r.x, 4 * id[u]);
#pragma unroll
  for (uint32_t u = 0; u < U; u++) {
    if (number(u) >= l.n) break;
    f(number(u), x[u], id[u]);
  }
}
// More tokens than LDS takes: how many each bucket has and their sums, up to each
__device__ __attribute__((noinline)) void tally(DrawShared &s, const Row r, const float *parts) {
  const Lists l = s.lists;
  const Series series_ = series();
  const uint32_t t = threadIdx.x;
  s.next[t] = 0;
  __syncthreads();
  for (uint32_t base = 0; base < l.n; base += MOST)
    each_listed<MOST / DRAW>(s, r, parts, l, base, [&](uint32_t, float x, uint32_t) {
      const double v = scaled(x, r.c);
      count_in(s.bucket, s.next, bucket_of(r, l, v), __builtin_bit_cast(uint32_t, x), fixed_weight(series_, r, v));
    });
  __syncthreads();
  uint64_t sum;
  uint32_t count;
  s.bucket[t] = block_scan((uint64_t)s.bucket[t], s.words, sum);
  ((uint32_t *)s.place[1])[2 * RANKED + t] = block_scan(s.next[t], s.counts, count);
  __syncthreads();
}
// and the tokens of bucket q, RANKED at most
__device__ __attribute__((noinline)) void collect(DrawShared &s, const Row r, const float *parts, uint32_t q) {
  const Lists l = s.lists;
  __syncthreads();
  if (threadIdx.x == 0) s.fill = 0;
  __syncthreads();
  for (uint32_t base = 0; base < l.n; base += MOST)
    each_listed<MOST / DRAW>(s, r, parts, l, base, [&](uint32_t, float x, uint32_t id) {
      if (bucket_of(r, l, scaled(x, r.c)) != q) return;
      const uint32_t to = atomicAdd(&s.fill, 1u);
      if (to < RANKED) s.place[1][to] = place(x, id);
    });
  __syncthreads();
}

}  // namespace

// A workgroup's row: its chunks' bins added up, the bins with the borders, and the tokens in these.  What it reads of the
// partials reaches no memory outside the row, whatever they hold.
// Of a row of 151936 tokens whose borders' bins hold 6 / 1050 / 6000 tokens (22 / 37 / 50 thousand cycles): the partials'
// heads 2400, their bins 5900, scans 1600, borders 3100 to 3700, the gather 4300 / 12000 / 22000 (two dependent loads a
// token, from memory), buckets and order 150 / 2700 / 4500, the borders among them 4200 / 8900 / 10400.  Bound by chains
// of loads and barriers and by the issue of the one workgroup that a row has.  Against all values put in order, as before
// (27.8 us for 128 rows), ordering the three borders' buckets alone took 26.1, and the gather's values spread evenly over
// the workgroup, not by their chunks, 22; a count of places by waves, or the same loads behind branches, changed
// nothing, and the bins on their way beside the heads, through LDS, cost 1 us.
extern "C" __global__ __launch_bounds__(DRAW) void logits_sample_draw(float *a, const uint32_t *ctl, DrawPush p) {
#pragma clang fp contract(off)
  __shared__ DrawShared s;
  const uint32_t row = blockIdx.y, t = threadIdx.x, n_chunks = (p.n_vocab + CHUNK - 1) / CHUNK;
  if (row >= ctl[2]) return;
  const uint32_t *words = ctl + p.ctrl_off + 8 * row;
  const float T = __builtin_bit_cast(float, words[0]), top_p = __builtin_bit_cast(float, words[1]),
              min_p = __builtin_bit_cast(float, words[2]);
  const float *parts = a + p.part_off + (size_t)row * n_chunks * PART;
  uint32_t *out = (uint32_t *)a + p.out_off + 4 * row;
  Row r{a + p.x_off + (size_t)row * p.x_stride, p.n_vocab, scale_of(T), -INFINITY};
  if (t < CHUNKS) {
    const float *part = parts + (size_t)min(t, n_chunks - 1) * PART;
    s.first[t] = *(const double *)part;
    s.largest[t] = part[2];
  }
  if (t < BINS) s.edge[t] = exp2(-0.125 * (double)t);
  s.bucket[t] = 0;
  if (t == 0) s.below = 0;
  __syncthreads();
  const float top = wave_max(fmaxf(s.largest[t & 63], s.largest[64 + (t & 63)]));
  if (!has_weight(top)) {
    if (t == 0) *(uint4 *)out = make_uint4(~0u, 0, 0xff800000u, 0);
    return;
  }
  const double t_top = scaled(top, r.c);
  r.edge = __builtin_rint(t_top);
  if (t < n_chunks) {
    const double d = r.edge - s.first[t];
    s.down[t] = d < BINS ? (uint32_t)(int)d : d < INFINITY ? BINS : ~0u;
  }
  __syncthreads();

  // the row's bins: thread t has bin t % BINS of every other chunk
  {
    const uint32_t b = t % BINS, first = __builtin_amdgcn_readfirstlane(t / BINS);  // (waves of one chunk each)
    uint32_t n = 0;  // tokens that end with it
    uint64_t sum = 0, below = 0;
    constexpr uint32_t U = 10, STEP = DRAW / BINS;  // chunks whose loads are in flight
    for (uint32_t i0 = first; i0 < n_chunks; i0 += U * STEP) {
      uint64_t w[U], low[U];
      uint32_t downs[U], deep = 0;
#pragma unroll
      for (uint32_t j = 0; j < U; j++) {
        const uint32_t i = min(i0 + j * STEP, n_chunks - 1);
        const void *bins = parts + (size_t)i * PART + HEAD;
        downs[j] = i0 + j * STEP < n_chunks ? __builtin_amdgcn_readfirstlane(s.down[i]) : ~0u;
        w[j] = past<uint64_t>(bins, b >= downs[j] ? 8 * (b - downs[j]) : 0);
        // the chunk's bin b, if it lies in the row's last
        low[j] = downs[j] != ~0u && b + downs[j] >= BINS - 1 ? past<uint64_t>(bins, 8 * b) : 0;
      }
#pragma unroll
      for (uint32_t j = 0; j < U; j++) {
        const uint32_t i = i0 + j * STEP;
        if (b < BINS - 1 && b >= downs[j]) {
          const uint32_t end = (uint32_t)(w[j] >> COUNT_AT);
          n += end;
          sum += w[j] & SUM;
          s.ends[i][b - downs[j]] = end;
        }
        if (b == BINS - 1) n += (uint32_t)(low[j] >> COUNT_AT);  // how many the chunk has
        if (low[j] & SUM) deep |= 1u << j;
      }
      for (; deep; deep &= deep - 1) {  // in weights of the last bin's middle (read again: few rows reach so deep)
        const uint32_t i = i0 + (uint32_t)__builtin_ctz(deep) * STEP;
        const uint64_t low = ((const uint64_t *)(parts + (size_t)i * PART + HEAD))[b];
        const double by = exp2(((double)(BINS - 1) - (double)b - (r.edge - s.first[i])) * 0.125);
        below += (uint64_t)__builtin_rint((double)(low & SUM) * by);
      }
    }
    if (below) atomicAdd(&s.below, (unsigned long long)below);
    if (t >= BINS) s.half_sum[b] = sum, s.half_n[b] = n;
    __syncthreads();
    double c = 0.0, c_all;
    if (t < BINS) {
      s.n[t + 1] = n + s.half_n[t];
      sum += s.half_sum[t];
      c = sum_of(b == BINS - 1 ? s.below : sum, s.edge[b]);
    }
    c = block_scan(c, s.sums, c_all);
    if (t < BINS) s.c[t + 1] = c;
    if (t == 0) s.n[0] = 0, s.c[0] = 0.0;
    __syncthreads();
  }

  // The bins with the borders, by the first wave.  What is known of C(n1) and C(n2) before these are looked at lies
  // between lo and hi.
  const uint32_t total = s.n[BINS];
  const bool by_p = top_p < 1.0f;
  const double share = fmax((double)top_p, 0.0), u = ((double)words[4] + 0.5) * 0x1p-32;
  if (t < 64) {
    const uint32_t k = !(T > 0.0f) || min_p > 1.0f ? 1 : words[3] && words[3] < total ? words[3] : total;
    const double least = min_p > 0.0f ? t_top + 8.0 * log2(fmin((double)min_p, 1.0)) : -INFINITY;
    const uint32_t bm = min_p > 0.0f ? bin_of(r, least) : BINS;
    const uint32_t bk = k < total ? first_bin(s.n, [&](uint32_t n) { return n >= k; }) : BINS;
    const uint32_t b1 = min(bm < BINS && s.n[bm] < total ? bm : BINS, bk);  // (BINS: all tokens stay)
    constexpr double MORE = 1.0 + 1e-9, LESS = 1.0 - 1e-9;
    double lo = s.c[BINS], hi = lo;
    if (b1 < BINS) {
      lo = s.c[b1], hi = s.c[b1 + 1];
      if (b1 == bk) {
        const double more = (double)(k - s.n[bk]) * s.edge[bk];
        hi = fmin(hi, lo + more * UP);
        if (bm != bk && bk < BINS - 1) lo += more * DOWN;
      }
      if (b1 == 0) lo = fmax(lo, DOWN * LESS);  // the largest stays
    }
    // where n1 lies, or past it
    const uint32_t b_last = min(b1, first_bin(s.n, [&](uint32_t n) { return n >= total; }));
    uint32_t p_lo = b_last, p_hi = b_last;  // where n2 lies
    if (by_p) {
      lo *= share * LESS, hi *= share * MORE;
      p_lo = min(first_bin(s.c, [&](double c) { return c >= lo; }), b_last);
      p_hi = min(first_bin(s.c, [&](double c) { return c >= hi; }), b_last);
      hi = fmin(s.c[p_hi + 1], hi + s.edge[p_lo] * UP);
      lo = fmax(lo, DOWN * LESS);
    }
    const uint32_t d_lo = min(first_bin(s.c, [&](double c) { return c > lo * u * LESS; }), p_hi);
    const uint32_t d_hi = min(first_bin(s.c, [&](double c) { return c > hi * u * MORE; }), p_hi);
    if (t == 0) s.at = {least, k, bm, bk, b1, p_lo, p_hi, d_lo, d_hi};
  }
  __syncthreads();
  const double least = s.at.least;
  const uint32_t k = s.at.k, bm = s.at.bm, bk = s.at.bk, b1 = s.at.b1, p_lo = s.at.p_lo, p_hi = s.at.p_hi;
  const uint32_t d_lo = s.at.d_lo, d_hi = s.at.d_hi;
  // up to three runs of bins [f, e], each below the one before (one that is not there: f = ~0)
  uint32_t f0 = d_lo, e0 = d_hi, f1 = ~0u, e1 = 0, f2 = ~0u, e2 = 0;
  if (by_p) {
    if (p_lo <= e0 + 1)
      e0 = max(e0, p_hi);
    else
      f1 = p_lo, e1 = p_hi;
  }
  if (b1 < BINS) {
    if (b1 <= e0 + 1)
      e0 = max(e0, b1);
    else if (f1 != ~0u && b1 <= e1 + 1)
      e1 = max(e1, b1);
    else
      f2 = e2 = b1;
  }
  // the bins and tokens before each run
  uint32_t n_spans = e0 - f0 + 1, n = s.n[e0 + 1] - s.n[f0], deepest = e0, span1 = n_spans, at1 = n, span2 = 0, at2 = 0;
  if (f1 != ~0u) n_spans += e1 - f1 + 1, n += s.n[e1 + 1] - s.n[f1], deepest = e1;
  span2 = n_spans, at2 = n;
  if (f2 != ~0u) n_spans++, n += s.n[e2 + 1] - s.n[f2], deepest = e2;
  n = min(n, r.n_vocab);  // (as it is, of this row's partials)
  Found n2, chosen;
  bool many = n_spans > SPANS || deepest == BINS - 1;
  if (!many) {
    // ---- few: from the chunks' lists into LDS, in buckets by t; more: sums of the buckets, then those with borders
    const bool few = n <= MOST;
    const uint32_t per = DRAW / n_spans;
    const float per_inverse = 1.0f / (float)per;
    const uint32_t runs = 1 + (f1 != ~0u) + (f2 != ~0u);
    const Series series_ = series();
    {
      uint2 run = make_uint2(0, 0);
      const uint32_t i = t % n_chunks, which = t / n_chunks;
      if (which < runs) {
        const uint32_t f = which == 0 ? f0 : which == 1 && f1 != ~0u ? f1 : f2;
        const uint32_t e = which == 0 ? e0 : which == 1 && f1 != ~0u ? e1 : e2, down = s.down[i];
        if (down <= e)
          run = make_uint2(f > down ? s.ends[i][f - down - 1] : 0, min((uint32_t)s.ends[i][e - down], CHUNK));
      }
      uint32_t all;
      const uint32_t end = block_scan(run.y - run.x, s.counts, all);
      if (t < RUNS) s.runs[t] = make_uint2(run.y - end, which < runs ? end : ~0u);
    }
    __syncthreads();
    uint32_t half = 1;
    while (2 * half < n_chunks * runs) half *= 2;
    const Lists lists{f0, f1, f2, span1, span2, per, n_chunks, half, n};
    auto take = [&](uint32_t i, float x, uint32_t id) {
      // (with the bucket above the id: it goes by the value, so that the order is the same)
      const double v = scaled(x, r.c);
      const uint32_t b = n > 64 ? bucket_of(r, lists, v) : 0;
      s.place[0][i] = place(x, id | b << ID_BITS);
      if (n > 64) atomicAdd(&s.bucket[b], (unsigned long long)fixed_weight(series_, r, v) + (1ull << COUNT_AT));
    };
    if (n <= DRAW) {
      each_listed<1>(s, r, parts, lists, 0, take);
    } else if (few) {
      each_listed<MOST / DRAW>(s, r, parts, lists, 0, take);
    } else {
      if (t == 0) s.lists = lists;
      __syncthreads();
      tally(s, r, parts);
    }
    __syncthreads();
    if (n > 64 && few) {
      uint64_t all;
      const uint64_t mine = s.bucket[t], end = block_scan(mine, s.words, all);
      s.bucket[t] = end;
      s.next[t] = (uint32_t)((end - mine) >> COUNT_AT);
      __syncthreads();
      for (uint32_t i = t; i < n; i += DRAW) {
        const uint64_t v = s.place[0][i];
        s.place[1][min(atomicAdd(&s.next[(uint32_t)v >> ID_BITS], 1u), MOST - 1)] = v;
      }
      __syncthreads();
    }
    if (t < 64 || !few) {  // the first wave alone, or every wave the same
      const uint32_t lane = t & 63;
      uint32_t o0 = 0, m = n;  // of the order here, the places whose tokens lie in order
      uint64_t *sorted = s.place[0];
      double *upto = (double *)(s.place[0] + RANKED);
      bool fits = true;
      auto weight_of = [&](uint64_t v) { return fixed_weight(series_, r, scaled(value_at(v), r.c)); };
      auto start_of = [&](uint32_t b) {  // bin b's first place in the order here
        return b >= f2 ? at2 + s.n[b] - s.n[f2] : b >= f1 ? at1 + s.n[b] - s.n[f1] : s.n[b] - s.n[f0];
      };
      auto span_of = [&](uint32_t b) { return b >= f2 ? span2 + b - f2 : b >= f1 ? span1 + b - f1 : b - f0; };
      // with bucket q
      auto count_to = [&](uint32_t q) {
        return few ? (uint32_t)(s.bucket[q] >> COUNT_AT) : ((const uint32_t *)s.place[1])[2 * RANKED + q];
      };
      auto sum_to = [&](uint32_t q) { return few ? s.bucket[q] & SUM : s.bucket[q]; };
      auto sum_before = [&](uint32_t q) { return q ? sum_to(q - 1) : 0; };
      if (n <= 64) {  // all of them
        const uint64_t v = t < n ? s.place[0][t] : ~0ull;
        uint32_t rank = 0;
        for (uint32_t i = 0; i < n; i++) rank += s.place[0][i] < v;
        if (t < n) sorted[rank] = v;
        uint64_t *raw = s.place[1];
        const uint64_t sum = wave_scan(t < n ? weight_of(sorted[t]) : 0);
        if (t < n) raw[t] = sum;
        if (t < n) {
          const uint32_t b = bin_of(r, scaled(value_at(sorted[t]), r.c)), i0 = start_of(b);
          upto[t] = s.c[b] + sum_of(sum - (i0 ? raw[i0 - 1] : 0), s.edge[b]);
        }
      } else {
        m = 0;
      }
      auto order = [&](uint32_t q) {  // bucket q's
        const uint32_t i0 = q ? count_to(q - 1) : 0, size = count_to(q) - i0;
        if (m && i0 == o0) return;
        fits = fits && size <= RANKED;  // (if not, nothing found from here on is used)
        o0 = i0, m = size <= RANKED ? size : 0;
        if (!few && m) collect(s, r, parts, q);
        const uint64_t *of = s.place[1] + (few ? o0 : 0);
        for (uint32_t j = lane; j < m; j += 64) {
          const uint64_t v = of[j];
          uint32_t rank = 0;
#pragma unroll 4
          for (uint32_t i = 0; i < m; i++) rank += of[i] < v;
          sorted[rank] = v;
        }
        const uint32_t span = q / per;
        const uint32_t b = span >= span2 ? f2 + span - span2 : span >= span1 ? f1 + span - span1 : f0 + span;
        uint64_t before = sum_before(q) - sum_before(span * per);
        for (uint32_t j0 = 0; j0 < m; j0 += 64) {
          const uint32_t j = j0 + lane;
          const uint64_t sum = before + wave_scan(j < m ? weight_of(sorted[j]) : 0);
          if (j < m) upto[j] = s.c[b] + sum_of(sum, s.edge[b]);
          before = __shfl(sum, 63);
        }
      };
      // the bucket with place i
      auto order_at = [&](uint32_t i) {
        if (n > 64) order(min(first_of(DRAW, [&](uint32_t q) { return count_to(q) > i; }), DRAW - 1));
      };
      // the token at place i of the order here (within a run of bins places and ranks go together), if it lies in order
      auto found_at = [&](uint32_t i) {
        const uint32_t rank = i >= at2 && f2 != ~0u   ? s.n[f2] + i - at2
                              : i >= at1 && f1 != ~0u ? s.n[f1] + i - at1
                                                      : s.n[f0] + i;
        const uint32_t j = min(i - o0, RANKED - 1);
        return Found{sorted[j], rank + 1, upto[j]};
      };
      // n1: of bin b1 those that stay
      Found n1{0, total, s.c[BINS]};
      if (b1 < BINS) {
        const uint32_t i0 = start_of(b1);
        uint32_t some = s.n[b1 + 1] - s.n[b1];
        if (b1 == bk) some = k - s.n[b1];
        if (b1 == bm) {  // (what lies in the buckets before `least`'s is larger, in those behind it smaller)
          if (n > 64) order(bucket_of(r, lists, least));
          const uint32_t at = max(o0, i0) - i0;
          some = min(some, at + first_of(o0 + m - max(o0, i0), [&](uint32_t i) {
            return scaled(value_at(sorted[i + max(o0, i0) - o0]), r.c) < least;
          }));
        }
        if (some) order_at(i0 + some - 1);
        n1 = some ? found_at(i0 + some - 1) : Found{0, s.n[b1], s.c[b1]};
      }
      // the first token of bins [f, e], not past the n-th, that meets `want`; the last of these if none does
      auto first = [&](Want want, double goal, uint32_t most, uint32_t f, uint32_t e) {
        const uint32_t i0 = start_of(f), i1 = min(i0 + max(min(s.n[e + 1], most), s.n[f] + 1) - s.n[f], n);
        auto ok = [&](double c) { return want == kReach ? c >= goal : c > goal; };
        if (n > 64) {
          const uint32_t q0 = span_of(f) * per, n_q = (span_of(e) + 1) * per - q0;
          const uint32_t q = q0 + first_of(n_q, [&](uint32_t i) {
            const uint32_t k = (uint32_t)(((float)i + 0.5f) * per_inverse);  // i / per
            return ok(s.c[f + k] + sum_of(sum_to(q0 + i) - sum_before(q0 + k * per), s.edge[f + k]));
          });
          const uint32_t i = q ? count_to(q - 1) : 0;
          if (q < q0 + n_q && i < i1 && i < count_to(q))
            order(q);
          else
            order_at(min(i, i1 - 1));
        }
        const uint32_t from = max(i0, o0), to = min(i1, o0 + m);
        const uint32_t i = from + first_of(to - from, [&](uint32_t i) { return ok(upto[from + i - o0]); });
        return found_at(min(i, to - 1));
      };
      n2 = by_p ? first(kReach, share * n1.sum, n1.n, p_lo, p_hi) : n1;
      chosen = first(kPass, u * n2.sum, n2.n, d_lo, d_hi);
      if (t == 0) s.fits = fits;
    }
    __syncthreads();
    many = !s.fits;
  }
  if (many) {
    Found n1{0, total, s.c[BINS]};
    if (b1 < BINS && b1 == bm) n1 = search_above(s, r, least, bm);
    if (b1 < BINS && b1 == bk) {
      const Found by_k = search(s, r, kCount, (double)k);
      if (by_k.n < n1.n) n1 = by_k;
    }
    n2 = n1;
    if (by_p) {
      const Found f = search(s, r, kReach, share * n1.sum);
      if (f.n < n1.n) n2 = f;
    }
    chosen = search(s, r, kPass, u * n2.sum);
    if (chosen.n > n2.n) chosen = search(s, r, kCount, (double)n2.n);
  }
  if (t == 0) {
    const double y = (scaled(value_at(chosen.place), r.c) - r.edge) * 0.125 * 0.69314718055994530942 - log(n2.sum);
    const uint32_t id = (uint32_t)chosen.place & ((1u << ID_BITS) - 1);
    *(uint4 *)out = make_uint4(id, n2.n, __builtin_bit_cast(uint32_t, n2.n == 1 ? 0.0f : (float)y), 0);
  }
}
