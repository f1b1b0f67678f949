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
// t = x 8 log2(e) / T, one floor(t) each, in which a weight is 2^((t - floor(t) - 1) / 8) of its bin's upper
// edge's.  A bin's count and sum of weights are integers (36 bits after the point: a weight is off by 7e-12
// of itself at most), the same in any order, and only the tokens of the bins in which a border lies (min_p's
// or top_k's, top_p's, the draw's) are looked at one by one, in f64.
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
constexpr uint32_t LIST = 256;  // a chunk's largest values that are listed, of whole bins
// a chunk's part: {floor(t) of its largest value (f64), that value, bins listed, values listed, 0, 0, 0}, bins, list
constexpr uint32_t HEAD = 8, PART = HEAD + 2 * BINS + 2 * LIST;
constexpr int COUNT_AT = 50;  // a bin's word: its count from this bit on, its weights' sum times 2^36 below
constexpr uint64_t SUM = (1ull << COUNT_AT) - 1;

// What both kernels take a logit for, to the same bits.
SK_DEV bool has_weight(float x) { return x > -INFINITY; }  // (not NaN)
SK_DEV double scale_of(float T) { return 11.541560327111707 / (T > 0.0f ? (double)T : 1.0); }  // 8 log2(e) / T
SK_DEV double scaled(float x, double c) { return (double)fminf(x, 3.402823466e38f) * c; }
// 2^36 2^((f - 1) / 8), f in [0, 1): a series in f - 1/2 of which what is left out is below 6e-14
SK_DEV double weight(double f) {
  constexpr double S = 0x1p36;
  const double s = f - 0.5;
  double y = S * 5.626858230225532679e-10;
  y = __builtin_fma(y, s, S * 3.896563422975180069e-8);
  y = __builtin_fma(y, s, S * 2.248621090734246650e-6);
  y = __builtin_fma(y, s, S * 1.038103838861001429e-4);
  y = __builtin_fma(y, s, S * 3.594401424606149610e-3);
  y = __builtin_fma(y, s, S * 8.297000176389627734e-2);
  return __builtin_fma(y, s, S * 9.576032806985736469e-1);
}
SK_DEV uint64_t whole(double v) { return (uint64_t)__builtin_rint(v); }
// What t adds to the sum of the bin floor(t), d bins below the first.
SK_DEV uint64_t fixed_weight(double t, double d) {
#pragma clang fp contract(off)
  const double y = weight(t - __builtin_floor(t));
  if (d < BINS) return __builtin_bit_cast(uint64_t, y + 0x1p52) - 0x4330000000000000ull;  // rounded there
  return whole(y * exp2(((double)(BINS - 1) - d) * 0.125));  // below the last bin's lower edge
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

template <typename T>
SK_DEV T wave_scan(T v, uint32_t lane) {  // inclusive
#pragma unroll
  for (uint32_t d = 1; d < 64; d <<= 1) {
    const T u = __shfl_up(v, d, 64);
    if (lane >= d) v += u;
  }
  return v;
}

}  // namespace

// A workgroup's CHUNK tokens of a row: their bins below its own largest value, and the values of the first bins.
extern "C" __global__ __launch_bounds__(THREADS) void logits_sample(float *a, const uint32_t *ctl, SamplePush p) {
#pragma clang fp contract(off)
  constexpr uint32_t WAVES = THREADS / 64;
  __shared__ unsigned long long bin[BINS];
  __shared__ float big[WAVES];
  __shared__ uint32_t counts[WAVES], n_list;
  const uint32_t row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (row >= ctl[2]) return;
  const uint32_t base = blockIdx.x * CHUNK, n = min(CHUNK, p.n_vocab - base);
  const float *x = a + p.x_off + (size_t)row * p.x_stride + base;
  float *part = a + p.part_off + ((size_t)row * gridDim.x + blockIdx.x) * PART;
  const double c = scale_of(__builtin_bit_cast(float, ctl[p.ctrl_off + 8 * row]));
  f32x4 v[EACH / 4];
#pragma unroll
  for (uint32_t k = 0; k < EACH / 4; k++) {  // tokens 4 (t + THREADS k) + [0, 4)
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
  float top = -INFINITY;
#pragma unroll
  for (uint32_t k = 0; k < EACH / 4; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) top = fmaxf(top, v[k][e]);  // (leaves NaN aside)
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
  if (lane == 0) big[wave] = top;
  bin[t] = 0;
  if (t == 0) n_list = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < WAVES; w++) top = fmaxf(top, big[w]);
  const double first = __builtin_floor(scaled(top, c));
  if (!has_weight(top)) {  // nothing here: no bins, and none are read
    if (t == 0) {
      *(double *)part = -INFINITY;
      ((uint32_t *)part)[3] = BINS;
      ((uint32_t *)part)[4] = 0;
    }
    return;
  }
  uint32_t at[EACH];
#pragma unroll
  for (uint32_t k = 0; k < EACH / 4; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      uint32_t &b = at[4 * k + e];
      b = BINS;
      if (!has_weight(v[k][e])) continue;
      const double s = scaled(v[k][e], c), d = first - __builtin_floor(s);
      b = d < BINS ? (uint32_t)(int)d : BINS - 1;
      const uint64_t word = fixed_weight(s, d);
      atomicAdd(&bin[b], (unsigned long long)(word + (1ull << COUNT_AT)));
    }
  __syncthreads();
  const uint64_t mine = bin[t];
  ((uint64_t *)(part + HEAD))[t] = mine;
  // the bins whose values, with those above them, are LIST at most (the last bin has values of any size)
  uint32_t sum = wave_scan((uint32_t)(mine >> COUNT_AT), lane);
  if (lane == 63) counts[wave] = sum;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < WAVES; w++)
    if (w < wave) sum += counts[w];
  const uint32_t listed = __syncthreads_count(sum <= LIST && t < BINS - 1);
  uint2 *list = (uint2 *)(part + HEAD + 2 * BINS);
#pragma unroll
  for (uint32_t i = 0; i < EACH; i++)
    if (at[i] < listed) {
      const float y = v[i / 4][i % 4];
      list[atomicAdd(&n_list, 1u)] = make_uint2(__builtin_bit_cast(uint32_t, y), base + 4 * (t + THREADS * (i / 4)) + i % 4);
    }
  __syncthreads();
  if (t == 0) {
    *(double *)part = first;
    part[2] = top;
    ((uint32_t *)part)[3] = listed;
    ((uint32_t *)part)[4] = n_list;
  }
}

namespace {

constexpr uint32_t DRAW = 1024, DRAW_WAVES = DRAW / 64;
constexpr uint32_t MOST = 8192;    // values of the bins with borders that are put in order in LDS
constexpr uint32_t SPANS = 64;     // such bins
constexpr uint32_t CHUNKS = 128;   // of a row
constexpr uint32_t DIGITS = 2048;  // buckets of the search that takes any number of them

struct DrawShared {
  union {
    uint64_t got[MOST];   // places as they came,
    uint64_t upto[MOST];  // and, of those in order, the sum behind each
    double largest[CHUNKS];
    struct {
      unsigned long long sum[DIGITS];
      uint32_t count[DIGITS];
    } digit;
  };
  uint64_t in_order[MOST];
  double c[BINS + 1];    // C before a bin, in weights of the row's upper edge
  uint32_t n[BINS + 1];  // tokens before it
  uint32_t span[BINS];   // a bin's place among those looked at (~0: none)
  uint32_t bucket[DRAW + 1];
  double first[CHUNKS];  // the chunks' parts: floor(t) of their largest values, bins and values listed
  uint32_t listed[CHUNKS], values[CHUNKS];
  double sums[DRAW_WAVES];
  uint64_t words[DRAW_WAVES];
  uint32_t counts[DRAW_WAVES];
  unsigned long long below;
  uint32_t fill, found[4];
};

// A row as its kernel sees it.
struct Row {
  const float *x;
  uint32_t n_vocab;
  double c, edge;  // t = x c; floor(t) of the largest value
};
SK_DEV uint32_t bin_of(const Row &r, double t) {
  const double d = r.edge - __builtin_floor(t);
  return d < BINS - 1 ? (uint32_t)(int)d : BINS - 1;
}
SK_DEV uint64_t fixed_weight(const Row &r, double t) { return fixed_weight(t, r.edge - __builtin_floor(t)); }
// the weight of a bin's upper edge, and a sum of its weights
SK_DEV double edge_weight(uint32_t b) { return exp2(-0.125 * (double)b); }
SK_DEV double sum_of(uint64_t fixed, double edge) { return (double)fixed * 0x1p-36 * edge; }

// Every value of the row that may lie in a bin above t = least, its place and t: f(place, t).
template <typename F>
SK_DEV void each_value(const Row &r, double least, F f) {
  // the f32 below least / c, with room for both roundings
  const float low = (float)(least / r.c), from = low - fabsf(low) * 1e-6f;
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
        if (has_weight(v[k][e]) && !(v[k][e] < from)) f(place(v[k][e], i0 + 4 * DRAW * k + e), scaled(v[k][e], r.c));
  }
}

// The first bin b whose end satisfies ok(end), BINS if none does; ok is false, then true.  The same in every wave.
template <typename A, typename F>
SK_DEV uint32_t first_bin(const A *before, F ok) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t m = __ballot(ok(before[8 * lane + 8]));
  if (!m) return BINS;
  const uint32_t b = 8 * (uint32_t)__builtin_ctzll(m);
  return b + (uint32_t)__builtin_ctzll(__ballot(lane >= 7 || ok(before[b + lane % 8 + 1])));
}

template <typename T>
SK_DEV T block_scan(T v, T *waves, T &total) {  // inclusive, over DRAW threads; a barrier at its start and one inside
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v, lane);
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
  const double edge = edge_weight(b);
  Found f{0, s.n[b], s.c[b]};
  constexpr int at[5] = {53, 42, 32, 10, 0}, bits[5] = {11, 11, 10, 22, 10};
  // (ids are below 2^20: 10 bits from bit 10 on, all 22 of them compared as a prefix)
  for (int k = 0; k < 5; k++) {
    __syncthreads();
    for (uint32_t i = t; i < DIGITS; i += DRAW) s.digit.sum[i] = 0, s.digit.count[i] = 0;
    __syncthreads();
    const int above = at[k] + bits[k];
    each_value(r, b < BINS - 1 ? r.edge - (double)b : -INFINITY, [&](uint64_t place, double v) {
      if (bin_of(r, v) != b || (above < 64 && place >> above != f.place >> above)) return;
      const uint32_t d = (uint32_t)(place >> at[k]) & (DIGITS - 1);
      atomicAdd(&s.digit.sum[d], (unsigned long long)fixed_weight(r, v));
      atomicAdd(&s.digit.count[d], 1u);
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

// Tokens of t >= least, all of them and their sum, least in bin b.
__device__ __attribute__((noinline)) Found search_above(DrawShared &s, const Row r, double least, uint32_t b) {
  unsigned long long sum = 0;
  uint32_t n = 0;
  each_value(r, least, [&](uint64_t, double v) {
    if (v >= least && bin_of(r, v) == b) sum += fixed_weight(r, v), n++;
  });
  uint64_t all;
  uint32_t count;
  block_scan((uint64_t)sum, s.words, all);
  block_scan(n, s.counts, count);
  return {0, s.n[b] + count, s.c[b] + sum_of(all, edge_weight(b))};
}

}  // namespace

// A workgroup's row: its chunks' bins added up, the bins with the borders, and the tokens in these.
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
  float top = -INFINITY;
  if (t < CHUNKS) {
    const float *part = parts + (size_t)min(t, n_chunks - 1) * PART;
    const double first = *(const double *)part;
    s.first[t] = first;
    if (first > -INFINITY) s.largest[t] = part[2];
    else s.largest[t] = -INFINITY;
    s.listed[t] = ((const uint32_t *)part)[3];
    s.values[t] = ((const uint32_t *)part)[4];
  }
  __syncthreads();
  {
    const uint32_t lane = t & 63;
    double big = fmax(s.largest[lane], s.largest[lane + 64]);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) big = fmax(big, __shfl_xor(big, d, 64));
    top = (float)big;
    r.edge = __builtin_floor(scaled(top, r.c));
  }
  if (!has_weight(top)) {
    if (t == 0) *(uint4 *)out = make_uint4(~0u, 0, 0xff800000u, 0);
    return;
  }

  // the row's bins: thread t has bin t % BINS of every other chunk
  {
    const uint32_t b = t % BINS;
    uint32_t n = 0;
    uint64_t sum = 0;
    if (t == 0) s.below = 0, s.fill = 0;
    __syncthreads();
    constexpr uint32_t U = 10, STEP = DRAW / BINS;  // chunks whose loads are in flight
    for (uint32_t i0 = t / BINS; i0 < n_chunks; i0 += U * STEP) {
      uint64_t w[U];
#pragma unroll
      for (uint32_t j = 0; j < U; j++) {
        const uint32_t i = min(i0 + j * STEP, n_chunks - 1);
        const double d = r.edge - s.first[i];  // the chunk's bins lie so many below the row's
        const uint32_t down = d < BINS ? (uint32_t)(int)d : BINS;
        w[j] = ((const uint64_t *)(parts + (size_t)i * PART + HEAD))[b >= down ? b - down : 0];
        if (i0 + j * STEP >= n_chunks || b < down || b == BINS - 1) w[j] = 0;
      }
#pragma unroll
      for (uint32_t j = 0; j < U; j++) {
        n += (uint32_t)(w[j] >> COUNT_AT);
        sum += w[j] & SUM;
      }
    }
    // a chunk's bins from the row's last on go there, in weights of that one's edge
    for (uint32_t i = t / BINS; i < n_chunks; i += STEP) {
      const double d = r.edge - s.first[i];
      if (!(d < INFINITY) || (double)b + d < (double)(BINS - 1)) continue;
      const uint64_t w = ((const uint64_t *)(parts + (size_t)i * PART + HEAD))[b];
      if (!w) continue;
      atomicAdd(&s.below, (unsigned long long)whole((double)(w & SUM) * exp2(((double)(BINS - 1) - (double)b - d) * 0.125)));
      atomicAdd(&s.fill, (uint32_t)(w >> COUNT_AT));
    }
    s.got[t] = sum;
    s.bucket[t] = n;
    __syncthreads();
    if (t < BINS) {
      n += s.bucket[t + BINS];
      sum += s.got[t + BINS];
      if (b == BINS - 1) n = s.fill, sum = s.below;
    } else {
      n = 0, sum = 0;
    }
    uint32_t n_all;
    double c_all;
    const uint32_t n_end = block_scan(n, s.counts, n_all);
    const double c_end = block_scan(sum_of(sum, edge_weight(b)), s.sums, c_all);
    if (t < BINS) s.n[t + 1] = n_end, s.c[t + 1] = c_end;
    if (t == 0) s.n[0] = 0, s.c[0] = 0.0, s.fill = 0;
    __syncthreads();
  }

  // The bins with the borders.  What is known of C(n1) and C(n2) before these are looked at lies between lo and hi.
  const uint32_t total = s.n[BINS];
  const double t_top = scaled(top, r.c);
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
      const double more = (double)(k - s.n[bk]) * edge_weight(bk);
      hi = fmin(hi, lo + more);
      if (bm != bk && bk < BINS - 1) lo += more * edge_weight(1);
    }
    if (b1 == 0) lo = fmax(lo, edge_weight(1));  // the largest stays
  }
  uint32_t p_lo = BINS, p_hi = 0;
  const bool by_p = top_p < 1.0f;
  const double share = fmax((double)top_p, 0.0);
  const uint32_t b_last = min(b1, first_bin(s.n, [&](uint32_t n) { return n >= total; }));  // where n1 lies
  if (by_p) {
    lo *= share * LESS, hi *= share * MORE;
    p_lo = min(first_bin(s.c, [&](double c) { return c >= lo; }), b_last);
    p_hi = min(first_bin(s.c, [&](double c) { return c >= hi; }), b_last);
    hi = fmin(s.c[p_hi + 1], hi + edge_weight(p_lo));
    lo = fmax(lo, s.n[p_lo] ? 0.0 : edge_weight(1) * LESS);
  }
  const double u = ((double)words[4] + 0.5) * 0x1p-32;
  const uint32_t d_lo = min(first_bin(s.c, [&](double c) { return c > lo * u * LESS; }), by_p ? p_hi : b_last);
  const uint32_t d_hi = min(first_bin(s.c, [&](double c) { return c > hi * u * MORE; }), by_p ? p_hi : b_last);
  auto looked_at = [&](uint32_t b) { return b == b1 || (b >= p_lo && b <= p_hi) || (b >= d_lo && b <= d_hi); };

  // their places, and how many
  uint32_t n_spans, n_values, deepest;
  {
    const bool yes = t < BINS && looked_at(t) && s.n[t + 1] > s.n[t];
    const uint32_t at = block_scan((uint32_t)yes, s.counts, n_spans);
    if (t < BINS) s.span[t] = yes ? at - 1 : ~0u;
    block_scan(yes ? s.n[t + 1] - s.n[t] : 0u, s.counts, n_values);
    deepest = b1 < BINS ? b1 : by_p ? p_hi : d_hi;
  }
  Found n1, n2, chosen;
  if (n_spans <= SPANS && n_values <= MOST && deepest < BINS - 1) {
    // ---- few: their values into LDS, from the chunks' lists where these go down far enough, in buckets by t
    const double down = t < n_chunks ? (double)deepest - (r.edge - s.first[t]) : -1.0;  // such a chunk's bin
    const bool listed = !__syncthreads_or(t < n_chunks && down >= (double)s.listed[t]);
    const uint32_t per = DRAW / max(n_spans, 1u);
    auto bucket_of = [&](uint32_t b, double v) {
      const double f = 1.0 - (v - __builtin_floor(v));
      return s.span[b] * per + min((uint32_t)(int)(f * (double)per), per - 1);
    };
    s.bucket[t] = 0;
    if (t == 0) s.bucket[DRAW] = 0;
    __syncthreads();
    auto take = [&](uint64_t place, double v) {
      const uint32_t b = bin_of(r, v);
      if (s.span[b] == ~0u) return;
      const uint32_t at = atomicAdd(&s.fill, 1u);
      if (at < MOST) s.got[at] = place;  // (always: so many were counted)
      atomicAdd(&s.bucket[bucket_of(b, v)], 1u);
    };
    if (listed) {
      constexpr uint32_t U = 5, STEP = DRAW / LIST;
      for (uint32_t i0 = t / LIST; i0 < n_chunks; i0 += U * STEP) {
        uint2 v[U];
        bool is[U];
#pragma unroll
        for (uint32_t j = 0; j < U; j++) {
          const uint32_t i = min(i0 + j * STEP, n_chunks - 1);
          is[j] = i0 + j * STEP < n_chunks && t % LIST < s.values[i];
          v[j] = is[j] ? ((const uint2 *)(parts + (size_t)i * PART + HEAD + 2 * BINS))[t % LIST] : make_uint2(0, 0);
        }
#pragma unroll
        for (uint32_t j = 0; j < U; j++)
          if (is[j]) {
            const float x = __builtin_bit_cast(float, v[j].x);
            take(place(x, v[j].y), scaled(x, r.c));
          }
      }
    } else {
      each_value(r, r.edge - (double)deepest, take);
    }
    __syncthreads();
    const uint32_t n = min(s.fill, MOST);
    uint32_t all;
    const uint32_t mine = s.bucket[t], end = block_scan(mine, s.counts, all);
    s.bucket[t] = end - mine;  // where the bucket starts
    __syncthreads();
    for (uint32_t i = t; i < n; i += DRAW) {
      const uint64_t v = s.got[i];
      const double at = scaled(value_at(v), r.c);
      s.in_order[atomicAdd(&s.bucket[bucket_of(bin_of(r, at), at)], 1u)] = v;
    }
    __syncthreads();  // a bucket's word is now its end, the one before it its start
    uint64_t v[MOST / DRAW];
    uint32_t rank[MOST / DRAW];
#pragma unroll
    for (uint32_t j = 0; j < MOST / DRAW; j++) {
      const uint32_t i = t + DRAW * j;
      if (i >= n) continue;
      v[j] = s.in_order[i];
      const double at = scaled(value_at(v[j]), r.c);
      const uint32_t b = bucket_of(bin_of(r, at), at), from = b ? s.bucket[b - 1] : 0, to = s.bucket[b];
      rank[j] = from;
      for (uint32_t o = from; o < to; o++) rank[j] += s.in_order[o] < v[j];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < MOST / DRAW; j++)
      if (t + DRAW * j < n) s.in_order[rank[j]] = v[j];
    __syncthreads();
    // the sum behind each: of thread t the values [8 t, 8 t + 8)
    constexpr uint32_t OF = MOST / DRAW;
    uint64_t w[OF], sum = 0, sum_all;
    uint32_t bin[OF];
#pragma unroll
    for (uint32_t j = 0; j < OF; j++) {
      const uint32_t i = OF * t + j;
      bin[j] = 0, w[j] = 0;
      if (i < n) {
        const double at = scaled(value_at(s.in_order[i]), r.c);
        bin[j] = bin_of(r, at);
        w[j] = fixed_weight(r, at);
      }
      sum += w[j];
    }
    uint64_t before = block_scan(sum, s.words, sum_all) - sum;
#pragma unroll
    for (uint32_t j = 0; j < OF; j++) {
      before += w[j];
      if (OF * t + j < n) s.upto[OF * t + j] = before;
    }
    __syncthreads();
    // of a looked-at bin the first place in the order; its sums start at the bin's C
    if (t < BINS && s.span[t] != ~0u) s.bucket[s.span[t]] = t;
    __syncthreads();
    if (t < 64) {
      const uint32_t b = t < n_spans ? s.bucket[t] : 0, c = t < n_spans ? s.n[b + 1] - s.n[b] : 0;
      const uint32_t start = wave_scan(c, t) - c;
      if (t < n_spans) s.span[b] = start;
    }
    __syncthreads();
    auto upto = [&](uint32_t i, uint32_t b) {
      const uint32_t start = s.span[b];
      return s.c[b] + sum_of(s.upto[i] - (start ? s.upto[start - 1] : 0), edge_weight(b));
    };
    auto rank_of = [&](uint32_t i, uint32_t b) { return s.n[b] + i - s.span[b] + 1; };
    auto found_at = [&](uint32_t i) {
      const uint64_t at = s.in_order[i];
      const uint32_t b = bin_of(r, scaled(value_at(at), r.c));
      return Found{at, rank_of(i, b), upto(i, b)};
    };
    // n1: the last place of bin b1 that stays
    n1 = {0, total, s.c[BINS]};
    if (b1 < BINS) {
      if (t == 0) s.found[0] = 0;
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < OF; j++) {
        const uint32_t i = OF * t + j;
        if (i < n && bin[j] == b1 && rank_of(i, b1) <= k && scaled(value_at(s.in_order[i]), r.c) >= least)
          atomicMax(&s.found[0], i + 1);
      }
      __syncthreads();
      n1 = s.found[0] ? found_at(s.found[0] - 1) : Found{0, s.n[b1], s.c[b1]};
    }
    // the first place in bins [from, to] that meets `want`, the last of them if none does
    auto first = [&](Want want, double goal, uint32_t most, uint32_t from, uint32_t to) {
      __syncthreads();
      if (t == 0) s.found[1] = ~0u, s.found[2] = 0;
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < OF; j++) {
        const uint32_t i = OF * t + j;
        if (i >= n || bin[j] < from || bin[j] > to || rank_of(i, bin[j]) > most) continue;
        if (meets(want, goal, 0, upto(i, bin[j]))) atomicMin(&s.found[1], i);
        atomicMax(&s.found[2], i);
      }
      __syncthreads();
      return found_at(s.found[1] != ~0u ? s.found[1] : s.found[2]);
    };
    n2 = by_p ? first(kReach, share * n1.sum, n1.n, p_lo, p_hi) : n1;
    chosen = first(kPass, u * n2.sum, n2.n, d_lo, d_hi);
  } else {
    // ---- many
    n1 = {0, total, s.c[BINS]};
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
    const double y = (scaled(value_at(chosen.place), r.c) - r.edge - 1.0) * 0.125 * 0.69314718055994530942 - log(n2.sum);
    *(uint4 *)out = make_uint4((uint32_t)chosen.place, n2.n, __builtin_bit_cast(uint32_t, n2.n == 1 ? 0.0f : (float)y), 0);
  }
}
