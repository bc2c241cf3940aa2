// fm_sample.hip -- one category of each row of logits, drawn with a given uniform number (include/factorysim.h
// fm_sample_logits).
//
// A row's categories are ranked by a 64-bit place: the logit's bits, mapped so that whole numbers compare as the logits
// do, above the complement of the index (the lower index first among equals).  Every setting keeps a leading part of
// that ranking, and so does the share u of the kept weight, so all of them are the same question: which category is
// the one where a running sum (of ones, or of weights) passes a number.
//
// Weights are exp((logit - largest) / T) in multiples of 2^-s of the largest's, as 64-bit integers: sums are exact,
// so no result depends on the order in which a launch happens to add, and a border that lies 2^-45 of the row's
// weight away is still told apart (fp32 sums over 10^5 categories lose 2^-20 and would draw another category).
#include "fm_ops_dev.hpp"

namespace fm {
namespace {

struct Settings {
  double temperature, top_p, min_p;
  int64_t top_k;
  const float *temperature_rows, *top_p_rows, *min_p_rows;
  const int32_t* top_k_rows;
  const void* u;
  int u64, shift;  // shift: s above
};

struct Row {
  double inv_t, top_p, min_p, min_w, u, one;
  int64_t top_k;
  bool greedy, nan;
};

__device__ __forceinline__ Row row_settings(const Settings& a, int64_t r) {
  Row o;
  const double t = a.temperature_rows ? (double)a.temperature_rows[r] : a.temperature;
  o.min_p = a.min_p_rows ? (double)a.min_p_rows[r] : a.min_p;
  o.top_p = a.top_p_rows ? (double)a.top_p_rows[r] : a.top_p;
  o.top_k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
  o.u = a.u64 ? ((const double*)a.u)[r] : (double)((const float*)a.u)[r];
  o.nan = t != t || o.min_p != o.min_p || o.top_p != o.top_p || o.u != o.u;
  o.greedy = t <= 0;
  o.inv_t = 1.0 / t;
  o.one = (double)(1ull << a.shift);
  o.min_w = ldexp(fmin(o.min_p, 1.0), a.shift);
  return o;
}

// a block's row has the same settings for all lanes: in scalar registers
__device__ __forceinline__ double uniform(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 |
                                          (uint32_t)__builtin_amdgcn_readfirstlane((int)b)));
}
__device__ __forceinline__ Row block_settings(const Settings& a, int64_t r) {
  Row o = row_settings(a, r);
  o.inv_t = uniform(o.inv_t);
  o.top_p = uniform(o.top_p);
  o.min_p = uniform(o.min_p);
  o.min_w = uniform(o.min_w);
  o.u = uniform(o.u);
  o.one = uniform(o.one);
  return o;
}

// ascending as the floats; -0 and +0 are the same
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}

// exp(x) for x <= 0 to 6e-15 of itself: x = n ln 2 + r with |r| <= ln(2) / 2, the Taylor polynomial of degree 11 for
// exp(r) (its rest is below r^12 / 12! = 6e-15), scaled by 2^n
__device__ __forceinline__ double exp_neg(double x) {
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0.69314718055994529, x);
  r = fma(n, -2.3190468138462996e-17, r);
  double p = 1.0 / 39916800.0;
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}

// the weight as a whole number of 2^-shift: adding 2^52 leaves it, rounded, in the low bits
__device__ __forceinline__ uint64_t weight_of(float v, float top, const Row& o) {
  if (v == top) return (uint64_t)o.one;
  const double x = fmax(((double)v - (double)top) * o.inv_t, -1000.0);
  return (uint64_t)__double_as_longlong(fma(exp_neg(x), o.one, 4503599627370496.0)) & 0xfffffffffffffull;
}

// the number to pass for the share u of `sum`
__device__ __forceinline__ uint64_t target_of(double u, uint64_t sum) {
  const double t = u * (double)sum;
  return t <= 0 ? 0 : t >= (double)sum ? sum - 1 : (uint64_t)t;
}
// the last category kept by top_p passes this number: its own weight starts below p times `sum`
__device__ __forceinline__ uint64_t border_of(double p, uint64_t sum) {
  const double t = ceil(p * (double)sum);
  return t <= 1 ? 0 : t >= (double)sum ? sum - 1 : (uint64_t)t - 1;
}

// The row's logits: `each` calls f(column, logit) for every category, with -inf where it is barred.  16-byte loads
// from any element on, U of them on their way at a time; f is called for one after the other (`ordered`: the weights of
// several at once would spill registers).
template <typename T, bool MASKED>
struct Source {
  const T* z;
  const uint8_t* mask;
  int cols;

  template <int NT, int U, bool ORDERED, typename F>
  __device__ __forceinline__ void each(F&& f) const {
    constexpr int N = 16 / (int)sizeof(T);
    const int vectors = cols / N;
    for (int i = threadIdx.x; i < vectors; i += NT * U) {
      T v[U][N];
      uint8_t m[U][N];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int c = (i + u * NT < vectors ? i + u * NT : i) * N;
        __builtin_memcpy(v[u], z + c, 16);
        if (MASKED) __builtin_memcpy(m[u], mask + c, N);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool in = i + u * NT < vectors;
#pragma unroll
        for (int n = 0; n < N; n++) {
          f((i + u * NT) * N + n, in && !(MASKED && !m[u][n]) ? to_f32(v[u][n]) : -INFINITY);
          if (ORDERED) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    const int c = vectors * N + (int)threadIdx.x;
    if (c < cols) f(c, !(MASKED && !mask[c]) ? to_f32(z[c]) : -INFINITY);
  }
};

__device__ __forceinline__ uint64_t place_of(float v, int c) { return (uint64_t)key_of(v) << 32 | (uint32_t)~c; }
__device__ __forceinline__ float logit_of(uint64_t place) { return of_key((uint32_t)(place >> 32)); }
__device__ __forceinline__ int64_t column_of(uint64_t place) { return (int64_t)(uint32_t)~(uint32_t)place; }

// ---------------------------------------------------------------------------------------------- up to 64 categories
// G lanes a row, one category each: sorted by exchanging places between lanes, then every setting is a prefix of the
// group's lanes.  Rows of two categories fill a wave 32 at a time.
template <typename T, int G>
__global__ __launch_bounds__(256) void sample_group(const T* logits, int64_t stride, const uint8_t* mask, int64_t mask_stride, Settings a, int64_t* out,
                                                    int64_t rows, int cols) {
  const int lane = threadIdx.x & 63, j = lane & (G - 1), base = lane - j;
  const uint64_t group = (G == 64 ? ~0ull : (1ull << G) - 1) << base;
  const int64_t step = (int64_t)gridDim.x * (256 / G);
  for (int64_t first = (int64_t)blockIdx.x * (256 / G); first < rows; first += step) {
    const int64_t row = first + threadIdx.x / G, r = row < rows ? row : rows - 1;
    const Row o = row_settings(a, r);
    const bool in = j < cols && !(mask && !mask[r * mask_stride + j]);
    const float v = in ? to_f32(logits[r * stride + j]) : -INFINITY;
    const bool nan = (__ballot(v != v) & group) != 0;
    uint64_t p = v == -INFINITY ? 0 : place_of(v, j);
#pragma unroll
    for (int k = 2; k <= G; k <<= 1)
#pragma unroll
      for (int m = k >> 1; m; m >>= 1) {
        const uint64_t q = __shfl_xor((unsigned long long)p, m);
        const bool larger = ((j & m) == 0) == ((j & k) == 0 || k == G);  // this lane keeps the larger one
        p = (p > q) == larger ? p : q;
      }
    const int n = __popcll(__ballot(p != 0) & group);
    const float top = __shfl(logit_of(p), base);
    const uint64_t w = p && !nan ? weight_of(logit_of(p), top, o) : 0;
    uint64_t sum = w;  // up to and with this lane's
#pragma unroll
    for (int m = 1; m < G; m <<= 1) {
      const uint64_t q = __shfl_up((unsigned long long)sum, m, G);
      if (j >= m) sum += q;
    }
    int kept = o.top_k > 0 && o.top_k < n ? (int)o.top_k : n;
    auto upto = [&](int k) { return (uint64_t)__shfl((unsigned long long)sum, base + (k > 0 ? k - 1 : 0)); };
    uint64_t s = upto(kept);
    if (o.top_p < 1) {
      const int k = __popcll(__ballot(sum <= border_of(o.top_p, s)) & group) + 1;
      kept = k < kept ? k : kept;
    }
    const int k = __popcll(__ballot(p && (double)w >= o.min_w) & group);
    kept = k < kept ? k : kept;
    s = upto(kept);
    int at = __popcll(__ballot(sum <= target_of(o.u, s)) & group);
    at = o.greedy ? 0 : at < kept ? at : kept - 1;
    const uint64_t found = __shfl((unsigned long long)p, base + (at > 0 ? at : 0));
    if (j == 0 && row < rows) out[row] = o.nan || nan || n == 0 ? -1 : column_of(found);
  }
}

// ---------------------------------------------------------------------------------------------- sorted lists
// A leading part of a row's ranking (or a stretch of it) in LDS: its places, sorted, and their weights' running sums.
template <int LN>
struct List {
  unsigned long long place[LN], upto[LN];
  unsigned long long wave[16];
  int at;
};

// Sorts the first n places (the larger first) and sums their weights.  Bitonic: pairs that are at most 64 apart stay
// within the 128 places of one wave, and need no barrier.  A place of 0 is none.
template <int NT, int LN>
__device__ void sort_list(List<LN>& l, int n, float top, const Row& o) {
  int m = 2;
  while (m < n) m <<= 1;
  for (int i = n + threadIdx.x; i < m; i += NT) l.place[i] = 0;
  __syncthreads();
  bool wide = false;
  for (int k = 2; k <= m; k <<= 1)
    for (int j = k >> 1; j; j >>= 1) {
      if (wide || j > 64)
        __syncthreads();
      else
        wave_sync();
      wide = j > 64;
      for (int i = threadIdx.x; i < m / 2; i += NT) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const unsigned long long p = l.place[a], q = l.place[b];
        if ((p < q) == ((a & k) == 0 || k == m)) {
          l.place[a] = q;
          l.place[b] = p;
        }
      }
    }
  __syncthreads();
  // each thread sums its share of the places, the shares are joined over lanes, then over waves
  const int each = (m + NT - 1) / NT, first = threadIdx.x * each;
  uint64_t own = 0;
  for (int i = first; i < first + each && i < m; i++)
    if (l.place[i]) own += weight_of(logit_of(l.place[i]), top, o);
  uint64_t run = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t x = __shfl_up((unsigned long long)run, d);
    if ((threadIdx.x & 63) >= d) run += x;
  }
  if ((threadIdx.x & 63) == 63) l.wave[threadIdx.x >> 6] = run;
  __syncthreads();
  uint64_t sum = run - own;
  for (int w = 0; w < (int)(threadIdx.x >> 6); w++) sum += l.wave[w];
  for (int i = first; i < first + each && i < m; i++) {
    if (l.place[i]) sum += weight_of(logit_of(l.place[i]), top, o);
    l.upto[i] = sum;
  }
  __syncthreads();
}

// the first of n whose running sum is over `number` (the last of them where none is)
template <int NT, int LN>
__device__ int first_over(List<LN>& l, int n, uint64_t number) {
  if (threadIdx.x == 0) l.at = n - 1;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT)
    if (l.upto[i] > number && (i == 0 || l.upto[i - 1] <= number)) l.at = i;
  __syncthreads();
  const int at = l.at;
  __syncthreads();
  return at;
}

// the category of a row whose list holds n > 0 of its categories from the first on: all that the settings can keep
template <int NT, int LN>
__device__ uint64_t draw_from(List<LN>& l, int n, const Row& o) {
  if (o.greedy) return l.place[0];
  int kept = o.top_k > 0 && o.top_k < n ? (int)o.top_k : n;
  if (o.top_p < 1) kept = first_over<NT>(l, kept, border_of(o.top_p, l.upto[kept - 1])) + 1;
  if (o.min_w > 0) {
    if (threadIdx.x == 0) l.at = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < kept; i += NT)  // the last of those that weigh enough: a prefix
      if ((double)(l.upto[i] - (i ? l.upto[i - 1] : 0)) >= o.min_w &&
          (i + 1 == kept || (double)(l.upto[i + 1] - l.upto[i]) < o.min_w))
        l.at = i;
    __syncthreads();
    kept = l.at + 1;
    __syncthreads();
  }
  return l.place[first_over<NT>(l, kept, target_of(o.u, l.upto[kept - 1]))];
}

// Rows of at most LN categories, a block each: the whole row is the list.
template <typename T, bool MASKED, int NT, int LN>
__global__ __launch_bounds__(NT) void sample_list(const T* logits, int64_t stride, const uint8_t* mask, int64_t mask_stride, Settings a, int64_t* out,
                                                  int64_t rows, int cols) {
  __shared__ List<LN> l;
  __shared__ float fbuf[NT / 64];
  const int64_t r = blockIdx.x + (int64_t)gridDim.x * blockIdx.y;
  if (r < rows) {
    const Source<T, MASKED> src{logits + r * stride, MASKED ? mask + r * mask_stride : nullptr, cols};
    const Row o = block_settings(a, r);
    for (int c = threadIdx.x; c < cols; c += NT) l.place[c] = 0;
    __syncthreads();
    float top = -INFINITY;
    int wrong = o.nan, n = 0;
    src.template each<NT, 1, false>([&](int c, float v) {
      wrong |= v != v;
      top = fmaxf(top, v);
      n += v != -INFINITY;
      if (v != -INFINITY) l.place[c] = place_of(v, c);
    });
    top = block_max<NT>(top, fbuf);
    wrong = __syncthreads_or(wrong);
    n = block_sum<NT>(n, (int*)l.wave);
    __syncthreads();
    uint64_t found = 0;
    if (!wrong && n > 0) {
      sort_list<NT>(l, cols, top, o);
      found = draw_from<NT>(l, n, o);
    }
    if (threadIdx.x == 0) out[r] = found ? column_of(found) : -1;
  }
}

// ---------------------------------------------------------------------------------------------- longer rows
// One block a row.  A pass finds the largest logit, a second one counts and weighs the categories by how far below it
// they lie (2048 steps of equal width); sums over steps then tell in which step a setting's border and the drawn
// category lie, and only the categories of such a step, or of the few steps up to it, are listed and sorted.
constexpr int NT = 1024, DIGIT = 11, BINS = 1 << DIGIT, LISTED = 2048;

struct Find {
  unsigned long long weight[BINS];
  uint32_t count[BINS];
  unsigned long long wave[NT / 64], ubuf[NT / 64];
  unsigned long long place, before, upto;  // the category found; the sum before it and with it
  float fbuf[2][NT / 64];
};

// adds a category to a bin; a wave whose categories all go to one bin adds them up first (one value in many places
// would otherwise be 64 turns at the same address)
__device__ __forceinline__ void add(Find& f, int b, uint64_t w) {
  const int b0 = __builtin_amdgcn_readfirstlane(b);
  if (__all(b == b0)) {
    const uint64_t active = __ballot(1);
    const uint64_t w0 = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(w >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)w);
    if (__all(w == w0)) {
      if ((threadIdx.x & 63) == __ffsll((unsigned long long)active) - 1) {
        atomicAdd(&f.count[b0], (uint32_t)__popcll(active));
        atomicAdd(&f.weight[b0], (unsigned long long)w0 * __popcll(active));
      }
      return;
    }
  }
  atomicAdd(&f.count[b], 1u);
  atomicAdd(&f.weight[b], (unsigned long long)w);
}

// Of rows that the steps do not tell apart: the category at which a sum passes a number, digit by digit of its place.
// Each pass over the row adds up its categories by the next 11 bits, among those that share the bits found so far.
// The first category (in rank) at which the running sum of weights (or, by_count, of ones) is over `number`, which the
// sum of all of them is.  f.place, f.before and f.upto (sums of weights) are set for every thread.
template <typename S>
__device__ __forceinline__ void find(bool by_count, const S& src, float top, const Row& o, uint64_t number, Find& f) {
  const int low = 64 - __clz((unsigned)(src.cols > 1 ? src.cols - 1 : 1)) - 32;  // bits of an index
  uint64_t place = 0, known = 0, before = 0, wbefore = 0;
  int at = 64;
  while (at > 0) {
    if (at == 32) {  // the index's upper bits are the same for all: ones, complemented
      const uint64_t upper = ~((1ull << low) - 1) & 0xffffffffull;
      known |= upper;
      place |= upper;
      at = low;
    }
    const int floor_ = at > 32 ? 32 : 0, d = at - floor_ < DIGIT ? at - floor_ : DIGIT, sh = at - d, bins = 1 << d;
    for (int i = threadIdx.x; i < bins; i += NT) {
      f.count[i] = 0;
      f.weight[i] = 0;
    }
    __syncthreads();
    src.template each<NT, 2, true>([&](int c, float v) {
      const uint64_t p = place_of(v, c);
      if (v > -INFINITY && (p & known) == place) add(f, (int)(p >> sh) & (bins - 1), weight_of(v, top, o));
    });
    __syncthreads();
    // thread i sums the i-th share of the bins from the top, then the bin is where the sum passes the number
    const int each = (bins + NT - 1) / NT, first = bins - 1 - (int)threadIdx.x * each;
    uint64_t own = 0, ownw = 0;
    for (int i = 0; i < each && first - i >= 0; i++) {
      own += by_count ? (uint64_t)f.count[first - i] : (uint64_t)f.weight[first - i];
      ownw += f.weight[first - i];
    }
    uint64_t run = own, runw = ownw;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const uint64_t x = __shfl_up((unsigned long long)run, m), y = __shfl_up((unsigned long long)runw, m);
      if ((threadIdx.x & 63) >= m) {
        run += x;
        runw += y;
      }
    }
    if ((threadIdx.x & 63) == 63) {
      f.wave[threadIdx.x >> 6] = run;
      f.ubuf[threadIdx.x >> 6] = runw;
    }
    __syncthreads();
    uint64_t base = before, basew = wbefore;
    for (int w = 0; w < (int)(threadIdx.x >> 6); w++) {
      base += f.wave[w];
      basew += f.ubuf[w];
    }
    uint64_t sum = base + run - own, sumw = basew + runw - ownw;
    if (sum <= number && number < sum + own) {  // one thread's
      for (int i = 0; i < each; i++) {
        const uint64_t val = by_count ? (uint64_t)f.count[first - i] : (uint64_t)f.weight[first - i];
        if (number < sum + val) {
          f.place = place | (uint64_t)(first - i) << sh;
          f.before = sum;
          f.upto = sumw;
          break;
        }
        sum += val;
        sumw += f.weight[first - i];
      }
    }
    __syncthreads();
    place = f.place;
    before = f.before;
    wbefore = f.upto;
    known |= (uint64_t)(bins - 1) << sh;
    at = sh;
    __syncthreads();
  }
  const uint64_t w = weight_of(logit_of(place), top, o);
  if (threadIdx.x == 0) {
    f.place = place;
    f.before = wbefore;
    f.upto = wbefore + w;
  }
  __syncthreads();
}

// the weight of the categories that min_p keeps: like every setting's, the leading part of the ranking
template <typename S>
__device__ __forceinline__ uint64_t weight_over(const S& src, float top, const Row& o, Find& f) {
  uint64_t own = 0;
  src.template each<NT, 2, true>([&](int, float v) {
    const uint64_t w = v > -INFINITY ? weight_of(v, top, o) : 0;
    own += (double)w >= o.min_w ? w : 0;
  });
  const uint64_t sum = block_sum<NT>((unsigned long long)own, f.ubuf);
  __syncthreads();
  return sum;
}

// the drawn category's place, with nothing but `find`: n categories are not barred, their weight is `sum`, of which min_p
// keeps at most `most`
template <typename S>
__device__ __forceinline__ uint64_t draw_by_digits(const S& src, float top, const Row& o, uint64_t n, uint64_t sum, uint64_t most, Find& f) {
  for (int stage = 0;; stage++) {  // top_k's border, top_p's, the draw
    if (stage == 0 && (o.greedy || o.top_k <= 0 || (uint64_t)o.top_k >= n)) continue;
    if (stage == 1 && (o.greedy || o.top_p >= 1)) continue;
    if (stage == 2 && most < sum) sum = most;
    find(stage == 0 || o.greedy, src, top, o, o.greedy ? 0 : stage == 0 ? (uint64_t)o.top_k - 1 : stage == 1 ? border_of(o.top_p, sum) : target_of(o.u, sum), f);
    if (stage == 2) return f.place;
    sum = f.upto;
    __syncthreads();
  }
}

// the step below the largest logit; a function that never falls as v does
struct Steps {
  float top, scale;
  __device__ __forceinline__ int operator()(float v) const {
    const float d = v == top ? 0.0f : (top - v) * scale;
    return d < (float)(BINS - 1) ? (int)d : BINS - 1;
  }
};

struct Long {
  Find f;
  List<LISTED> l;
  int listed, step;
  unsigned long long categories, weight;
};

// Lists and sorts the categories of steps `from` .. `to`.  False, for all threads, where they are too many.
template <typename S>
__device__ __forceinline__ bool list_steps(const S& src, const Steps& steps, int from, int to, const Row& o, Long& g) {
  const uint32_t n = (to + 1 < BINS ? g.f.count[to + 1] : (uint32_t)g.categories) - g.f.count[from];
  if (n > LISTED) return false;
  __syncthreads();
  if (threadIdx.x == 0) g.listed = 0;
  __syncthreads();
  src.template each<NT, 4, false>([&](int c, float v) {
    const int b = steps(v);
    if (b >= from && b <= to && v > -INFINITY) g.l.place[atomicAdd(&g.listed, 1)] = place_of(v, c);
  });
  __syncthreads();
  sort_list<NT>(g.l, (int)n, steps.top, o);
  return true;
}

// the step in which the running count (or weight) passes `number`
__device__ __forceinline__ int step_of(bool by_count, Long& g, uint64_t number) {
  for (int b = threadIdx.x; b < BINS; b += NT) {
    const uint64_t from = by_count ? (uint64_t)g.f.count[b] : (uint64_t)g.f.weight[b];
    const uint64_t to = b + 1 == BINS ? (by_count ? g.categories : g.weight) : by_count ? (uint64_t)g.f.count[b + 1] : (uint64_t)g.f.weight[b + 1];
    if (from <= number && number < to) g.step = b;
  }
  __syncthreads();
  const int b = g.step;
  __syncthreads();
  return b;
}

template <typename T, bool MASKED>
__global__ __launch_bounds__(NT) void sample_long(const T* logits, int64_t stride, const uint8_t* mask, int64_t mask_stride, Settings a, int64_t* out,
                                                  int64_t rows, int cols) {
  __shared__ Long g;
  const int64_t r = blockIdx.x + (int64_t)gridDim.x * blockIdx.y;
  if (r < rows) {
    const Source<T, MASKED> src{logits + r * stride, MASKED ? mask + r * mask_stride : nullptr, cols};
    const Row o = block_settings(a, r);
    float top = -INFINITY, least = INFINITY;
    int wrong = o.nan;
    src.template each<NT, 4, false>([&](int, float v) {
      wrong |= v != v;
      top = fmaxf(top, v);
      least = fminf(least, v > -INFINITY ? v : INFINITY);
    });
    for (int b = threadIdx.x; b < BINS; b += NT) {
      g.f.count[b] = 0;
      g.f.weight[b] = 0;
    }
    top = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(block_max<NT>(top, g.f.fbuf[0]))));
    least = -block_max<NT>(-least, g.f.fbuf[1]);
    wrong = __syncthreads_or(wrong);
    uint64_t found = 0;
    if (!wrong && top > -INFINITY) {
      // steps of 1/64 of the temperature reach down to weights of e^-32; narrower where the whole row is closer
      const float wanted = fmaxf(64.0f * (float)fabs(o.inv_t), (float)BINS / (top - least));
      const Steps steps{top, wanted < 1e30f ? wanted : 1e30f};
      src.template each<NT, 2, true>([&](int, float v) {
        if (v > -INFINITY) add(g.f, steps(v), weight_of(v, top, o));
      });
      __syncthreads();
      {  // counts and weights to sums of the steps before; two steps a thread
        const int b = threadIdx.x * 2;
        const uint32_t c0 = g.f.count[b], c1 = g.f.count[b + 1];
        const uint64_t w0 = g.f.weight[b], w1 = g.f.weight[b + 1];
        uint64_t c = c0 + c1, w = w0 + w1;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
          const uint64_t x = __shfl_up((unsigned long long)c, m), y = __shfl_up((unsigned long long)w, m);
          if ((threadIdx.x & 63) >= m) {
            c += x;
            w += y;
          }
        }
        if ((threadIdx.x & 63) == 63) {
          g.f.wave[threadIdx.x >> 6] = c;
          g.f.ubuf[threadIdx.x >> 6] = w;
        }
        __syncthreads();
        for (int v = 0; v < (int)(threadIdx.x >> 6); v++) {
          c += g.f.wave[v];
          w += g.f.ubuf[v];
        }
        g.f.count[b] = (uint32_t)c - c0 - c1;
        g.f.count[b + 1] = (uint32_t)c - c1;
        g.f.weight[b] = w - w0 - w1;
        g.f.weight[b + 1] = w - w1;
        if (threadIdx.x == NT - 1) {
          g.categories = c;
          g.weight = w;
        }
        __syncthreads();
      }
      const uint64_t n = g.categories, all = g.weight;
      const bool cut = o.top_k > 0 && (uint64_t)o.top_k < n;
      uint64_t sum = all, most = all;
      bool ok = false;
      // First, one list of every step that can hold a kept category: few categories, as a rule.  Else a list for each
      // border, of its own step: top_k's, top_p's, the draw's.
      for (int stage = 0; stage < 4; stage++) {
        int from = 0, to = BINS - 1;
        uint64_t number = 0;
        if (stage == 0) {
          if (o.greedy)
            to = 0;
          else if (cut)
            to = step_of(true, g, (uint64_t)o.top_k - 1);
          else if (o.top_p < 1)
            to = step_of(false, g, border_of(o.top_p, all));
          if (o.min_p > 1e-9 && !o.greedy && !(cut && o.top_p < 1)) {
            // min_p keeps logits over top + T ln(min_p); a step more than that, and some float32 roundings, are let in.
            // (With both others, top_p's share is of all that top_k keeps: none of it can be left out.)
            const double reach = log(fmin(o.min_p, 1.0)) / o.inv_t, least_kept = (double)top + reach * 1.000001 - 1e-6 * fabs((double)top);
            const int last = steps((float)least_kept) + 1;
            to = last < to ? last : to;
          }
        } else if (stage == 1) {
          if (!cut) continue;
          from = to = step_of(true, g, (uint64_t)o.top_k - 1);
        } else {
          if (stage == 2 && o.top_p >= 1) continue;
          if (stage == 3 && o.min_w > 0) {
            most = weight_over(src, top, o, g.f);
            sum = most < sum ? most : sum;
          }
          number = stage == 2 ? border_of(o.top_p, sum) : target_of(o.u, sum);
          from = to = step_of(false, g, number);
        }
        ok = list_steps(src, steps, from, to, o, g);
        if (!ok) {
          if (stage == 0 && !o.greedy) continue;
          break;
        }
        const int listed = g.listed;
        if (stage == 0) {
          Row rest = o;
          int m = listed;
          if (!cut && o.top_p < 1 && !o.greedy) {  // top_p's share is of the whole row, which the list is not
            m = first_over<NT>(g.l, listed, border_of(o.top_p, all)) + 1;
            rest.top_p = 1;
          }
          found = draw_from<NT>(g.l, m, rest);
          break;
        }
        if (stage == 1) {
          sum = g.f.weight[from] + g.l.upto[o.top_k - 1 - g.f.count[from]];
        } else {
          const int at = first_over<NT>(g.l, listed, number - g.f.weight[from]);
          if (stage == 2)
            sum = g.f.weight[from] + g.l.upto[at];
          else
            found = g.l.place[at];
        }
      }
      if (!ok) {
        __syncthreads();
        if (o.min_w > 0 && !o.greedy) most = weight_over(src, top, o, g.f);
        found = draw_by_digits(src, top, o, n, all, most, g.f);
      }
    }
    if (threadIdx.x == 0) out[r] = found ? column_of(found) : -1;
  }
}

int shift_of(int64_t cols) {  // the sum of cols weights of at most 2^s stays below 2^63
  int s = 51;
  while (s > 0 && (cols - 1) >> (62 - s)) s--;
  return s;
}

// Up to 64 categories a group of lanes holds a row; up to 2048 a block sorts it whole (fewer threads for fewer
// categories: their barriers cost more than the idle lanes); longer rows are narrowed down first.
template <typename T, bool MASKED>
void launch(const fm_sample_args& a) {
  const Settings s{a.temperature, a.top_p, a.min_p, a.top_k, a.temperature_rows, a.top_p_rows, a.min_p_rows, a.top_k_rows, a.u, a.u_dtype == FM_DTYPE_F64, shift_of(a.cols)};
  hipStream_t st = (hipStream_t)a.stream;
  const int cols = (int)a.cols;
  auto blocks = [&](int rows_each) {
    const int64_t n = (a.rows + rows_each - 1) / rows_each;
    return (int)(n < (1 << 20) ? n : 1 << 20);
  };
  const dim3 each(blocks(1), (unsigned)((a.rows + (1 << 20) - 1) >> 20));
#define ARGS (const T*)a.logits, a.stride, a.mask, a.mask_stride, s, a.out, a.rows, cols
  if (cols <= 2)
    sample_group<T, 2><<<blocks(128), 256, 0, st>>>(ARGS);
  else if (cols <= 4)
    sample_group<T, 4><<<blocks(64), 256, 0, st>>>(ARGS);
  else if (cols <= 8)
    sample_group<T, 8><<<blocks(32), 256, 0, st>>>(ARGS);
  else if (cols <= 16)
    sample_group<T, 16><<<blocks(16), 256, 0, st>>>(ARGS);
  else if (cols <= 32)
    sample_group<T, 32><<<blocks(8), 256, 0, st>>>(ARGS);
  else if (cols <= 64)
    sample_group<T, 64><<<blocks(4), 256, 0, st>>>(ARGS);
  else if (cols <= 256)
    sample_list<T, MASKED, 64, 256><<<each, 64, 0, st>>>(ARGS);
  else if (cols <= 512)
    sample_list<T, MASKED, 128, 512><<<each, 128, 0, st>>>(ARGS);
  else if (cols <= 1024)
    sample_list<T, MASKED, 256, 1024><<<each, 256, 0, st>>>(ARGS);
  else if (cols <= 2048)
    sample_list<T, MASKED, 512, 2048><<<each, 512, 0, st>>>(ARGS);
  else
    sample_long<T, MASKED><<<each, NT, 0, st>>>(ARGS);
#undef ARGS
}
}  // namespace
}  // namespace fm

using namespace fm;
extern "C" {
int64_t fm_sample_workspace(int64_t rows, int64_t cols) { return 0; }

int fm_sample_logits(const fm_sample_args* a) {
  return guarded([&] {
    if (int rc = check_sample(a)) return rc;
    if (a->rows == 0) return FM_OK;
    if (a->device < 0) {
      cpu_sample(*a);
      return FM_OK;
    }
    OnDevice on(a->device);
    if (on.err == hipSuccess)
      with_type(a->dtype, [&](auto tag) {
        typedef typename decltype(tag)::type T;
        if (a->mask)
          launch<T, true>(*a);
        else
          launch<T, false>(*a);
      });
    return on.status("sample");
  });
}
}
