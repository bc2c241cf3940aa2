// fm_sample.hip -- one category of each row of logits, drawn with a given uniform number (include/factorysim.h
// fm_sample_logits).
//
// A row's categories are ranked by a 64-bit place: the logit's bits, mapped so that whole numbers compare as the logits do,
// above the complement of the index (the lower index first among equals).  Every setting keeps a leading part of that ranking,
// and so does the share u of the kept weight, so all of them are the same question: which category is the one where a running
// sum (of ones, or of weights) passes a number.
//
// Weights are exp((logit - largest) / T) in multiples of 2^-s of the largest's (s = 51 up to 2048 categories, 45 for 2^17), as
// 64-bit integers whose sums do not depend on the order in which a launch happens to add: a call gives the same on every run.
// A weight is good to 6e-15 of itself (exp_neg), beyond 2048 categories the sums that find a border's step to 5e-13 (2^-41; fp32
// sums over 10^5 categories lose 2^-20 and would draw another category).  Where a border lies as near as that to one between two
// categories, another kernel or backend may draw the neighbour.  Shares of equal logits that hold all the weight are exact.
//
// Measured on an MI355X: 16384 x 2 fp32 3.3 us, 65536 x 33 42, 16384 x 1000 74, 1 x 32768 15, 37 x 50021 with a mask 25,
// 256 x 131072 bf16, top_p 0.9, 57, of which reading it once would take 13.  Short rows are bound by their launch, 33 to 64
// categories by the 21 exchanges that sort them, rows of hundreds by a float64 exponential and an LDS atomic a logit, long ones by
// float64 instructions (17 a logit) and a second read.
#include <type_traits>

#include "fm_ops_dev.hpp"

#define GLOBAL __attribute__((address_space(1)))
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
  o.inv_t = fmin(1.0 / t, 1e290);
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
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}
template <typename V>
__device__ __forceinline__ const GLOBAL V* uniform(const V* v) {
  const uint64_t b = (uint64_t)v;
  return (const GLOBAL V*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32))
      << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)b));
}
__device__ __forceinline__ Row uniform(Row o) {
  o.inv_t = uniform(o.inv_t);
  o.top_p = uniform(o.top_p);
  o.min_p = uniform(o.min_p);
  o.min_w = uniform(o.min_w);
  o.u = uniform(o.u);
  o.one = uniform(o.one);
  o.top_k = ((int64_t)uniform((int)(o.top_k >> 32)) << 32) | (uint32_t)uniform((int)o.top_k);
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

// the number to pass for the share u of `sum` (a NaN, whose row is not drawn, gives 0)
__device__ __forceinline__ uint64_t target_of(double u, uint64_t sum) {
  const double t = u * (double)sum;
  return !(t > 0) ? 0 : t >= (double)sum ? sum - 1 : (uint64_t)t;
}
// the last category kept by top_p passes this number: its own weight starts below p times `sum`
__device__ __forceinline__ uint64_t border_of(double p, uint64_t sum) {
  const double t = ceil(p * (double)sum);
  return !(t > 1) ? 0 : t >= (double)sum ? sum - 1 : (uint64_t)t - 1;
}

// The row's logits, -inf where a category is barred.  The pointers say that they are to global memory, also in functions of
// their own.
typedef uint32_t Vec16 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t Vec8 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t Vec4 __attribute__((aligned(1)));

template <typename T, bool MASKED>
struct Source {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef typename std::conditional<N == 8, Vec8, Vec4>::type Bytes;
  const GLOBAL T* z;
  const GLOBAL uint8_t* mask;
  int cols;

  __device__ __forceinline__ float operator()(int c) const { return MASKED && !mask[c] ? -INFINITY : to_f32(z[c]); }

  // f(first column, N logits) by 16-byte loads from any element on, U of them on their way at a time; g(column, logit) for
  // what is left at the end
  template <int NT, int U, typename F, typename G>
  __device__ __forceinline__ void vectors(F&& f, G&& g) const {
    const int count = cols / N;
    for (int i = threadIdx.x; i < count; i += NT * U) {
      Vec16 v[U];
      Bytes m[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int c = (i + u * NT < count ? i + u * NT : i) * N;
        v[u] = *(const GLOBAL Vec16*)(z + c);
        if (MASKED) m[u] = *(const GLOBAL Bytes*)(mask + c);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i + u * NT >= count) break;
        T raw[N];
        uint8_t open[N];
        float x[N];
        __builtin_memcpy(raw, &v[u], 16);
        if (MASKED) __builtin_memcpy(open, &m[u], N);
#pragma unroll
        for (int n = 0; n < N; n++) x[n] = MASKED && !open[n] ? -INFINITY : to_f32(raw[n]);
        f((i + u * NT) * N, x);
      }
    }
    const int c = count * N + (int)threadIdx.x;
    if (c < cols) g(c, (*this)(c));
  }
  // f(column, logit), one at a time: for rare passes, in little code
  template <int NT, typename F>
  __device__ __forceinline__ void each(F&& f) const {
    for (int c = threadIdx.x; c < cols; c += NT) f(c, (*this)(c));
  }
};

__device__ __forceinline__ uint64_t place_of(float v, int c) { return (uint64_t)key_of(v) << 32 | (uint32_t)~c; }
__device__ __forceinline__ float logit_of(uint64_t place) { return of_key((uint32_t)(place >> 32)); }
__device__ __forceinline__ int64_t column_of(uint64_t place) { return (int64_t)(uint32_t)~(uint32_t)place; }

// sorts G lanes' places, the larger first (bitonic, by exchanges between lanes); j: the lane's number among them
template <int G, int K = 2, int M = 1>
__device__ __forceinline__ uint64_t sort_lanes(uint64_t p, int j) {
  if constexpr (K <= G) {
    const uint64_t q = lane_xor<M>(p);
    const bool larger = ((j & M) == 0) == ((j & K) == 0 || K == G);  // this lane keeps the larger one
    p = (p > q) == larger ? p : q;
    if constexpr (M > 1)
      return sort_lanes<G, K, M / 2>(p, j);
    else
      return sort_lanes<G, 2 * K, K>(p, j);
  } else {
    return p;
  }
}

// ---------------------------------------------------------------------------------------------- up to 64 categories
// G lanes a row, one category each: sorted by exchanging places between lanes, then every setting is a prefix of the
// group's lanes.  Rows of two categories fill a wave 32 at a time: 65536 of them take 5 us, of 33 categories 42.
template <typename T, int G>
__global__ __launch_bounds__(256) void sample_group(const T* logits, int64_t stride, const uint8_t* mask,
    int64_t mask_stride, Settings a, int64_t* out, int64_t rows, int cols) {
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
    p = sort_lanes<G>(p, j);
    const int n = __popcll(__ballot(p != 0) & group);
    const float top = __shfl(logit_of(p), base);
    const uint64_t w = p && !nan ? weight_of(logit_of(p), top, o) : 0;
    const uint64_t sum = sum_lanes<G>(w, j);  // up to and with this lane's
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

// Sorts the first n places (the larger first) and sums their weights.  Up to 256, with as many threads as there are for
// each, every place is compared with all (n^2 steps, but without a barrier between them: 200 places take 3 us, sorting them 9);
// more are sorted by bitonic exchanges in LDS, where pairs that are at most 64 apart stay within the 128 places of one wave and
// need no barrier.  A place below 2^32 (above it is the logit, never 0) is none; up to n all places differ.
template <int NT, int LN>
__device__ __forceinline__ void sort_list(List<LN>& l, int n, float top, const Row& o) {
  constexpr int Q = NT > 256 ? NT / 256 : 1;  // threads for each place
  if (n <= NT / Q) {
    __syncthreads();
    if ((int)threadIdx.x < n) {
      const uint64_t p = l.place[threadIdx.x];
      l.upto[threadIdx.x] = p >> 32 ? weight_of(logit_of(p), top, o) : 0;
    }
    __syncthreads();
    const int i = threadIdx.x / Q;
    uint64_t own = 0, sum = 0;
    int before = 0;
    if (i < n) {
      own = l.place[i];
#pragma unroll 8
      for (int k = threadIdx.x % Q; k < n; k += Q) {
        const uint64_t p = l.place[k], w = l.upto[k];
        sum += p > own ? w : 0;
        before += p > own;
      }
      sum = group_sum<Q>(sum) + l.upto[i];
      before = group_sum<Q>(before);
    }
    __syncthreads();
    if (i < n && threadIdx.x % Q == 0) {
      l.place[before] = own;
      l.upto[before] = sum;
    }
    __syncthreads();
    return;
  }
  int m = 128;
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
  for (int i = first; i < first + each && i < m; i++) {
    own += l.place[i] >> 32 ? weight_of(logit_of(l.place[i]), top, o) : 0;
    l.upto[i] = own;
  }
  const uint64_t run = sum_lanes<64>(own, threadIdx.x & 63);
  if ((threadIdx.x & 63) == 63) l.wave[threadIdx.x >> 6] = run;
  __syncthreads();
  uint64_t before = run - own;
  for (int w = 0; w < (int)(threadIdx.x >> 6); w++) before += l.wave[w];
  for (int i = first; i < first + each && i < m; i++) l.upto[i] += before;
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

// ---------------------------------------------------------------------------------------------- up to 2048 categories
// A wave a row, R logits a lane in registers, no barriers.  Weights go to 256 steps of the logit in LDS; the step in which a
// sum passes a number is found by the lanes' running sums, and its categories, at most 64 as a rule, are compared with each
// other, one a lane.  16384 x 1000 takes 72 us, sorting the rows in LDS, a block each, 296.
constexpr int WBINS = 256;

__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane)
      << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

template <typename T, bool MASKED, int R>
struct WaveRow {
  static constexpr int N = 16 / (int)sizeof(T), V = R / N;
  struct Lds {
    unsigned long long weight[WBINS], place[64];
    uint32_t count[WBINS];
    int listed;
  };
  float x[V][N];
  float top, scale;
  int lane;
  uint64_t wbefore, wbin[WBINS / 64];  // this lane's steps: the weight of all before, and each one's
  uint32_t cbefore, cbin[WBINS / 64];

  // f(column, logit) over the lane's categories, -inf where one is barred
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int n = 0; n < N; n++) {
        f((i * 64 + lane) * N + n, x[i][n]);
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  __device__ __forceinline__ int step_of(float v) const {
    const float d = v == top ? 0.0f : (top - v) * scale;
    return d < (float)(WBINS - 1) ? (int)d : WBINS - 1;
  }
  // the step in which the running sum passes `number`, and that sum before it (by_count: of ones; wsum: of weights)
  __device__ __forceinline__ int find_step(bool by_count, uint64_t number, uint64_t& sum, uint64_t& wsum) const {
    uint64_t s = by_count ? cbefore : wbefore, w = wbefore, at_s = 0, at_w = 0;
    int found = -1;
#pragma unroll
    for (int k = 0; k < WBINS / 64; k++) {
      const uint64_t own = by_count ? (uint64_t)cbin[k] : wbin[k];
      if (s <= number && number < s + own) {
        found = lane * (WBINS / 64) + k;
        at_s = s;
        at_w = w;
      }
      s += own;
      w += wbin[k];
    }
    const int l = __ffsll((unsigned long long)__ballot(found >= 0)) - 1;
    sum = read_lane(at_s, l);
    wsum = read_lane(at_w, l);
    return __builtin_amdgcn_readlane(found, l);
  }
  // The category at which the running sum (of ones, or of weights) passes `number`: its place, and the weight up to and with
  // it.
  __device__ __forceinline__ uint64_t find(bool by_count, uint64_t number, Lds& g, const Row& o, uint64_t& upto) const {
    uint64_t sum, wsum;
    const int step = find_step(by_count, number, sum, wsum);
    if (lane == 0) g.listed = 0;
    wave_sync();
    each([&](int c, float v) {
      if (v > -INFINITY && step_of(v) == step) {
        const int i = atomicAdd(&g.listed, 1);
        if (i < 64) g.place[i] = place_of(v, c);
      }
    });
    wave_sync();
    const int n = uniform(g.listed);
    if (n <= 64) {
      const uint64_t p = lane < n ? g.place[lane] : 0, w = p ? weight_of(logit_of(p), top, o) : 0;
      uint64_t own = 0, ownw = wsum;  // up to and with this lane's
      for (int k = 0; k < n; k++) {
        const bool over = read_lane(p, k) >= p;
        own += over;
        ownw += over ? read_lane(w, k) : 0;
      }
      own = by_count ? sum + own : ownw;
      // the first one over the number: of those, the one with the largest place (the last of all, should rounding leave none)
      uint64_t best = p && own > number ? p : 0;
      best = sort_lanes<64>(best, lane);
      best = read_lane(best, 0);
      const uint64_t hit = __ballot(p && p == best);
      const int l = hit ? __ffsll((unsigned long long)hit) - 1 : 0;
      if (best) {
        upto = read_lane(ownw, l);
        return best;
      }
      uint64_t last = sort_lanes<64>(p ? ~p : 0, lane);
      last = ~read_lane(last, 0);
      upto = read_lane(ownw, __ffsll((unsigned long long)__ballot(p == last)) - 1);
      return last;
    }
    // more: bit by bit of its place, the largest one up to which the row's sum is over the number
    uint64_t place = 0, total = 0;
    for (int bit = 63; bit >= 0; bit--) {
      const uint64_t test = place | 1ull << bit;
      uint64_t s = 0, w = 0;
      each([&](int c, float v) {
        if (v > -INFINITY && place_of(v, c) >= test) {
          const uint64_t own = weight_of(v, top, o);
          w += own;
          s += by_count ? 1 : own;
        }
      });
      s = group_sum<64>(s);
      w = group_sum<64>(w);
      if (s > number) {
        place = test;
        total = w;
      }
    }
    upto = total;
    return place;
  }
};

template <typename T, bool MASKED, int R>
__global__ __launch_bounds__(256, R > 16 ? 2 : 4) void sample_wave(const T* logits, int64_t stride, const uint8_t* mask,
    int64_t mask_stride, Settings a, int64_t* out, int64_t rows, int cols) {
  typedef WaveRow<T, MASKED, R> W;
  constexpr int N = W::N;
  __shared__ typename W::Lds lds[4];
  const int64_t r = ((int64_t)blockIdx.x + (int64_t)gridDim.x * blockIdx.y) * 4 + uniform((int)(threadIdx.x >> 6));
  if (r >= rows) return;
  typename W::Lds& g = lds[threadIdx.x >> 6];
  const Row o = uniform(row_settings(a, r));
  W w;
  w.lane = threadIdx.x & 63;
  const Source<T, MASKED> src{(const GLOBAL T*)(logits + r * stride),
      (const GLOBAL uint8_t*)(MASKED ? mask + r * mask_stride : nullptr), cols};
#pragma unroll
  for (int i = 0; i < W::V; i++) {  // whole vectors; the row's last elements one at a time
    const int c = (i * 64 + w.lane) * N;
    Vec16 v;
    typename Source<T, MASKED>::Bytes m;
    const bool whole = c + N <= cols;
    if (whole) {
      v = *(const GLOBAL Vec16*)(src.z + c);
      if (MASKED) m = *(const GLOBAL typename Source<T, MASKED>::Bytes*)(src.mask + c);
    }
    T raw[N];
    uint8_t open[N];
    __builtin_memcpy(raw, &v, 16);
    if (MASKED) __builtin_memcpy(open, &m, N);
#pragma unroll
    for (int n = 0; n < N; n++) w.x[i][n] = whole && !(MASKED && !open[n]) ? to_f32(raw[n]) : -INFINITY;
    if (!whole && c < cols)
#pragma unroll
      for (int n = 0; n < N; n++)
        if (c + n < cols) w.x[i][n] = src(c + n);
  }
  float top = -INFINITY, least = INFINITY;
  int wrong = 0;
  uint32_t n = 0;
  w.each([&](int, float v) {
    wrong |= v != v;
    n += v > -INFINITY;
    top = fmaxf(top, v);
    least = fminf(least, v > -INFINITY ? v : INFINITY);
  });
  w.top = uniform(group_max<64>(top));
  least = -group_max<64>(-least);
  uint64_t found = 0;
  if (!__ballot(wrong) && !o.nan && w.top > -INFINITY) {
    if (o.greedy) {
      w.each([&](int c, float v) {
        const uint64_t p = v == w.top ? place_of(v, c) : 0;
        found = p > found ? p : found;
      });
      found = read_lane(sort_lanes<64>(found, w.lane), 0);
    } else {
      // steps down to weights of e^-32 (with a T of next to nothing, to what float32 can tell apart), or to the row's least
      // logit
      const float range = w.top - least, reach = fminf(range, fmaxf((float)(32.0 / o.inv_t), range / 4096.0f));
      w.scale = uniform(reach > 0 ? fminf((float)WBINS / reach, 3e38f) : 0.0f);
      const bool counted = o.top_k > 0 && o.top_k < cols;
#pragma unroll
      for (int k = 0; k < WBINS / 64; k++) {
        g.weight[k * 64 + w.lane] = 0;
        g.count[k * 64 + w.lane] = 0;
      }
      wave_sync();
      uint64_t heavy = 0;  // the weight of those that min_p keeps: a leading part, like every setting's
      w.each([&](int, float v) {
        if (v == -INFINITY) return;
        const int b = w.step_of(v);
        const uint64_t own = weight_of(v, w.top, o);
        atomicAdd(&g.weight[b], (unsigned long long)own);
        if (counted) atomicAdd(&g.count[b], 1u);
        heavy += (double)own >= o.min_w ? own : 0;
      });
      wave_sync();
      uint64_t sum = 0;
      uint32_t sumc = 0;
#pragma unroll
      for (int k = 0; k < WBINS / 64; k++) {
        w.wbin[k] = g.weight[w.lane * (WBINS / 64) + k];
        w.cbin[k] = g.count[w.lane * (WBINS / 64) + k];
        sum += w.wbin[k];
        sumc += w.cbin[k];
      }
      uint64_t all = sum_lanes<64>(sum, w.lane);
      const uint32_t allc = sum_lanes<64>(sumc, w.lane);
      w.wbefore = all - sum;
      w.cbefore = allc - sumc;
      sum = read_lane(all, 63);
      n = __builtin_amdgcn_readlane(allc, 63);
      const bool cut = counted && (uint64_t)o.top_k < n;
#pragma unroll 1
      for (int stage = 0; stage < 3; stage++) {  // top_k's border, top_p's, the draw
        if ((stage == 0 && !cut) || (stage == 1 && o.top_p >= 1)) continue;
        if (stage == 2 && o.min_w > 0) {
          const uint64_t kept = group_sum<64>(heavy);
          sum = kept < sum ? kept : sum;
        }
        uint64_t upto;
        found = w.find(stage == 0, stage == 0 ? (uint64_t)o.top_k - 1 : stage == 1 ? border_of(o.top_p, sum)
            : target_of(o.u, sum), g, o, upto);
        sum = upto < sum ? upto : sum;
      }
    }
  }
  if (w.lane == 0) out[r] = found ? column_of(found) : -1;
}

// ---------------------------------------------------------------------------------------------- longer rows
// One block a row, two passes over it as a rule.  The first counts or weighs the categories by steps of their logit, the second
// lists and sorts those of the few steps in which a border and the drawn category lie.
//
// Steps are `scale` to a logit, counted down from HEAD at the largest logit of the row's first vectors (one for each thread),
// so that no pass is needed to find the row's own largest; should one lie above step 0, the pass is made again. With t = (first
// - v) scale + HEAD, step b = floor(t) and r = t - b, a category weighs exp(-r width) times what the top of its step does,
// width = 1 / (scale T) <= 0.022 (32 steps to a power of two; more where the first vectors are closer together).  A polynomial
// of degree 4 in r gives that to 5e-13 (four operations, 15 with the step's), and only the steps' sums are scaled by a proper
// exp.  Equal logits weigh the same, but not quite what a list's weigh: draw_by_steps takes care where that could show.
//
// 256 rows of 131072 bf16, a CU each: first vectors 3 us, first pass 21, sums of steps 2, second pass 10 (7 TB/s over all CUs),
// list 3, the rest 5.  What every thread does for the row as a whole is 16 waves' work: 100 operations take 0.7 us.
constexpr int BINS = 2048, HEAD = 512, DIGIT = 11;

struct Steps {
  double first, scale, inv, width;  // inv: 1 / scale; width: 1 / (scale T)
  double base;                 // first * scale + HEAD
  __device__ __forceinline__ double at(float v) const { return fma(-(double)v, scale, base); }
  // never falls as v falls; -1 above the steps, the last step takes all that lies below
  __device__ __forceinline__ static int of(double t) { return (int)floor(fmin(fmax(t, -1.0), (double)(BINS - 1))); }
  __device__ __forceinline__ int operator()(float v) const { return of(at(v)); }
  // whether all that the last step holds weighs less than 2^-47 of the row's largest: nothing
  __device__ __forceinline__ bool past() const { return (BINS - 1 - HEAD) * width >= 33.0; }
  // all logits of steps b0 .. b1 (and a few others) lie within `half` of `mid`
  __device__ __forceinline__ void around(int b0, int b1, float& mid, float& half) const {
    const double d0 = (double)(HEAD - b0) * inv, d1 = (double)(HEAD - b1 - 1) * inv;
    const double slack = 4e-7 * (fabs(first) + fabs(d0) + fabs(d1));
    mid = (float)(first + 0.5 * (d0 + d1));
    half = b0 > b1 ? -1.0f : b1 == BINS - 1 ? INFINITY : (float)(0.5 * (d0 - d1) + slack);
  }
};

template <int NT>
struct Long {
  static constexpr int LISTED = NT == 1024 ? 2048 : 1024;  // categories of one list (with the rest, within 64 KB)
  List<LISTED> l;
  unsigned long long weight[BINS + 1 + 64];
  uint32_t count[BINS + 1 + 64];
  unsigned long long wave[NT / 64], ubuf[NT / 64];
  unsigned long long place, before, upto;  // find: the category found; the weight before it and with it
  float fbuf[2][NT / 64];
  unsigned long long tail;
  int listed, step, seen, total;
  // what the functions below, which are not inlined (each is called from several places), work on
  const void* z;
  const uint8_t* mask;
  int cols;
  float top;
  Row o;
  Steps steps;
};
static_assert(sizeof(Long<1024>) < 64000 && sizeof(Long<256>) < 64000, "dynamic LDS of a launch");
template <int NT>
__device__ __forceinline__ Long<NT>& shared() {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  return *(Long<NT>*)lds;
}
template <typename T, bool MASKED, int NT>
__device__ __forceinline__ Source<T, MASKED> shared_source() {
  const Long<NT>& g = shared<NT>();
  return Source<T, MASKED>{uniform((const T*)g.z), MASKED ? uniform(g.mask) : nullptr, uniform(g.cols)};
}
// exclusive sums of `mine` over the block's threads, in order; `all` gets the sum of all
template <int NT>
__device__ __forceinline__ uint64_t block_before(uint64_t mine, unsigned long long* buf, uint64_t& all) {
  const uint64_t run = sum_lanes<64>(mine, threadIdx.x & 63);
  if ((threadIdx.x & 63) == 63) buf[threadIdx.x >> 6] = run;
  __syncthreads();
  constexpr int W = NT / 64;
  const uint64_t waves = sum_lanes<W>((uint64_t)buf[threadIdx.x % W], threadIdx.x % W);
  const int wave = uniform((int)threadIdx.x >> 6);
  all = read_lane(waves, W - 1);
  __syncthreads();
  return (wave ? read_lane(waves, wave - 1) : 0) + run - mine;
}

// The first pass: counts and / or mantissas of every step.  Returns what only the row as a whole shows: its largest logit
// (which tells whether one lay above the steps: those went to step 0, and the pass is made again), the number of its
// categories (COUNT), and in `seen` a NaN.  The last step's count is what the others leave, its weight is g.tail.
template <int NT, bool COUNT, bool WEIGH, typename S>
__device__ __forceinline__ void weigh_steps(const S& src, const Steps& steps, double one, Long<NT>& g, float& top,
    int& categories, int& seen) {
  const bool far = WEIGH && !steps.past();
  // exp(-r width) = 1 + r (c1 + r (c2 + r (c3 + r c4))), exact at r = 0: its series with the term of r^5 put into the lower
  // ones by r^4 = 2 r^3 - 5/4 r^2 + r/4 - 1/128, which Chebyshev's polynomial of degree 4 on 0 .. 1 gives to 1/128; 5e-13 in
  // all. In units of 2^-s, and with 2^52 added, which leaves the whole number in the low bits
  const double w = steps.width, e5 = -w * w * w * w * w / 120;
  const double c1 = uniform(one * (-w - e5 / 128)), c2 = uniform(one * (w * w / 2 + e5 / 4)),
      c4 = uniform(one * (w * w * w * w / 24 + e5 * 2));
  // an operation takes one operand from scalar registers: the others stay in vector registers
  double c3 = one * (-w * w * w / 6 - e5 * 1.25), c0 = one + 4503599627370496.0, base = steps.base;
  asm volatile("" : "+v"(c3), "+v"(c0), "+v"(base));
  // where the weight of what lies below the steps goes, each lane's its own
  const uint32_t spare = BINS + 1 + (threadIdx.x & 63);
  auto weigh = [&](float v) {
    top = fmaxf(top, v);
    seen |= v != v;
    if (COUNT) categories += v > -INFINITY;
    const double t = fma(-(double)v, steps.scale, base);
    uint32_t at;  // by the instruction, which gives 0 for less than 0 and NaN, the most for more: in C++ that is undefined
    asm("v_cvt_u32_f64 %0, %1" : "=v"(at) : "v"(t));
    const uint32_t b = at < BINS - 1 ? at : spare;
    if (COUNT) atomicAdd(&g.count[b], 1u);
    if (WEIGH) {
      const double r = __builtin_amdgcn_fract(t);
      double e = fma(r, c4, c3);
      e = fma(e, r, c2);
      e = fma(e, r, c1);
      e = fma(e, r, c0);
      atomicAdd(&g.weight[b], (unsigned long long)__double_as_longlong(e) & 0xfffffffffffffull);
    }
  };
  auto below = [&](float v) {  // where the last step can still weigh: its categories
    const double t = steps.at(v);
    if (!(t >= (double)(BINS - 1)) || v == -INFINITY) return;
    const double e = exp_neg(fmax(((double)(BINS - 1) - t) * steps.width, -1000.0));
    atomicAdd(&g.tail, (unsigned long long)__double_as_longlong(fma(e, one, 4503599627370496.0)) & 0xfffffffffffffull);
  };
  src.template vectors<NT, 2>(
      [&](int c, const float* v) {
        float least = v[0];
#pragma unroll
        for (int i = 0; i < S::N; i++) {
          weigh(v[i]);
          if (WEIGH) least = fminf(least, v[i]);
          __builtin_amdgcn_sched_barrier(0);  // one after the other: several at once spill registers
        }
        if (far && steps.at(least) >= (double)(BINS - 1))
#pragma unroll 1
          for (int i = 0; i < S::N; i++) below(src(c + i));
      },
      [&](int, float v) {
        weigh(v);
        if (far) below(v);
      });
}

// the step in which the running sum passes `number`
template <int NT, typename V>
__device__ __forceinline__ int step_of(Long<NT>& g, const V* sums, uint64_t number) {
  for (int b = threadIdx.x; b < BINS; b += NT)
    if (sums[b] <= number && number < sums[b + 1]) g.step = b;
  __syncthreads();
  const int b = g.step;
  __syncthreads();
  return b < 0 ? 0 : b < BINS ? b : BINS - 1;
}

// Lists and sorts the categories of steps a0 .. a1 and b0 .. b1.  False, for all threads, where they are too many.
template <typename T, bool MASKED, int NT>
__device__ __noinline__ bool list_steps(int a0, int a1, int b0, int b1) {
  Long<NT>& g = shared<NT>();
  const Source<T, MASKED> src = shared_source<T, MASKED, NT>();
  const Steps steps{uniform(g.steps.first), uniform(g.steps.scale), uniform(g.steps.inv), 0.0, uniform(g.steps.base)};
  a0 = uniform(a0), a1 = uniform(a1), b0 = uniform(b0), b1 = uniform(b1);
  if (threadIdx.x == 0) g.listed = 0;
  __syncthreads();
  // those near the wanted steps are listed; the few that lie in a step beside them are then taken out, in parallel (looked at
  // where they are found, each held up its wave: 37 x 50021 took 2.7 us longer)
  float am, ah, bm, bh;
  steps.around(a0, a1, am, ah);
  steps.around(b0, b1, bm, bh);
  const bool below = (a1 == BINS - 1 && a0 > 0 && a0 <= a1) || (b1 == BINS - 1 && b0 > 0 && b0 <= b1);
  auto take = [&](int c, float v) {
    if (!(fabsf(v - am) <= ah || fabsf(v - bm) <= bh)) return;
    const int i = atomicAdd(&g.listed, 1);
    if (i < Long<NT>::LISTED) g.l.place[i] = place_of(v, c);
  };
  if (below) {
    // the last step, which has no lower end to be near to, but not all: each category's step (rare: it can still weigh only
    // where the first vectors are much closer together than the rest)
    src.template each<NT>([&](int c, float v) {
      const int b = steps(v);
      if (v > -INFINITY && ((b >= a0 && b <= a1) || (b >= b0 && b <= b1))) {
        const int i = atomicAdd(&g.listed, 1);
        if (i < Long<NT>::LISTED) g.l.place[i] = place_of(v, c);
      }
    });
  } else {
    src.template vectors<NT, 4>(
        [&](int c, const float* v) {
          float a = fabsf(v[0] - am), b = fabsf(v[0] - bm);
#pragma unroll
          for (int i = 1; i < src.N; i++) {
            a = fminf(a, fabsf(v[i] - am));
            b = fminf(b, fabsf(v[i] - bm));
          }
          if (!(a <= ah || b <= bh)) return;
#pragma unroll
          for (int i = 0; i < src.N; i++) take(c + i, v[i]);
        },
        take);
  }
  __syncthreads();
  const int n = uniform(g.listed);
  __syncthreads();  // all have read it: the next list begins by clearing it
  if (n > Long<NT>::LISTED) return false;
  for (int i = threadIdx.x; i < n; i += NT) {
    const float v = logit_of(g.l.place[i]);
    const int b = steps(v);
    if (v > -INFINITY && ((b >= a0 && b <= a1) || (b >= b0 && b <= b1))) continue;
    g.l.place[i] = i;  // sorted behind the others
    atomicSub(&g.listed, 1);
  }
  sort_list<NT>(g.l, n, uniform(g.top), uniform(g.o));
  return true;
}

// adds a category to a bin; a wave whose categories all go to one bin adds them up first (one value in many places
// would otherwise be 64 turns at the same address)
template <int NT>
__device__ __forceinline__ void add(Long<NT>& f, int b, uint64_t w) {
  const int b0 = __builtin_amdgcn_readfirstlane(b);
  if (__all(b == b0)) {
    const uint64_t active = __ballot(1);
    const uint64_t w0 = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(w >> 32))
        << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)w);
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

// Of rows that the steps do not tell apart (more than a list of equal or nearly equal logits): the category at which a sum
// passes a number, digit by digit of its place.  Each pass over the row adds up its categories by the next 11 bits,
// among those that share the bits found so far.  Found is the first category (in rank) at which the running sum of
// weights (or, by_count, of ones) is over `number`, which the sum of all of them is.  f.place, f.before and f.upto (sums of
// weights) are set for every thread.
template <int NT, typename S>
__device__ __forceinline__ void find(bool by_count, const S& src, float top, const Row& o, uint64_t number, Long<NT>& f) {
  const int low = 32 - __clz((unsigned)(src.cols - 1));  // bits of an index
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
    src.template each<NT>([&](int c, float v) {
      const uint64_t p = place_of(v, c);
      if (v > -INFINITY && (p & known) == place) add(f, (int)(p >> sh) & (bins - 1), weight_of(v, top, o));
    });
    __syncthreads();
    // thread i sums the i-th share of the bins from the top, then the bin is where the sum passes the number
    const int each = (bins + NT - 1) / NT, last = bins - 1 - (int)threadIdx.x * each;
    uint64_t own = 0, ownw = 0, all;
    for (int i = 0; i < each && last - i >= 0; i++) {
      own += by_count ? (uint64_t)f.count[last - i] : (uint64_t)f.weight[last - i];
      ownw += f.weight[last - i];
    }
    uint64_t sum = before + block_before<NT>(own, f.wave, all), sumw = wbefore + block_before<NT>(ownw, f.ubuf, all);
    if (sum <= number && number < sum + own) {  // one thread's
      for (int i = 0; i < each; i++) {
        const uint64_t val = by_count ? (uint64_t)f.count[last - i] : (uint64_t)f.weight[last - i];
        if (number < sum + val) {
          f.place = place | (uint64_t)(last - i) << sh;
          f.before = sum;
          f.upto = sumw;
          break;
        }
        sum += val;
        sumw += f.weight[last - i];
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

// the drawn category's place, with nothing but `find`
template <typename T, bool MASKED, int NT>
__device__ __noinline__ uint64_t draw_by_digits() {
  Long<NT>& f = shared<NT>();
  const Source<T, MASKED> src = shared_source<T, MASKED, NT>();
  const float top = uniform(f.top);
  const Row o = uniform(f.o);
  // categories, their weight, the weight of those that min_p keeps (a leading part, as every setting's)
  uint64_t n = 0, all = 0, most = 0;
  src.template each<NT>([&](int, float v) {
    const uint64_t w = v > -INFINITY ? weight_of(v, top, o) : 0;
    n += v > -INFINITY;
    all += w;
    most += (double)w >= o.min_w ? w : 0;
  });
  n = block_sum<NT>((unsigned long long)n, f.ubuf);
  __syncthreads();
  all = block_sum<NT>((unsigned long long)all, f.ubuf);
  __syncthreads();
  most = block_sum<NT>((unsigned long long)most, f.ubuf);
  __syncthreads();
  uint64_t sum = all;
  for (int stage = 0;; stage++) {  // top_k's border, top_p's, the draw
    if (stage == 0 && (o.top_k <= 0 || (uint64_t)o.top_k >= n)) continue;
    if (stage == 1 && o.top_p >= 1) continue;
    if (stage == 2 && most < sum) sum = most;
    find<NT>(stage == 0, src, top, o, stage == 0 ? (uint64_t)o.top_k - 1 : stage == 1 ? border_of(o.top_p, sum)
        : target_of(o.u, sum), f);
    if (stage == 2) return f.place;
    sum = f.upto;
    __syncthreads();
  }
}

// The drawn category's place from the steps' sums; 0 where a list is too short for it.
template <typename T, bool MASKED, int NT>
__device__ __forceinline__ uint64_t draw_by_steps(const Steps& steps, float top, const Row& o, bool counted, bool weighed) {
  Long<NT>& g = shared<NT>();
  const uint64_t n = counted ? g.count[BINS] : 0, all = weighed ? g.weight[BINS] : 0;
  const bool cut = counted && (uint64_t)o.top_k < n;
  uint64_t sum = all;
  if (counted && !weighed) {  // top_k, and few: one list of all that it keeps (of all, where there are fewer)
    int to = cut ? step_of(g, g.count, (uint64_t)o.top_k - 1) : BINS - 1;
    if (to == BINS - 1 && steps.past()) to--;  // what lies below weighs nothing
    if (!list_steps<T, MASKED, NT>(0, to, 0, -1) || !g.listed) return 0;
    return draw_from<NT>(g.l, g.listed, o);
  }
  const int b = cut ? step_of(g, g.count, (uint64_t)o.top_k - 1) : BINS - 1;
  const bool shorter = cut && !(b == BINS - 1 && steps.past());
  if (shorter) {
    if (!list_steps<T, MASKED, NT>(b, b, 0, -1)) return 0;
    const int i = (int)(o.top_k - 1 - g.count[b]);
    if (!g.listed) return 0;
    sum = g.weight[b] + g.l.upto[i < g.listed ? i : g.listed - 1];
    sum = sum < all ? sum : all;  // (the steps' weights and their categories' differ by roundings)
    __syncthreads();
  }
  // the steps of the border behind which nothing is kept: top_p's, or, where it comes first, min_p's (its logit is known
  // but for rounding: three steps)
  int b0 = BINS, b1 = -1;
  if (o.top_p < 1) b0 = b1 = step_of(g, g.weight, border_of(o.top_p, sum));
  if (o.min_w > 0) {
    double least = o.min_p;
    asm volatile("" : "+v"(least));  // the logarithm stays here: every row would pay for it ahead of the passes
    const double lowest = (double)top + (least < 1 ? log(fmax(least, 1e-300)) / o.inv_t : 0.0);
    const int m = Steps::of((steps.first - lowest) * steps.scale + HEAD);
    const int m0 = m > 1 ? m - 1 : 0, m1 = m + 1 < BINS ? m + 1 : BINS - 1;
    if (g.weight[m0] >= sum) {
      // all that is kept weighs more than that: no border (its list would often be the last step's, all that lies below)
    } else if (b1 < 0 || m1 < b0) {
      b0 = m0;
      b1 = m1;
    } else if (m0 <= b1) {
      b0 = m0 < b0 ? m0 : b0;
      b1 = m1 > b1 ? m1 : b1;
    }
  }
  const bool border = b1 >= 0;
  // the draw's step is known but for how much of the border's steps is kept
  int t0 = step_of(g, g.weight, target_of(o.u, border && g.weight[b0] ? (uint64_t)g.weight[b0] : border ? 1 : sum));
  int t1 = border ? step_of(g, g.weight, target_of(o.u, (uint64_t)g.weight[b1 + 1] < sum ? (uint64_t)g.weight[b1 + 1] : sum))
      : t0;
  for (int turn = 0; turn < 2; turn++) {
    // first both in one list, then, should they be too many, the border alone and the one step of the draw
    if (turn && !border) return 0;
    const bool together = turn == 0;
    const bool joined = together && border && b0 <= t1 + 1;  // one stretch of steps
    if (together ? list_steps<T, MASKED, NT>(t0, border && t1 > b1 ? b1 : t1, b0, b1)
        : list_steps<T, MASKED, NT>(b0, b1, 0, -1)) {
      int split = 0;  // where the border's steps begin
      uint64_t base = g.weight[border ? (joined ? (t0 < b0 ? t0 : b0) : b0) : t0];
      const uint64_t tbase = joined ? base : g.weight[t0];
      if (together && border && !joined) {
        if (threadIdx.x == 0) g.step = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < g.listed; i += NT)
          if (steps(logit_of(g.l.place[i])) <= t1) atomicMax(&g.step, i + 1);
        __syncthreads();
        split = g.step;
        __syncthreads();
      }
      // Where the list holds all that weighs, the row's sum is the list's, in which equal logits weigh exactly as much.  The
      // steps' sums are off by up to 5e-13 of themselves: a share of 256 equal logits' weight could end one of them later.
      if (together && g.weight[joined ? (t0 < b0 ? t0 : b0) : t0] == 0 && !shorter &&
          g.weight[(border ? b1 : t1) + 1] == g.weight[BINS] && (!border || joined || g.weight[t1 + 1] == g.weight[b0]) &&
          g.listed)
        sum = g.l.upto[g.listed - 1];
      const uint64_t off = split ? g.l.upto[split - 1] : 0;  // of the list's sum, what belongs to the draw's steps
      if (border) {
        int end = g.listed;  // what is kept of the list
        if (o.top_p < 1) {
          const uint64_t number = border_of(o.top_p, sum);
          end = number < base ? split : first_over<NT>(g.l, end, number - base + off) + 1;
        }
        if (o.min_w > 0) {
          if (threadIdx.x == 0) g.step = 0;
          __syncthreads();
          for (int i = threadIdx.x; i < end; i += NT)
            if ((double)(g.l.upto[i] - (i ? g.l.upto[i - 1] : 0)) >= o.min_w) atomicMax(&g.step, i + 1);
          __syncthreads();
          end = g.step;
          __syncthreads();
        }
        const uint64_t kept = base + (end > split ? g.l.upto[end - 1] - off : 0);
        sum = kept < sum ? kept : sum;
        if (!sum) return 0;
      }
      const uint64_t number = target_of(o.u, sum);
      if (together) {
        const int n = border && !joined ? split : g.listed;
        return n ? g.l.place[first_over<NT>(g.l, n, number < tbase ? 0 : number - tbase)] : 0;
      }
      const int b = step_of(g, g.weight, number);
      if (!list_steps<T, MASKED, NT>(b, b, 0, -1) || !g.listed) return 0;
      return g.l.place[first_over<NT>(g.l, g.listed, number - g.weight[b])];
    }
  }
  return 0;
}

template <typename T, bool MASKED, int NT>
__global__ __launch_bounds__(NT, 4) void sample_long(const T* logits, int64_t stride, const uint8_t* mask,
    int64_t mask_stride, Settings a, int64_t* out, int64_t rows, int cols) {
  Long<NT>& g = shared<NT>();
  const int64_t r = blockIdx.x + (int64_t)gridDim.x * blockIdx.y;
  if (r >= rows) return;
  const Source<T, MASKED> src{(const GLOBAL T*)(logits + r * stride),
      (const GLOBAL uint8_t*)(MASKED ? mask + r * mask_stride : nullptr), cols};
  const Row o = uniform(row_settings(a, r));
  float top = -INFINITY;
  int wrong = o.nan;
  uint64_t found = 0;
  if (o.greedy || wrong) {
    unsigned long long best = 0;
    auto larger = [&](int c, float v) {
      wrong |= v != v;
      const unsigned long long p = v > -INFINITY ? place_of(v, c) : 0;
      best = p > best ? p : best;
    };
    src.template vectors<NT, 2>(
        [&](int c, const float* v) {
#pragma unroll
          for (int i = 0; i < src.N; i++) larger(c + i, v[i]);
        },
        larger);
    best = sort_lanes<64>(best, threadIdx.x & 63);  // the largest to lane 0
    if ((threadIdx.x & 63) == 0) g.wave[threadIdx.x >> 6] = best;
    wrong = __syncthreads_or(wrong);
    for (int w = 0; w < NT / 64; w++) best = g.wave[w] > best ? g.wave[w] : best;
    if (threadIdx.x == 0) out[r] = wrong || !best ? -1 : column_of(best);
    return;
  }
  for (int b = threadIdx.x; b < BINS; b += NT) {
    g.count[b] = 0;
    g.weight[b] = 0;
  }
  // the first vectors: where the steps start and how narrow they can be
  const Source<T, MASKED> start{src.z, src.mask, cols < NT * (16 / (int)sizeof(T)) ? cols : NT * (16 / (int)sizeof(T))};
  float first = -INFINITY, least = INFINITY;
  int open = 0;
  auto look = [&](int, float v) {
    first = fmaxf(first, v);
    least = fminf(least, v > -INFINITY ? v : INFINITY);
    open += v > -INFINITY;
  };
  start.template vectors<NT, 1>(
      [&](int c, const float* v) {
#pragma unroll
        for (int i = 0; i < src.N; i++) look(c + i, v[i]);
      },
      look);
  first = group_max<64>(first);
  least = -group_max<64>(-least);
  open = group_sum<64>(open);
  if ((threadIdx.x & 63) == 0) {
    g.fbuf[0][threadIdx.x >> 6] = first;
    g.fbuf[1][threadIdx.x >> 6] = least;
    g.wave[threadIdx.x >> 6] = open;
  }
  __syncthreads();
  constexpr int W = NT / 64;
  first = group_max<W>(g.fbuf[0][threadIdx.x % W]);
  least = -group_max<W>(-g.fbuf[1][threadIdx.x % W]);
  open = group_sum<W>((int)g.wave[threadIdx.x % W]);
  const bool counted = o.top_k > 0 && o.top_k < cols, weighed = !counted || o.top_k > Long<NT>::LISTED / 2;
  for (int turn = 0; turn < 2; turn++) {
    // a power of two of the weight in 32 steps; narrower where the first vectors (enough of them that are not barred) lie
    // within 1024 T counts as 2^-35 |first| at least: the next float32 below would still weigh e^-2048, and first * scale stays
    // below 2^41
    // (to some 2^-20: they choose the scale, whose own bits are what counts)
    const double most = 34359738368.0 * __builtin_amdgcn_rcp(fabs((double)first)), inv_t = fmin(o.inv_t, most);
    const double close = open < 256 ? 0.0 : 1024.0 * __builtin_amdgcn_rcp((double)first - (double)least);
    const double wanted = fmin(fmin(fmax(fmax(32.0 * 1.4426950408889634 * inv_t, close), 1e-30), 64.0 * most), 1e300);
    Steps steps;
    steps.first = uniform(first);
    steps.scale = uniform(__longlong_as_double(__double_as_longlong(wanted) >> 37 << 37));  // 16 bits: first * scale is exact
    steps.inv = uniform(1.0 / steps.scale);
    steps.width = uniform(inv_t * steps.inv);
    steps.base = uniform(steps.first * steps.scale + HEAD);
    if (turn)
      for (int b = threadIdx.x; b < BINS; b += NT) {
        g.count[b] = 0;
        g.weight[b] = 0;
      }
    if (threadIdx.x == 0) g.tail = g.total = 0;
    __syncthreads();
    int seen = 0;
    top = -INFINITY;
    int categories = 0;
    if (!(first > -INFINITY && first < INFINITY)) {  // nothing to start from, or nothing but infinity counts
      for (int c = threadIdx.x; c < cols; c += NT) {
        const float v = src(c);
        seen |= v != v;
        top = fmaxf(top, v);
      }
    } else if (!weighed) {
      weigh_steps<NT, true, false>(src, steps, o.one, g, top, categories, seen);
    } else if (!counted) {
      weigh_steps<NT, false, true>(src, steps, o.one, g, top, categories, seen);
    } else {
      weigh_steps<NT, true, true>(src, steps, o.one, g, top, categories, seen);
    }
    if (threadIdx.x == 0) {
      g.z = (const void*)src.z;
      g.mask = (const uint8_t*)src.mask;
      g.cols = cols;
      g.o = o;
      g.steps = steps;
      g.seen = 0;
    }
    __syncthreads();
    if (seen) atomicOr(&g.seen, seen);
    if (counted) {
      categories = group_sum<64>(categories);
      if ((threadIdx.x & 63) == 0) atomicAdd(&g.total, categories);
    }
    top = block_max<NT>(top, g.fbuf[0]);  // (a barrier)
    if (threadIdx.x == 0) g.top = top;
    seen = uniform(g.seen);
    if (seen || top == -INFINITY) break;
    if (!(first > -INFINITY && first < INFINITY) || steps.at(top) < 0) {
      // again from the row's largest logit; rows of infinities are left to the digits
      if (turn == 0 && top < INFINITY) {
        least = fminf(least, top);
        first = top;
        __syncthreads();
        continue;
      }
      __syncthreads();
      found = draw_by_digits<T, MASKED, NT>();
      break;
    }
    // the steps' mantissas to weights; counts and weights to sums of the steps before
    constexpr int EACH = BINS / NT;
    const int b0 = threadIdx.x * EACH;
    uint64_t all;
    if (weighed) {
      const double shift = ((double)top - steps.first) * inv_t;
      uint64_t sum = 0;
      for (int i = 0; i < EACH; i++) {
        const uint64_t m = b0 + i < BINS - 1 ? g.weight[b0 + i] : g.tail;
        const uint64_t w = m ? (uint64_t)rint((double)m * exp_neg(fmax((double)(HEAD - b0 - i) * steps.width - shift,
            -1000.0))) : 0;
        g.weight[b0 + i] = sum;
        sum += w;
      }
      sum = block_before<NT>(sum, g.wave, all);
      for (int i = 0; i < EACH; i++) g.weight[b0 + i] += sum;
      if (threadIdx.x == 0) g.weight[BINS] = all;
    }
    if (counted) {
      uint32_t sum = 0;
      for (int i = 0; i < EACH; i++) {
        const uint32_t c = g.count[b0 + i];
        g.count[b0 + i] = sum;
        sum += c;
      }
      sum = (uint32_t)block_before<NT>(sum, g.ubuf, all);
      for (int i = 0; i < EACH; i++) g.count[b0 + i] += sum;
      if (threadIdx.x == 0) g.count[BINS] = (uint32_t)g.total;
    }
    __syncthreads();
    found = draw_by_steps<T, MASKED, NT>(steps, top, o, counted, weighed);
    __syncthreads();
    if (!found) found = draw_by_digits<T, MASKED, NT>();
    break;
  }
  if (threadIdx.x == 0) out[r] = found ? column_of(found) : -1;
}

int shift_of(int64_t cols) {  // the sum of cols weights of at most 2^s stays below 2^63
  int s = 51;
  while (s > 0 && (cols - 1) >> (62 - s)) s--;
  return s;
}

// Up to 64 categories a group of lanes holds a row, up to 2048 a wave, longer rows take a block: of 256 threads (three to a
// CU by their LDS) where there are rows enough or the row has little for more, else of 1024 (one to a CU).  Measured with
// top_p 0.9, us with 256 / 1024 threads: rows of 2100 fp32 16 / 14 for 16 of them, 19 / 27 for 512, 32 / 51 for 1024; of 9001
// 22 / 18 for 256, 25 / 33 for 512, 47 / 62 for 1024; of 65536 86 / 48 for 256, 83 / 87 for 512, 145 / 159 for 1024; of 131072
// 131 / 71, 148 / 133 and 300 / 261.  So the one border could lie at 512 rows, and rows up to 4096 would gain 2 us by 1024
// threads where they are few.
template <typename T, bool MASKED>
void launch(const fm_sample_args& a) {
  const Settings s{a.temperature, a.top_p, a.min_p, a.top_k, a.temperature_rows, a.top_p_rows, a.min_p_rows, a.top_k_rows, a.u,
      a.u_dtype == FM_DTYPE_F64, shift_of(a.cols)};
  hipStream_t st = (hipStream_t)a.stream;
  const int cols = (int)a.cols;
  auto blocks = [&](int rows_each) {
    const int64_t n = (a.rows + rows_each - 1) / rows_each;
    return (int)(n < (1 << 20) ? n : 1 << 20);
  };
  const dim3 fours(blocks(4), (unsigned)((a.rows + (1 << 22) - 1) >> 22));
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
  else if (cols <= 512)
    sample_wave<T, MASKED, 8><<<fours, 256, 0, st>>>(ARGS);
  else if (cols <= 1024)
    sample_wave<T, MASKED, 16><<<fours, 256, 0, st>>>(ARGS);
  else if (cols <= 2048)
    sample_wave<T, MASKED, 32><<<fours, 256, 0, st>>>(ARGS);
  else if (cols <= 4096 || (a.rows >= 1024 && cols <= 65536))
    sample_long<T, MASKED, 256><<<each, 256, sizeof(Long<256>), st>>>(ARGS);
  else
    sample_long<T, MASKED, 1024><<<each, 1024, sizeof(Long<1024>), st>>>(ARGS);
#undef ARGS
}
}  // namespace
}  // namespace fm

using namespace fm;
extern "C" {
int64_t fm_sample_workspace(int64_t, int64_t) { return 0; }

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
