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
  double inv_t, top_p, min_w, u, one;
  int64_t top_k;
  bool greedy, nan;
};

__device__ __forceinline__ Row row_settings(const Settings& a, int64_t r) {
  Row o;
  const double t = a.temperature_rows ? (double)a.temperature_rows[r] : a.temperature;
  const double m = a.min_p_rows ? (double)a.min_p_rows[r] : a.min_p;
  o.top_p = a.top_p_rows ? (double)a.top_p_rows[r] : a.top_p;
  o.top_k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
  o.u = a.u64 ? ((const double*)a.u)[r] : (double)((const float*)a.u)[r];
  o.nan = t != t || m != m || o.top_p != o.top_p || o.u != o.u;
  o.greedy = t <= 0;
  o.inv_t = 1.0 / t;
  o.one = (double)(1ull << a.shift);
  o.min_w = ldexp(fmin(m, 1.0), a.shift);
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

// ---------------------------------------------------------------------------------------------- rows of any length
// One block a row.  The category at which a sum passes a number is found digit by digit of its place: each pass over
// the row adds up its categories by the next 11 bits, among those that share the bits found so far.
constexpr int NT = 256, DIGIT = 11, BINS = 1 << DIGIT;

struct Find {
  uint32_t count[BINS];
  unsigned long long weight[BINS];
  unsigned long long wave[NT / 64];
  unsigned long long place, before, upto;  // the category found; the sum before it and with it
  float fbuf[NT / 64];
  unsigned long long ubuf[NT / 64];
};

template <typename T>
struct Source {
  const T* z;
  const uint8_t* mask;
  int cols;
  // logit of column c; -inf where it is barred
  __device__ __forceinline__ float operator()(int c) const { return mask && !mask[c] ? -INFINITY : to_f32(z[c]); }
};

// The first category (in rank) at which the running sum of weights (or, BY_COUNT, of ones) is over `number`, which the
// sum of all of them is.  f.place, f.before and f.upto (sums of weights) are set for every thread.
template <bool BY_COUNT, typename T>
__device__ void find(const Source<T>& src, float top, const Row& o, uint64_t number, Find& f) {
  const int low = 64 - __clz((unsigned)(src.cols > 1 ? src.cols - 1 : 1)) - 32;  // bits of an index
  uint64_t place = 0, known = 0, before = 0, wbefore = 0;
  int at = 64;
  while (at > 32 || (at > 0 && low > 0)) {
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
    for (int c = threadIdx.x; c < src.cols; c += NT) {
      const float v = src(c);
      if (v == -INFINITY) continue;
      const uint64_t p = (uint64_t)key_of(v) << 32 | (uint32_t)~c;
      if ((p & known) != place) continue;
      const int b = (int)(p >> sh) & (bins - 1);
      atomicAdd(&f.count[b], 1u);
      atomicAdd(&f.weight[b], (unsigned long long)weight_of(v, top, o));
    }
    __syncthreads();
    // thread i sums the i-th share of the bins from the top, then the bin is where the sum passes the number
    const int each = (bins + NT - 1) / NT, first = bins - 1 - (int)threadIdx.x * each;
    uint64_t own = 0, ownw = 0;
    for (int i = 0; i < each && first - i >= 0; i++) {
      own += BY_COUNT ? (uint64_t)f.count[first - i] : (uint64_t)f.weight[first - i];
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
        const uint64_t val = BY_COUNT ? (uint64_t)f.count[first - i] : (uint64_t)f.weight[first - i];
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
  const uint64_t w = weight_of(of_key((uint32_t)(place >> 32)), top, o);
  if (threadIdx.x == 0) {
    f.place = place;
    f.before = wbefore;
    f.upto = wbefore + w;
  }
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(NT) void sample_any(const T* logits, int64_t stride, const uint8_t* mask, int64_t mask_stride, Settings a, int64_t* out,
                                                 int64_t rows, int cols) {
  __shared__ Find f;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const Source<T> src{logits + r * stride, mask ? mask + r * mask_stride : nullptr, cols};
    const Row o = row_settings(a, r);
    float top = -INFINITY;
    int wrong = o.nan;
    for (int c = threadIdx.x; c < cols; c += NT) {
      const float v = src(c);
      wrong |= v != v;
      top = fmaxf(top, v);
    }
    top = block_max<NT>(top, f.fbuf);
    wrong = __syncthreads_or(wrong);
    int64_t token = -1;
    if (!wrong && top > -INFINITY) {
      uint64_t place;
      if (o.greedy) {
        find<true>(src, top, o, 0, f);
        place = f.place;
      } else {
        uint64_t sum, last = 0;  // what is kept: places from `last` up, and their weight
        if (o.top_k > 0 && o.top_k < cols) {
          uint64_t n = 0;
          for (int c = threadIdx.x; c < cols; c += NT) n += src(c) > -INFINITY;
          n = block_sum<NT>((unsigned long long)n, f.ubuf);
          __syncthreads();
          find<true>(src, top, o, (uint64_t)o.top_k < n ? (uint64_t)o.top_k - 1 : n - 1, f);
          last = f.place;
          sum = f.upto;
        } else {
          uint64_t n = 0;
          for (int c = threadIdx.x; c < cols; c += NT) {
            const float v = src(c);
            n += v > -INFINITY ? weight_of(v, top, o) : 0;
          }
          sum = block_sum<NT>((unsigned long long)n, f.ubuf);
          __syncthreads();
        }
        if (o.top_p < 1) {
          find<false>(src, top, o, border_of(o.top_p, sum), f);
          last = f.place;
          sum = f.upto;
          __syncthreads();
        }
        if (o.min_w > 0) {
          uint64_t n = 0;
          for (int c = threadIdx.x; c < cols; c += NT) {
            const float v = src(c);
            if (v == -INFINITY || ((uint64_t)key_of(v) << 32 | (uint32_t)~c) < last) continue;
            const uint64_t w = weight_of(v, top, o);
            n += (double)w >= o.min_w ? w : 0;
          }
          sum = block_sum<NT>((unsigned long long)n, f.ubuf);
          __syncthreads();
        }
        find<false>(src, top, o, target_of(o.u, sum), f);
        place = f.place;
      }
      token = (int64_t)(uint32_t)~(uint32_t)place;
    }
    if (threadIdx.x == 0) out[r] = token;
    __syncthreads();
  }
}

int shift_of(int64_t cols) {  // the sum of cols weights of at most 2^s stays below 2^63
  int s = 51;
  while (s > 0 && (cols - 1) >> (62 - s)) s--;
  return s;
}

template <typename T>
void launch(const fm_sample_args& a) {
  Settings s{a.temperature, a.top_p, a.min_p, a.top_k, a.temperature_rows, a.top_p_rows, a.min_p_rows, a.top_k_rows, a.u, a.u_dtype == FM_DTYPE_F64, shift_of(a.cols)};
  sample_any<T><<<(int)(a.rows < (1 << 20) ? a.rows : 1 << 20), NT, 0, (hipStream_t)a.stream>>>((const T*)a.logits, a.stride, a.mask, a.mask_stride, s, a.out,
                                                                                                a.rows, (int)a.cols);
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
      with_type(a->dtype, [&](auto tag) { launch<typename decltype(tag)::type>(*a); });
    return on.status("sample");
  });
}
}
