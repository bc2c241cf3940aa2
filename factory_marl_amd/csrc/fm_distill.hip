// fm_distill.hip -- distillation from a teacher's top logits (include/factorysim.h fm_distill_*).
//
//   loss = T^2 sum over the listed entries of p (log p - log q[index]),  q = softmax(z / T),  p = softmax(teacher / T)
//   dz_j = grad T (q_j - sum of p over the entries that list j)
//
// The forward pass reads z once (a running maximum and sum), the backward pass reads it again and writes dz: memory bounds both
// on long rows, the launches (3 us each) on short ones.  Measured on an MI355X: 4096 x 131072 bf16, k 64, 229 us forward
// (4.7 TB/s; the exponentials come close to the loads there, fp32 reaches 5.9) and 396 us backward (5.4 TB/s, as a copy);
// 1021 x 50021 bf16, k 37, 27 and 41 us (22 and 36 with z still in the cache); 32768 x 2, k 2, 3.4 and 3.6 us; 65536 x 64, k 64,
// 39 and 27 us: one row in flight a wave, and a float64 logarithm in each listed lane.
#include <cfloat>
#include <type_traits>

#include "fm_ops_dev.hpp"

namespace fm {
namespace {
constexpr int NT = 256;
constexpr int SHORT = 2048;   // columns of a row that a group of lanes takes
constexpr int SPLIT = 32768;  // columns of a row that a block takes, backward

struct Teacher {
  const void* index;
  int64_t index_stride;
  const void* logit;
  int64_t logit_stride;
  int index64, logit_type, k, cols;
  float temperature, c;  // c: log2(e) / T
  double inv_t, t2;
};

__device__ __forceinline__ int64_t index_at(const Teacher& t, int64_t row, int i) {
  const int64_t o = row * t.index_stride + i;
  return t.index64 ? ((const int64_t*)t.index)[o] : ((const int32_t*)t.index)[o];
}
__device__ __forceinline__ float logit_at(const Teacher& t, int64_t row, int i) {
  const int64_t o = row * t.logit_stride + i;
  return t.logit_type == FM_DTYPE_F32 ? ((const float*)t.logit)[o] : t.logit_type == FM_DTYPE_F16
      ? (float)((const f16*)t.logit)[o] : (float)((const bf16*)t.logit)[o];
}

// exp2 of at most 0; the hardware's, to one unit in the last place
__device__ __forceinline__ float exp2_neg(float x) { return __builtin_amdgcn_exp2f(x); }

// The row's entries into LDS: at[i] (-1: not listed) and p[i].  Returns 1, 0 where none is listed, NaN where an
// index is too large or a logit NaN or +inf.  top, total: the teacher's largest logit and its sum of exp.
__device__ float load_teacher(const Teacher& t, int64_t row, int* at, float* p, float* buf, float& top, float& total) {
  float m = -INFINITY, s = 0;
  float wrong = 0;
  for (int i = threadIdx.x; i < t.k; i += NT) {
    const int64_t j = index_at(t, row, i);
    const float l = j < 0 ? -INFINITY : logit_at(t, row, i);
    if (j >= t.cols || !(l < INFINITY)) wrong = 1;
    at[i] = l == -INFINITY || j >= t.cols ? -1 : (int)j;
    p[i] = l;
    m = fmaxf(m, l);
  }
  top = block_max<NT>(m, buf);
  wrong = block_max<NT>(wrong, buf + NT / 64);
  for (int i = threadIdx.x; i < t.k; i += NT) {
    const float e = at[i] < 0 ? 0.0f : exp2_neg((p[i] - top) * t.c);
    p[i] = e;
    s += e;
  }
  total = block_sum<NT>(s, buf + 2 * (NT / 64));
  const float inv = 1.0f / total;
  for (int i = threadIdx.x; i < t.k; i += NT) p[i] *= inv;
  __syncthreads();
  return wrong > 0 ? NAN : total > 0 ? 1.0f : 0.0f;
}

// Largest logit and sum of exp((z - largest) / T), one pass: the sum is scaled down where a larger logit comes along.
// The difference comes before the scaling: both may be near the type's lowest value.
struct Softmax {
  float m = -FLT_MAX, s = 0;
  template <int N>
  __device__ __forceinline__ void add(const float* v, float c) {
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < N; i++) mx = fmaxf(mx, v[i]);
    if (mx > m) {
      s *= exp2_neg((m - mx) * c);
      m = mx;
    }
#pragma unroll
    for (int i = 0; i < N; i++) s += exp2_neg((v[i] - m) * c);
  }
  __device__ __forceinline__ void rescale(float top, float c) {
    s *= exp2_neg((m - top) * c);
    m = top;
  }
};

// f(first column, N logits as floats) over columns [from, to) by `threads` threads, of which this is `t`: U 16-byte
// loads on their way at a time, from any element on; g(column, logit) for the elements that are left
template <int U, typename T, typename F, typename G>
__device__ __forceinline__ void each(const T* z, int from, int to, int t, int threads, F&& f, G&& g) {
  constexpr int N = 16 / (int)sizeof(T);
  const int vectors = (to - from) / N;
  int i = t;
  for (; i + (U - 1) * threads < vectors; i += U * threads) {
    T v[U][N];
#pragma unroll
    for (int u = 0; u < U; u++) __builtin_memcpy(v[u], z + from + (i + u * threads) * N, 16);
#pragma unroll
    for (int u = 0; u < U; u++) {
      float x[N];
#pragma unroll
      for (int n = 0; n < N; n++) x[n] = to_f32(v[u][n]);
      f(from + (i + u * threads) * N, x);
    }
  }
  for (; i < vectors; i += threads) {
    T v[N];
    __builtin_memcpy(v, z + from + i * N, 16);
    float x[N];
#pragma unroll
    for (int n = 0; n < N; n++) x[n] = to_f32(v[n]);
    f(from + i * N, x);
  }
  const int c = from + vectors * N + t;
  if (c < to) g(c, to_f32(z[c]));
}

// ---------------------------------------------------------------------------------------------- short rows and lists
// G lanes a row, k <= G: each lane has an entry of the list, and one column (or, WIDE with G = 64, vectors of them).  No
// barriers and no LDS but for the bits: rows of two columns go 32 to a wave (a block a row took 67 us for 32768 of them
// instead of 3.5).
struct Entry {
  int at;  // its column; -1: not listed
  float p, logit, top, total, mass;
};
template <int G>
__device__ __forceinline__ Entry entry_of(const Teacher& t, int64_t row, int j, uint64_t group) {
  Entry e;
  const int64_t at = j < t.k ? index_at(t, row, j) : -1;
  e.logit = at < 0 ? -INFINITY : logit_at(t, row, j);
  const bool wrong = (__ballot(at >= t.cols || !(e.logit < INFINITY)) & group) != 0;
  e.at = e.logit == -INFINITY || at >= t.cols ? -1 : (int)at;
  e.top = group_max<G>(e.logit);
  const float x = e.at < 0 ? 0.0f : exp2_neg((e.logit - e.top) * t.c);
  e.total = group_sum<G>(x);
  e.p = x / e.total;
  e.mass = wrong ? NAN : e.total > 0 ? 1.0f : 0.0f;
  return e;
}

template <typename T, int G, bool WIDE>
__device__ __forceinline__ Softmax softmax_of(const T* zr, int j, const Teacher& t) {
  Softmax q;
  if (WIDE) {
    each<2>(zr, 0, t.cols, j, 64, [&](int, const float* v) { q.add<16 / (int)sizeof(T)>(v, t.c); },
        [&](int, float v) { q.add<1>(&v, t.c); });
  } else if (j < t.cols) {
    const float v = to_f32(zr[j]);
    q.add<1>(&v, t.c);
  }
  q.rescale(group_max<G>(q.m), t.c);
  q.s = group_sum<G>(q.s);
  return q;
}

// one entry's part of the loss; log_ratio: log of the student's sum of exp over the teacher's
__device__ __forceinline__ double term_of(float p, float teacher, float top, float z, float m, double log_ratio,
    const Teacher& t) {
  return (double)p * ((((double)teacher - top) - ((double)z - m)) * t.inv_t + log_ratio);
}

template <typename T, int G, bool WIDE>
__global__ __launch_bounds__(NT) void distill_fwd_group(const T* z, int64_t stride, Teacher t, float* loss, float* stats,
    int64_t rows) {
  const int lane = threadIdx.x & 63, j = lane & (G - 1);
  const uint64_t group = (G == 64 ? ~0ull : (1ull << G) - 1) << (lane - j);
  for (int64_t first = (int64_t)blockIdx.x * (NT / G); first < rows; first += (int64_t)gridDim.x * (NT / G)) {
    const int64_t row = first + threadIdx.x / G, r = row < rows ? row : rows - 1;
    const T* zr = z + r * stride;
    const Entry e = entry_of<G>(t, r, j, group);
    const Softmax q = softmax_of<T, G, WIDE>(zr, j, t);
    double sum = 0;
    if (e.p > 0) sum = term_of(e.p, e.logit, e.top, to_f32(zr[e.at]), q.m, log((double)q.s / e.total), t);
    sum = group_sum<G>(sum);
    if (j || row >= rows) continue;
    loss[row] = e.mass != e.mass ? e.mass : e.mass == 0 ? 0.0f : (float)(t.t2 * sum);
    if (stats) {
      stats[2 * row] = q.m;
      stats[2 * row + 1] = q.s;
    }
  }
}

// Everything first as if nothing were listed, then the listed columns again, each by the lanes whose entries list it: by p of
// the one entry, or, where a column is listed twice (a bit of it is set twice), by all entries' sum, the same for each of them.
template <typename T, int G, bool WIDE>
__global__ __launch_bounds__(NT) void distill_bwd_group(const T* z, int64_t stride, Teacher t, const float* stats,
    const float* grad, int64_t grad_stride, T* dz, int64_t rows) {
  constexpr int N = 16 / (int)sizeof(T), WORDS = WIDE ? SHORT / 32 : G / 32 + (G < 32);
  __shared__ uint32_t bits[NT / G][WORDS];
  const int lane = threadIdx.x & 63, j = lane & (G - 1), base = lane - j;
  const uint64_t group = (G == 64 ? ~0ull : (1ull << G) - 1) << base;
  uint32_t* seen = bits[threadIdx.x / G];
  for (int64_t first = (int64_t)blockIdx.x * (NT / G); first < rows; first += (int64_t)gridDim.x * (NT / G)) {
    const int64_t row = first + threadIdx.x / G, r = row < rows ? row : rows - 1;
    const T* zr = z + r * stride;
    T* dr = dz + r * (int64_t)t.cols;
    const Entry e = entry_of<G>(t, r, j, group);
    for (int i = j; i < WORDS; i += G) seen[i] = 0;
    wave_sync();
    bool twice = false;
    if (e.at >= 0) twice = atomicOr(&seen[e.at >> 5], 1u << (e.at & 31)) >> (e.at & 31) & 1;
    const float m = stats[2 * r], inv = 1.0f / stats[2 * r + 1], scale = e.mass == 0 ? 0.0f
        : e.mass * grad[r * grad_stride] * t.temperature;
    auto part = [&](float v, float listed) { return e.mass == 0 ? 0.0f : scale * (exp2_neg((v - m) * t.c) * inv - listed); };
    if (row < rows) {
      if (WIDE) {
        each<2>(
            zr, 0, t.cols, j, 64,
            [&](int c, const float* v) {
              T o[N];
#pragma unroll
              for (int n = 0; n < N; n++) o[n] = from_f32<T>(part(v[n], 0.0f));
              __builtin_memcpy(dr + c, o, 16);
            },
            [&](int c, float v) { dr[c] = from_f32<T>(part(v, 0.0f)); });
      } else if (j < t.cols) {
        dr[j] = from_f32<T>(part(to_f32(zr[j]), 0.0f));
      }
    }
    float listed = e.p;
    if (__ballot(twice)) {  // in any of the wave's rows
      listed = 0;
      for (int i = 0; i < t.k; i++) {
        int at;
        float p;
        if (G == 64) {
          at = __builtin_amdgcn_readlane(e.at, i);
          p = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e.p), i));
        } else {
          at = __shfl(e.at, base + i);
          p = __shfl(e.p, base + i);
        }
        listed += at == e.at ? p : 0.0f;
      }
    }
    wave_sync();
    if (e.at >= 0 && e.mass == 1 && row < rows) dr[e.at] = from_f32<T>(part(to_f32(zr[e.at]), listed));
  }
}

// ---------------------------------------------------------------------------------------------- long rows and lists
// Columns [from, to) of split y of a row: of vectors, so that each starts where the loads do.
template <typename T>
__device__ __forceinline__ void split_of(int cols, int y, int splits, int& from, int& to) {
  constexpr int N = 16 / (int)sizeof(T);
  const int each = ((cols + splits - 1) / splits + N - 1) / N * N;
  from = min(y * each, cols);
  to = min(from + each, cols);
}

template <typename T>
__device__ __forceinline__ Softmax block_softmax(const T* zr, int from, int to, const Teacher& t, float* buf) {
  Softmax q;
  each<4>(zr, from, to, threadIdx.x, NT, [&](int, const float* v) { q.add<16 / (int)sizeof(T)>(v, t.c); },
      [&](int, float v) { q.add<1>(&v, t.c); });
  q.rescale(block_max<NT>(q.m, buf), t.c);
  q.s = block_sum<NT>(q.s, buf + NT / 64);
  return q;
}

template <typename T>
__device__ __forceinline__ void write_loss(const T* zr, const Teacher& t, int64_t r, const Softmax& q, float* loss,
    float* stats, int* at, float* p, float* buf, double* dbuf) {
  float top, total;
  const float mass = load_teacher(t, r, at, p, buf, top, total);
  const double log_ratio = log((double)q.s / total);
  double sum = 0;
  for (int i = threadIdx.x; i < t.k; i += NT)
    if (p[i] > 0) sum += term_of(p[i], logit_at(t, r, i), top, to_f32(zr[at[i]]), q.m, log_ratio, t);
  sum = block_sum<NT>(sum, dbuf);
  if (threadIdx.x) return;
  loss[r] = mass != mass ? mass : mass == 0 ? 0.0f : (float)(t.t2 * sum);
  if (stats) {
    stats[2 * r] = q.m;
    stats[2 * r + 1] = q.s;
  }
}

// a block a row
template <typename T>
__global__ __launch_bounds__(NT) void distill_fwd(const T* z, int64_t stride, Teacher t, float* loss, float* stats,
    int64_t rows) {
  __shared__ int at[FM_DISTILL_MAX_K];
  __shared__ float p[FM_DISTILL_MAX_K], buf[5 * (NT / 64)];
  __shared__ double dbuf[NT / 64];
  const int64_t r = blockIdx.x + (int64_t)gridDim.x * blockIdx.y;
  if (r >= rows) return;
  const Softmax q = block_softmax(z + r * stride, 0, t.cols, t, buf + 3 * (NT / 64));
  write_loss(z + r * stride, t, r, q, loss, stats, at, p, buf, dbuf);
}

// Few rows: a block for each of a row's splits, whose softmax goes to part [rows][splits][2], then a block a row: 1 x 131072
// takes 6.6 us, which one block alone would read for 15.
template <typename T>
__global__ __launch_bounds__(NT) void distill_fwd_split(const T* z, int64_t stride, Teacher t, float* part) {
  __shared__ float buf[2 * (NT / 64)];
  int from, to;
  split_of<T>(t.cols, blockIdx.x, gridDim.x, from, to);
  const Softmax q = block_softmax(z + (int64_t)blockIdx.y * stride, from, to, t, buf);
  if (threadIdx.x == 0) {
    float* o = part + 2 * ((int64_t)blockIdx.y * gridDim.x + blockIdx.x);
    o[0] = q.m;
    o[1] = q.s;
  }
}
template <typename T>
__global__ __launch_bounds__(NT) void distill_fwd_join(const T* z, int64_t stride, Teacher t, const float* part, int splits,
    float* loss, float* stats) {
  __shared__ int at[FM_DISTILL_MAX_K];
  __shared__ float p[FM_DISTILL_MAX_K], buf[5 * (NT / 64)];
  __shared__ double dbuf[NT / 64];
  const int64_t r = blockIdx.x;
  Softmax q;
  if ((int)threadIdx.x < splits) {  // at most 64: every wave joins them
    q.m = part[2 * (r * splits + threadIdx.x)];
    q.s = part[2 * (r * splits + threadIdx.x) + 1];
  }
  q.rescale(block_max<NT>(q.m, buf + 3 * (NT / 64)), t.c);
  q.s = block_sum<NT>(q.s, buf + 4 * (NT / 64));
  write_loss(z + r * stride, t, r, q, loss, stats, at, p, buf, dbuf);
}

// dlogits of a split of a row a block: everything first as if nothing were listed, then the listed columns of the split
// again, as above (whoever lists the same one writes the same value).
template <typename T>
__global__ __launch_bounds__(NT) void distill_bwd(const T* z, int64_t stride, Teacher t, const float* stats,
    const float* grad, int64_t grad_stride, T* dz, int64_t rows, int splits) {
  __shared__ int at[FM_DISTILL_MAX_K];
  __shared__ float p[FM_DISTILL_MAX_K], buf[3 * (NT / 64)];
  __shared__ uint32_t seen[SPLIT / 32 + 1], dup[SPLIT / 32 + 1];  // columns of the split that are listed, and listed twice
  const int64_t b = blockIdx.x + (int64_t)gridDim.x * blockIdx.y, r = b / splits;
  if (r >= rows) return;
  const T* zr = z + r * stride;
  T* dr = dz + r * (int64_t)t.cols;
  int from, to;
  split_of<T>(t.cols, (int)(b - r * splits), splits, from, to);
  for (int i = threadIdx.x; i < SPLIT / 32 + 1; i += NT) seen[i] = dup[i] = 0;
  float top, total;
  const float mass = load_teacher(t, r, at, p, buf, top, total);
  int twice = 0;  // whether a column of the split is listed twice
  for (int i = threadIdx.x; i < t.k; i += NT) {
    const int c = at[i] - from;
    if (at[i] >= from && at[i] < to && (atomicOr(&seen[c >> 5], 1u << (c & 31)) >> (c & 31) & 1)) {
      twice = 1;
      atomicOr(&dup[c >> 5], 1u << (c & 31));
    }
  }
  const float m = stats[2 * r], inv = 1.0f / stats[2 * r + 1], scale = mass == 0 ? 0.0f
      : mass * grad[r * grad_stride] * t.temperature;
  auto part = [&](float v, float listed) { return mass == 0 ? 0.0f : scale * (exp2_neg((v - m) * t.c) * inv - listed); };
  constexpr int N = 16 / (int)sizeof(T);
  each<4>(
      zr, from, to, threadIdx.x, NT,
      [&](int c, const float* v) {
        T o[N];
#pragma unroll
        for (int n = 0; n < N; n++) o[n] = from_f32<T>(part(v[n], 0.0f));
        __builtin_memcpy(dr + c, o, 16);
      },
      [&](int c, float v) { dr[c] = from_f32<T>(part(v, 0.0f)); });
  if (mass != 1) return;
  twice = __syncthreads_or(twice);
  for (int first = threadIdx.x & ~63; first < t.k; first += NT) {  // a wave at a time: 64 entries
    const int i = first + (threadIdx.x & 63), c = i < t.k ? at[i] : -1;
    const bool mine = c >= from && c < to;
    float listed = mine ? p[i] : 0.0f;
    if (twice) {
      // the entries whose column is listed twice, one after the other: all of the wave's lanes look for it
      uint64_t left = __ballot(mine && (dup[(c - from) >> 5] >> ((c - from) & 31) & 1));
      for (; left; left &= left - 1) {
        const int lane = __ffsll((unsigned long long)left) - 1, column = __builtin_amdgcn_readlane(c, lane);
        float sum = 0;
        for (int n = threadIdx.x & 63; n < t.k; n += 64) sum += at[n] == column ? p[n] : 0.0f;
        sum = group_sum<64>(sum);
        if ((threadIdx.x & 63) == lane) listed = sum;
      }
    }
    if (mine) dr[c] = from_f32<T>(part(to_f32(zr[c]), listed));
  }
}

// ---------------------------------------------------------------------------------------------- the choice
Teacher teacher_of(const fm_distill_args& a) {
  return Teacher{a.index, a.index_stride, a.teacher, a.teacher_stride, a.index_dtype == FM_DTYPE_I64, a.teacher_dtype, (int)a.k,
                 (int)a.cols, (float)a.temperature, (float)(1.4426950408889634 / a.temperature), 1.0 / a.temperature,
                 a.temperature * a.temperature};
}

// splits of a row in the forward pass: where there are fewer rows than fill the chip (4 blocks a CU), of 4096 columns or more.
// Measured, us without / with them, bf16: 1 x 131072 12.8 / 7.0, 64 x 131072 13.4 / 9.3, 256 x 131072 18.6 / 18.3; but 1 x 8192
// 5.0 / 6.9, 1 x 32768 6.6 / 6.8, 512 x 32768 10.4 / 13.0, 512 x 131072 25.3 / 30.0: the second launch costs 2 us, so they could
// begin at some 32768 columns and end at 256 rows.  (backward, which needs no second launch: 1 x 32768 8.2 / 5.5, 256 x 32768
// 11.8 / 10.8, 512 x 32768 16.7 / 15.4)
int splits_of(int64_t rows, int64_t cols) {
  if (rows < 1 || rows >= 1024) return 1;
  const int64_t wanted = 1024 / rows, most = cols / 4096;
  const int64_t n = wanted < most ? wanted : most;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

// f(lanes, wide) for rows and lists that a group of lanes holds; false for longer ones
template <typename F>
bool with_group(int64_t cols, int64_t k, F&& f) {
  if (k > 64 || cols > SHORT) return false;
#define GROUP(g, w) f(std::integral_constant<int, g>(), std::integral_constant<bool, w>())
  const int64_t n = cols > k ? cols : k;
  if (n <= 2)
    GROUP(2, false);
  else if (n <= 4)
    GROUP(4, false);
  else if (n <= 8)
    GROUP(8, false);
  else if (n <= 16)
    GROUP(16, false);
  else if (n <= 32)
    GROUP(32, false);
  else if (n <= 64)
    GROUP(64, false);
  else
    GROUP(64, true);
#undef GROUP
  return true;
}

template <typename T>
void forward(const fm_distill_args& a) {
  hipStream_t st = (hipStream_t)a.stream;
  const Teacher t = teacher_of(a);
  const T* z = (const T*)a.logits;
  if (with_group(a.cols, a.k, [&](auto g, auto w) {
        const int64_t n = (a.rows + NT / g - 1) / (NT / g);
        distill_fwd_group<T, decltype(g)::value, decltype(w)::value><<<(int)(n < (1 << 20) ? n : 1 << 20), NT, 0, st>>>(z,
            a.stride, t, a.loss, a.stats, a.rows);
      }))
    return;
  const int splits = splits_of(a.rows, a.cols);
  if (splits > 1) {
    distill_fwd_split<T><<<dim3(splits, (int)a.rows), NT, 0, st>>>(z, a.stride, t, (float*)a.workspace);
    distill_fwd_join<T><<<(int)a.rows, NT, 0, st>>>(z, a.stride, t, (const float*)a.workspace, splits, a.loss, a.stats);
  } else {
    distill_fwd<T><<<grid_of(a.rows), NT, 0, st>>>(z, a.stride, t, a.loss, a.stats, a.rows);
  }
}

template <typename T>
void backward(const fm_distill_args& a) {
  hipStream_t st = (hipStream_t)a.stream;
  const Teacher t = teacher_of(a);
  const T* z = (const T*)a.logits;
  if (with_group(a.cols, a.k, [&](auto g, auto w) {
        const int64_t n = (a.rows + NT / g - 1) / (NT / g);
        distill_bwd_group<T, decltype(g)::value, decltype(w)::value><<<(int)(n < (1 << 20) ? n : 1 << 20), NT, 0, st>>>(z,
            a.stride, t, a.stats, a.grad, a.grad_stride, (T*)a.dlogits, a.rows);
      }))
    return;
  // a block for every SPLIT columns (the list is read again for each), for fewer where that leaves CUs without work
  int64_t splits = (a.cols + SPLIT - 1) / SPLIT;
  if (a.rows * splits < 1024) splits = splits_of(a.rows, a.cols) > splits ? splits_of(a.rows, a.cols) : splits;
  distill_bwd<T><<<grid_of(a.rows * splits), NT, 0, st>>>(z, a.stride, t, a.stats, a.grad, a.grad_stride, (T*)a.dlogits,
      a.rows, (int)splits);
}
}  // namespace
}  // namespace fm

using namespace fm;
extern "C" {
int64_t fm_distill_workspace(int64_t rows, int64_t cols) {
  const int n = splits_of(rows, cols);
  return n > 1 ? rows * n * 8 : 0;
}

int fm_distill_forward(const fm_distill_args* a) {
  return guarded([&] {
    if (int rc = check_distill(a, false)) return rc;
    if (a->rows == 0) return FM_OK;
    if (a->device < 0) {
      cpu_distill_forward(*a);
      return FM_OK;
    }
    OnDevice on(a->device);
    if (on.err == hipSuccess) with_type(a->dtype, [&](auto tag) { forward<typename decltype(tag)::type>(*a); });
    return on.status("distill");
  });
}

int fm_distill_backward(const fm_distill_args* a) {
  return guarded([&] {
    if (int rc = check_distill(a, true)) return rc;
    if (a->rows == 0) return FM_OK;
    if (a->device < 0) {
      cpu_distill_backward(*a);
      return FM_OK;
    }
    OnDevice on(a->device);
    if (on.err == hipSuccess) with_type(a->dtype, [&](auto tag) { backward<typename decltype(tag)::type>(*a); });
    return on.status("distill backward");
  });
}
}
