// fm_norm.hip -- layer norm over the last dimension, forward and backward (include/factorysim.h fm_layer_norm_*).
//
//   y  = h weight + bias,  h = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - h mean(g h)),  g = dy weight;  dweight = sum over rows of dy h,  dbias = sum of dy
//
// Some 20 operations an element against 4 to 16 bytes: memory bounds all of it but the smallest calls, which a launch does
// (3 us).  Forward reads x and writes y, backward reads x and dy and writes dx: five passes.  Measured on an MI355X, where a
// copy of 1 GiB moves 5.1 TB/s: 16384 x 8192 bf16 91 us forward (5.9 TB/s) and 155 + 5 us backward (5.2 TB/s);
// 32768 x 512 fp32 21 and 36 us; 5003 x 1001 fp16, no row aligned, 6.9 and 15.5 us (5003 x 1024, all aligned, 6.3 and 14.9: it is
// the size, a few rows a block, and not the alignment that keeps it from its 4 and 6); 8192 x 128 fp32 4 and 8 us.
#include <type_traits>

#include "fm_ops_dev.hpp"

namespace fm {
namespace {
constexpr int NT = 256;

// ---------------------------------------------------------------------------------------------- vectors of a row
template <typename T, int N>
struct Raw {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load(const T* p) {
  Raw<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float* from) {
  Raw<T, N> r;
#pragma unroll
  for (int i = 0; i < N; i++) r.v[i] = from_f32<T>(from[i]);
  __builtin_memcpy(p, &r, sizeof(r));
}
// N of a parameter's elements; `other` for all where there is none
template <typename P, int N>
__device__ __forceinline__ void load_param(const P* p, int at, float other, float* to) {
  if (p) {
    const Raw<P, N> r = load<P, N>(p + at);
#pragma unroll
    for (int i = 0; i < N; i++) to[i] = to_f32(r.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) to[i] = other;
  }
}

// ---------------------------------------------------------------------------------------------- rows beyond 16384
// One block a row, the row read again (from the cache) for each of its sums.  Vectors as below: whole, the last one moved back
// to the row's end; `skip` of its elements are another thread's too.  1024 x 20000 bf16: 27 us forward (3.1 TB/s), 28 + 24 + 4
// backward: x is read three times forward, x and dy three times backward.
constexpr int WT = 1024;
template <typename T, typename F>
__device__ __forceinline__ void each_vector(int cols, F&& f) {
  constexpr int N = 16 / (int)sizeof(T);
  for (int c = threadIdx.x * N; c < cols; c += WT * N) {
    const int at = c < cols - N ? c : cols - N;
    f(at, c - at);
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(WT) void norm_fwd_wide(const T* x, int64_t x_stride, const P* weight, const P* bias, T* y,
    float* mean_out, float* rstd_out, int64_t rows, int cols, float eps) {
  constexpr int N = 16 / (int)sizeof(T);
  __shared__ float buf[2][WT / 64];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    float s = 0;
    each_vector<T>(cols, [&](int at, int skip) {
      const Raw<T, N> v = load<T, N>(xr + at);
#pragma unroll
      for (int i = 0; i < N; i++) s += i >= skip ? to_f32(v.v[i]) : 0.0f;
    });
    const float mean = block_sum<WT>(s, buf[0]) / (float)cols;
    s = 0;
    each_vector<T>(cols, [&](int at, int skip) {
      const Raw<T, N> v = load<T, N>(xr + at);
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float d = to_f32(v.v[i]) - mean;
        s += i >= skip ? d * d : 0.0f;
      }
    });
    const float rstd = 1.0f / sqrtf(block_sum<WT>(s, buf[1]) / (float)cols + eps);
    each_vector<T>(cols, [&](int at, int) {
      const Raw<T, N> v = load<T, N>(xr + at);
      float w[N], b[N];
      load_param<P, N>(weight, at, 1.0f, w);
      load_param<P, N>(bias, at, 0.0f, b);
#pragma unroll
      for (int i = 0; i < N; i++) b[i] += (to_f32(v.v[i]) - mean) * rstd * w[i];
      store<T, N>(y + r * (int64_t)cols + at, b);
    });
    if (mean_out && threadIdx.x == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    __syncthreads();
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(WT) void norm_dx_wide(const T* x, int64_t x_stride, const T* dy, int64_t dy_stride,
    const P* weight, const float* mean_in, const float* rstd_in, T* dx, int64_t rows, int cols) {
  constexpr int N = 16 / (int)sizeof(T);
  __shared__ float buf[2][WT / 64];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    const T* gr = dy + r * dy_stride;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float sg = 0, sgh = 0;
    each_vector<T>(cols, [&](int at, int skip) {
      const Raw<T, N> v = load<T, N>(xr + at), d = load<T, N>(gr + at);
      float w[N];
      load_param<P, N>(weight, at, 1.0f, w);
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float g = to_f32(d.v[i]) * w[i];
        sg += i >= skip ? g : 0.0f;
        sgh += i >= skip ? g * ((to_f32(v.v[i]) - mean) * rstd) : 0.0f;
      }
    });
    sg = block_sum<WT>(sg, buf[0]) / (float)cols;
    sgh = block_sum<WT>(sgh, buf[1]) / (float)cols;
    each_vector<T>(cols, [&](int at, int) {
      const Raw<T, N> v = load<T, N>(xr + at), d = load<T, N>(gr + at);
      float w[N];
      load_param<P, N>(weight, at, 1.0f, w);
#pragma unroll
      for (int i = 0; i < N; i++) w[i] = rstd * (to_f32(d.v[i]) * w[i] - sg - (to_f32(v.v[i]) - mean) * rstd * sgh);
      store<T, N>(dx + r * (int64_t)cols + at, w);
    });
    __syncthreads();
  }
}

// Sums over a stretch of rows, 64 columns a block, 4 rows at a time: part[stretch] = dweight, dbias of the stretch.
template <typename T>
__global__ __launch_bounds__(NT) void norm_dparam_wide(const T* x, int64_t x_stride, const T* dy, int64_t dy_stride,
    const float* mean_in, const float* rstd_in, float* part, int64_t rows, int cols) {
  __shared__ float buf[2][4][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), lane = threadIdx.x >> 6;
  const int64_t each = (rows + gridDim.y - 1) / gridDim.y, first = blockIdx.y * each;
  const int64_t end = first + each < rows ? first + each : rows;
  float dw = 0, db = 0;
  if (c < cols)
    for (int64_t r = first + lane; r < end; r += 4) {
      const float d = to_f32(dy[r * dy_stride + c]);
      dw += d * ((to_f32(x[r * x_stride + c]) - mean_in[r]) * rstd_in[r]);
      db += d;
    }
  buf[0][lane][threadIdx.x & 63] = dw;
  buf[1][lane][threadIdx.x & 63] = db;
  __syncthreads();
  if (threadIdx.x < 64 && c < cols) {
    float* to = part + (int64_t)blockIdx.y * 2 * cols;
    const int t = threadIdx.x;
    to[c] = (buf[0][0][t] + buf[0][1][t]) + (buf[0][2][t] + buf[0][3][t]);
    to[cols + c] = (buf[1][0][t] + buf[1][1][t]) + (buf[1][2][t] + buf[1][3][t]);
  }
}

// ---------------------------------------------------------------------------------------------- rows up to 16384
// TPR threads hold a row in registers, V vectors of N elements each (16 bytes; N = 1 for rows shorter than that); a
// block of NT threads holds NT / TPR rows and goes on to later ones, its weights (and, backward, its columns' sums for dweight
// and dbias) staying in registers and the next row on its way while one is worked on.  Every load is a whole vector
// and unconditional, so that a wave waits for all of its loads at once: vectors start at the row, not at a 16-byte
// border (the hardware loads them from any element), and one that would pass the row's end is moved back to end there.
// Its first `skip` elements are then another thread's too: they are left out of the sums, and stored twice with the
// same value.
template <int N, int TPR, int V>
struct Place {
  int at[V], skip[V];  // where vector j starts; its elements that are not this thread's (N: none is)
  __device__ __forceinline__ Place(int t, int cols) {
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int c = (j * TPR + t) * N;
      at[j] = c < cols - N ? c : cols - N;
      skip[j] = c < cols ? c - at[j] : N;
    }
  }
};

// f(i) added up over the elements that are this thread's
template <int N, typename F>
__device__ __forceinline__ float own_sum(int skip, F&& f) {
  float s = 0;
#pragma unroll
  for (int i = 0; i < N; i++) s += f(i);
  if (skip) {
    s = 0;
#pragma unroll
    for (int i = 0; i < N; i++) s += i >= skip ? f(i) : 0.0f;
  }
  return s;
}

// sum over the TPR threads of a row; `buf` holds a value of each of the block's waves
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  if constexpr (TPR <= 64) {
    return group_sum<TPR>(v);
  } else {
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    const float* own = buf + threadIdx.x / TPR * (TPR / 64);
    float s = own[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; i++) s += own[i];
    return s;
  }
}

template <typename T, typename P, int NT_, int TPR, int V, int N>
__global__ __launch_bounds__(NT_) void norm_fwd(const T* x, int64_t x_stride, const P* weight, const P* bias, T* y,
    float* mean_out, float* rstd_out, int64_t rows, int cols, float eps) {
  constexpr int RPB = NT_ / TPR;
  __shared__ float buf[2][2][NT_ / 64];
  const int t = threadIdx.x % TPR;
  const Place<N, TPR, V> at(t, cols);
  float w[V][N], b[V][N];
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  Raw<T, N> next[V];
#pragma unroll
  for (int j = 0; j < V; j++) next[j] = load<T, N>(x + (r < rows ? r : rows - 1) * x_stride + at.at[j]);
#pragma unroll
  for (int j = 0; j < V; j++) {
    load_param<P, N>(weight, at.at[j], 1.0f, w[j]);
    load_param<P, N>(bias, at.at[j], 0.0f, b[j]);
  }
  const float inv = 1.0f / (float)cols;
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < rows; base += step, r += step, turn ^= 1) {
    float v[V][N], s = 0;
#pragma unroll
    for (int j = 0; j < V; j++)
#pragma unroll
      for (int i = 0; i < N; i++) v[j][i] = to_f32(next[j].v[i]);
    if (base + step < rows) {
      const int64_t n = r + step < rows ? r + step : rows - 1;
#pragma unroll
      for (int j = 0; j < V; j++) next[j] = load<T, N>(x + n * x_stride + at.at[j]);
    }
#pragma unroll
    for (int j = 0; j < V; j++) s += own_sum<N>(at.skip[j], [&](int i) { return v[j][i]; });
    const float mean = row_sum<TPR>(s, buf[turn][0]) * inv;
    s = 0;
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int i = 0; i < N; i++) v[j][i] -= mean;
      s += own_sum<N>(at.skip[j], [&](int i) { return v[j][i] * v[j][i]; });
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(s, buf[turn][1]) * inv + eps);
    if (r >= rows) continue;
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int i = 0; i < N; i++) v[j][i] = v[j][i] * rstd * w[j][i] + b[j][i];
      if (at.skip[j] < N) store<T, N>(y + r * (int64_t)cols + at.at[j], v[j]);
    }
    if (mean_out && t == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

// dx of each row and, at the end, the block's sums for dweight and dbias (part: [blocks][2][cols]; NULL = not wanted): x and dy
// are read once for all three.  With the vectors' tails tested before each load a wave waited for one load after the other
// (16384 x 8192 bf16: 266 us), whole ones and the next row ahead take 152.
// The columns' sums of a block's rows are joined over its wave's lanes, then over its waves through LDS, in order.
template <typename T, typename P, int NT_, int TPR, int V, int N>
__global__ __launch_bounds__(NT_) void norm_bwd(const T* x, int64_t x_stride, const T* dy, int64_t dy_stride,
    const P* weight, const float* mean_in, const float* rstd_in, T* dx, float* part, int64_t rows, int cols) {
  constexpr int RPB = NT_ / TPR;
  __shared__ float buf[2][2][NT_ / 64];
  extern __shared__ float sums[];  // [groups of rows][cols], for one of the two at a time
  const int t = threadIdx.x % TPR;
  const Place<N, TPR, V> at(t, cols);
  float w[V][N], dw[V][N], db[V][N];
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  Raw<T, N> nx[V], ny[V];
  float nmean, nrstd;
  auto fetch = [&](int64_t row) {
    const int64_t n = row < rows ? row : rows - 1;
#pragma unroll
    for (int j = 0; j < V; j++) {
      nx[j] = load<T, N>(x + n * x_stride + at.at[j]);
      ny[j] = load<T, N>(dy + n * dy_stride + at.at[j]);
    }
    nmean = mean_in[n];
    nrstd = rstd_in[n];
  };
  // 1024 threads have 128 registers each: no room for the next row beside 16 elements of this one
  constexpr bool AHEAD = NT_ < 1024 || V * N <= 8;
  if (AHEAD) fetch(r);
#pragma unroll
  for (int j = 0; j < V; j++) {
    load_param<P, N>(weight, at.at[j], 1.0f, w[j]);
#pragma unroll
    for (int i = 0; i < N; i++) dw[j][i] = db[j][i] = 0;
  }
  const float inv = 1.0f / (float)cols;
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < rows; base += step, r += step, turn ^= 1) {
    const bool there = r < rows;
    if (!AHEAD) fetch(r);
    const float mean = nmean, rstd = nrstd;
    float h[V][N], g[V][N], sg = 0, sgh = 0;
#pragma unroll
    for (int j = 0; j < V; j++)
#pragma unroll
      for (int i = 0; i < N; i++) {
        h[j][i] = (to_f32(nx[j].v[i]) - mean) * rstd;
        g[j][i] = there ? to_f32(ny[j].v[i]) : 0.0f;
      }
    if (AHEAD && base + step < rows) fetch(r + step);
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        dw[j][i] += g[j][i] * h[j][i];
        db[j][i] += g[j][i];
        g[j][i] *= w[j][i];
      }
      sg += own_sum<N>(at.skip[j], [&](int i) { return g[j][i]; });
      sgh += own_sum<N>(at.skip[j], [&](int i) { return g[j][i] * h[j][i]; });
    }
    if (!dx) continue;
    sg = row_sum<TPR>(sg, buf[turn][0]) * inv;
    sgh = row_sum<TPR>(sgh, buf[turn][1]) * inv;
    if (!there) continue;
#pragma unroll
    for (int j = 0; j < V; j++) {
#pragma unroll
      for (int i = 0; i < N; i++) g[j][i] = rstd * (g[j][i] - sg - h[j][i] * sgh);
      if (at.skip[j] < N) store<T, N>(dx + r * (int64_t)cols + at.at[j], g[j]);
    }
  }
  if (!part) return;
  if (TPR < 64) {
#pragma unroll
    for (int m = TPR; m < 64; m <<= 1)
#pragma unroll
      for (int j = 0; j < V; j++)
#pragma unroll
        for (int i = 0; i < N; i++) {
          dw[j][i] += __shfl_xor(dw[j][i], m);
          db[j][i] += __shfl_xor(db[j][i], m);
        }
  }
  constexpr int GROUPS = TPR < 64 ? NT_ / 64 : RPB;
  const int group = TPR < 64 ? threadIdx.x / 64 : threadIdx.x / TPR;
  const bool writes = TPR >= 64 || (threadIdx.x & 63) < TPR;
  float* to = part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int which = 0; which < 2; which++) {
    float* own = GROUPS == 1 ? to + which * cols : sums + group * cols;
    if (which && GROUPS > 1) __syncthreads();
    if (writes)
#pragma unroll
      for (int j = 0; j < V; j++) {
        const float* from = which ? db[j] : dw[j];
        if (at.skip[j] == 0)
          __builtin_memcpy(own + at.at[j], from, N * sizeof(float));
        else
#pragma unroll
          for (int i = 0; i < N; i++)
            if (i >= at.skip[j]) own[at.at[j] + i] = from[i];
      }
    if (GROUPS == 1) continue;
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += NT_) {
      float a = sums[c];
#pragma unroll
      for (int k = 1; k < GROUPS; k++) a += sums[k * cols + c];
      to[which * cols + c] = a;
    }
  }
}

// The blocks' sums added up in a fixed order: 64 columns a block, C adjacent ones a thread, 1024 C / 64 of the sums at a
// time.  As above, a thread's columns are moved back where they would pass the end.
constexpr int ST = 1024;
template <typename P, int C>
__global__ __launch_bounds__(ST) void norm_dparam_sum(const float* part, int parts, P* dweight, P* dbias, int cols) {
  constexpr int LANES = ST * C / 64;
  __shared__ float buf[LANES][65];
  // over dweight's and dbias's columns in turn
  const int all = 2 * cols, from = (int)(blockIdx.x + gridDim.x * blockIdx.y) * 64;
  if (from >= all) return;
  const int c = threadIdx.x % (64 / C) * C, lane = threadIdx.x / (64 / C);
  const int o = from + c, at = o < all - C ? o : all - C;
  float s[C] = {};
#pragma unroll 8
  for (int p = lane; p < parts; p += LANES) {
    float v[C];
    __builtin_memcpy(v, part + (int64_t)p * all + at, sizeof(v));
#pragma unroll
    for (int i = 0; i < C; i++) s[i] += v[i];
  }
#pragma unroll
  for (int i = 0; i < C; i++) buf[lane][c + i] = s[i];
  __syncthreads();
  // 16 threads a column
  const int k = threadIdx.x & 15, d = threadIdx.x >> 4;
  float a = 0;
#pragma unroll
  for (int i = k; i < LANES; i += 16) a += buf[i][d];
  a = group_sum<16>(a);
  const int od = from + d / C * C;  // as at, of column d
  const int to = (od < all - C ? od : all - C) + d % C;
  if (k == 0) {
    if (to < cols && dweight) dweight[to] = from_f32<P>(a);
    if (to >= cols && dbias) dbias[to - cols] = from_f32<P>(a);
  }
}

// ---------------------------------------------------------------------------------------------- the choice
constexpr int WIDEST = 16384;  // columns that a block holds in registers

// f(block, threads per row, vectors per thread, elements per vector) of the narrowest shape that holds a row
template <typename T, typename F>
void with_shape(int64_t cols, F&& f) {
  constexpr int N = 16 / (int)sizeof(T);
  const int64_t v = (cols + N - 1) / N;
#define SHAPE(nt, tpr, n, e) \
  return f(std::integral_constant<int, nt>(), std::integral_constant<int, tpr>(), std::integral_constant<int, n>(), \
           std::integral_constant<int, e>())
  if (cols < N) SHAPE(256, N, 1, 1);
  if (v <= 4) SHAPE(256, 4, 1, N);
  if (v <= 16) SHAPE(256, 16, 1, N);
  if (v <= 32) SHAPE(256, 32, 1, N);
  if (v <= 64) SHAPE(256, 64, 1, N);
  if (v <= 128) SHAPE(256, 64, 2, N);
  if (v <= 256) SHAPE(256, 256, 1, N);
  if (v <= 512) SHAPE(256, 256, 2, N);
  if (v <= 1024) SHAPE(512, 512, 2, N);
  if (v <= 2048) SHAPE(1024, 1024, 2, N);
  if constexpr (sizeof(T) == 4) SHAPE(1024, 1024, 4, N);
#undef SHAPE
}

// Blocks of the backward pass, each with sums of its own: one for each of the 256 CUs; of 256 threads twice as many
// (their registers let two or three share a CU) where a block still gets 8 rows, so that writing and adding up its sums
// stays small beside them.  Measured with 256 / 512 blocks, bf16, us: 1024 x 2048 11.3 / 12.8, 8192 x 2048 32.9 / 26.1, 2048 x
// 1001 10.7 / 12.7, 32768 x 1001 38.9 / 38.0 (256 threads); 1024 x 16384 35.4 / 50.2, 8192 x 16384 163 / 176 (more threads).
int blocks_of(int64_t rows, int rpb, int threads) {
  const int64_t turns = (rows + rpb - 1) / rpb, most = threads == 256 ? 512 : 256;
  const int64_t blocks = rows / 8 < 256 ? 256 : rows / 8 < most ? rows / 8 : most;
  return (int)(turns < blocks ? turns : blocks);
}

int wide_parts(int64_t rows) { return (int)(rows < 1 ? 0 : rows < 16 * 256 ? (rows + 15) / 16 : 256); }

template <typename T, typename P>
void forward(const fm_layer_norm_args& a) {
  hipStream_t st = (hipStream_t)a.stream;
  const int cols = (int)a.cols;
  if (cols > WIDEST) {
    norm_fwd_wide<T, P><<<(int)(a.rows < (1 << 20) ? a.rows : 1 << 20), WT, 0, st>>>((const T*)a.x, a.x_stride,
        (const P*)a.weight, (const P*)a.bias, (T*)a.y, a.mean, a.rstd, a.rows, cols, (float)a.eps);
    return;
  }
  with_shape<T>(a.cols, [&](auto nt, auto tpr, auto n, auto e) {
    constexpr int B = decltype(nt)::value, TPR = decltype(tpr)::value, V = decltype(n)::value, N = decltype(e)::value;
    const int64_t turns = (a.rows + B / TPR - 1) / (B / TPR), most = 256 * 2048 / B;
    norm_fwd<T, P, B, TPR, V, N><<<(int)(turns < most ? turns : most), B, 0, st>>>((const T*)a.x, a.x_stride,
        (const P*)a.weight, (const P*)a.bias, (T*)a.y, a.mean, a.rstd, a.rows, cols, (float)a.eps);
  });
}

template <typename T, typename P>
void backward(const fm_layer_norm_args& a) {
  hipStream_t st = (hipStream_t)a.stream;
  const int cols = (int)a.cols;
  const bool sums = a.dweight || a.dbias;
  int parts = 0;
  if (a.rows > 0 && cols > WIDEST) {
    if (a.dx)
      norm_dx_wide<T, P><<<(int)(a.rows < (1 << 20) ? a.rows : 1 << 20), WT, 0, st>>>((const T*)a.x, a.x_stride,
          (const T*)a.dy, a.dy_stride, (const P*)a.weight, a.mean, a.rstd, (T*)a.dx, a.rows, cols);
    parts = wide_parts(a.rows);
    if (sums)
      norm_dparam_wide<T><<<dim3((cols + 63) / 64, parts), NT, 0, st>>>((const T*)a.x, a.x_stride, (const T*)a.dy,
          a.dy_stride, a.mean, a.rstd, (float*)a.workspace, a.rows, cols);
  } else if (a.rows > 0 && (a.dx || sums)) {
    with_shape<T>(a.cols, [&](auto nt, auto tpr, auto n, auto e) {
      constexpr int B = decltype(nt)::value, TPR = decltype(tpr)::value, V = decltype(n)::value, N = decltype(e)::value;
      parts = blocks_of(a.rows, B / TPR, B);
      norm_bwd<T, P, B, TPR, V, N><<<parts, B, B > TPR ? 4 * cols * (TPR < 64 ? B / 64 : B / TPR) : 0, st>>>((const T*)a.x,
          a.x_stride, (const T*)a.dy, a.dy_stride, (const P*)a.weight, a.mean, a.rstd, (T*)a.dx,
          sums ? (float*)a.workspace : nullptr, a.rows, cols);
    });
  }
  if (!sums) return;
  if (cols > 1)
    norm_dparam_sum<P, 4><<<grid_of((2 * (int64_t)cols + 63) / 64), ST, 0, st>>>((const float*)a.workspace, parts,
        (P*)a.dweight, (P*)a.dbias, cols);
  else
    norm_dparam_sum<P, 1><<<1, ST, 0, st>>>((const float*)a.workspace, parts, (P*)a.dweight, (P*)a.dbias, cols);
}
}  // namespace
}  // namespace fm

using namespace fm;
extern "C" {
int64_t fm_layer_norm_workspace(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return 0;
  // which shape holds a row of this width depends on its type: the most blocks that any would take
  return (cols > WIDEST ? wide_parts(rows) : blocks_of(rows, 1, 256)) * 8 * cols;
}

int fm_layer_norm_forward(const fm_layer_norm_args* a) {
  return guarded([&] {
    if (int rc = check_norm(a, false)) return rc;
    if (a->rows == 0) return FM_OK;
    if (a->device < 0) {
      cpu_norm_forward(*a);
      return FM_OK;
    }
    OnDevice on(a->device);
    if (on.err == hipSuccess)
      with_type(a->x_dtype, [&](auto t) {
        typedef typename decltype(t)::type T;
        if (a->param_dtype == FM_DTYPE_F32)
          forward<T, float>(*a);
        else
          forward<T, T>(*a);
      });
    return on.status("layer norm");
  });
}

int fm_layer_norm_backward(const fm_layer_norm_args* a) {
  return guarded([&] {
    if (int rc = check_norm(a, true)) return rc;
    if (a->device < 0) {
      cpu_norm_backward(*a);
      return FM_OK;
    }
    OnDevice on(a->device);
    if (on.err == hipSuccess)
      with_type(a->x_dtype, [&](auto t) {
        typedef typename decltype(t)::type T;
        if (a->param_dtype == FM_DTYPE_F32)
          backward<T, float>(*a);
        else
          backward<T, T>(*a);
      });
    return on.status("layer norm backward");
  });
}
}
