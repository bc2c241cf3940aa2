// fm_norm.hip -- layer norm over the last dimension, forward and backward (include/factorysim.h fm_layer_norm_*).
//
//   y  = h weight + bias,  h = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - h mean(g h)),  g = dy weight;  dweight = sum over rows of dy h,  dbias = sum of dy
#include "fm_ops_dev.hpp"

namespace fm {
namespace {
constexpr int NT = 256;

// One block a row at a time, the row read again from the cache for each of its sums.
template <typename T, typename P>
__global__ __launch_bounds__(NT) void norm_fwd_wide(const T* x, int64_t x_stride, const P* weight, const P* bias, T* y, float* mean_out,
                                                    float* rstd_out, int64_t rows, int cols, float eps) {
  __shared__ float buf[2][NT / 64];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    T* yr = y + r * (int64_t)cols;
    float s = 0;
    for (int c = threadIdx.x; c < cols; c += NT) s += to_f32(xr[c]);
    const float mean = block_sum<NT>(s, buf[0]) / (float)cols;
    s = 0;
    for (int c = threadIdx.x; c < cols; c += NT) {
      const float d = to_f32(xr[c]) - mean;
      s += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum<NT>(s, buf[1]) / (float)cols + eps);
    for (int c = threadIdx.x; c < cols; c += NT) {
      const float h = (to_f32(xr[c]) - mean) * rstd;
      yr[c] = from_f32<T>(h * (weight ? to_f32(weight[c]) : 1.0f) + (bias ? to_f32(bias[c]) : 0.0f));
    }
    if (mean_out && threadIdx.x == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    __syncthreads();
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(NT) void norm_dx_wide(const T* x, int64_t x_stride, const T* dy, int64_t dy_stride, const P* weight, const float* mean_in,
                                                   const float* rstd_in, T* dx, int64_t rows, int cols) {
  __shared__ float buf[2][NT / 64];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    const T* gr = dy + r * dy_stride;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float sg = 0, sgh = 0;
    for (int c = threadIdx.x; c < cols; c += NT) {
      const float g = to_f32(gr[c]) * (weight ? to_f32(weight[c]) : 1.0f);
      sg += g;
      sgh += g * ((to_f32(xr[c]) - mean) * rstd);
    }
    sg = block_sum<NT>(sg, buf[0]) / (float)cols;
    sgh = block_sum<NT>(sgh, buf[1]) / (float)cols;
    for (int c = threadIdx.x; c < cols; c += NT) {
      const float g = to_f32(gr[c]) * (weight ? to_f32(weight[c]) : 1.0f);
      const float h = (to_f32(xr[c]) - mean) * rstd;
      dx[r * (int64_t)cols + c] = from_f32<T>(rstd * (g - sg - h * sgh));
    }
    __syncthreads();
  }
}

// Sums over a stretch of rows, 64 columns a block, 4 rows at a time: part[stretch] = dweight, dbias of the stretch.
template <typename T>
__global__ __launch_bounds__(NT) void norm_dparam_wide(const T* x, int64_t x_stride, const T* dy, int64_t dy_stride, const float* mean_in,
                                                       const float* rstd_in, float* part, int64_t rows, int cols) {
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

// The stretches' sums added up, in their order: 64 columns a block, 4 stretches at a time.
template <typename P>
__global__ __launch_bounds__(NT) void norm_dparam_sum(const float* part, int parts, P* dweight, P* dbias, int cols) {
  __shared__ float buf[4][64];
  const int i = blockIdx.x * 64 + (threadIdx.x & 63), lane = threadIdx.x >> 6;  // over dweight's and dbias's columns in turn
  float s = 0;
  if (i < 2 * cols)
    for (int p = lane; p < parts; p += 4) s += part[(int64_t)p * 2 * cols + i];
  buf[lane][threadIdx.x & 63] = s;
  __syncthreads();
  if (threadIdx.x < 64 && i < 2 * cols) {
    const int t = threadIdx.x;
    P* to = i < cols ? dweight : dbias;
    if (to) to[i < cols ? i : i - cols] = from_f32<P>((buf[0][t] + buf[1][t]) + (buf[2][t] + buf[3][t]));
  }
}

int64_t parts_of(int64_t rows) { return rows < 1 ? 0 : rows < 16 * 256 ? (rows + 15) / 16 : 256; }

template <typename T, typename P>
void forward(const fm_layer_norm_args& a) {
  const int grid = (int)(a.rows < (1 << 20) ? a.rows : 1 << 20);
  norm_fwd_wide<T, P><<<grid, NT, 0, (hipStream_t)a.stream>>>((const T*)a.x, a.x_stride, (const P*)a.weight, (const P*)a.bias, (T*)a.y, a.mean,
                                                              a.rstd, a.rows, (int)a.cols, (float)a.eps);
}

template <typename T, typename P>
void backward(const fm_layer_norm_args& a) {
  hipStream_t st = (hipStream_t)a.stream;
  const int grid = (int)(a.rows < (1 << 20) ? a.rows : 1 << 20), cols = (int)a.cols, parts = (int)parts_of(a.rows);
  if (a.dx && a.rows > 0)
    norm_dx_wide<T, P><<<grid, NT, 0, st>>>((const T*)a.x, a.x_stride, (const T*)a.dy, a.dy_stride, (const P*)a.weight, a.mean, a.rstd, (T*)a.dx,
                                            a.rows, cols);
  if (!a.dweight && !a.dbias) return;
  if (parts)
    norm_dparam_wide<T><<<dim3((cols + 63) / 64, parts), NT, 0, st>>>((const T*)a.x, a.x_stride, (const T*)a.dy, a.dy_stride, a.mean, a.rstd,
                                                                      (float*)a.workspace, a.rows, cols);
  norm_dparam_sum<P><<<(2 * cols + 63) / 64, NT, 0, st>>>((const float*)a.workspace, parts, (P*)a.dweight, (P*)a.dbias, cols);
}
}  // namespace
}  // namespace fm

using namespace fm;
extern "C" {
int64_t fm_layer_norm_workspace(int64_t rows, int64_t cols) { return cols < 1 ? 0 : parts_of(rows) * 2 * cols * 4; }

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
