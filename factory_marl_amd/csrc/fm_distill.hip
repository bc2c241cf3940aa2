// fm_distill.hip -- distillation from a teacher's top logits (include/factorysim.h fm_distill_*).
//
//   loss = T^2 sum over the listed entries of p (log p - log q[index]),  q = softmax(z / T),  p = softmax(teacher / T)
//   dz_j = grad T (q_j - sum of p over the entries that list j)
#include "fm_ops_dev.hpp"

namespace fm {
namespace {
constexpr int NT = 256;

struct Teacher {
  const void* index;
  int64_t index_stride;
  const void* logit;
  int64_t logit_stride;
  int index64, logit_type, k, cols;
  float inv_t;
};

__device__ __forceinline__ int64_t index_at(const Teacher& t, int64_t row, int i) {
  const int64_t o = row * t.index_stride + i;
  return t.index64 ? ((const int64_t*)t.index)[o] : ((const int32_t*)t.index)[o];
}
__device__ __forceinline__ float logit_at(const Teacher& t, int64_t row, int i) {
  const int64_t o = row * t.logit_stride + i;
  return t.logit_type == FM_DTYPE_F32 ? ((const float*)t.logit)[o] : t.logit_type == FM_DTYPE_F16 ? (float)((const f16*)t.logit)[o] : (float)((const bf16*)t.logit)[o];
}

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
    const float e = at[i] < 0 ? 0.0f : expf((p[i] - top) * t.inv_t);
    p[i] = e;
    s += e;
  }
  total = block_sum<NT>(s, buf + 2 * (NT / 64));
  const float inv = 1.0f / total;
  for (int i = threadIdx.x; i < t.k; i += NT) p[i] *= inv;
  __syncthreads();
  return wrong > 0 ? NAN : total > 0 ? 1.0f : 0.0f;
}

template <typename T>
__global__ __launch_bounds__(NT) void distill_fwd(const T* z, int64_t stride, Teacher t, float temperature, float* loss, float* stats, int64_t rows) {
  __shared__ int at[FM_DISTILL_MAX_K];
  __shared__ float p[FM_DISTILL_MAX_K];
  __shared__ float buf[5 * (NT / 64)];
  __shared__ double dbuf[NT / 64];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* zr = z + r * stride;
    float m = -INFINITY;
    for (int c = threadIdx.x; c < t.cols; c += NT) m = fmaxf(m, to_f32(zr[c]));
    m = block_max<NT>(m, buf + 3 * (NT / 64));
    float s = 0;
    for (int c = threadIdx.x; c < t.cols; c += NT) {
      const float v = to_f32(zr[c]);
      s += v == -INFINITY ? 0.0f : expf((v - m) * t.inv_t);
    }
    s = block_sum<NT>(s, buf + 4 * (NT / 64));
    float top, total;
    const float mass = load_teacher(t, r, at, p, buf, top, total);
    const double log_s = log((double)s), log_total = log((double)total);
    double sum = 0;
    for (int i = threadIdx.x; i < t.k; i += NT)
      if (p[i] > 0) {
        const float v = to_f32(zr[at[i]]);
        const double logp = ((double)logit_at(t, r, i) - top) * t.inv_t - log_total;
        sum += (double)p[i] * (logp - ((double)v - m) * t.inv_t + log_s);
      }
    sum = block_sum<NT>(sum, dbuf);
    if (threadIdx.x == 0) {
      loss[r] = mass != mass ? mass : mass == 0 ? 0.0f : (float)((double)temperature * temperature * sum);
      if (stats) {
        stats[2 * r] = m;
        stats[2 * r + 1] = s;
      }
    }
    __syncthreads();
  }
}

// dlogits of one row a block: everything first as if nothing were listed, then the listed places again, each with all
// of the entries that list it (whoever writes the same place writes the same value).
template <typename T>
__global__ __launch_bounds__(NT) void distill_bwd(const T* z, int64_t stride, Teacher t, float temperature, const float* stats, const float* grad,
                                                  int64_t grad_stride, T* dz, int64_t rows) {
  __shared__ int at[FM_DISTILL_MAX_K];
  __shared__ float p[FM_DISTILL_MAX_K];
  __shared__ float buf[3 * (NT / 64)];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* zr = z + r * stride;
    T* dr = dz + r * (int64_t)t.cols;
    float top, total;
    const float mass = load_teacher(t, r, at, p, buf, top, total);
    const float m = stats[2 * r], inv = 1.0f / stats[2 * r + 1], scale = mass == 0 ? 0.0f : grad[r * grad_stride] * temperature;
    for (int c = threadIdx.x; c < t.cols; c += NT) {
      const float v = to_f32(zr[c]);
      const float q = v == -INFINITY ? 0.0f * inv : expf((v - m) * t.inv_t) * inv;
      dr[c] = from_f32<T>(mass == 0 ? 0.0f : mass * scale * q);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < t.k; i += NT) {
      const int j = at[i];
      if (j < 0 || mass == 0) continue;
      float listed = 0;
      for (int n = 0; n < t.k; n++) listed += at[n] == j ? p[n] : 0.0f;
      const float v = to_f32(zr[j]);
      const float q = v == -INFINITY ? 0.0f * inv : expf((v - m) * t.inv_t) * inv;
      dr[j] = from_f32<T>(mass * scale * (q - listed));
    }
    __syncthreads();
  }
}

Teacher teacher_of(const fm_distill_args& a) {
  return Teacher{a.index, a.index_stride, a.teacher, a.teacher_stride, a.index_dtype == FM_DTYPE_I64, a.teacher_dtype, (int)a.k, (int)a.cols, (float)(1.0 / a.temperature)};
}
}  // namespace
}  // namespace fm

using namespace fm;
extern "C" {
int64_t fm_distill_workspace(int64_t rows, int64_t cols) { return 0; }

int fm_distill_forward(const fm_distill_args* a) {
  return guarded([&] {
    if (int rc = check_distill(a, false)) return rc;
    if (a->rows == 0) return FM_OK;
    if (a->device < 0) {
      cpu_distill_forward(*a);
      return FM_OK;
    }
    OnDevice on(a->device);
    if (on.err == hipSuccess)
      with_type(a->dtype, [&](auto tag) {
        typedef typename decltype(tag)::type T;
        distill_fwd<T><<<(int)(a->rows < (1 << 20) ? a->rows : 1 << 20), NT, 0, (hipStream_t)a->stream>>>(
            (const T*)a->logits, a->stride, teacher_of(*a), (float)a->temperature, a->loss, a->stats, a->rows);
      });
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
    if (on.err == hipSuccess)
      with_type(a->dtype, [&](auto tag) {
        typedef typename decltype(tag)::type T;
        distill_bwd<T><<<(int)(a->rows < (1 << 20) ? a->rows : 1 << 20), NT, 0, (hipStream_t)a->stream>>>(
            (const T*)a->logits, a->stride, teacher_of(*a), (float)a->temperature, a->stats, a->grad, a->grad_stride, (T*)a->dlogits, a->rows);
      });
    return on.status("distill backward");
  });
}
}
