// fm_ops_cpu.cpp -- the policy-head operators' argument checks and their CPU backend (device = -1): one thread, sums in
// double.  Each function is the operator's definition written out; the GPU kernels are held to the same statements.
#include <algorithm>
#include <cstring>
#include <limits>
#include <numeric>
#include <vector>

#include "fm_ops.hpp"

namespace fm {
namespace {
float half_to_float(uint16_t h) {
  const uint32_t sign = (uint32_t)(h & 0x8000) << 16, exp = (h >> 10) & 31, man = h & 1023;
  if (exp == 0) return std::ldexp((float)man, -24) * (sign ? -1.f : 1.f);
  const uint32_t bits = sign | (exp == 31 ? 0x7f800000u : (exp + 112) << 23) | man << 13;
  float f;
  std::memcpy(&f, &bits, 4);
  return f;
}

float bf16_to_float(uint16_t h) {
  const uint32_t bits = (uint32_t)h << 16;
  float f;
  std::memcpy(&f, &bits, 4);
  return f;
}

double load(const void* p, int type, int64_t i) {
  switch (type) {
    case FM_DTYPE_F16: return half_to_float(((const uint16_t*)p)[i]);
    case FM_DTYPE_BF16: return bf16_to_float(((const uint16_t*)p)[i]);
    case FM_DTYPE_F64: return ((const double*)p)[i];
    default: return ((const float*)p)[i];
  }
}

int64_t load_index(const void* p, int type, int64_t i) {
  return type == FM_DTYPE_I64 ? ((const int64_t*)p)[i] : ((const int32_t*)p)[i];
}

// the nearest value of a 16-bit format (digits significant bits, exponents down to emin), ties to even: one rounding
// from double; v's magnitude is scaled so that the kept digits are an integer
uint16_t round16(double v, int digits, int emin, int emax, int man_bits) {
  const uint16_t sign = std::signbit(v) ? 0x8000 : 0;
  const uint16_t inf = (uint16_t)(((1u << (15 - man_bits)) - 1) << man_bits);
  if (std::isnan(v)) return sign | inf | (uint16_t)(1u << (man_bits - 1));
  double m = std::fabs(v);
  if (std::isinf(m)) return sign | inf;
  if (m == 0) return sign;
  int e = std::ilogb(m);
  if (e < emin) e = emin;
  double q = std::nearbyint(std::ldexp(m, digits - 1 - e));  // 0 .. 2^digits
  if (q >= std::ldexp(1.0, digits)) {
    q /= 2;
    e++;
  }
  if (e > emax) return sign | inf;
  const double one = std::ldexp(1.0, digits - 1);
  if (q < one) return sign | (uint16_t)q;  // subnormal
  return sign | (uint16_t)((uint16_t)(e - emin + 1) << man_bits) | (uint16_t)(q - one);
}

void store(void* p, int type, int64_t i, double v) {
  switch (type) {
    case FM_DTYPE_F16: ((uint16_t*)p)[i] = round16(v, 11, -14, 15, 10); break;
    case FM_DTYPE_BF16: ((uint16_t*)p)[i] = round16(v, 8, -126, 127, 7); break;
    default: ((float*)p)[i] = (float)v;
  }
}

int bad(const char* msg) { return report(FM_EINVAL, msg); }
}  // namespace

// ------------------------------------------------------------------ argument checks
int check_norm(const fm_layer_norm_args* a, bool backward) {
  if (!a) return bad("layer norm: null argument");
  if (a->device < -1) return bad("layer norm: device is a GPU ordinal or -1");
  if (!is_float_type(a->x_dtype)) return bad("layer norm: x_dtype is F32, F16 or BF16");
  if (a->param_dtype != a->x_dtype && a->param_dtype != FM_DTYPE_F32) return bad("layer norm: param_dtype is x_dtype or F32");
  if (a->rows < 0 || a->cols < 1) return bad("layer norm: rows >= 0 and cols >= 1 are needed");
  if (a->x_stride < 0 || (backward && a->dy_stride < 0)) return bad("layer norm: negative row stride");
  if (!fits(a->rows, a->cols, a->x_stride) || (backward && !fits(a->rows, a->cols, a->dy_stride)) || a->cols > FM_MAX_COLS)
    return bad("layer norm: too many elements");
  const int xs = type_size(a->x_dtype), ps = type_size(a->param_dtype);
  if (!aligned(a->x, xs) || !aligned(a->weight, ps)) return bad("layer norm: misaligned pointer");
  if (a->rows > 0 && !a->x) return bad("layer norm: x is NULL");
  if (!backward) {
    if (!(a->eps >= 0) || std::isinf(a->eps)) return bad("layer norm: eps is finite and >= 0");
    if (a->rows > 0 && !a->y) return bad("layer norm: y is NULL");
    if (!a->mean != !a->rstd) return bad("layer norm: mean and rstd are kept together");
    if (!aligned(a->bias, ps) || !aligned(a->y, xs) || !aligned(a->mean, 4) || !aligned(a->rstd, 4))
      return bad("layer norm: misaligned pointer");
    return FM_OK;
  }
  if (a->rows > 0 && (!a->dy || !a->mean || !a->rstd)) return bad("layer norm: dy, mean and rstd are needed");
  if (!aligned(a->dy, xs) || !aligned(a->dx, xs) || !aligned(a->dweight, ps) || !aligned(a->dbias, ps) ||
      !aligned(a->mean, 4) || !aligned(a->rstd, 4))
    return bad("layer norm: misaligned pointer");
  if (a->device >= 0 && a->rows > 0 && (a->dweight || a->dbias) &&
      (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < fm_layer_norm_workspace(a->rows, a->cols)))
    return bad("layer norm: the workspace is NULL, misaligned or smaller than fm_layer_norm_workspace says");
  return FM_OK;
}

int check_sample(const fm_sample_args* a) {
  if (!a) return bad("sample: null argument");
  if (a->device < -1) return bad("sample: device is a GPU ordinal or -1");
  if (!is_float_type(a->dtype)) return bad("sample: dtype is F32, F16 or BF16");
  if (a->u_dtype != FM_DTYPE_F32 && a->u_dtype != FM_DTYPE_F64) return bad("sample: u_dtype is F32 or F64");
  if (a->rows < 0 || a->cols < 1 || a->cols > FM_MAX_COLS) return bad("sample: rows >= 0 and 1 <= cols <= 2^28 are needed");
  if (a->stride < 0 || a->mask_stride < 0) return bad("sample: negative row stride");
  if (!fits(a->rows, a->cols, a->stride) || !fits(a->rows, a->cols, a->mask_stride) || a->rows >> 35)
    return bad("sample: too many elements");
  if (a->rows > 0 && (!a->logits || !a->u || !a->out)) return bad("sample: logits, u and out are needed");
  if (!aligned(a->logits, type_size(a->dtype)) || !aligned(a->u, type_size(a->u_dtype)) || !aligned(a->out, 8) ||
      !aligned(a->temperature_rows, 4) || !aligned(a->top_p_rows, 4) || !aligned(a->min_p_rows, 4) ||
      !aligned(a->top_k_rows, 4))
    return bad("sample: misaligned pointer");
  if ((!a->temperature_rows && std::isnan(a->temperature)) || (!a->top_p_rows && std::isnan(a->top_p)) ||
      (!a->min_p_rows && std::isnan(a->min_p)))
    return bad("sample: a setting is NaN");
  return FM_OK;
}

int check_distill(const fm_distill_args* a, bool backward) {
  if (!a) return bad("distill: null argument");
  if (a->device < -1) return bad("distill: device is a GPU ordinal or -1");
  if (!is_float_type(a->dtype) || !is_float_type(a->teacher_dtype))
    return bad("distill: dtype and teacher_dtype are F32, F16 or BF16");
  if (a->index_dtype != FM_DTYPE_I32 && a->index_dtype != FM_DTYPE_I64) return bad("distill: index_dtype is I32 or I64");
  if (a->rows < 0 || a->cols < 1 || a->cols > FM_MAX_COLS) return bad("distill: rows >= 0 and 1 <= cols <= 2^28 are needed");
  if (a->k < 1 || a->k > FM_DISTILL_MAX_K) return bad("distill: 1 <= k <= 1024 is needed");
  if (a->stride < 0 || a->index_stride < 0 || a->teacher_stride < 0 || (backward && a->grad_stride < 0))
    return bad("distill: negative row stride");
  if (!fits(a->rows, a->cols, a->stride) || !fits(a->rows, a->k, a->index_stride) || !fits(a->rows, a->k, a->teacher_stride) ||
      (backward && !fits(a->rows, 1, a->grad_stride)))
    return bad("distill: too many elements");
  if (a->rows >> 35) return bad("distill: too many rows");
  if (!(a->temperature >= 1e-30 && a->temperature <= 1e30))
    return bad("distill: temperature is positive and within 1e-30 .. 1e30");
  if (a->rows > 0 && (!a->logits || !a->index || !a->teacher)) return bad("distill: logits, index and teacher are needed");
  if (a->rows > 0 && !backward && !a->loss) return bad("distill: loss is NULL");
  if (a->rows > 0 && backward && (!a->stats || !a->grad || !a->dlogits))
    return bad("distill: stats, grad and dlogits are needed");
  if (!aligned(a->logits, type_size(a->dtype)) || !aligned(a->index, type_size(a->index_dtype)) ||
      !aligned(a->teacher, type_size(a->teacher_dtype)) || !aligned(a->stats, 4) || !aligned(a->loss, 4) ||
      (backward && (!aligned(a->grad, 4) || !aligned(a->dlogits, type_size(a->dtype)))))
    return bad("distill: misaligned pointer");
  const int64_t need = fm_distill_workspace(a->rows, a->cols);
  if (a->device >= 0 && !backward && need > 0 && (!a->workspace || !aligned(a->workspace, 16) || a->workspace_bytes < need))
    return bad("distill: the workspace is NULL, misaligned or smaller than fm_distill_workspace says");
  return FM_OK;
}

// ------------------------------------------------------------------ layer norm
void cpu_norm_forward(const fm_layer_norm_args& a) {
  for (int64_t r = 0; r < a.rows; r++) {
    const int64_t o = r * a.x_stride;
    double mean = 0, var = 0;
    for (int64_t c = 0; c < a.cols; c++) mean += load(a.x, a.x_dtype, o + c);
    mean /= (double)a.cols;
    for (int64_t c = 0; c < a.cols; c++) {
      const double d = load(a.x, a.x_dtype, o + c) - mean;
      var += d * d;
    }
    const double rstd = 1.0 / std::sqrt(var / (double)a.cols + a.eps);
    for (int64_t c = 0; c < a.cols; c++) {
      const double h = (load(a.x, a.x_dtype, o + c) - mean) * rstd;
      store(a.y, a.x_dtype, r * a.cols + c,
            h * (a.weight ? load(a.weight, a.param_dtype, c) : 1.0) + (a.bias ? load(a.bias, a.param_dtype, c) : 0.0));
    }
    if (a.mean) {
      a.mean[r] = (float)mean;
      a.rstd[r] = (float)rstd;
    }
  }
}

void cpu_norm_backward(const fm_layer_norm_args& a) {
  std::vector<double> dw(a.cols, 0.0), db(a.cols, 0.0);
  for (int64_t r = 0; r < a.rows; r++) {
    const int64_t o = r * a.x_stride, g = r * a.dy_stride;
    const double mean = a.mean[r], rstd = a.rstd[r];
    double sg = 0, sgh = 0;
    for (int64_t c = 0; c < a.cols; c++) {
      const double h = (load(a.x, a.x_dtype, o + c) - mean) * rstd, d = load(a.dy, a.x_dtype, g + c);
      const double t = a.weight ? d * load(a.weight, a.param_dtype, c) : d;
      sg += t;
      sgh += t * h;
      dw[c] += d * h;
      db[c] += d;
    }
    if (!a.dx) continue;
    for (int64_t c = 0; c < a.cols; c++) {
      const double h = (load(a.x, a.x_dtype, o + c) - mean) * rstd, d = load(a.dy, a.x_dtype, g + c);
      const double t = a.weight ? d * load(a.weight, a.param_dtype, c) : d;
      store(a.dx, a.x_dtype, r * a.cols + c, rstd * (t - sg / (double)a.cols - h * (sgh / (double)a.cols)));
    }
  }
  for (int64_t c = 0; c < a.cols; c++) {
    if (a.dweight) store(a.dweight, a.param_dtype, c, dw[c]);
    if (a.dbias) store(a.dbias, a.param_dtype, c, db[c]);
  }
}

// ------------------------------------------------------------------ drawing categories
static int64_t sample_row(const fm_sample_args& a, int64_t r, std::vector<int64_t>& order, std::vector<double>& z,
                          std::vector<double>& w) {
  const double t = a.temperature_rows ? a.temperature_rows[r] : a.temperature;
  const double p = a.top_p_rows ? a.top_p_rows[r] : a.top_p, m = a.min_p_rows ? a.min_p_rows[r] : a.min_p;
  const int64_t k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
  const double u = load(a.u, a.u_dtype, r);
  if (std::isnan(t) || std::isnan(p) || std::isnan(m) || std::isnan(u)) return -1;
  order.clear();
  for (int64_t c = 0; c < a.cols; c++) {
    if (a.mask && !a.mask[r * a.mask_stride + c]) continue;
    z[c] = load(a.logits, a.dtype, r * a.stride + c);
    if (std::isnan(z[c])) return -1;
    if (z[c] != -INFINITY) order.push_back(c);
  }
  if (order.empty()) return -1;
  std::stable_sort(order.begin(), order.end(), [&](int64_t i, int64_t j) { return z[i] > z[j]; });
  if (t <= 0) return order[0];
  const double top = z[order[0]];
  size_t n = order.size();
  if (k > 0 && (size_t)k < n) n = (size_t)k;
  // as on the GPU, weights are whole multiples of 2^-s: s as large as 62 bits for the sum allow, at most 51
  int s = 51;
  while (s > 0 && (a.cols - 1) >> (62 - s)) s--;
  w.resize(n);
  uint64_t total = 0;
  auto fixed = [&](int64_t c) {
    const double x = z[c] == top ? 0.0 : std::fmax((z[c] - top) * (1.0 / t), -1000.0);
    return (uint64_t)std::nearbyint(std::ldexp(std::exp(x), s));
  };
  for (size_t i = 0; i < n; i++) {
    w[i] = (double)fixed(order[i]);
    total += (uint64_t)w[i];
  }
  if (p < 1) {
    uint64_t sum = 0;
    size_t kept = 0;
    while (kept < n && (kept == 0 || (double)sum < p * (double)total)) sum += (uint64_t)w[kept++];
    n = kept;
  }
  const double floor_w = std::ldexp(std::fmin(m, 1.0), s);
  uint64_t sum = 0;
  size_t kept = 0;
  while (kept < n && (kept == 0 || w[kept] >= floor_w)) sum += (uint64_t)w[kept++];
  const double target = u * (double)sum;
  const uint64_t at = target <= 0 ? 0 : target >= (double)sum ? sum - 1 : (uint64_t)target;
  uint64_t before = 0;
  for (size_t i = 0; i < kept; i++) {
    before += (uint64_t)w[i];
    if (before > at) return order[i];
  }
  return order[0];
}

void cpu_sample(const fm_sample_args& a) {
  std::vector<int64_t> order;
  std::vector<double> z(a.cols), w;
  order.reserve(a.cols);
  w.reserve(a.cols);
  for (int64_t r = 0; r < a.rows; r++) a.out[r] = sample_row(a, r, order, z, w);
}

// ------------------------------------------------------------------ distillation
// the teacher's probabilities of row r's listed entries (0 elsewhere); returns their sum (1; 0 for an empty list), NaN
// where an index is too large
static double teacher_row(const fm_distill_args& a, int64_t r, std::vector<double>& p, std::vector<double>& logp) {
  double top = -INFINITY, sum = 0;
  bool nan = false;
  for (int64_t i = 0; i < a.k; i++) {
    const int64_t j = load_index(a.index, a.index_dtype, r * a.index_stride + i);
    logp[i] = j < 0 ? -INFINITY : load(a.teacher, a.teacher_dtype, r * a.teacher_stride + i) / a.temperature;
    if (j >= a.cols || std::isnan(logp[i]) || logp[i] == INFINITY) nan = true;
    top = std::fmax(top, logp[i]);
  }
  if (nan) return std::numeric_limits<double>::quiet_NaN();
  for (int64_t i = 0; i < a.k; i++) sum += p[i] = logp[i] == -INFINITY ? 0.0 : std::exp(logp[i] - top);
  for (int64_t i = 0; i < a.k; i++) {
    if (sum > 0) p[i] /= sum;
    logp[i] -= top + std::log(sum);
  }
  return sum > 0 ? 1.0 : 0.0;
}

void cpu_distill_forward(const fm_distill_args& a) {
  std::vector<double> p(a.k), logp(a.k);
  for (int64_t r = 0; r < a.rows; r++) {
    double top = -INFINITY, sum = 0;
    for (int64_t c = 0; c < a.cols; c++) top = std::fmax(top, load(a.logits, a.dtype, r * a.stride + c));
    for (int64_t c = 0; c < a.cols; c++) {
      const double z = load(a.logits, a.dtype, r * a.stride + c);
      if (z != -INFINITY) sum += std::exp((z - top) / a.temperature);
    }
    const double mass = teacher_row(a, r, p, logp);
    double loss = std::isnan(mass) ? mass : 0.0;
    for (int64_t i = 0; i < a.k && mass > 0; i++) {
      if (p[i] <= 0) continue;
      const double z = load(a.logits, a.dtype, r * a.stride + load_index(a.index, a.index_dtype, r * a.index_stride + i));
      loss += p[i] * (logp[i] - (z == -INFINITY ? -INFINITY : (z - top) / a.temperature) + std::log(sum));
    }
    a.loss[r] = (float)(a.temperature * a.temperature * loss);
    if (a.stats) {
      a.stats[2 * r] = (float)top;
      a.stats[2 * r + 1] = (float)sum;
    }
  }
}

void cpu_distill_backward(const fm_distill_args& a) {
  std::vector<double> p(a.k), logp(a.k), d(a.cols);
  for (int64_t r = 0; r < a.rows; r++) {
    const double top = a.stats[2 * r], sum = a.stats[2 * r + 1];
    const double mass = teacher_row(a, r, p, logp), scale = a.grad[r * a.grad_stride] * a.temperature;
    for (int64_t c = 0; c < a.cols; c++) {
      const double z = load(a.logits, a.dtype, r * a.stride + c);
      d[c] = mass == 0 ? 0 : mass * ((z == -INFINITY ? 0.0 : std::exp((z - top) / a.temperature)) / sum);
    }
    for (int64_t i = 0; i < a.k && mass > 0; i++)
      if (p[i] > 0) d[load_index(a.index, a.index_dtype, r * a.index_stride + i)] -= p[i];
    for (int64_t c = 0; c < a.cols; c++) store(a.dlogits, a.dtype, r * a.cols + c, mass == 0 ? 0.0 : scale * d[c]);
  }
}
}  // namespace fm
