// fm_torch.cpp -- the operators' calls from tensors: factory_marl_amd/ops.py checks and shapes the arguments and calls
// torch.ops.factorysim.*, whose backward passes run here without the interpreter (a Python node waits for it on the
// engine's thread: a layer norm of 64 x 128, forward and backward, took 105 us of host time with one and takes 60 like this).
// All computing is the library's; its entry points are handed over once, by `bind`.
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include "../../include/factorysim.h"

namespace {
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Entries {
  decltype(&fm_layer_norm_forward) norm_forward;
  decltype(&fm_layer_norm_backward) norm_backward;
  decltype(&fm_layer_norm_workspace) norm_workspace;
  decltype(&fm_distill_forward) distill_forward;
  decltype(&fm_distill_backward) distill_backward;
  decltype(&fm_distill_workspace) distill_workspace;
  decltype(&fm_sample_logits) sample_logits;
  decltype(&fm_sample_workspace) sample_workspace;
  decltype(&fm_last_error) last_error;
} fm;

void bind(at::IntArrayRef addresses) {
  TORCH_CHECK(addresses.size() * sizeof(void*) == sizeof(fm), "factorysim: entry points");
  std::memcpy(&fm, addresses.data(), sizeof(fm));
}

void check(int rc) { TORCH_CHECK(rc == 0, "factorysim error ", rc, ": ", fm.last_error()); }

int32_t code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FM_DTYPE_F32;
    case at::kHalf: return FM_DTYPE_F16;
    case at::kBFloat16: return FM_DTYPE_BF16;
    case at::kInt: return FM_DTYPE_I32;
    case at::kLong: return FM_DTYPE_I64;
    default: TORCH_CHECK_TYPE(false, "factorysim: element type ", t.scalar_type());
  }
}

// device and stream of a call on t: the current stream of its device, which inside a backward pass the engine has set to the
// forward pass's
template <typename Args>
void place(Args& a, const Tensor& t) {
  a.device = t.is_cpu() ? -1 : (int32_t)t.device().index();
  a.stream = t.is_cpu() ? nullptr : (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }
void* data(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

// [rows, cols] with adjacent columns
Tensor rows_of(const Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }

template <typename Args>
Tensor workspace(Args& a, int64_t bytes, const Tensor& like) {
  if (a.device < 0 || bytes <= 0) return Tensor();
  Tensor t = at::empty({bytes}, like.options().dtype(at::kByte));
  a.workspace = data(t);
  a.workspace_bytes = bytes;
  return t;
}

// A tensor that a node keeps.  What comes back may be another one (hooks on saved tensors pack and unpack as they like): its
// values are taken in any layout, another shape, type or device is refused.
struct Kept {
  SavedVariable saved;
  std::vector<int64_t> sizes;
  at::ScalarType type;
  at::Device device = at::kCPU;
  bool defined = false;

  void keep(const Tensor& t) {
    saved = SavedVariable(t, false);
    if (!(defined = t.defined())) return;
    sizes = t.sizes().vec();
    type = t.scalar_type();
    device = t.device();
  }
  Tensor get() const {
    const Tensor t = saved.unpack();
    if (!defined) return t;
    TORCH_CHECK(t.defined() && t.sizes() == at::IntArrayRef(sizes) && t.scalar_type() == type && t.device() == device,
                "factorysim: a tensor kept for the backward pass was unpacked with another shape, type or device");
    return t.dim() == 2 ? rows_of(t) : t.contiguous();
  }
  void drop() { saved.reset_data(); }
};

// a backward pass's results; differentiating them is refused, where a graph of them is being made
variable_list once(variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  auto refuse = std::make_shared<torch::autograd::DelayedError>("factorysim: this operator is differentiable once",
      (int)out.size());
  return (*refuse)(std::move(out));
}

// a forward-mode derivative would be lost without a word
void no_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(),
                              "factorysim: this operator has no forward-mode derivative");
}

// ------------------------------------------------------------------ layer norm
struct LayerNormBackward : public torch::autograd::Node {
  Kept x, weight, stats;
  at::ScalarType param;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const Tensor x_ = x.get(), w = weight.get(), s = stats.get().contiguous(), dy = rows_of(grads[0]);
    const auto parameter = x_.options().dtype(param);
    if (task_should_compute_output(0)) out[0] = at::empty(x_.sizes(), x_.options());
    if (task_should_compute_output(1)) out[1] = at::empty({x_.size(1)}, parameter);
    if (task_should_compute_output(2)) out[2] = at::empty({x_.size(1)}, parameter);
    fm_layer_norm_args a = {};
    place(a, x_);
    a.x_dtype = code(x_);
    a.param_dtype = param == x_.scalar_type() ? a.x_dtype : FM_DTYPE_F32;
    a.rows = x_.size(0);
    a.cols = x_.size(1);
    a.x = data(x_);
    a.x_stride = row_stride(x_);
    a.weight = data(w);
    a.mean = (float*)data(s);
    a.rstd = a.mean + a.rows;
    a.dy = data(dy);
    a.dy_stride = row_stride(dy);
    a.dx = data(out[0]);
    a.dweight = data(out[1]);
    a.dbias = data(out[2]);
    const Tensor work = workspace(a, out[1].defined() || out[2].defined() ? fm.norm_workspace(a.rows, a.cols) : 0, x_);
    check(fm.norm_backward(&a));
    return once(std::move(out));
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.drop();
    weight.drop();
    stats.drop();
  }
  std::string name() const override { return "LayerNormBackward"; }
};

// x [rows, cols] with adjacent columns; weight, bias [cols], contiguous
Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  const bool graph = torch::autograd::compute_requires_grad(x, w, b);
  no_tangent(x), no_tangent(w), no_tangent(b);
  const int64_t n = x.size(0);
  Tensor y = at::empty({n, x.size(1)}, x.options().requires_grad(false)), stats;
  fm_layer_norm_args a = {};
  place(a, x);
  a.x_dtype = code(x);
  a.param_dtype = w.defined() ? code(w) : b.defined() ? code(b) : a.x_dtype;
  a.rows = n;
  a.cols = x.size(1);
  a.x = data(x);
  a.x_stride = row_stride(x);
  a.weight = data(w);
  a.bias = data(b);
  a.eps = eps;
  a.y = data(y);
  if (graph) {
    stats = at::empty({2, n}, x.options().dtype(at::kFloat).requires_grad(false));
    a.mean = (float*)data(stats);
    a.rstd = n ? a.mean + n : nullptr;
  }
  check(fm.norm_forward(&a));
  if (!graph) return y;
  auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
  node->x.keep(x);
  node->weight.keep(w);
  node->stats.keep(stats);
  node->param = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
  torch::autograd::set_history(y, node);
  return y;
}

// ------------------------------------------------------------------ distillation
fm_distill_args distill_args(const Tensor& z, const Tensor& index, const Tensor& teacher, double temperature) {
  fm_distill_args a = {};
  place(a, z);
  a.dtype = code(z);
  a.index_dtype = code(index);
  a.teacher_dtype = code(teacher);
  a.rows = z.size(0);
  a.cols = z.size(1);
  a.k = index.size(1);
  a.logits = data(z);
  a.stride = row_stride(z);
  a.index = data(index);
  a.index_stride = row_stride(index);
  a.teacher = data(teacher);
  a.teacher_stride = row_stride(teacher);
  a.temperature = temperature;
  return a;
}

struct DistillBackward : public torch::autograd::Node {
  Kept z, index, teacher, stats;
  double temperature;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    if (!grads[0].defined()) return out;
    const Tensor z_ = z.get(), i = index.get(), t = teacher.get(), s = stats.get().contiguous(), &g = grads[0];
    out[0] = at::empty(z_.sizes(), z_.options());
    fm_distill_args a = distill_args(z_, i, t, temperature);
    a.stats = (float*)data(s);
    a.grad = (const float*)data(g);
    a.grad_stride = row_stride(g);
    a.dlogits = data(out[0]);
    check(fm.distill_backward(&a));
    return once(std::move(out));
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    z.drop();
    index.drop();
    teacher.drop();
    stats.drop();
  }
  std::string name() const override { return "DistillBackward"; }
};

// z [rows, cols], index and teacher [rows, k], all with adjacent columns
Tensor distill_loss(const Tensor& z, const Tensor& index, const Tensor& teacher, double temperature) {
  const bool graph = torch::autograd::compute_requires_grad(z);
  no_tangent(z), no_tangent(teacher);
  fm_distill_args a = distill_args(z, index, teacher, temperature);
  const auto floats = z.options().dtype(at::kFloat).requires_grad(false);
  Tensor loss = at::empty({a.rows}, floats), stats;
  if (graph) stats = at::empty({a.rows, 2}, floats);
  a.loss = (float*)data(loss);
  a.stats = (float*)data(stats);
  const Tensor work = workspace(a, fm.distill_workspace(a.rows, a.cols), z);
  check(fm.distill_forward(&a));
  if (!graph) return loss;
  auto node = std::shared_ptr<DistillBackward>(new DistillBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(z));
  node->z.keep(z);
  node->index.keep(index);
  node->teacher.keep(teacher);
  node->stats.keep(stats);
  node->temperature = temperature;
  torch::autograd::set_history(loss, node);
  return loss;
}
// ------------------------------------------------------------------ drawing categories
// z [rows, cols] and mask (rows or one row of them) with adjacent columns, u and the settings of each row [rows], contiguous
Tensor sample_logits(const Tensor& z, const Tensor& u, const std::optional<Tensor>& mask, double temperature, int64_t top_k,
                     double top_p, double min_p, const std::optional<Tensor>& temperature_rows,
                     const std::optional<Tensor>& top_k_rows, const std::optional<Tensor>& top_p_rows,
                     const std::optional<Tensor>& min_p_rows) {
  fm_sample_args a = {};
  place(a, z);
  a.dtype = code(z);
  a.u_dtype = u.scalar_type() == at::kDouble ? FM_DTYPE_F64 : FM_DTYPE_F32;
  a.rows = z.size(0);
  a.cols = z.size(1);
  a.logits = data(z);
  a.stride = row_stride(z);
  if (mask) {
    a.mask = (const uint8_t*)data(*mask);
    a.mask_stride = row_stride(*mask);
  }
  a.u = data(u);
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  if (temperature_rows) a.temperature_rows = (const float*)data(*temperature_rows);
  if (top_k_rows) a.top_k_rows = (const int32_t*)data(*top_k_rows);
  if (top_p_rows) a.top_p_rows = (const float*)data(*top_p_rows);
  if (min_p_rows) a.min_p_rows = (const float*)data(*min_p_rows);
  const Tensor out = at::empty({a.rows}, z.options().dtype(at::kLong).requires_grad(false));
  a.out = (int64_t*)data(out);
  const Tensor work = workspace(a, fm.sample_workspace(a.rows, a.cols), z);
  check(fm.sample_logits(&a));
  return out;
}
}  // namespace

TORCH_LIBRARY(factorysim, m) {
  m.def("bind(int[] addresses) -> ()", &bind);
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", &layer_norm);
  m.def("distill_loss(Tensor logits, Tensor teacher_index, Tensor teacher_logits, float temperature) -> Tensor", &distill_loss);
  m.def("sample_logits(Tensor logits, Tensor u, Tensor? mask, float temperature, int top_k, float top_p, float min_p, "
        "Tensor? temperature_rows, Tensor? top_k_rows, Tensor? top_p_rows, Tensor? min_p_rows) -> Tensor", &sample_logits);
}
