// fm_torch.cpp -- the operators' calls from tensors: factory_marl_amd/ops.py checks and shapes the arguments and calls
// torch.ops.factorysim.*, whose backward passes run here without the interpreter (a Python node waits for it on the
// engine's thread: a layer norm of 64 x 128, forward and backward, took 105 us of host time with one and takes 60 like this).
// All computing is the library's; its entry points are handed over once, by fm_torch_bind.
//
// Each operator is registered for the dispatch keys that it has a form of its own for: CPU and CUDA compute, Meta gives the
// results' shapes, Autograd makes the graph and calls what is below it through the dispatcher again.  So whatever stands
// between (tracing, fake tensors, function transforms) sees every call that writes memory, backward passes among them.
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cstring>
#include <initializer_list>
#include <optional>
#include <tuple>
#include <vector>

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
  decltype(&fm_last_error) last_error;
} fm;

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

// A call's arguments are checked here too, since the operators can be called directly: kernels read and write what these say.
// t: on x's device, of these sizes, of one of the types
void need(const char* name, const Tensor& t, const Tensor& x, at::IntArrayRef sizes, std::initializer_list<at::ScalarType> types) {
  TORCH_CHECK(t.device() == x.device(), "factorysim: ", name, " is on ", t.device(), ", the first input on ", x.device());
  TORCH_CHECK(t.sizes() == sizes, "factorysim: ", name, " has shape ", t.sizes(), ", not ", sizes);
  TORCH_CHECK_TYPE(std::find(types.begin(), types.end(), t.scalar_type()) != types.end(), "factorysim: ", name, " is ",
                   t.scalar_type());
}
void need_rows(const char* name, const Tensor& x) {
  TORCH_CHECK(x.dim() == 2 && x.size(1) > 0, "factorysim: ", name, " is [rows, columns], not ", x.sizes());
}
void need_parameter(const char* name, const std::optional<Tensor>& p, const Tensor& x) {
  if (p) need(name, *p, x, {x.size(1)}, {x.scalar_type(), at::kFloat});
}

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
  c10::SymDimVector sizes;
  at::ScalarType type;
  at::Device device = at::kCPU;
  bool defined = false;

  void keep(const Tensor& t) {
    saved = SavedVariable(t, false);
    if (!(defined = t.defined())) return;
    const auto now = t.sym_sizes();
    sizes.assign(now.begin(), now.end());
    type = t.scalar_type();
    device = t.device();
  }
  Tensor get() const {
    const Tensor t = saved.unpack();
    TORCH_CHECK(!defined || (t.defined() && t.sym_sizes() == c10::SymIntArrayRef(sizes.data(), sizes.size()) && t.scalar_type() == type &&
                             t.device() == device),
                "factorysim: a tensor kept for the backward pass was unpacked with another shape, type or device");
    return t;
  }
  void drop() { saved.reset_data(); }
};

template <typename N>
std::shared_ptr<N> new_node() {
  return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// the results of a backward pass on `inputs`: differentiating them is refused
template <typename... T>
void once(std::vector<Tensor>& out, const T&... inputs) {
  if (!torch::autograd::compute_requires_grad(inputs...)) return;
  auto node = std::shared_ptr<torch::autograd::Error>(
      new torch::autograd::Error("factorysim: this operator is differentiable once",
                                 torch::autograd::collect_next_edges(inputs...)),
      torch::autograd::deleteNode);
  torch::autograd::set_history(out, node);
}

// a forward-mode derivative would be lost without a word
void no_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(),
                              "factorysim: this operator has no forward-mode derivative");
}

// an operator by its name, called through the dispatcher
template <typename F>
c10::TypedOperatorHandle<F> find(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define CALL(f, ...) ([&] { static const auto op = find<decltype(f)>("factorysim::" #f); return op.call(__VA_ARGS__); }())

typedef std::optional<Tensor> Maybe;
typedef std::array<bool, 3> Three;
typedef std::tuple<Tensor, Tensor> Two;
Tensor or_none(const Maybe& t) { return t.value_or(Tensor()); }

// ------------------------------------------------------------------ computing (CPU, CUDA)
// Rows are [rows, cols], as tensors of any layout.
Tensor norm_run(const Tensor& x_, const Maybe& weight, const Maybe& bias, double eps, Tensor* stats) {
  need_rows("x", x_);
  need_parameter("weight", weight, x_);
  need_parameter("bias", bias, x_);
  TORCH_CHECK_TYPE(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "factorysim: weight and bias differ in type");
  const Tensor x = rows_of(x_), w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
  const int64_t n = x.size(0);
  Tensor y = at::empty({n, x.size(1)}, x.options());
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
  if (stats) {
    *stats = at::empty({2, n}, x.options().dtype(at::kFloat));
    a.mean = (float*)data(*stats);
    a.rstd = n ? a.mean + n : nullptr;
  }
  check(fm.norm_forward(&a));
  return y;
}

Tensor layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  return norm_run(x, weight, bias, eps, nullptr);
}

// and the rows' mean and 1 / deviation, [2, rows]
Two layer_norm_stats(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  Tensor stats;
  Tensor y = norm_run(x, weight, bias, eps, &stats);
  return Two(y, stats);
}

// of dx, dweight, dbias (of type param) those that are wanted
std::vector<Tensor> layer_norm_backward(const Tensor& dy_, const Tensor& x_, const Maybe& weight, const Tensor& stats,
                                        at::ScalarType param, Three wanted) {
  need_rows("x", x_);
  need("dy", dy_, x_, x_.sizes(), {x_.scalar_type()});
  need("stats", stats, x_, {2, x_.size(0)}, {at::kFloat});
  TORCH_CHECK_TYPE(param == x_.scalar_type() || param == at::kFloat, "factorysim: param is float32 or x's type");
  if (weight) need("weight", *weight, x_, {x_.size(1)}, {param});
  const Tensor x = rows_of(x_), dy = rows_of(dy_), s = stats.contiguous(), w = weight ? weight->contiguous() : Tensor();
  const auto parameter = x.options().dtype(param);
  Tensor dx, dw, db;
  if (wanted[0]) dx = at::empty(x.sizes(), x.options());
  if (wanted[1]) dw = at::empty({x.size(1)}, parameter);
  if (wanted[2]) db = at::empty({x.size(1)}, parameter);
  fm_layer_norm_args a = {};
  place(a, x);
  a.x_dtype = code(x);
  a.param_dtype = param == x.scalar_type() ? a.x_dtype : FM_DTYPE_F32;
  a.rows = x.size(0);
  a.cols = x.size(1);
  a.x = data(x);
  a.x_stride = row_stride(x);
  a.weight = data(w);
  a.mean = (float*)data(s);
  a.rstd = a.mean + a.rows;
  a.dy = data(dy);
  a.dy_stride = row_stride(dy);
  a.dx = data(dx);
  a.dweight = data(dw);
  a.dbias = data(db);
  const Tensor work = workspace(a, dw.defined() || db.defined() ? fm.norm_workspace(a.rows, a.cols) : 0, x);
  check(fm.norm_backward(&a));
  std::vector<Tensor> out;
  for (const Tensor& t : {dx, dw, db})
    if (t.defined()) out.push_back(t);
  return out;
}

void check_distill(const Tensor& z, const Tensor& index, const Tensor& teacher) {
  need_rows("logits", z);
  need_rows("teacher_index", index);
  need("teacher_index", index, z, {z.size(0), index.size(1)}, {at::kInt, at::kLong});
  need("teacher_logits", teacher, z, index.sizes(), {at::kFloat, at::kHalf, at::kBFloat16});
}

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

Tensor distill_run(const Tensor& z_, const Tensor& index_, const Tensor& teacher_, double temperature, Tensor* stats) {
  check_distill(z_, index_, teacher_);
  const Tensor z = rows_of(z_), index = rows_of(index_), teacher = rows_of(teacher_);
  fm_distill_args a = distill_args(z, index, teacher, temperature);
  const auto floats = z.options().dtype(at::kFloat);
  Tensor loss = at::empty({a.rows}, floats);
  a.loss = (float*)data(loss);
  if (stats) {
    *stats = at::empty({a.rows, 2}, floats);
    a.stats = (float*)data(*stats);
  }
  const Tensor work = workspace(a, fm.distill_workspace(a.rows, a.cols), z);
  check(fm.distill_forward(&a));
  return loss;
}

Tensor distill_loss(const Tensor& z, const Tensor& index, const Tensor& teacher, double temperature) {
  return distill_run(z, index, teacher, temperature, nullptr);
}

// and the rows' largest logit and sum of exp, [rows, 2]
Two distill_loss_stats(const Tensor& z, const Tensor& index, const Tensor& teacher, double temperature) {
  Tensor stats;
  Tensor loss = distill_run(z, index, teacher, temperature, &stats);
  return Two(loss, stats);
}

Tensor distill_backward(const Tensor& grad, const Tensor& z_, const Tensor& index_, const Tensor& teacher_, const Tensor& stats,
                        double temperature) {
  check_distill(z_, index_, teacher_);
  need("grad", grad, z_, {z_.size(0)}, {at::kFloat});
  need("stats", stats, z_, {z_.size(0), 2}, {at::kFloat});
  const Tensor z = rows_of(z_), index = rows_of(index_), teacher = rows_of(teacher_), s = stats.contiguous();
  Tensor dz = at::empty(z.sizes(), z.options());
  fm_distill_args a = distill_args(z, index, teacher, temperature);
  a.stats = (float*)data(s);
  a.grad = (const float*)data(grad);
  a.grad_stride = row_stride(grad);
  a.dlogits = data(dz);
  check(fm.distill_backward(&a));
  return dz;
}

// mask: as the logits, or one row of them; u and the settings of each row: [rows]
Tensor sample_logits(const Tensor& z_, const Tensor& u_, const Maybe& mask_, double temperature, int64_t top_k, double top_p,
                     double min_p, const Maybe& temperature_rows, const Maybe& top_k_rows, const Maybe& top_p_rows,
                     const Maybe& min_p_rows) {
  need_rows("logits", z_);
  const int64_t n = z_.size(0);
  need("u", u_, z_, {n}, {at::kFloat, at::kDouble});
  if (mask_) need("mask", *mask_, z_, {mask_->dim() && mask_->size(0) == 1 ? 1 : n, z_.size(1)}, {at::kBool});
  if (temperature_rows) need("temperature", *temperature_rows, z_, {n}, {at::kFloat});
  if (top_k_rows) need("top_k", *top_k_rows, z_, {n}, {at::kInt});
  if (top_p_rows) need("top_p", *top_p_rows, z_, {n}, {at::kFloat});
  if (min_p_rows) need("min_p", *min_p_rows, z_, {n}, {at::kFloat});
  const Tensor z = rows_of(z_), u = u_.contiguous(), mask = mask_ ? rows_of(*mask_) : Tensor();
  auto flat = [](const Maybe& t) { return t ? t->contiguous() : Tensor(); };
  const Tensor t_rows = flat(temperature_rows), k_rows = flat(top_k_rows), p_rows = flat(top_p_rows), m_rows = flat(min_p_rows);
  fm_sample_args a = {};
  place(a, z);
  a.dtype = code(z);
  a.u_dtype = u.scalar_type() == at::kDouble ? FM_DTYPE_F64 : FM_DTYPE_F32;
  a.rows = n;
  a.cols = z.size(1);
  a.logits = data(z);
  a.stride = row_stride(z);
  if (mask.defined()) {
    a.mask = (const uint8_t*)data(mask);
    a.mask_stride = row_stride(mask);
  }
  a.u = data(u);
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.temperature_rows = (const float*)data(t_rows);
  a.top_k_rows = (const int32_t*)data(k_rows);
  a.top_p_rows = (const float*)data(p_rows);
  a.min_p_rows = (const float*)data(m_rows);
  Tensor out = at::empty({a.rows}, z.options().dtype(at::kLong));
  a.out = (int64_t*)data(out);
  check(fm.sample_logits(&a));
  return out;
}

// ------------------------------------------------------------------ shapes (Meta)
namespace meta {
Tensor of(const Tensor& like, std::vector<c10::SymInt> sizes, at::ScalarType type) {
  return at::empty_symint(sizes, like.options().dtype(type));
}
Tensor layer_norm(const Tensor& x, const Maybe&, const Maybe&, double) { return of(x, x.sym_sizes().vec(), x.scalar_type()); }
Two layer_norm_stats(const Tensor& x, const Maybe& w, const Maybe& b, double eps) {
  return Two(layer_norm(x, w, b, eps), of(x, {2, x.sym_size(0)}, at::kFloat));
}
std::vector<Tensor> layer_norm_backward(const Tensor&, const Tensor& x, const Maybe&, const Tensor&, at::ScalarType param,
                                        Three wanted) {
  std::vector<Tensor> out;
  if (wanted[0]) out.push_back(of(x, x.sym_sizes().vec(), x.scalar_type()));
  for (int i = 1; i < 3; i++)
    if (wanted[i]) out.push_back(of(x, {x.sym_size(1)}, param));
  return out;
}
Tensor distill_loss(const Tensor& z, const Tensor&, const Tensor&, double) { return of(z, {z.sym_size(0)}, at::kFloat); }
Two distill_loss_stats(const Tensor& z, const Tensor& index, const Tensor& teacher, double temperature) {
  return Two(distill_loss(z, index, teacher, temperature), of(z, {z.sym_size(0), 2}, at::kFloat));
}
Tensor distill_backward(const Tensor&, const Tensor& z, const Tensor&, const Tensor&, const Tensor&, double) {
  return of(z, z.sym_sizes().vec(), z.scalar_type());
}
Tensor sample_logits(const Tensor& z, const Tensor&, const Maybe&, double, int64_t, double, double, const Maybe&, const Maybe&,
                     const Maybe&, const Maybe&) {
  return of(z, {z.sym_size(0)}, at::kLong);
}
}  // namespace meta

// ------------------------------------------------------------------ graphs (Autograd)
namespace graph {
struct LayerNormBackward : public torch::autograd::Node {
  Kept x, weight, stats;
  at::ScalarType param;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const Three wanted = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
    const Tensor x_ = x.get(), w = weight.get(), s = stats.get();
    std::optional<at::AutoDispatchBelowADInplaceOrView> below;
    if (!at::GradMode::is_enabled()) below.emplace();  // no graph of the results is being made
    const std::vector<Tensor> got =
        CALL(layer_norm_backward, grads[0], x_, w.defined() ? Maybe(w) : Maybe(), s, param, wanted);
    size_t next = 0;
    for (int i = 0; i < 3; i++)
      if (wanted[i]) out[i] = got[next++];
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.drop();
    weight.drop();
    stats.drop();
  }
  std::string name() const override { return "LayerNormBackward"; }
};

Two layer_norm_stats(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  const Tensor w = or_none(weight), b = or_none(bias);
  no_tangent(x), no_tangent(w), no_tangent(b);
  const bool wanted = torch::autograd::compute_requires_grad(x, w, b);
  Two out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = CALL(layer_norm_stats, x, weight, bias, eps);
  }
  if (!wanted) return out;
  auto node = new_node<LayerNormBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
  node->x.keep(x);
  node->weight.keep(w);
  node->stats.keep(std::get<1>(out));
  node->param = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
  torch::autograd::set_history(std::get<0>(out), node);
  return out;
}

Tensor layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  if (torch::autograd::compute_requires_grad(x, or_none(weight), or_none(bias)))
    return std::get<0>(layer_norm_stats(x, weight, bias, eps));
  no_tangent(x), no_tangent(or_none(weight)), no_tangent(or_none(bias));
  at::AutoDispatchBelowADInplaceOrView below;
  return CALL(layer_norm, x, weight, bias, eps);
}

std::vector<Tensor> layer_norm_backward(const Tensor& dy, const Tensor& x, const Maybe& weight, const Tensor& stats,
                                        at::ScalarType param, Three wanted) {
  std::vector<Tensor> out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = CALL(layer_norm_backward, dy, x, weight, stats, param, wanted);
  }
  once(out, dy, x, or_none(weight), stats);
  return out;
}

struct DistillBackward : public torch::autograd::Node {
  Kept z, index, teacher, stats;
  double temperature;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    const Tensor z_ = z.get(), i = index.get(), t = teacher.get(), s = stats.get();
    std::optional<at::AutoDispatchBelowADInplaceOrView> below;
    if (!at::GradMode::is_enabled()) below.emplace();
    return {CALL(distill_backward, grads[0], z_, i, t, s, temperature)};
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

// the teacher's logits are constants: their gradient would be lost without a word
void constant(const Tensor& teacher) {
  TORCH_CHECK(!torch::autograd::compute_requires_grad(teacher),
              "factorysim: teacher_logits requires a gradient, which this loss does not give: detach it");
}

Two distill_loss_stats(const Tensor& z, const Tensor& index, const Tensor& teacher, double temperature) {
  no_tangent(z), no_tangent(teacher), constant(teacher);
  const bool wanted = torch::autograd::compute_requires_grad(z);
  Two out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = CALL(distill_loss_stats, z, index, teacher, temperature);
  }
  if (!wanted) return out;
  auto node = new_node<DistillBackward>();
  node->set_next_edges(torch::autograd::collect_next_edges(z));
  node->z.keep(z);
  node->index.keep(index);
  node->teacher.keep(teacher);
  node->stats.keep(std::get<1>(out));
  node->temperature = temperature;
  torch::autograd::set_history(std::get<0>(out), node);
  return out;
}

Tensor distill_loss(const Tensor& z, const Tensor& index, const Tensor& teacher, double temperature) {
  if (torch::autograd::compute_requires_grad(z)) return std::get<0>(distill_loss_stats(z, index, teacher, temperature));
  no_tangent(z), no_tangent(teacher), constant(teacher);
  at::AutoDispatchBelowADInplaceOrView below;
  return CALL(distill_loss, z, index, teacher, temperature);
}

Tensor distill_backward(const Tensor& grad, const Tensor& z, const Tensor& index, const Tensor& teacher, const Tensor& stats,
                        double temperature) {
  std::vector<Tensor> out(1);
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out[0] = CALL(distill_backward, grad, z, index, teacher, stats, temperature);
  }
  once(out, grad, z, stats);
  return out[0];
}
}  // namespace graph
}  // namespace

// the library's entry points, in the order of Entries; false: not as many
extern "C" bool fm_torch_bind(void* const* addresses, int64_t count) {
  if (count * sizeof(void*) != sizeof(fm)) return false;
  std::memcpy(&fm, addresses, sizeof(fm));
  return true;
}

TORCH_LIBRARY(factorysim, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_stats(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor stats, ScalarType param, bool[3] wanted) -> Tensor[]");
  m.def("distill_loss(Tensor logits, Tensor teacher_index, Tensor teacher_logits, float temperature) -> Tensor");
  m.def("distill_loss_stats(Tensor logits, Tensor teacher_index, Tensor teacher_logits, float temperature) -> (Tensor, Tensor)");
  m.def("distill_backward(Tensor grad, Tensor logits, Tensor teacher_index, Tensor teacher_logits, Tensor stats, "
        "float temperature) -> Tensor");
  m.def("sample_logits(Tensor logits, Tensor u, Tensor? mask, float temperature, int top_k, float top_p, float min_p, "
        "Tensor? temperature_rows, Tensor? top_k_rows, Tensor? top_p_rows, Tensor? min_p_rows) -> Tensor");
}
#define ALL_OF(m, from) \
  m.impl("layer_norm", from layer_norm); \
  m.impl("layer_norm_stats", from layer_norm_stats); \
  m.impl("layer_norm_backward", from layer_norm_backward); \
  m.impl("distill_loss", from distill_loss); \
  m.impl("distill_loss_stats", from distill_loss_stats); \
  m.impl("distill_backward", from distill_backward)
TORCH_LIBRARY_IMPL(factorysim, CPU, m) {
  ALL_OF(m, &);
  m.impl("sample_logits", &sample_logits);
}
TORCH_LIBRARY_IMPL(factorysim, CUDA, m) {
  ALL_OF(m, &);
  m.impl("sample_logits", &sample_logits);
}
TORCH_LIBRARY_IMPL(factorysim, Meta, m) {
  ALL_OF(m, &meta::);
  m.impl("sample_logits", &meta::sample_logits);
}
TORCH_LIBRARY_IMPL(factorysim, Autograd, m) {
  ALL_OF(m, &graph::);
  m.impl("sample_logits", torch::CppFunction::makeFallthrough());  // whole numbers: no gradient
}
