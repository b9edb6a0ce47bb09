// Passes of the token operators (layer norm, attention, rotary positions, dropout): checks, allocations, launches and their nodes of the autograd graph, without a return to
// Python in between.  (A forward and a backward pass of a layer norm of 16471 x 387 tokens, with the node in Python 122 us, all of it host time.)
#include "host.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/dynamo/compiled_autograd.h>

#include <pybind11/stl.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <cmath>

#include <ATen/cuda/CUDAGeneratorImpl.h>
#include <ATen/cuda/EmptyTensor.h>

#include "attention.cuh"
#include "dropout.cuh"
#include "layer_norm.cuh"
#include "rotary.cuh"

namespace {

using mkh::Tensor;
using OptTensor = c10::optional<Tensor>;

Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
template <typename T>
T* ptr_or_null(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
bool is_f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
bool native_type(const Tensor& t) { return is_f32(t) || t.scalar_type() == at::kBFloat16; }

using torch::autograd::variable_list;

// A dense tensor, without the dispatcher's way there (half a microsecond each, of which a backward pass has seven)
Tensor room(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
Tensor room(const Tensor& like) { return room(like.sizes(), like, like.scalar_type()); }

bool records(std::initializer_list<const Tensor*> ts) {
  bool any = false;
  for (const Tensor* t : ts) any = any || (t->defined() && t->requires_grad());
  return any && at::GradMode::is_enabled();
}

// Whether these tensors are no more than their memory and their autograd graph, so that kernels may take them.  Not so in `torch.func`'s transforms,
// forward-mode differentiation, tracing and dispatch modes, and for subclasses: what stands for a tensor there has no memory, or somebody has to see each
// operation.
bool plain(std::initializer_list<const Tensor*> ts) {
  using K = c10::DispatchKey;
  const c10::DispatchKeySet watched({K::Python, K::PythonTLSSnapshot, K::Tracer, K::FuncTorchDynamicLayerFrontMode, K::VmapMode, K::Functionalize});
  const c10::DispatchKeySet wrapped({K::Python, K::FuncTorchGradWrapper, K::FuncTorchBatched, K::Batched, K::Functionalize});
  if (c10::impl::tls_local_dispatch_key_set().included_.has_any(watched)) return false;
  for (const Tensor* t : ts)
    if (t->defined() && (t->key_set().has_any(wrapped) || t->_fw_grad(0).defined())) return false;
  return true;
}

// Launches of backward passes, which autograd runs in threads of its own, and of calls that nobody counts from outside
std::atomic<int64_t> background{0};
struct Backward {
  int64_t before = mkh::launches();
  ~Backward() {
    background += mkh::launches() - before;
    mkh::launches() = before;
  }
};
// Gradients that a graph is to be made of (create_graph) raise where that is differentiated
variable_list once_differentiable(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  const int n = static_cast<int>(grads.size());
  return (*std::make_shared<torch::autograd::DelayedError>("makani_b200: this operator has no second derivatives", n))(std::move(grads));
}

// A node with fields for operators whose inputs are all they keep beside numbers: `Op::gradients(grads, saved, fields, need)`; `need` of every edge.  (Torch's
// Function for extensions finds what it keeps by name: 11 us more of a forward and a backward pass on the host, now 64 for the rotation of 64 tokens.)
struct Fields {
  std::array<int64_t, 8> whole{};
  std::array<double, 2> real{};
};
template <typename Op>
struct FieldNode : torch::autograd::Node {
  Fields fields;
  std::vector<torch::autograd::SavedVariable> saved;

  // Behind `outputs`, with an edge to each of `inputs`
  static void record(const variable_list& outputs, const variable_list& inputs, const variable_list& kept, const Fields& f) {
    const std::shared_ptr<FieldNode> node(new FieldNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs));
    node->fields = f;
    node->saved.reserve(kept.size());
    for (const Tensor& t : kept) node->saved.emplace_back(t, false);
    for (const Tensor& t : outputs) torch::autograd::set_history(t, node);
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (auto& v : saved) v.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    variable_list kept;
    kept.reserve(saved.size());
    for (const auto& v : saved) kept.push_back(v.unpack());
    return gradients(grads, kept, fields, needed());
  }
  std::vector<bool> needed() const {
    std::vector<bool> n(num_outputs());
    for (size_t i = 0; i < n.size(); ++i) n[i] = next_edge(i).is_valid() && task_should_compute_output(i);
    return n;
  }
  static variable_list gradients(const variable_list& grads, const variable_list& kept, const Fields& f, const std::vector<bool>& need) {
    const Backward count;
    return Op::gradients(grads, kept, f, need);
  }

  // A compiled backward pass calls `gradients` as one opaque operation, as it does with nodes of torch's Function
  static variable_list call(const variable_list& grads, const std::vector<c10::IValue>& args) {
    torch::dynamo::autograd::PackedArgs packed(args);
    const auto kept = packed.unpack<variable_list>();
    Fields f;
    for (auto& v : f.whole) v = packed.unpack<int64_t>();
    for (auto& v : f.real) v = packed.unpack<double>();
    return gradients(grads, kept, f, packed.unpack<std::vector<bool>>());
  }
  void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
    for (const auto& v : saved) args.collect(v, false);
    for (const auto v : fields.whole) args.collect(v);
    for (const auto v : fields.real) args.collect(v);
  }
  variable_list apply_with_saved(const variable_list& grads, torch::dynamo::autograd::SwapSavedVariables& swap) override {
    using namespace torch::dynamo::autograd;
    variable_list kept;
    for (auto& v : saved) {
      swap.before(v);
      kept.push_back(v.unpack());
    }
    PackedArgs packed;
    packed.pack(kept);
    for (const auto v : fields.whole) packed.pack(v);
    for (const auto v : fields.real) packed.pack(v);
    packed.pack(needed());
    const auto metadata = IValuePacker<std::vector<std::optional<torch::autograd::InputMetadata>>>::pack(get_input_metadata(next_edges()));
    const auto args = std::move(packed).vec();
    std::vector<at::TypePtr> schema;
    for (const auto& v : args) schema.emplace_back(v.isTensor() ? at::TypePtr(at::TensorType::get()) : v.type());
    const auto& python = getPyCompilerInterface();
    const auto name = python->bind_function(swap.get_py_compiler(), Op::NAME, call, schema, /*is_custom_function=*/true, /*is_traceable=*/false);
    auto out = python->call_function(swap.get_py_compiler(), "apply_functional", name, grads, args, metadata);
    for (auto& v : saved) swap.after(v);
    return out;
  }
};

// ------------------------------------------------------------------------------------------ layer norm

// Rows of a tensor whose last dimension is dense, as two nested strides; a copy where it takes more
struct Rows {
  Tensor t;
  int64_t rows = 0, C = 0, inner = 1, outer_stride = 0, inner_stride = 0;
  explicit Rows(const Tensor& x) : t(x), C(x.size(-1)) {
    rows = C ? x.numel() / C : 0;
    if (!collapse()) {
      t = x.contiguous();
      MK_CHECK(collapse(), "layer norm: dense rows expected");
    }
  }

 private:
  bool collapse() {
    if (C > 1 && t.stride(-1) != 1) return false;
    int64_t size[2] = {1, 1}, stride[2] = {0, 0};      // innermost first
    int n = 0;
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
      if (t.size(d) == 1) continue;
      if (n > 0 && t.stride(d) == size[n - 1] * stride[n - 1]) {
        size[n - 1] *= t.size(d);
      } else {
        if (n == 2) return false;
        size[n] = t.size(d);
        stride[n++] = t.stride(d);
      }
    }
    inner = std::max<int64_t>(1, size[0]);
    inner_stride = stride[0];
    outer_stride = stride[1];
    return true;
  }
};

// A weight or a bias as the kernels read it: dense, in a type of theirs
Tensor channel_values(const OptTensor& t, const Tensor& x, const char* what) {
  if (!t.has_value() || !t->defined()) return Tensor();
  MK_CHECK(t->device() == x.device(), "layer norm: tensors must be on one CUDA device");
  MK_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), "layer norm: one ", what, " per channel expected");
  if (is_f32(*t) || (native_type(*t) && t->size(0) <= mk::LN_HALF_PARAMS)) return t->is_contiguous() ? *t : t->detach().contiguous();
  return t->detach().to(at::kFloat).contiguous();
}

// (s, y, statistics, weight as the kernel reads it): s and the statistics where they are asked for
std::tuple<OptTensor, Tensor, OptTensor, OptTensor> layer_norm_forward(const Tensor& x, const OptTensor& residual, const OptTensor& weight,
                                                                       const OptTensor& bias, double eps, bool out_f32, bool train) {
  MK_CHECK(x.is_cuda() && native_type(x) && x.dim() >= 1, "layer norm: bf16 or fp32 CUDA tensors expected");
  c10::cuda::CUDAGuard guard(x.device());
  const Rows in(x);
  MK_CHECK(in.C >= 1 && in.C <= mk::LN_CHANNELS, "layer norm: 1 to ", mk::LN_CHANNELS, " channels expected");
  const Tensor w = channel_values(weight, x, "weight"), b = channel_values(bias, x, "bias");
  Tensor r, s, stats, y = at::empty(x.sizes(), x.options().dtype(out_f32 ? at::kFloat : at::kBFloat16));
  if (residual.has_value() && residual->defined()) {
    MK_CHECK(residual->device() == x.device() && residual->sizes() == x.sizes() && native_type(*residual) && (is_f32(x) || !is_f32(*residual)),
             "layer norm: the residual must have the shape and device of x, and no wider type");
    r = residual->contiguous();
    s = at::empty(x.sizes(), x.options());
  }
  if (train) stats = at::empty({in.rows, 2}, x.options().dtype(at::kFloat));
  mk::LnForward p{};
  p.x = in.t.data_ptr();
  p.r = ptr_or_null<void>(r);
  p.s = ptr_or_null<void>(s);
  p.y = y.data_ptr();
  p.w = ptr_or_null<void>(w);
  p.b = ptr_or_null<void>(b);
  p.w_f32 = w.defined() && is_f32(w);
  p.b_f32 = b.defined() && is_f32(b);
  p.stats = ptr_or_null<float2>(stats);
  p.rows = in.rows;
  p.C = static_cast<int>(in.C);
  p.inner = in.inner;
  p.outer_stride = in.outer_stride;
  p.inner_stride = in.inner_stride;
  p.eps = static_cast<float>(eps);
  p.x_f32 = is_f32(x);
  p.r_f32 = r.defined() && is_f32(r);
  p.y_f32 = out_f32;
  mkh::launches() += in.rows > 0;
  mkh::check(mk::layer_norm_fwd(p, mkh::stream()), "layer_norm_fwd");
  return {maybe(s), y, maybe(stats), maybe(w)};
}

// (dx, dr, dweight, dbias); `half_copy`: dr, dx in bf16; `half_dw`, `half_db`: these in bf16
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& x, const Tensor& dy, const OptTensor& ds, const OptTensor& weight,
                                                                        const Tensor& stats, bool need_params, bool half_dw, bool half_db, bool half_copy) {
  MK_CHECK(x.is_cuda() && native_type(x) && native_type(dy) && dy.device() == x.device() && dy.sizes() == x.sizes(),
           "layer norm: gradients in the shape of x and on its device expected");
  c10::cuda::CUDAGuard guard(x.device());
  const Rows in(x);
  MK_CHECK(stats.is_cuda() && is_f32(stats) && stats.is_contiguous() && stats.numel() == 2 * in.rows, "layer norm: statistics of every row expected");
  const Tensor w = channel_values(weight, x, "weight"), g = dy.contiguous();
  Tensor d, dr, dw, db, part, dx = at::empty(x.sizes(), x.options());
  if (ds.has_value() && ds->defined()) {
    MK_CHECK(ds->device() == x.device() && ds->sizes() == x.sizes() && ds->scalar_type() == x.scalar_type(),
             "layer norm: the gradient of the sum must be like the sum");
    d = ds->contiguous();
  }
  if (half_copy) dr = at::empty(x.sizes(), x.options().dtype(at::kBFloat16));
  if (need_params) {
    // (no rows: no kernel that writes them)
    auto room = [&](bool half) {
      const auto options = x.options().dtype(half ? at::kBFloat16 : at::kFloat);
      return in.rows ? at::empty({in.C}, options) : at::zeros({in.C}, options);
    };
    dw = room(half_dw);
    db = room(half_db);
    const int64_t n = mk::layer_norm_scratch(in.rows, static_cast<int>(in.C));
    if (n) part = at::empty({n}, x.options().dtype(at::kFloat));
  }
  mk::LnBackward p{};
  p.x = in.t.data_ptr();
  p.dy = g.data_ptr();
  p.ds = ptr_or_null<void>(d);
  p.dx = dx.data_ptr();
  p.dr = ptr_or_null<void>(dr);
  p.w = ptr_or_null<void>(w);
  p.w_f32 = w.defined() && is_f32(w);
  p.stats = static_cast<const float2*>(stats.data_ptr());
  p.dw = ptr_or_null<void>(dw);
  p.db = ptr_or_null<void>(db);
  p.dw_f32 = !half_dw;
  p.db_f32 = !half_db;
  p.part = ptr_or_null<float>(part);
  p.rows = in.rows;
  p.C = static_cast<int>(in.C);
  p.inner = in.inner;
  p.outer_stride = in.outer_stride;
  p.inner_stride = in.inner_stride;
  p.x_f32 = is_f32(x);
  p.y_f32 = is_f32(g);
  int n = 0;
  mkh::check(mk::layer_norm_bwd(p, &n, mkh::stream()), "layer_norm_bwd");
  mkh::launches() += n;
  return {dx, maybe(dr), maybe(dw), maybe(db)};
}

// The same in torch's operations, for gradients that are to be differentiated in their turn or are not for kernels: (dx, dweight, dbias) in fp32, dx with `ds`
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward_graph(const Tensor& x, const Tensor& dy, const Tensor& ds, const Tensor& weight, double eps) {
  const Tensor xf = x.to(at::kFloat), dyf = dy.to(at::kFloat), off = xf - xf.mean(-1, true);
  const Tensor rstd = ((off * off).mean(-1, true) + eps).rsqrt(), xh = off * rstd, g = weight.defined() ? dyf * weight.to(at::kFloat) : dyf;
  Tensor dx = rstd * (g - g.mean(-1, true) - xh * (g * xh).mean(-1, true));
  if (ds.defined()) dx = dx + ds.to(at::kFloat);
  const int64_t C = x.size(-1), rows = x.numel() / C;
  return {dx, (dyf * xh).reshape({rows, C}).sum(0), dyf.reshape({rows, C}).sum(0)};
}

// The node behind s, if there is a sum, and y; its edges lead to x, the residual, weight and bias.  (A node with fields: torch's Function for extensions, which
// finds them by name, took 77 us where this takes 69, forward and backward of 256 x 32 in fp32; torch's own norm takes 68.)
struct LayerNormNode : torch::autograd::Node {
  // What it keeps beside tensors.  half: a residual in bf16 beside an fp32 x takes its gradient in its own type; half_dw, half_db: as the parameters;
  // own_weight: the kernels read the weight as it is, else a copy that is saved too
  struct Form {
    double eps = 0.0;
    bool added = false, half = false, half_dw = false, half_db = false, own_weight = false;
  };
  Form form;
  torch::autograd::SavedVariable source, weight, read_weight, stats;      // source: x, or s

  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (auto* v : {&source, &weight, &read_weight, &stats}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    return gradients(grads, {source.unpack(form.added ? getptr() : nullptr), weight.unpack(), read_weight.unpack(), stats.unpack()}, form, needed());
  }
  std::vector<bool> needed() const {
    return {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2), task_should_compute_output(3)};
  }

  // `saved`: source, weight, read_weight, stats; `need`: of x, the residual, weight and bias
  static variable_list gradients(const variable_list& grads, const variable_list& saved, const Form& f, const std::vector<bool>& need) {
    const Backward count;
    const Tensor &x = saved[0], &dy = grads.back(), ds = f.added ? grads[0] : Tensor();
    variable_list out(4);
    if (!dy.defined()) {
      if (need[0]) out[0] = ds;
      if (need[1] && ds.defined()) out[1] = f.half ? ds.to(at::kBFloat16) : ds;
      return out;
    }
    if (at::GradMode::is_enabled() || !plain({&x, &dy, &ds})) {      // (create_graph, batches of gradients, a traced backward pass)
      auto [dx, dw, db] = layer_norm_backward_graph(x, dy, ds, saved[1], f.eps);
      if (need[0]) out[0] = dx.to(x.scalar_type());
      if (need[1]) out[1] = dx.to(f.half ? at::kBFloat16 : x.scalar_type());
      if (need[2]) out[2] = dw;
      if (need[3]) out[3] = db;
      return out;
    }
    const at::AutoDispatchBelowAutograd below;
    auto [dx, dr, dw, db] = layer_norm_backward(x, dy, maybe(ds), maybe(saved[f.own_weight ? 1 : 2]), saved[3], need[2] || need[3], f.half_dw, f.half_db,
                                                f.half && need[1]);
    if (need[0]) out[0] = dx;
    if (need[1]) out[1] = f.half ? *dr : dx;
    if (need[2]) out[2] = *dw;
    if (need[3]) out[3] = *db;
    return out;
  }

  // A compiled backward pass calls `gradients` as one opaque operation, as it does with nodes of torch's Function
  static variable_list call(const variable_list& grads, const std::vector<c10::IValue>& args) {
    torch::dynamo::autograd::PackedArgs packed(args);
    const auto saved = packed.unpack<variable_list>();
    Form f;
    f.eps = packed.unpack<double>();
    for (bool* b : {&f.added, &f.half, &f.half_dw, &f.half_db, &f.own_weight}) *b = packed.unpack<bool>();
    return gradients(grads, saved, f, packed.unpack<std::vector<bool>>());
  }
  void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
    args.collect(source, form.added);
    for (auto* v : {&weight, &read_weight, &stats}) args.collect(*v, false);
    args.collect(form.eps);
    for (const bool b : {form.added, form.half, form.half_dw, form.half_db, form.own_weight}) args.collect(b);
  }
  variable_list apply_with_saved(const variable_list& grads, torch::dynamo::autograd::SwapSavedVariables& saved) override {
    using namespace torch::dynamo::autograd;
    torch::autograd::SavedVariable* const all[] = {&source, &weight, &read_weight, &stats};
    variable_list tensors;
    for (auto* v : all) {
      saved.before(*v);
      tensors.push_back(v->unpack(v == &source && form.added ? getptr() : nullptr));
    }
    PackedArgs packed;
    packed.pack(tensors);
    packed.pack(form.eps);
    for (const bool b : {form.added, form.half, form.half_dw, form.half_db, form.own_weight}) packed.pack(b);
    packed.pack(needed());
    const auto metadata = IValuePacker<std::vector<std::optional<torch::autograd::InputMetadata>>>::pack(get_input_metadata(next_edges()));
    const auto args = std::move(packed).vec();
    std::vector<at::TypePtr> schema;
    for (const auto& v : args) schema.emplace_back(v.isTensor() ? at::TypePtr(at::TensorType::get()) : v.type());
    const auto& python = getPyCompilerInterface();
    const auto name = python->bind_function(saved.get_py_compiler(), "LayerNormNode", call, schema, /*is_custom_function=*/true, /*is_traceable=*/false);
    auto out = python->call_function(saved.get_py_compiler(), "apply_functional", name, grads, args, metadata);
    for (auto* v : all) saved.after(*v);
    return out;
  }
};

// (s and) y; nothing where the tensors are not for kernels
variable_list layer_norm(const Tensor& x, const OptTensor& residual, const OptTensor& weight, const OptTensor& bias, double eps, bool out_f32) {
  const Tensor r = value(residual), w = value(weight), b = value(bias);
  if (!plain({&x, &r, &w, &b})) return {};
  const bool train = records({&x, &r, &w, &b});
  Tensor s, y, stats, read;
  {
    const at::AutoDispatchBelowAutograd below;
    auto [sum, out, statistics, read_weight] = layer_norm_forward(x, residual, weight, bias, eps, out_f32, train);
    s = value(sum), y = out, stats = value(statistics), read = value(read_weight);
  }
  if (train) {
    const std::shared_ptr<LayerNormNode> node(new LayerNormNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, r, w, b));
    node->form = {eps, s.defined(), s.defined() && r.scalar_type() != x.scalar_type(), w.defined() && w.scalar_type() == at::kBFloat16,
                  b.defined() && b.scalar_type() == at::kBFloat16, read.is_same(w)};
    if (s.defined()) torch::autograd::set_history(s, node);
    torch::autograd::set_history(y, node);
    using torch::autograd::SavedVariable;
    node->source = SavedVariable(s.defined() ? s : x, s.defined());
    node->weight = SavedVariable(w, false);
    if (!node->form.own_weight) node->read_weight = SavedVariable(read, false);
    node->stats = SavedVariable(stats, false);
  }
  if (s.defined()) return {s, y};
  return {y};
}

// ------------------------------------------------------------------------------------------ attention

__nv_bfloat16* bf(const Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }

// (what a dimension of size one has for a stride says nothing: torch lets it be anything, in a contiguous tensor too)
mk::AttnTensor view_of(const Tensor& t) {
  auto stride = [&](int d) { return t.size(d) == 1 ? t.size(3) : t.stride(d); };
  return {bf(t), stride(1), stride(2), stride(0)};
}

// [B, N, heads, D] as the kernels read it: dense channels, strides of whole 16-byte vectors, none of them zero; a copy where it is not
Tensor readable(const Tensor& t) {
  bool fits = t.stride(3) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  for (int d = 0; d < 3; ++d) fits = fits && (t.size(d) == 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0 && t.stride(d) < (1ll << 34)));
  if (fits) return t;
  const Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
}

// Which tokens see which: `left` and `right` below zero are without end
struct Mask {
  bool causal = false;
  int64_t left = -1, right = -1, sinks = 0;
};

mk::AttnShape shape_of(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets, const Mask& mask, double scale) {
  auto bf16 = [](const Tensor& t) { return t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 4; };
  MK_CHECK(bf16(q) && bf16(k) && bf16(v), "attention: bf16 CUDA tensors [B, N, heads, D] expected");
  MK_CHECK(k.device() == q.device() && v.device() == q.device(), "attention: tensors must be on one CUDA device");
  MK_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3),
           "attention: queries, keys and values must be of the same tokens and channels");
  MK_CHECK(q.size(2) > 0 && k.size(2) > 0 && q.size(2) % k.size(2) == 0, "attention: heads of keys must divide those of queries");
  MK_CHECK(q.size(3) > 0 && q.size(3) % 8 == 0 && q.size(3) <= mk::ATTN_WIDTH, "attention: 8, 16, .., ", mk::ATTN_WIDTH, " channels of a head expected");
  MK_CHECK(scale > 0.0 && std::isfinite(scale), "attention: a positive scale expected");
  MK_CHECK(q.size(0) * q.size(1) * q.size(2) < (1ll << 31) - (1ll << 24), "attention: too many rows");
  mk::AttnShape p{};
  p.B = static_cast<int>(q.size(0));
  p.N = static_cast<int>(q.size(1));
  p.H = static_cast<int>(q.size(2));
  p.Hk = static_cast<int>(k.size(2));
  p.D = static_cast<int>(q.size(3));
  p.causal = mask.causal;
  // (a window over everything is none)
  const int64_t most = p.N, left = mask.left < 0 ? most : std::min(mask.left, most), right = mask.causal ? 0 : mask.right < 0 ? most : std::min(mask.right, most);
  MK_CHECK(mask.sinks >= 0, "attention: no negative number of sinks");
  p.window = left < most - 1 || (!mask.causal && right < most - 1);
  p.left = static_cast<int>(left);
  p.right = static_cast<int>(right);
  p.sinks = static_cast<int>(std::min(mask.sinks, most));
  p.scale = static_cast<float>(scale);
  if (offsets.has_value() && offsets->defined()) {
    MK_CHECK(offsets->device() == q.device() && offsets->scalar_type() == at::kInt && offsets->dim() == 1 && offsets->is_contiguous() && offsets->size(0) >= 1,
             "attention: offsets must be int32 [sequences + 1] on the device of the queries");
    MK_CHECK(p.B == 1, "attention: packed sequences have no batch");
    p.offsets = offsets->data_ptr<int>();
    p.sequences = static_cast<int>(offsets->size(0) - 1);
  }
  return p;
}

// (o, what its rounding left out, L): the last two with `train`
std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const OptTensor& offsets, const Mask& mask,
                                                     double scale, bool train) {
  const mk::AttnShape p = shape_of(q_in, k_in, v_in, offsets, mask, scale);
  c10::cuda::CUDAGuard guard(q_in.device());
  Tensor o = room(q_in), rest, lse;
  if (train) {
    rest = room(q_in);
    lse = room({p.B, p.H, p.N}, q_in, at::kFloat);
  }
  if (o.numel() == 0) return {o, rest, lse};
  const Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in);
  Tensor scratch;
  if (const int64_t floats = mk::attention_scratch(p)) scratch = room({floats}, q, at::kFloat);
  int launches = 0;
  mkh::check(mk::attention_fwd(p, view_of(q), view_of(k), view_of(v), bf(o), ptr_or_null<__nv_bfloat16>(rest), ptr_or_null<float>(lse),
                               ptr_or_null<float>(scratch), &launches, mkh::error_word(q), mkh::stream()),
             "attention_fwd");
  mkh::launches() += launches;
  return {o, rest, lse};
}

// gradients into tensors [B, N, heads, D] (strides as `readable` has them)
void attention_backward(const Tensor& d_out, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& o, const Tensor& rest,
                        const Tensor& lse, const OptTensor& offsets, const Mask& mask, double scale, const Tensor& dq, const Tensor& dk, const Tensor& dv) {
  const mk::AttnShape p = shape_of(q_in, k_in, v_in, offsets, mask, scale);
  c10::cuda::CUDAGuard guard(q_in.device());
  MK_CHECK(plain({&d_out}), "attention: the backward pass takes no batches of gradients, and is not traced");
  MK_CHECK(d_out.device() == o.device() && d_out.sizes() == o.sizes() && d_out.scalar_type() == at::kBFloat16,
           "attention: a gradient like the output expected");
  if (o.numel() == 0) return;
  Tensor g = d_out.contiguous();
  if (reinterpret_cast<uintptr_t>(g.data_ptr()) & 15) g = g.clone();
  const Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in), delta = room(lse);
  Tensor scratch;
  if (const int64_t floats = mk::attention_bwd_scratch(p)) scratch = room({floats}, q, at::kFloat);
  int launches = 0;
  mkh::check(mk::attention_bwd(p, view_of(q), view_of(k), view_of(v), bf(o), bf(rest), bf(g), lse.data_ptr<float>(), delta.data_ptr<float>(), view_of(dq),
                               view_of(dk), view_of(dv), ptr_or_null<float>(scratch), &launches, mkh::error_word(q), mkh::stream()),
             "attention_bwd");
  mkh::launches() += launches;
}

// Numbers of a mask in a node's fields, from `at` on
void keep_mask(Fields& f, size_t at, const Mask& m) {
  f.whole[at] = m.causal;
  f.whole[at + 1] = m.left;
  f.whole[at + 2] = m.right;
  f.whole[at + 3] = m.sinks;
}
Mask kept_mask(const Fields& f, size_t at) { return {f.whole[at] != 0, f.whole[at + 1], f.whole[at + 2], f.whole[at + 3]}; }

struct AttentionOp {
  static constexpr const char* NAME = "AttentionNode";
  // fields: mask; scale.  kept: q, k, v, what the forward pass left, offsets.  edges: q, k, v
  static variable_list gradients(const variable_list& grads, const variable_list& s, const Fields& f, const std::vector<bool>&) {
    if (!grads[0].defined()) return variable_list(3);
    const at::AutoDispatchBelowAutograd below;
    const Tensor dq = room(s[0]), dk = room(s[1]), dv = room(s[2]);
    attention_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], maybe(s[6]), kept_mask(f, 0), f.real[0], dq, dk, dv);
    return once_differentiable({dq, dk, dv});
  }
};

// (o; nothing where the tensors are not for kernels)
OptTensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets, bool causal, double scale, int64_t left, int64_t right,
                    int64_t sinks) {
  const Backward count;
  const Tensor at = value(offsets);
  if (!plain({&q, &k, &v, &at})) return {};
  const bool train = records({&q, &k, &v});
  const Mask mask{causal, left, right, sinks};
  Tensor o, rest, lse;
  {
    const at::AutoDispatchBelowAutograd below;
    std::tie(o, rest, lse) = attention_forward(q, k, v, offsets, mask, scale, train);
  }
  if (train) {
    Fields f;
    keep_mask(f, 0, mask);
    f.real[0] = scale;
    FieldNode<AttentionOp>::record({o}, {q, k, v}, {q, k, v, o.detach(), rest, lse, at}, f);
  }
  return o;
}

// The same for [B, N, heads, D], or packed [T, heads, D] with offsets; nothing where the arguments are not for kernels as they are either, or wrong
OptTensor attention_call(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets, bool causal, std::optional<double> scale, int64_t left,
                         int64_t right, int64_t sinks) {
  const bool packed = offsets.has_value();
  const int64_t dim = packed ? 3 : 4;
  auto fits = [&](const Tensor& t) { return t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == dim && t.device() == q.device(); };
  if (!fits(q) || !fits(k) || !fits(v) || k.sizes() != v.sizes() || sinks < 0) return {};
  for (int64_t d = 0; d < dim; ++d)
    if (d != dim - 2 && k.size(d) != q.size(d)) return {};
  const int64_t H = q.size(-2), Hk = k.size(-2), D = q.size(-1);
  if (H < 1 || Hk < 1 || H % Hk || D < 8 || D % 8 || D > mk::ATTN_WIDTH) return {};
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D));
  if (!(s > 0.0) || !std::isfinite(s)) return {};
  if (!packed) return attention(q, k, v, offsets, causal, s, left, right, sinks);
  if (!offsets->is_cuda() || offsets->device() != q.device() || offsets->scalar_type() != at::kInt || offsets->dim() != 1 || offsets->size(0) < 1 ||
      !offsets->is_contiguous())
    return {};
  const OptTensor o = attention(q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0), offsets, causal, s, left, right, sinks);
  return o.has_value() ? OptTensor(o->squeeze(0)) : o;
}

// The output of a fused projection: [B, N, (q heads | k heads | v heads) x D], dense; its gradient is written as one tensor
struct Parts {
  Tensor q, k, v;
  Parts(const Tensor& qkv, int64_t heads, int64_t kv_heads) {
    MK_CHECK(qkv.dim() == 3 && heads > 0 && kv_heads > 0 && qkv.size(2) % (heads + 2 * kv_heads) == 0,
             "attention: [B, N, (heads + 2 kv_heads) * D] expected");
    const Tensor t = qkv.contiguous().view({qkv.size(0), qkv.size(1), heads + 2 * kv_heads, qkv.size(2) / (heads + 2 * kv_heads)});
    q = t.narrow(2, 0, heads);
    k = t.narrow(2, heads, kv_heads);
    v = t.narrow(2, heads + kv_heads, kv_heads);
  }
};

struct AttentionQkvOp {
  static constexpr const char* NAME = "AttentionQkvNode";
  // fields: heads, heads of keys, mask; scale.  kept: projection, what the forward pass left, offsets.  edge: projection
  static variable_list gradients(const variable_list& grads, const variable_list& s, const Fields& f, const std::vector<bool>&) {
    if (!grads[0].defined()) return variable_list(1);
    const at::AutoDispatchBelowAutograd below;
    const int64_t heads = f.whole[0], kv_heads = f.whole[1];
    const Tensor dqkv = room(s[0]);
    const Parts p(s[0], heads, kv_heads), d(dqkv, heads, kv_heads);
    attention_backward(grads[0], p.q, p.k, p.v, s[1], s[2], s[3], maybe(s[4]), kept_mask(f, 2), f.real[0], d.q, d.k, d.v);
    return once_differentiable({dqkv});
  }
};

OptTensor attention_qkv(const Tensor& qkv, int64_t heads, int64_t kv_heads, const OptTensor& offsets, bool causal, double scale, int64_t left, int64_t right,
                        int64_t sinks) {
  const Backward count;
  const Tensor at = value(offsets);
  if (!plain({&qkv, &at})) return {};
  const bool train = records({&qkv});
  const Mask mask{causal, left, right, sinks};
  Tensor o, rest, lse;
  {
    const at::AutoDispatchBelowAutograd below;
    const Parts p(qkv, heads, kv_heads);
    std::tie(o, rest, lse) = attention_forward(p.q, p.k, p.v, offsets, mask, scale, train);
  }
  if (train) {
    Fields f;
    f.whole[0] = heads;
    f.whole[1] = kv_heads;
    keep_mask(f, 2, mask);
    f.real[0] = scale;
    FieldNode<AttentionQkvOp>::record({o}, {qkv}, {qkv, o.detach(), rest, lse, at}, f);
  }
  return o;
}

// ------------------------------------------------------------------------------------------ rotary positions

// How channels turn, as a tensor of doubles on the host that autograd can keep: (interleaved, axes, bands of channels, turns per unit of position of every pair)
struct RotaryPlan {
  Tensor numbers;
  RotaryPlan(const std::vector<int64_t>& bands, const std::vector<double>& turns, bool interleaved) {
    std::vector<double> v{interleaved ? 1.0 : 0.0, static_cast<double>(bands.size())};
    v.insert(v.end(), bands.begin(), bands.end());
    v.insert(v.end(), turns.begin(), turns.end());
    numbers = at::tensor(v, at::kDouble);
  }
};

mk::RotTensor rot_view(const Tensor& t) {
  auto stride = [&](int d) { return t.size(d) == 1 ? t.size(3) : t.stride(d); };
  return {t.data_ptr(), stride(1), stride(2), stride(0)};
}

// Tensors of a pass: queries and, perhaps, keys, with weights and biases of their norms; positions
struct RotInputs {
  Tensor x[2], w[2], b[2], positions;
};

mk::RotShape rot_shape(const Tensor& like, const RotInputs& in, const Tensor& plan, int64_t norm, double eps, bool inverse) {
  MK_CHECK(like.is_cuda() && native_type(like) && like.dim() == 4, "rotary positions: bf16 or fp32 CUDA tensors [B, N, heads, D] expected");
  MK_CHECK(like.size(3) % 8 == 0 && like.size(3) >= 8 && like.size(3) <= mk::ROT_WIDTH, "rotary positions: 8, 16, .., ", mk::ROT_WIDTH,
           " channels of a head expected");
  MK_CHECK(like.size(0) * like.size(1) < (1ll << 31) - (1ll << 24), "rotary positions: too many tokens");
  MK_CHECK(norm >= 0 && norm <= 2, "rotary positions: an unknown norm");
  mk::RotShape p{};
  p.B = static_cast<int>(like.size(0));
  p.N = static_cast<int>(like.size(1));
  p.D = static_cast<int>(like.size(3));
  p.f32 = is_f32(like);
  p.norm = static_cast<uint8_t>(norm);
  p.inverse = inverse;
  p.eps = static_cast<float>(eps);
  if (in.positions.defined()) {
    const Tensor& at = in.positions;
    const double* const v = plan.data_ptr<double>();
    p.interleaved = v[0] != 0.0;
    p.axes = static_cast<int>(v[1]);
    MK_CHECK(p.axes >= 1 && p.axes <= mk::ROT_AXES && at.device() == like.device() && at.is_contiguous() && (at.dim() == 2 || at.dim() == 3) &&
                 at.size(-1) == p.axes && at.size(-2) == p.N && (at.dim() == 2 || at.size(0) == p.B),
             "rotary positions: positions [N, axes] or [B, N, axes] expected");
    int channels = 0;
    for (int a = 0; a < p.axes; ++a) {
      p.band[a] = static_cast<int>(v[2 + a]);
      MK_CHECK(p.band[a] >= 2 && p.band[a] % 2 == 0 && p.band[a] <= p.D, "rotary positions: bands of even widths expected");
      channels += p.band[a];
    }
    MK_CHECK(channels <= p.D && plan.numel() == 2 + p.axes + channels / 2, "rotary positions: ", channels, " channels of ", p.D, " turned");
    std::copy_n(v + 2 + p.axes, channels / 2, p.turns);
    switch (at.scalar_type()) {
      case at::kInt: p.position_type = mk::ROT_POS_I32; break;
      case at::kLong: p.position_type = mk::ROT_POS_I64; break;
      case at::kFloat: p.position_type = mk::ROT_POS_F32; break;
      case at::kDouble: p.position_type = mk::ROT_POS_F64; break;
      default: MK_CHECK(false, "rotary positions: positions in int32, int64, fp32 or fp64 expected");
    }
    p.positions = at.data_ptr();
    p.position_batch = at.dim() == 3 ? at.size(1) * at.size(2) : 0;
  }
  return p;
}

void rot_weights(mk::RotPart& part, const Tensor& w, const Tensor& b, const Tensor& like) {
  for (const Tensor* t : {&w, &b})
    MK_CHECK(!t->defined() || (t->is_cuda() && t->device() == like.device() && is_f32(*t) && t->is_contiguous() && t->dim() == 1 && t->size(0) == like.size(3)),
             "rotary positions: weights and biases [D] of the norm expected");
  part.w = ptr_or_null<float>(w);
  part.b = ptr_or_null<float>(b);
}
Tensor rot_param(const Tensor& t) {
  if (!t.defined()) return t;
  return (is_f32(t) && t.is_contiguous()) ? t : t.detach().to(at::kFloat).contiguous();
}

// Results into `out`, tensors [B, N, heads, D]
void rotary_into(const RotInputs& in, const Tensor (&out)[2], const Tensor& plan, int64_t norm, double eps, bool inverse) {
  c10::cuda::CUDAGuard guard(in.x[0].device());
  mk::RotShape p = rot_shape(in.x[0], in, plan, norm, eps, inverse);
  Tensor x[2];
  for (int i = 0; i < 2; ++i) {
    if (!in.x[i].defined() || in.x[i].numel() == 0) continue;
    MK_CHECK(in.x[i].dim() == 4 && in.x[i].device() == in.x[0].device() && in.x[i].scalar_type() == in.x[0].scalar_type() && in.x[i].size(0) == p.B &&
                 in.x[i].size(1) == p.N && in.x[i].size(3) == p.D,
             "rotary positions: queries and keys of the same tokens and channels expected");
    x[i] = readable(in.x[i]);
    MK_CHECK(x[i].size(0) * x[i].size(1) * x[i].size(2) < (1ll << 31) - (1ll << 24), "rotary positions: too many rows");
    mk::RotPart& part = p.part[p.parts++];
    part.x = rot_view(x[i]);
    part.out = rot_view(out[i]);
    part.heads = static_cast<int>(x[i].size(2));
    rot_weights(part, in.w[i], in.b[i], x[i]);
  }
  if (p.parts == 0) return;
  ++mkh::launches();
  mkh::check(mk::rotary_fwd(p, mkh::stream()), "rotary_fwd");
}
// Gradients of x into `out` (which may be `dy`), and of weights and biases; parts whose gradient is not defined are left out
void rotary_back(const RotInputs& in, const Tensor (&dy)[2], const Tensor (&out)[2], const Tensor& plan, int64_t norm, double eps, bool inverse,
                 const bool (&sums)[2], Tensor (&dw)[2], Tensor (&db)[2], const int* limit = nullptr) {
  const Tensor& like = dy[0].defined() ? dy[0] : dy[1];
  c10::cuda::CUDAGuard guard(like.device());
  mk::RotShape p = rot_shape(like, in, plan, norm, eps, inverse);
  p.limit = limit;
  Tensor x[2], d[2], scratch;
  for (int i = 0; i < 2; ++i) {
    if (!dy[i].defined()) continue;
    if (dy[i].numel() == 0) {
      for (Tensor* t : {&dw[i], &db[i]})
        if (sums[i]) *t = at::zeros({p.D}, dy[i].options().dtype(at::kFloat));
      continue;
    }
    mk::RotPart& part = p.part[p.parts++];
    d[i] = out[i].is_same(dy[i]) ? dy[i] : readable(dy[i]);
    part.dy = rot_view(d[i]);
    part.out = rot_view(out[i]);
    part.heads = static_cast<int>(d[i].size(2));
    if (norm) {
      x[i] = readable(in.x[i]);
      part.x = rot_view(x[i]);
    }
    rot_weights(part, in.w[i], in.b[i], d[i]);
    if (sums[i]) {
      dw[i] = room({p.D}, dy[i], at::kFloat);
      db[i] = room({p.D}, dy[i], at::kFloat);
      part.dw = dw[i].data_ptr<float>();
      part.db = db[i].data_ptr<float>();
    }
  }
  if (p.parts == 0) return;
  if (sums[0] || sums[1]) scratch = room({mk::rotary_scratch(p)}, like, at::kFloat);
  int launches = 0;
  mkh::check(mk::rotary_bwd(p, ptr_or_null<float>(scratch), &launches, mkh::stream()), "rotary_bwd");
  mkh::launches() += launches;
}

// Gradients of parameters in their own types, where they are asked for
Tensor param_grad(const Tensor& g, const Tensor& param, bool needed) {
  if (!needed || !param.defined() || !g.defined()) return Tensor();
  return g.scalar_type() == param.scalar_type() ? g : g.to(param.scalar_type());
}

// Queries and, perhaps, keys; edges: q, k, weights of q and k, biases of q and k
variable_list rotary_pass(const Tensor& q, const Tensor& k, const Tensor (&w)[2], const Tensor (&b)[2], const Tensor& positions, const Tensor& plan, int64_t norm,
                          double eps, bool inverse);
struct RotaryOp {
  static constexpr const char* NAME = "RotaryNode";
  // fields: norm, inverse; eps.  kept: positions, plan, and with a norm q, k, weights and biases
  static variable_list gradients(const variable_list& grads, const variable_list& s, const Fields& f, const std::vector<bool>& need) {
    const int64_t norm = f.whole[0];
    const bool inverse = f.whole[1] != 0;
    const Tensor dy[2] = {grads[0], grads.size() > 1 ? grads[1] : Tensor()};
    variable_list out(6);
    if (!dy[0].defined() && !dy[1].defined()) return out;
    MK_CHECK(plain({&dy[0], &dy[1]}), "rotary positions: the backward pass takes no batches of gradients, and is not traced");
    if (norm == 0 && at::GradMode::is_enabled()) {      // (the same again, the other way round: it can be differentiated as often as one likes)
      const int first = dy[0].defined() ? 0 : 1;
      auto g = rotary_pass(dy[first], first == 0 ? dy[1] : Tensor(), {}, {}, s[0], s[1], 0, 0.0, !inverse);
      out[first] = g[0];
      if (g.size() > 1) out[1] = g[1];
      return out;
    }
    const at::AutoDispatchBelowAutograd below;
    RotInputs in;
    in.positions = s[0];
    Tensor dx[2], dw[2], db[2];
    bool sums[2] = {false, false};
    for (int i = 0; i < 2; ++i) {
      if (!dy[i].defined()) continue;
      if (norm) {
        in.x[i] = s[2 + i];
        in.w[i] = rot_param(s[4 + i]);
        sums[i] = need[2 + i] || need[4 + i];
      }
      dx[i] = room(dy[i]);
    }
    rotary_back(in, dy, dx, s[1], norm, f.real[0], inverse, sums, dw, db);
    for (int i = 0; i < 2; ++i) {
      if (need[i]) out[i] = dx[i];
      if (norm) {
        out[2 + i] = param_grad(dw[i], s[4 + i], need[2 + i]);
        out[4 + i] = param_grad(db[i], s[6 + i], need[4 + i]);
      }
    }
    return once_differentiable(out);
  }
};
variable_list rotary_pass(const Tensor& q, const Tensor& k, const Tensor (&w)[2], const Tensor (&b)[2], const Tensor& positions, const Tensor& plan, int64_t norm,
                          double eps, bool inverse) {
  variable_list results;
  {
    const at::AutoDispatchBelowAutograd below;
    RotInputs in{{q, k}, {rot_param(w[0]), rot_param(w[1])}, {rot_param(b[0]), rot_param(b[1])}, positions};
    Tensor out[2];
    for (int i = 0; i < 2; ++i)
      if (in.x[i].defined()) {
        out[i] = room(in.x[i]);
        results.push_back(out[i]);
      }
    rotary_into(in, out, plan, norm, eps, inverse);
  }
  if (records({&q, &k, &w[0], &w[1], &b[0], &b[1]})) {
    Fields f;
    f.whole[0] = norm;
    f.whole[1] = inverse;
    f.real[0] = eps;
    variable_list kept{positions, plan};
    if (norm) kept.insert(kept.end(), {q, k, w[0], w[1], b[0], b[1]});
    FieldNode<RotaryOp>::record(results, {q, k, w[0], w[1], b[0], b[1]}, kept, f);
  }
  return results;
}

// (results; nothing where the tensors are not for kernels)
variable_list rotary(const Tensor& q, const OptTensor& k, const OptTensor& qw, const OptTensor& kw, const OptTensor& qb, const OptTensor& kb,
                     const OptTensor& positions, const RotaryPlan& plan, int64_t norm, double eps, bool inverse) {
  const Backward count;
  const Tensor keys = value(k), w[2] = {value(qw), value(kw)}, b[2] = {value(qb), value(kb)}, at = value(positions);
  if (!plain({&q, &keys, &w[0], &w[1], &b[0], &b[1], &at})) return {};
  return rotary_pass(q, keys, w, b, at, plan.numbers, norm, eps, inverse);
}

// The same for queries (and keys) [B, N, heads, D] or packed [T, heads, D]; nothing where the arguments are not for kernels either, or wrong: the caller looks closer then
variable_list rotary_call(const Tensor& q, const OptTensor& k, const OptTensor& qw, const OptTensor& kw, const OptTensor& qb, const OptTensor& kb,
                          const OptTensor& positions, const RotaryPlan& plan, int64_t norm, double eps, bool inverse) {
  const bool packed = q.dim() == 3;
  if (!q.is_cuda() || !native_type(q) || !(packed || q.dim() == 4) || norm < 0 || norm > 2 || !(eps >= 0.0)) return {};
  const int64_t D = q.size(-1);
  if (D < 8 || D > mk::ROT_WIDTH || D % 8) return {};
  const auto device = q.device();
  if (k.has_value()) {
    if (k->dim() != q.dim() || k->scalar_type() != q.scalar_type() || k->device() != device) return {};
    for (int64_t d = 0; d < q.dim(); ++d)
      if (d != q.dim() - 2 && k->size(d) != q.size(d)) return {};
  }
  for (const OptTensor* t : {&qw, &kw, &qb, &kb})
    if (t->has_value() && (norm == 0 || (*t)->dim() != 1 || (*t)->size(0) != D || (*t)->device() != device || !(*t)->is_floating_point())) return {};
  const double* const numbers = plan.numbers.data_ptr<double>();
  const int64_t axes = static_cast<int64_t>(numbers[1]);
  if (positions.has_value() != (axes > 0)) return {};
  OptTensor at = positions;
  if (axes > 0) {
    const Tensor& t = *positions;
    const auto type = t.scalar_type();
    if (t.device() != device || t.requires_grad() || (type != at::kInt && type != at::kLong && type != at::kFloat && type != at::kDouble)) return {};
    const bool shared = t.dim() == 2, own = !packed && t.dim() == 3 && t.size(0) == q.size(0);
    if (!(shared || own) || t.size(-1) != axes || t.size(-2) != q.size(-3) || 2 * (plan.numbers.numel() - 2 - axes) > D) return {};
    if (!t.is_contiguous()) at = t.contiguous();
  }
  if (!packed) return rotary(q, k, qw, kw, qb, kb, at, plan, norm, eps, inverse);
  variable_list out = rotary(q.unsqueeze(0), k.has_value() ? OptTensor(k->unsqueeze(0)) : k, qw, kw, qb, kb, at, plan, norm, eps, inverse);
  for (Tensor& t : out) t = t.squeeze(0);
  return out;
}

// A fused projection's queries and keys normed and turned, then attention: one tensor for both, the gradient of the projection written as one
struct RotaryAttentionOp {
  static constexpr const char* NAME = "RotaryAttentionNode";
  // fields: heads, heads of keys, norm, mask; eps, scale.  kept: projection, weights and biases, positions, offsets, plan, queries and keys as attention took
  // them, and what it keeps.  edges: projection, weights and biases
  static variable_list gradients(const variable_list& grads, const variable_list& s, const Fields& f, const std::vector<bool>& need) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const int64_t heads = f.whole[0], kv_heads = f.whole[1], norm = f.whole[2];
    const Tensor &qkv = s[0], &offsets = s[6], &qk = s[8];
    const at::AutoDispatchBelowAutograd below;
    const Parts p(qkv, heads, kv_heads);
    const Tensor dqkv = room(qkv);
    const Parts d(dqkv, heads, kv_heads);
    attention_backward(grads[0], qk.narrow(2, 0, heads), qk.narrow(2, heads, kv_heads), p.v, s[9], s[10], s[11], maybe(offsets),
                       kept_mask(f, 3), f.real[1], d.q, d.k, d.v);
    RotInputs in;
    in.positions = s[5];
    const Tensor dx[2] = {d.q, d.k};
    Tensor dw[2], db[2];
    bool sums[2] = {false, false};
    for (int i = 0; i < 2; ++i) {
      in.x[i] = i ? p.k : p.q;
      if (norm) {
        in.w[i] = rot_param(s[1 + i]);
        sums[i] = need[1 + i] || need[3 + i];
      }
    }
    // (in place: a lane writes what it alone has read; tokens of no sequence have the zeros that attention left)
    const int* limit = offsets.defined() ? offsets.data_ptr<int>() + offsets.size(0) - 1 : nullptr;
    rotary_back(in, dx, dx, s[7], norm, f.real[0], false, sums, dw, db, limit);
    if (need[0]) out[0] = dqkv;
    for (int i = 0; i < 2; ++i) {
      out[1 + i] = param_grad(dw[i], s[1 + i], need[1 + i]);
      out[3 + i] = param_grad(db[i], s[3 + i], need[3 + i]);
    }
    return once_differentiable(out);
  }
};

OptTensor rotary_attention_qkv(const Tensor& qkv, int64_t heads, int64_t kv_heads, const OptTensor& qw, const OptTensor& kw, const OptTensor& qb,
                               const OptTensor& kb, const OptTensor& positions, const OptTensor& offsets, const RotaryPlan& plan, int64_t norm, double eps,
                               bool causal, double scale, int64_t left, int64_t right, int64_t sinks) {
  const Backward count;
  const Tensor w[2] = {value(qw), value(kw)}, b[2] = {value(qb), value(kb)}, at = value(positions), off = value(offsets);
  if (!plain({&qkv, &w[0], &w[1], &b[0], &b[1], &at, &off})) return {};
  const bool train = records({&qkv, &w[0], &w[1], &b[0], &b[1]});
  Tensor o, rest, lse, qk;
  {
    const at::AutoDispatchBelowAutograd below;
    const Parts p(qkv, heads, kv_heads);
    const RotInputs in{{p.q, p.k}, {rot_param(w[0]), rot_param(w[1])}, {rot_param(b[0]), rot_param(b[1])}, at};
    qk = room({qkv.size(0), qkv.size(1), heads + kv_heads, p.q.size(3)}, qkv, qkv.scalar_type());
    const Tensor out[2] = {qk.narrow(2, 0, heads), qk.narrow(2, heads, kv_heads)};
    rotary_into(in, out, plan.numbers, norm, eps, false);
    std::tie(o, rest, lse) = attention_forward(out[0], out[1], p.v, offsets, Mask{causal, left, right, sinks}, scale, train);
  }
  if (train) {
    Fields f;
    f.whole = {heads, kv_heads, norm, causal, left, right, sinks, 0};
    f.real = {eps, scale};
    FieldNode<RotaryAttentionOp>::record({o}, {qkv, w[0], w[1], b[0], b[1]}, {qkv, w[0], w[1], b[0], b[1], at, off, plan.numbers, qk, o.detach(), rest, lse}, f);
  }
  return o;
}

// ------------------------------------------------------------------------------------------ dropout

// x (and a residual) dense; the mask from `seed` [2] (key, number of the call), or, where there is none, from torch's generator of the device, whose key and
// position are then written to `kept`
std::tuple<Tensor, Tensor> dropout_pass(const Tensor& x_in, const Tensor& residual, const Tensor& seed, const Tensor& kept, double p, at::ScalarType out_type,
                                        bool copy) {
  c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = x_in.contiguous(), r = residual.defined() ? residual.contiguous() : Tensor();
  const Tensor out = room(x.sizes(), x, out_type), half = copy ? room(x.sizes(), x, at::kBFloat16) : Tensor();
  mk::DropParams d{};
  d.x = x.data_ptr();
  d.r = ptr_or_null<void>(r);
  d.out = out.data_ptr();
  d.copy = ptr_or_null<void>(half);
  d.n = x.numel();
  const double words = std::nearbyint(p * 4294967296.0);
  MK_CHECK(p >= 0.0 && p <= 1.0 && words >= 1.0, "dropout: a probability of 2^-32 to 1 expected");
  d.last = static_cast<uint32_t>(words - 1.0);
  d.factor = p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.f;
  if (seed.defined()) {
    MK_CHECK(seed.device() == x.device() && seed.scalar_type() == at::kLong && seed.is_contiguous() && seed.numel() == 2,
             "dropout: a seed of two int64 (key, number of the call) on the device of x expected");
    d.source.key_at = seed.data_ptr<int64_t>();
    d.source.offset_at = d.source.key_at + 1;
  } else {
    // (a call takes four of the positions of every subsequence, as a call of torch's own generator with one block of words does, so that none is used twice)
    auto* generator = at::get_generator_or_default<at::CUDAGeneratorImpl>(std::nullopt, at::cuda::detail::getDefaultCUDAGenerator());
    at::PhiloxCudaState state;
    {
      const std::lock_guard<std::mutex> lock(generator->mutex_);
      state = generator->philox_cuda_state(4);
    }
    d.source.shift = 2;
    if (state.captured_) {
      d.source.key_at = state.seed_.ptr;
      d.source.offset_at = state.offset_.ptr;
      d.source.more = state.offset_intragraph_;
    } else {
      d.source.key = state.seed_.val;
      d.source.more = state.offset_.val;
    }
    d.source.kept = ptr_or_null<int64_t>(kept);
  }
  d.x_f32 = is_f32(x);
  d.r_f32 = r.defined() && is_f32(r);
  d.out_f32 = out_type == at::kFloat;
  mkh::launches() += d.n > 0;
  mkh::check(mk::dropout(d, mkh::stream()), "dropout");
  return {out, half};
}

Tensor dropout_run(const Tensor& x, const Tensor& residual, const Tensor& seed, double p, bool out_f32);
struct DropoutOp {
  static constexpr const char* NAME = "DropoutNode";
  // fields: x in fp32, the residual in fp32; p.  kept: seed.  edges: x, residual
  static variable_list gradients(const variable_list& grads, const variable_list& s, const Fields& f, const std::vector<bool>& need) {
    const Tensor &seed = s[0], &dy = grads[0];
    const bool x_f32 = f.whole[0] != 0, r_f32 = f.whole[1] != 0;
    variable_list out(2);
    if (!dy.defined()) return out;
    MK_CHECK(plain({&dy}), "dropout: the backward pass takes no batches of gradients, and is not traced");
    const bool half = need[1] && !r_f32 && is_f32(dy);
    if (at::GradMode::is_enabled()) {      // (the same mask on the gradient, which can be differentiated again)
      if (need[0]) {
        out[0] = dropout_run(dy, Tensor(), seed, f.real[0], is_f32(dy));
        if (is_f32(dy) && !x_f32) out[0] = out[0].to(at::kBFloat16);
      }
      if (need[1]) out[1] = half ? dy.to(at::kBFloat16) : dy;
      return out;
    }
    const at::AutoDispatchBelowAutograd below;
    if (need[0]) {
      auto [dx, copy] = dropout_pass(dy, Tensor(), seed, Tensor(), f.real[0], x_f32 ? at::kFloat : at::kBFloat16, half);
      out[0] = dx;
      if (half) out[1] = copy;
    } else if (half) {
      out[1] = dy.to(at::kBFloat16);
    }
    if (need[1] && !half) out[1] = dy;
    return out;
  }
};
Tensor dropout_run(const Tensor& x, const Tensor& residual, const Tensor& seed, double p, bool out_f32) {
  const bool train = records({&x, &residual});
  Tensor kept, y;
  {
    const at::AutoDispatchBelowAutograd below;
    if (!seed.defined() && train) kept = room({2}, x, at::kLong);
    y = std::get<0>(dropout_pass(x, residual, seed, kept, p, out_f32 ? at::kFloat : at::kBFloat16, false));
  }
  if (train) {
    Fields f;
    f.whole[0] = is_f32(x);
    f.whole[1] = residual.defined() && is_f32(residual);
    f.real[0] = p;
    FieldNode<DropoutOp>::record({y}, {x, residual}, {seed.defined() ? seed : kept}, f);
  }
  return y;
}

// (nothing where the tensors or arguments are not for the kernel, or wrong: the caller looks closer then)
OptTensor dropout_call(const Tensor& x, const OptTensor& residual, const OptTensor& seed, double p) {
  if (!x.is_cuda() || !native_type(x) || !(p >= 0.0 && p <= 1.0)) return {};
  const auto device = x.device();
  if (residual.has_value() && (!native_type(*residual) || residual->device() != device || residual->sizes() != x.sizes())) return {};
  if (seed.has_value() && (seed->scalar_type() != at::kLong || seed->dim() != 1 || seed->size(0) != 2 || seed->device() != device)) return {};
  const Backward count;
  const Tensor r = value(residual), s = seed.has_value() ? seed->contiguous() : Tensor();
  if (!plain({&x, &r, &s})) return {};
  return dropout_run(x, r, s, p, is_f32(x) || (r.defined() && is_f32(r)));
}

}  // namespace

namespace mkh {

void bind_tokens(pybind11::module_& m) {
  using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("background_launches", []() { return background.load(); }, "kernel launches of backward passes that autograd ran");
  m.def("layer_norm", &layer_norm, Free());
  using pybind11::arg;
  m.def("attention", &attention, arg("q"), arg("k"), arg("v"), arg("offsets"), arg("causal"), arg("scale"), arg("left") = -1, arg("right") = -1,
        arg("sinks") = 0, Free());
  m.def("attention_qkv", &attention_qkv, arg("qkv"), arg("heads"), arg("kv_heads"), arg("offsets"), arg("causal"), arg("scale"), arg("left") = -1,
        arg("right") = -1, arg("sinks") = 0, Free());
  pybind11::class_<RotaryPlan>(m, "RotaryPlan")
      .def(pybind11::init<const std::vector<int64_t>&, const std::vector<double>&, bool>());
  m.def("rotary", &rotary, Free());
  m.def("rotary_call", &rotary_call, Free());
  m.def("attention_call", &attention_call, Free());
  m.def("dropout_call", &dropout_call, Free());
  m.def("rotary_attention_qkv", &rotary_attention_qkv, Free());
}

}  // namespace mkh
