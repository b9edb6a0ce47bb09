// Passes of the token operators (layer norm, attention): checks, allocations, launches and their nodes of the autograd graph, without a return to
// Python in between.  (A forward and a backward pass of a layer norm of 16471 x 387 tokens, with the node in Python 122 us, all of it host time.)
#include "host.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/dynamo/compiled_autograd.h>

#include <pybind11/stl.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "attention.cuh"
#include "layer_norm.cuh"

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

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

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

// Launches of backward passes, which autograd runs in threads of its own
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

mk::AttnShape shape_of(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets, bool causal, double scale) {
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
  p.causal = causal;
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
std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const OptTensor& offsets, bool causal,
                                                double scale, bool train) {
  const mk::AttnShape p = shape_of(q_in, k_in, v_in, offsets, causal, scale);
  c10::cuda::CUDAGuard guard(q_in.device());
  Tensor o = at::empty(q_in.sizes(), q_in.options()), rest, lse;
  if (train) {
    rest = at::empty(q_in.sizes(), q_in.options());
    lse = at::empty({p.B, p.H, p.N}, q_in.options().dtype(at::kFloat));
  }
  if (o.numel() == 0) return {o, rest, lse};
  const Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in);
  Tensor scratch;
  if (const int64_t floats = mk::attention_scratch(p)) scratch = at::empty({floats}, q.options().dtype(at::kFloat));
  int launches = 0;
  mkh::check(mk::attention_fwd(p, view_of(q), view_of(k), view_of(v), bf(o), ptr_or_null<__nv_bfloat16>(rest), ptr_or_null<float>(lse),
                               ptr_or_null<float>(scratch), &launches, mkh::error_word(q), mkh::stream()),
             "attention_fwd");
  mkh::launches() += launches;
  return {o, rest, lse};
}

// gradients into tensors [B, N, heads, D] (strides as `readable` has them)
void attention_backward(const Tensor& d_out, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& o, const Tensor& rest,
                        const Tensor& lse, const OptTensor& offsets, bool causal, double scale, const Tensor& dq, const Tensor& dk, const Tensor& dv) {
  const mk::AttnShape p = shape_of(q_in, k_in, v_in, offsets, causal, scale);
  c10::cuda::CUDAGuard guard(q_in.device());
  MK_CHECK(plain({&d_out}), "attention: the backward pass takes no batches of gradients, and is not traced");
  MK_CHECK(d_out.device() == o.device() && d_out.sizes() == o.sizes() && d_out.scalar_type() == at::kBFloat16,
           "attention: a gradient like the output expected");
  if (o.numel() == 0) return;
  Tensor g = d_out.contiguous();
  if (reinterpret_cast<uintptr_t>(g.data_ptr()) & 15) g = g.clone();
  const Tensor q = readable(q_in), k = readable(k_in), v = readable(v_in), delta = at::empty_like(lse);
  Tensor scratch;
  if (const int64_t floats = mk::attention_bwd_scratch(p)) scratch = at::empty({floats}, q.options().dtype(at::kFloat));
  int launches = 0;
  mkh::check(mk::attention_bwd(p, view_of(q), view_of(k), view_of(v), bf(o), bf(rest), bf(g), lse.data_ptr<float>(), delta.data_ptr<float>(), view_of(dq),
                               view_of(dk), view_of(dv), ptr_or_null<float>(scratch), &launches, mkh::error_word(q), mkh::stream()),
             "attention_bwd");
  mkh::launches() += launches;
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets, bool causal, double scale,
                        bool train) {
    auto [o, rest, lse] = attention_forward(q, k, v, offsets, causal, scale, train);
    if (train) {
      ctx->save_for_backward({q, k, v, o, rest, lse, value(offsets)});
      ctx->saved_data["causal"] = causal;
      ctx->saved_data["scale"] = scale;
    }
    return o;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const Backward count;
    const variable_list s = ctx->get_saved_variables();
    const Tensor dq = at::empty(s[0].sizes(), s[0].options()), dk = at::empty(s[1].sizes(), s[1].options()), dv = at::empty(s[2].sizes(), s[2].options());
    attention_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], maybe(s[6]), ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), dq, dk,
                       dv);
    return once_differentiable({dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// (o; nothing where the tensors are not for kernels)
OptTensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets, bool causal, double scale) {
  const Tensor at = value(offsets);
  if (!plain({&q, &k, &v, &at})) return {};
  return Attention::apply(q, k, v, offsets, causal, scale, records({&q, &k, &v}));
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

struct AttentionQkv : torch::autograd::Function<AttentionQkv> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, int64_t heads, int64_t kv_heads, const OptTensor& offsets, bool causal, double scale,
                        bool train) {
    const Parts p(qkv, heads, kv_heads);
    auto [o, rest, lse] = attention_forward(p.q, p.k, p.v, offsets, causal, scale, train);
    if (train) {
      ctx->save_for_backward({qkv, o, rest, lse, value(offsets)});
      ctx->saved_data["heads"] = heads;
      ctx->saved_data["kv_heads"] = kv_heads;
      ctx->saved_data["causal"] = causal;
      ctx->saved_data["scale"] = scale;
    }
    return o;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const Backward count;
    const variable_list s = ctx->get_saved_variables();
    const int64_t heads = ctx->saved_data["heads"].toInt(), kv_heads = ctx->saved_data["kv_heads"].toInt();
    const Tensor dqkv = at::empty(s[0].sizes(), s[0].options());
    const Parts p(s[0], heads, kv_heads), d(dqkv, heads, kv_heads);
    attention_backward(grads[0], p.q, p.k, p.v, s[1], s[2], s[3], maybe(s[4]), ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), d.q, d.k,
                       d.v);
    return once_differentiable({dqkv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

OptTensor attention_qkv(const Tensor& qkv, int64_t heads, int64_t kv_heads, const OptTensor& offsets, bool causal, double scale) {
  const Tensor at = value(offsets);
  if (!plain({&qkv, &at})) return {};
  return AttentionQkv::apply(qkv, heads, kv_heads, offsets, causal, scale, records({&qkv}));
}

}  // namespace

namespace mkh {

void bind_tokens(pybind11::module_& m) {
  using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("background_launches", []() { return background.load(); }, "kernel launches of backward passes that autograd ran");
  m.def("layer_norm", &layer_norm, Free());
  m.def("attention", &attention, Free());
  m.def("attention_qkv", &attention_qkv, Free());
}

}  // namespace mkh
