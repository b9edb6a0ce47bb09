// Passes of the token operators (layer norm, attention): checks, allocations and launches without a return to Python in between.
#include "host.h"

#include <pybind11/stl.h>

#include <algorithm>

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

Tensor channel_f32(const OptTensor& t, const Tensor& x, const char* what) {
  if (!t.has_value() || !t->defined()) return Tensor();
  MK_CHECK(t->device() == x.device(), "layer norm: tensors must be on one CUDA device");
  MK_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), "layer norm: one ", what, " per channel expected");
  return t->detach().to(at::kFloat).contiguous();
}

// (s, y, statistics, weight in fp32): s and the statistics where they are asked for
std::tuple<OptTensor, Tensor, OptTensor, OptTensor> layer_norm_forward(const Tensor& x, const OptTensor& residual, const OptTensor& weight,
                                                                       const OptTensor& bias, double eps, bool out_f32, bool train) {
  MK_CHECK(x.is_cuda() && native_type(x) && x.dim() >= 1, "layer norm: bf16 or fp32 CUDA tensors expected");
  c10::cuda::CUDAGuard guard(x.device());
  const Rows in(x);
  MK_CHECK(in.C >= 1 && in.C <= mk::LN_CHANNELS, "layer norm: 1 to ", mk::LN_CHANNELS, " channels expected");
  const Tensor w = channel_f32(weight, x, "weight"), b = channel_f32(bias, x, "bias");
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
  p.w = ptr_or_null<float>(w);
  p.b = ptr_or_null<float>(b);
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

// (dx, dr, dweight, dbias); `half_copy`: dr, dx in bf16
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& x, const Tensor& dy, const OptTensor& ds, const OptTensor& weight,
                                                                        const Tensor& stats, bool need_params, bool half_copy) {
  MK_CHECK(x.is_cuda() && native_type(x) && native_type(dy) && dy.device() == x.device() && dy.sizes() == x.sizes(),
           "layer norm: gradients in the shape of x and on its device expected");
  c10::cuda::CUDAGuard guard(x.device());
  const Rows in(x);
  MK_CHECK(stats.is_cuda() && is_f32(stats) && stats.is_contiguous() && stats.numel() == 2 * in.rows, "layer norm: statistics of every row expected");
  const Tensor w = channel_f32(weight, x, "weight"), g = dy.contiguous();
  Tensor d, dr, dw, db, part, dx = at::empty(x.sizes(), x.options());
  if (ds.has_value() && ds->defined()) {
    MK_CHECK(ds->device() == x.device() && ds->sizes() == x.sizes() && ds->scalar_type() == x.scalar_type(),
             "layer norm: the gradient of the sum must be like the sum");
    d = ds->contiguous();
  }
  if (half_copy) dr = at::empty(x.sizes(), x.options().dtype(at::kBFloat16));
  if (need_params) {
    // (no rows: no kernel that writes them)
    const Tensor both = in.rows ? at::empty({2, in.C}, x.options().dtype(at::kFloat)) : at::zeros({2, in.C}, x.options().dtype(at::kFloat));
    dw = both.select(0, 0);
    db = both.select(0, 1);
    const int64_t n = mk::layer_norm_scratch(in.rows, static_cast<int>(in.C));
    if (n) part = at::empty({n}, x.options().dtype(at::kFloat));
  }
  mk::LnBackward p{};
  p.x = in.t.data_ptr();
  p.dy = g.data_ptr();
  p.ds = ptr_or_null<void>(d);
  p.dx = dx.data_ptr();
  p.dr = ptr_or_null<void>(dr);
  p.w = ptr_or_null<float>(w);
  p.stats = static_cast<const float2*>(stats.data_ptr());
  p.dw = ptr_or_null<float>(dw);
  p.db = ptr_or_null<float>(db);
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

}  // namespace

namespace mkh {

void bind_tokens(pybind11::module_& m) {
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
}

}  // namespace mkh
