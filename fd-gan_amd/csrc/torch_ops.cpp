// torch_ops.cpp -- the torch side of fdgan_hip.norm.layer_norm and of fdgan_hip.optim's gradient lists and Adam step.
//
// The library itself knows no torch (include/fdgan_hip.h); this module takes layouts, allocates and calls its C entries where Python would
// cost more than the work.  A small layer norm's forward and backward are a few microseconds on the GPU, and a Python autograd node cost 60 us
// of host time around them, most of it in the engine's own thread (1777 x 1001 fp32: 122 us a pass with it, 68 with this one); a list of 287
// gradients is clipped by 20 us of GPU work and took 145 us with the list walked in Python.  The entries' addresses come from the binding
// (fdgan_hip/lib.py), which has checked the library's identity.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <unordered_set>
#include <vector>

#include "../../include/fdgan_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
  decltype(&fdgan_layer_norm_fwd) fwd = nullptr;
  decltype(&fdgan_layer_norm_bwd) bwd = nullptr;
  decltype(&fdgan_layer_norm_workspace) workspace = nullptr;
  decltype(&fdgan_grad_norm_workspace) norm_workspace = nullptr;
  decltype(&fdgan_grad_norm) grad_norm = nullptr;
  decltype(&fdgan_grad_clip) grad_clip = nullptr;
  decltype(&fdgan_adam_step) adam = nullptr;
  decltype(&fdgan_adam_step_clipped) adam_clipped = nullptr;
  decltype(&fdgan_last_error) last_error = nullptr;
} entries;

int dtype_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? FD_F32 : t.scalar_type() == at::kHalf ? FD_F16 : FD_BF16;
}

// Elements from one row of `c` values to the next; -1 if the rows do not lie at one pitch with their values next to each other
int64_t pitch_of(const Tensor& t, int64_t lead, int64_t c) {
  if (t.is_contiguous()) return c;
  int64_t have = 1;
  for (int64_t d = t.dim() - 1; d >= lead; --d) {
    if (t.size(d) != 1 && t.stride(d) != have) return -1;
    have *= t.size(d);
  }
  int64_t pitch = c;
  have = 1;
  for (int64_t d = lead - 1; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (have == 1) pitch = t.stride(d);
    else if (t.stride(d) != pitch * have) return -1;
    have *= t.size(d);
  }
  return pitch;
}

struct Rows {
  Tensor t;          // what is read: the tensor itself, or its copy where the layout is no rows at one pitch
  FdTensor fd;
};
Rows rows_of(const Tensor& x, int64_t lead, int64_t c, int64_t rows) {
  Rows r;
  int64_t pitch = pitch_of(x, lead, c);
  r.t = pitch < 0 ? x.contiguous() : x;
  if (pitch < 0) pitch = c;
  r.fd = FdTensor{r.t.data_ptr(), rows, 1, 1, c, {pitch, pitch, pitch, 1}, dtype_of(x), 0};
  return r;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void check(int rc, const char* what) {
  TORCH_CHECK(rc == FD_OK, "libfdgan_hip ", what, " failed (", rc, "): ", entries.last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

struct Result {
  Tensor y, x, stats;
};

Result forward_rows(const Tensor& x, const Tensor& w, const Tensor& b, int64_t lead, int64_t c, double eps, bool keep) {
  const c10::DeviceGuard guard(x.device());
  const int64_t rows = x.numel() / c;
  Result r;
  r.y = at::empty(x.sizes(), x.options());
  if (keep) r.stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
  r.x = x;
  if (rows == 0) return r;
  const Rows in = rows_of(x, lead, c, rows);
  r.x = in.t;
  const FdTensor out{r.y.data_ptr(), rows, 1, 1, c, {c, c, c, 1}, in.fd.dtype, 0};
  const int64_t floats = entries.workspace(rows, c, 0);
  TORCH_CHECK_VALUE(floats >= 0, "layer_norm: ", rows, " rows of ", c, " values are too many for one call");
  const Tensor ws = floats > 0 ? at::empty({floats}, x.options().dtype(at::kFloat)) : Tensor();
  float* mean = keep ? r.stats.data_ptr<float>() : nullptr;
  const Tensor& wt = w.defined() ? w : b;
  check(entries.fwd(&in.fd, ptr(w), ptr(b), wt.defined() ? dtype_of(wt) : FD_F32, (float)eps, &out, mean, keep ? mean + rows : nullptr,
                    static_cast<float*>(ptr(ws)), floats, stream_of(x)),
        "layer_norm_fwd");
  return r;
}

struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& w, const std::optional<Tensor>& b, int64_t lead, int64_t c, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
    Result r = forward_rows(x, weight.defined() ? weight.contiguous() : weight, bias.defined() ? bias.contiguous() : bias, lead, c, eps, true);
    ctx->save_for_backward({r.x, weight, r.stats});
    ctx->saved_data["lead"] = lead;
    ctx->saved_data["c"] = c;
    if (bias.defined()) {
      ctx->saved_data["bias"] = bias.sizes().vec();
      ctx->saved_data["btype"] = (int64_t)bias.scalar_type();
    }
    return r.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const variable_list saved = ctx->get_saved_variables();
      const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2], &dy = grads[0];
      if (!dy.defined()) return out;
      const c10::DeviceGuard guard(x.device());
      const int64_t lead = ctx->saved_data["lead"].toInt(), c = ctx->saved_data["c"].toInt(), rows = x.numel() / c;
      const bool has_bias = ctx->saved_data.count("bias") > 0;
      const auto wtype = weight.defined() ? weight.scalar_type() : has_bias ? (at::ScalarType)ctx->saved_data["btype"].toInt() : at::kFloat;
      // the edges count the tensors that were given
      if (ctx->needs_input_grad(0)) out[0] = at::empty(x.sizes(), x.options());
      if (weight.defined() && ctx->needs_input_grad(1)) out[1] = at::empty(weight.sizes(), x.options().dtype(wtype));
      if (has_bias && ctx->needs_input_grad(weight.defined() ? 2 : 1)) out[2] = at::empty(ctx->saved_data["bias"].toIntVector(), x.options().dtype(wtype));
      if (rows == 0) {
        for (int k = 1; k < 3; ++k)
          if (out[k].defined()) out[k].zero_();
      } else if (out[0].defined() || out[1].defined() || out[2].defined()) {
        const Rows rx = rows_of(x, lead, c, rows), rdy = rows_of(dy, lead, c, rows);
        const Tensor w = weight.defined() ? weight.contiguous() : weight;
        const int64_t floats = entries.workspace(rows, c, 1);
        TORCH_CHECK_VALUE(floats >= 0, "layer_norm: the gradients of ", rows, " rows of ", c, " values are too many for one call");
        const Tensor ws = at::empty({floats}, x.options().dtype(at::kFloat));
        const FdTensor dx{ptr(out[0]), rows, 1, 1, c, {c, c, c, 1}, rx.fd.dtype, 0};
        const float* mean = stats.data_ptr<float>();
        check(entries.bwd(&rx.fd, &rdy.fd, ptr(w), wtype == at::kFloat ? FD_F32 : wtype == at::kHalf ? FD_F16 : FD_BF16, mean, mean + rows,
                          out[0].defined() ? &dx : nullptr, ptr(out[1]), ptr(out[2]), 0, ws.data_ptr<float>(), floats, stream_of(x)),
              "layer_norm_bwd");
      }
    }
    if (again) {      // the results were formed outside autograd: a second derivative must raise, not come out as zero
      variable_list have;
      for (const Tensor& t : out)
        if (t.defined()) have.push_back(t.requires_grad_(true).view_as(t));
      auto error = std::make_shared<torch::autograd::DelayedError>("layer_norm can be differentiated once", (int64_t)have.size());
      have = (*error)(std::move(have));
      size_t k = 0;
      for (Tensor& t : out)
        if (t.defined()) t = have[k++];
    }
    return out;
  }
};

Tensor layer_norm(const Tensor& x, const std::vector<int64_t>& shape, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  TORCH_CHECK(entries.fwd, "fdgan::layer_norm: the library's entries are not bound (fdgan_hip.lib.torch_ops)");
  // a tangent would be dropped: below, only requires_grad is asked for
  const auto dual = [](const std::optional<Tensor>& t) { return t && t->defined() && t->_fw_grad(0).defined(); };
  TORCH_CHECK(!x._fw_grad(0).defined() && !dual(weight) && !dual(bias), "layer_norm: forward-mode derivatives are not offered (the gradient is, once)");
  TORCH_CHECK(x.is_cuda(), "layer_norm: the FD-GAN HIP path needs a tensor on an MI355X (`cuda`) device; there is no CPU fallback");
  const int64_t k = (int64_t)shape.size(), lead = x.dim() - k;
  TORCH_CHECK_VALUE(k > 0 && lead >= 0 && x.sizes().slice(lead) == at::IntArrayRef(shape), "layer_norm: a tensor of shape ", x.sizes(),
                    " does not end in normalized_shape ", at::IntArrayRef(shape));
  double many = 1;
  for (int64_t n : shape) many *= (double)n;
  TORCH_CHECK_VALUE(many >= 1 && many <= (double)(1 << 29), "layer_norm: rows of ", many, " values");
  const int64_t c = (int64_t)many;
  const auto type = x.scalar_type();
  TORCH_CHECK_TYPE((type == at::kFloat || type == at::kHalf || type == at::kBFloat16) && x.layout() == at::kStrided, "layer_norm: fp32, fp16 or bf16 expected, got ", type);
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps ", eps);
  for (const auto* t : {&weight, &bias}) {
    if (!t->has_value()) continue;
    const Tensor& v = **t;
    TORCH_CHECK_VALUE(v.sizes() == at::IntArrayRef(shape), "layer_norm: weight or bias of shape ", v.sizes(), " for normalized_shape ", at::IntArrayRef(shape));
    TORCH_CHECK(v.device() == x.device(), "layer_norm: weight or bias is on ", v.device(), " but the input is on ", x.device());
    TORCH_CHECK_TYPE(v.scalar_type() == at::kFloat || v.scalar_type() == type, "layer_norm: weight or bias of ", v.scalar_type(), " for an input of ", type,
                     " (fp32 or the input's type expected)");
  }
  TORCH_CHECK_TYPE(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "layer_norm: weight and bias differ in type");
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad())))
    return LayerNormFn::apply(x, weight, bias, lead, c, eps);
  return forward_rows(x, w.defined() ? w.contiguous() : w, b.defined() ? b.contiguous() : b, lead, c, eps, false).y;
}

// ---- gradient lists --------------------------------------------------------------------------------------------------------------
struct Spans {
  std::vector<FdGradSpan> table;
  std::vector<std::pair<Tensor, Tensor>> copies;      // a tensor with gaps, and the dense copy that is worked on
};

Spans spans_of(const std::vector<Tensor>& ts, const char* what, bool in_place) {
  TORCH_CHECK(entries.grad_clip, "fdgan: the library's entries are not bound (fdgan_hip.lib.torch_ops)");
  Spans s;
  s.table.reserve(ts.size());
  for (const Tensor& t : ts) {
    TORCH_CHECK(t.is_cuda(), what, ": the FD-GAN HIP path needs a tensor on an MI355X (`cuda`) device; there is no CPU fallback");
    TORCH_CHECK_VALUE(t.device() == ts[0].device(), what, ": tensors on ", ts[0].device(), " and ", t.device(), " (one process drives one GPU)");
    const auto st = t.scalar_type();
    TORCH_CHECK_TYPE(t.layout() == at::kStrided && (st == at::kFloat || st == at::kHalf || st == at::kBFloat16), what,
                     ": dense fp32, fp16 or bf16 tensors expected, got ", t.layout(), " ", st);
    Tensor d = t;
    if (!t.is_non_overlapping_and_dense()) {
      if (in_place)
        for (int64_t k = 0; k < t.dim(); ++k)
          TORCH_CHECK_VALUE(t.stride(k) != 0 || t.size(k) < 2, what, ": an expanded tensor of shape ", t.sizes(), " cannot be scaled in place");
      d = t.contiguous();
      s.copies.emplace_back(t, d);
    }
    s.table.push_back({d.data_ptr(), d.numel(), dtype_of(d)});
  }
  if (in_place && s.table.size() > 1) {
    std::vector<std::pair<char*, char*>> held;
    held.reserve(s.table.size());
    for (const FdGradSpan& g : s.table)
      if (g.n > 0) held.emplace_back(static_cast<char*>(g.ptr), static_cast<char*>(g.ptr) + g.n * (g.dtype == FD_F32 ? 4 : 2));
    std::sort(held.begin(), held.end());
    for (size_t k = 1; k < held.size(); ++k) TORCH_CHECK_VALUE(held[k - 1].second <= held[k].first, what, ": two of the tensors share memory");
  }
  return s;
}

// max_norm < 0: the norm alone
Tensor norm_of(const Spans& s, const Tensor& like, int64_t kind, double max_norm, const char* what) {
  const c10::DeviceGuard guard(like.device());
  const int64_t n = (int64_t)s.table.size(), room = entries.norm_workspace(s.table.data(), n);
  TORCH_CHECK(room > 0, what, ": a tensor is too long");
  const auto options = at::TensorOptions().device(like.device());
  const Tensor partial = at::empty({room}, options.dtype(at::kDouble)), out = at::empty({}, options.dtype(at::kFloat));
  double* p = partial.data_ptr<double>();
  float* o = out.data_ptr<float>();
  if (max_norm < 0) check(entries.grad_norm(s.table.data(), n, (int)kind, p, room, o, stream_of(like)), what);
  else check(entries.grad_clip(s.table.data(), n, (int)kind, (float)max_norm, p, room, o, stream_of(like)), what);
  return out;
}

Tensor grad_norm(const at::TensorList tensors, int64_t kind) {
  if (tensors.empty()) return at::zeros({});
  at::NoGradGuard off;
  const std::vector<Tensor> ts = tensors.vec();
  return norm_of(spans_of(ts, "grad_norm", false), ts[0], kind, -1.0, "grad_norm");
}

Tensor clip_grad_norm(const at::TensorList parameters, double max_norm, int64_t kind, bool finite) {
  at::NoGradGuard off;
  std::vector<Tensor> grads;
  grads.reserve(parameters.size());
  std::unordered_set<const void*> seen;
  seen.reserve(parameters.size());
  for (const Tensor& p : parameters)
    if (p.grad().defined() && seen.insert(p.unsafeGetTensorImpl()).second) grads.push_back(p.grad());
  if (grads.empty()) return at::zeros({});
  const Spans s = spans_of(grads, "clip_grad_norm_", true);
  if (finite) {
    const double total = norm_of(s, grads[0], kind, -1.0, "clip_grad_norm_").item<double>();
    TORCH_CHECK(std::isfinite(total), "clip_grad_norm_: the gradients' norm is ", total, ": nothing was clipped");
  }
  const Tensor total = norm_of(s, grads[0], kind, max_norm, "clip_grad_norm_");
  for (const auto& c : s.copies) c.first.copy_(c.second);
  for (const Tensor& g : grads)
    if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
  return total;
}

// ---- Adam -----------------------------------------------------------------------------------------------------------------------
// max_norm: absent, no clipping; the result is then undefined (None)
std::optional<Tensor> adam_step(const Tensor& p, const Tensor& g, const Tensor& m, const Tensor& v, int64_t step, double lr, double b1, double b2, double eps,
                                const std::optional<double>& max_norm) {
  TORCH_CHECK(entries.adam, "fdgan: the library's entries are not bound (fdgan_hip.lib.torch_ops)");
  TORCH_CHECK(p.is_cuda(), "adam_step_: the FD-GAN HIP path needs a tensor on an MI355X (`cuda`) device; there is no CPU fallback");
  const int64_t n = p.numel();
  const char* name = "pgmv";
  for (const Tensor* t : {&p, &g, &m, &v}) {
    TORCH_CHECK_VALUE(t->device() == p.device() && t->scalar_type() == at::kFloat && t->layout() == at::kStrided && t->numel() == n && t->is_contiguous(),
                      "adam_step_: ", *name, ": contiguous fp32 tensors of one length on one device expected, got ", t->scalar_type(), " ", t->sizes(), " on ", t->device());
    TORCH_CHECK_VALUE(n == 0 || ((uintptr_t)t->data_ptr() & 15) == 0, "adam_step_: ", *name, " does not begin at a multiple of 16 bytes");
    ++name;
  }
  const char* at[4] = {static_cast<char*>(p.data_ptr()), static_cast<char*>(g.data_ptr()), static_cast<char*>(m.data_ptr()), static_cast<char*>(v.data_ptr())};
  std::sort(at, at + 4);
  for (int k = 1; k < 4; ++k) TORCH_CHECK_VALUE(n == 0 || at[k] - at[k - 1] >= 4 * n, "adam_step_: two of the tensors share memory");
  TORCH_CHECK_VALUE(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1, "adam_step_: betas ", b1, ", ", b2, " (0 <= beta < 1)");
  TORCH_CHECK_VALUE(step >= 1, "adam_step_: step ", step, " (counts from 1)");
  TORCH_CHECK_VALUE(!max_norm || *max_norm >= 0, "adam_step_: max_norm ", max_norm.value_or(0));
  at::NoGradGuard off;
  const c10::DeviceGuard guard(p.device());
  const auto options = at::TensorOptions().device(p.device());
  std::optional<Tensor> norm;
  if (n == 0) {
    if (max_norm) norm = at::zeros({}, options.dtype(at::kFloat));
    return norm;
  }
  float *pp = p.data_ptr<float>(), *mp = m.data_ptr<float>(), *vp = v.data_ptr<float>();
  const float* gp = g.data_ptr<float>();
  if (!max_norm) {
    check(entries.adam(pp, gp, mp, vp, n, (float)lr, b1, b2, (float)eps, step, stream_of(p)), "adam_step");
  } else {
    const FdGradSpan s{const_cast<float*>(gp), n, FD_F32};
    const int64_t room = entries.norm_workspace(&s, 1);
    TORCH_CHECK(room > 0, "adam_step_: the tensors are too long");
    const Tensor partial = at::empty({room}, options.dtype(at::kDouble));
    norm = at::empty({}, options.dtype(at::kFloat));
    check(entries.adam_clipped(pp, gp, mp, vp, n, (float)lr, b1, b2, (float)eps, step, (float)*max_norm, partial.data_ptr<double>(), room,
                               norm->data_ptr<float>(), stream_of(p)),
          "adam_step_clipped");
  }
  for (const Tensor* t : {&p, &m, &v})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return norm;
}

void bind(int64_t version, const std::vector<int64_t>& address) {
  TORCH_CHECK(version == FDGAN_ABI_VERSION, "fdgan torch module built for ABI ", FDGAN_ABI_VERSION, ", library has ", version);
  TORCH_CHECK(address.size() == 9, "fdgan torch module: 9 entries expected");
  entries.fwd = reinterpret_cast<decltype(entries.fwd)>(address[0]);
  entries.bwd = reinterpret_cast<decltype(entries.bwd)>(address[1]);
  entries.workspace = reinterpret_cast<decltype(entries.workspace)>(address[2]);
  entries.norm_workspace = reinterpret_cast<decltype(entries.norm_workspace)>(address[3]);
  entries.grad_norm = reinterpret_cast<decltype(entries.grad_norm)>(address[4]);
  entries.grad_clip = reinterpret_cast<decltype(entries.grad_clip)>(address[5]);
  entries.adam = reinterpret_cast<decltype(entries.adam)>(address[6]);
  entries.adam_clipped = reinterpret_cast<decltype(entries.adam_clipped)>(address[7]);
  entries.last_error = reinterpret_cast<decltype(entries.last_error)>(address[8]);
}

}  // namespace

TORCH_LIBRARY(fdgan, m) {
  m.def("layer_norm(Tensor x, int[] normalized_shape, Tensor? weight, Tensor? bias, float eps) -> Tensor",
        [](const Tensor& x, const std::vector<int64_t>& shape, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
          return layer_norm(x, shape, weight, bias, eps);
        });
  m.def("adam_step(Tensor p, Tensor g, Tensor m, Tensor v, int step, float lr, float beta1, float beta2, float eps, float? max_norm) -> Tensor?", &adam_step);
  m.def("grad_norm(Tensor[] tensors, int kind) -> Tensor", [](const std::vector<Tensor>& t, int64_t kind) { return grad_norm(t, kind); });
  m.def("clip_grad_norm(Tensor[] parameters, float max_norm, int kind, bool finite) -> Tensor",
        [](const std::vector<Tensor>& t, double max_norm, int64_t kind, bool finite) { return clip_grad_norm(t, max_norm, kind, finite); });
  m.def("bind(int version, int[] address) -> ()", [](int64_t version, const std::vector<int64_t>& address) { bind(version, address); });
  m.def("build_id() -> str", [] { return std::string(FDGAN_TORCH_ID); });
}
