// The operators' host path in C++: the same checks, allocations and C calls as
// decode.py, block_norm.py and sampling.py make, for calls of a few
// microseconds where the interpreter's share is the larger one.  A call that
// does not pass the checks returns None and the Python path takes it (it
// raises the error, or brings unusual strides into order).
//
// The C entry points come from the library that _native.py loaded (bind).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>

#include "../../../../include/kdn_b200.h"

namespace {

using at::Tensor;
using Optional = std::optional<Tensor>;

struct Entries {
  int (*step)(const KdnStepArgs*, kdn_stream_t);
  int (*norm_fwd)(const KdnBlockNormArgs*, kdn_stream_t);
  int (*norm_bwd)(const KdnBlockNormArgs*, kdn_stream_t);
  size_t (*norm_workspace)(int64_t, int64_t);
  int (*sample)(const KdnSampleArgs*, kdn_stream_t);
  const char* (*last_error)();
} entry{};

void bind(uintptr_t step, uintptr_t norm_fwd, uintptr_t norm_bwd, uintptr_t norm_workspace, uintptr_t sample,
          uintptr_t last_error) {
  entry.step = reinterpret_cast<decltype(entry.step)>(step);
  entry.norm_fwd = reinterpret_cast<decltype(entry.norm_fwd)>(norm_fwd);
  entry.norm_bwd = reinterpret_cast<decltype(entry.norm_bwd)>(norm_bwd);
  entry.norm_workspace = reinterpret_cast<decltype(entry.norm_workspace)>(norm_workspace);
  entry.sample = reinterpret_cast<decltype(entry.sample)>(sample);
  entry.last_error = reinterpret_cast<decltype(entry.last_error)>(last_error);
}

template <class Args>
void launch(int (*fn)(const Args*, kdn_stream_t), const Args& args, const Tensor& on, const char* what) {
  const c10::cuda::CUDAGuard guard(on.device());
  const int rc = fn(&args, reinterpret_cast<kdn_stream_t>(c10::cuda::getCurrentCUDAStream(on.get_device()).stream()));
  if (rc != KDN_OK)
    throw std::runtime_error("kdn_b200 " + std::string(what) + " failed (" + std::to_string(rc) + "): " + entry.last_error());
}

bool is_bf16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
bool is_float(const Tensor& t) { return is_bf16(t) || t.scalar_type() == at::kFloat; }
// carries a forward-mode tangent, which no operator here propagates: the Python path refuses it
bool is_dual(const Tensor& t) { return t.unsafeGetTensorImpl()->autograd_meta() && t._fw_grad(0).defined(); }
const void* ptr(const Optional& t) { return t ? t->const_data_ptr() : nullptr; }

// rows [B, width] of a type and device, their values contiguous
bool rows_of(const Tensor& t, int64_t B, int64_t width, const Tensor& like) {
  return t.dim() == 2 && t.size(0) == B && t.size(1) == width && t.scalar_type() == like.scalar_type() &&
         t.device() == like.device() && (t.stride(1) == 1 || width == 1);
}

// ---- the token step (decode.py) ----
// args: the step's parameters laid out by decode.py; omega and r: of the isotropic step one tensor [B, 2 H]
std::optional<Tensor> step(const std::string& args, const Tensor& memory, const Tensor& covariance, const Tensor& window,
                           const Tensor& qkv, const Tensor& decay, const Tensor& omega, const Optional& r,
                           const Tensor& gate, const Optional& slots) {
  if (args.size() != sizeof(KdnStepArgs)) return std::nullopt;
  KdnStepArgs a;
  std::memcpy(&a, args.data(), sizeof(a));
  const int64_t channels = a.H * a.D;
  if (qkv.dim() != 2 || !qkv.is_cuda() || !is_float(qkv)) return std::nullopt;
  const int64_t B = qkv.size(0);
  const bool iso = a.variant == KDN_ISO;
  if (!rows_of(qkv, B, 3 * channels, qkv) || !rows_of(decay, B, channels, qkv) || !rows_of(gate, B, channels, qkv) ||
      !rows_of(omega, B, iso ? 2 * a.H : channels, qkv) || (!iso && (!r || !rows_of(*r, B, a.H, qkv))))
    return std::nullopt;
  // the Python path says that the step has no derivative
  const bool grad = at::GradMode::is_enabled();
  for (const Tensor* t : {&qkv, &decay, &omega, iso ? nullptr : &*r, &gate})
    if (t && t->unsafeGetTensorImpl()->autograd_meta() && ((grad && t->requires_grad()) || is_dual(*t))) return std::nullopt;
  if (window.scalar_type() != qkv.scalar_type() || memory.device() != qkv.device()) return std::nullopt;
  if (slots) {
    if (slots->dim() != 1 || slots->size(0) != B || !slots->is_contiguous() || slots->device() != qkv.device() ||
        (slots->scalar_type() != at::kInt && slots->scalar_type() != at::kLong))
      return std::nullopt;
    a.slots = slots->const_data_ptr();
    a.slots_i64 = slots->scalar_type() == at::kLong;
  } else if (memory.size(0) < B) {
    return std::nullopt;
  }
  Tensor y = at::empty({B, channels}, qkv.options());
  a.act_bf16 = is_bf16(qkv);
  a.B = B;
  a.num_slots = memory.size(0);
  a.qkv = qkv.const_data_ptr();
  a.qkv_stride = qkv.stride(0);
  a.decay_raw = decay.const_data_ptr();
  a.decay_stride = decay.stride(0);
  a.omega_raw = omega.const_data_ptr();
  a.omega_stride = omega.stride(0);
  if (iso) {  // the row's second half
    a.r_raw = static_cast<const char*>(omega.const_data_ptr()) + a.H * omega.element_size();
    a.r_stride = omega.stride(0);
  } else {
    a.r_raw = r->const_data_ptr();
    a.r_stride = r->stride(0);
  }
  a.gate = gate.const_data_ptr();
  a.gate_stride = gate.stride(0);
  a.memory = static_cast<float*>(memory.data_ptr());
  a.covariance = static_cast<float*>(covariance.data_ptr());
  a.window = window.data_ptr();
  a.y = y.data_ptr();
  launch(entry.step, a, qkv, "kdn_step");
  return y;
}

// ---- the norms around a block (block_norm.py) ----
KdnBlockNormArgs norm_args(const Tensor& x, const Tensor& y, const Optional& gate, const Tensor& weight,
                           const Optional& post_weight, const Optional& scale, double alpha, int64_t swish, double eps) {
  KdnBlockNormArgs a{};
  a.stream_bf16 = is_bf16(x);
  a.act_bf16 = is_bf16(y);
  a.weights_bf16 = is_bf16(weight);
  a.swish = (int32_t)swish;
  a.rows = x.size(0);
  a.D = x.size(1);
  a.alpha = (float)alpha;
  a.eps = (float)eps;
  a.x = x.const_data_ptr();
  a.y = y.const_data_ptr();
  a.gate = ptr(gate);
  a.x_stride = x.stride(0);
  a.y_stride = y.stride(0);
  a.gate_stride = gate ? gate->stride(0) : 0;
  a.weight = weight.const_data_ptr();
  a.post_weight = ptr(post_weight);
  a.scale = ptr(scale);
  return a;
}

std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& y, const Optional& gate,
                                                const Tensor& weight, const Optional& post_weight, const Optional& scale,
                                                double alpha, int64_t swish, double eps, bool keep) {
  KdnBlockNormArgs a = norm_args(x, y, gate, weight, post_weight, scale, alpha, swish, eps);
  Tensor z = at::empty(x.sizes(), x.options()), h = at::empty(x.sizes(), y.options()), rstd;
  a.z = z.data_ptr();
  a.h = h.data_ptr();
  if (keep) {
    rstd = at::empty({2, a.rows}, x.options().dtype(at::kFloat));
    a.rstd = static_cast<float*>(rstd.data_ptr());
  }
  launch(entry.norm_fwd, a, x, "kdn_block_norm_fwd");
  return {z, h, rstd};
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& y,
                                                const Optional& gate, const Tensor& weight, const Optional& post_weight,
                                                const Optional& scale, double alpha, int64_t swish, double eps) {
    auto [z, h, rstd] = norm_forward(x, y, gate, weight, post_weight, scale, alpha, swish, eps, true);
    ctx->save_for_backward({x, y, gate.value_or(Tensor()), weight, post_weight.value_or(Tensor()),
                            scale.value_or(Tensor()), rstd});
    ctx->saved_data["alpha"] = alpha;
    ctx->saved_data["swish"] = swish;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return {z, h};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list cotangents) {
    const bool again = at::GradMode::is_enabled();
    torch::autograd::variable_list grads(9);
    {
      at::AutoGradMode off(false);
      const auto saved = ctx->get_saved_variables();
      const Tensor dz = cotangents[0].defined() ? cotangents[0].contiguous() : Tensor(),
                   dh = cotangents[1].defined() ? cotangents[1].contiguous() : Tensor();
      if (!dz.defined() && !dh.defined()) return grads;
      auto present = [&](int i) { return saved[i].defined() ? Optional(saved[i]) : std::nullopt; };
      KdnBlockNormArgs a =
          norm_args(saved[0], saved[1], present(2), saved[3], present(4), present(5), ctx->saved_data["alpha"].toDouble(),
                    ctx->saved_data["swish"].toInt(), ctx->saved_data["eps"].toDouble());
      a.rstd = static_cast<float*>(saved[6].data_ptr());
      if (dz.defined()) a.dz = dz.const_data_ptr();
      if (dh.defined()) a.dh = dh.const_data_ptr();
      void** const out[6] = {&a.dx, &a.dy, &a.dgate, &a.dweight, &a.dpost, &a.dscale};
      bool weights = false;
      for (int i = 0; i < 6; ++i) {
        // z does not depend on the weight: without dh it has no gradient
        if (!saved[i].defined() || !ctx->needs_input_grad(index_of(ctx, saved, i)) || (i == 3 && !dh.defined())) continue;
        grads[i] = at::empty(saved[i].sizes(), saved[i].options());
        *out[i] = grads[i].data_ptr();
        weights = weights || i >= 3;
      }
      Tensor workspace;
      if (weights) {
        a.workspace_bytes = entry.norm_workspace(a.rows, a.D);
        workspace = at::empty({(int64_t)a.workspace_bytes}, saved[0].options().dtype(at::kByte));
        a.workspace = workspace.data_ptr();
      }
      launch(entry.norm_bwd, a, saved[0], "kdn_block_norm_bwd");
    }
    if (again) {  // as once_differentiable: differentiating the gradients is an error
      torch::autograd::variable_list some;
      for (auto& g : grads)
        if (g.defined()) some.push_back(g.detach().set_requires_grad(true));
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "trying to differentiate twice a function that was marked with @once_differentiable", (int)some.size());
      some = (*error)(std::move(some));
      size_t k = 0;
      for (auto& g : grads)
        if (g.defined()) g = some[k++];
    }
    return grads;
  }

  // the edge of input i: absent tensors have none
  static size_t index_of(torch::autograd::AutogradContext*, const torch::autograd::variable_list& saved, int i) {
    size_t k = 0;
    for (int j = 0; j < i; ++j) k += saved[j].defined();
    return k;
  }
};

// [rows, D] with contiguous rows that do not overlap, or one row for all
bool apart(const Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= t.size(1) || t.stride(0) == 0);
}

// rows [rows, D] as apart() wants them; the gate and the block's output as x
std::optional<std::tuple<Tensor, Tensor>> block_norm(const Tensor& x, const Tensor& y, const Tensor& weight,
                                                     const Optional& post_weight, const Optional& gate,
                                                     const Optional& scale, double alpha, int64_t swish, double eps,
                                                     int64_t least, int64_t most) {
  if (x.dim() < 1 || !x.is_cuda() || !is_float(x) || !is_float(y) || y.sizes() != x.sizes()) return std::nullopt;
  const int64_t D = x.size(-1);
  if (D < least || D > most || x.numel() == 0) return std::nullopt;
  if (is_bf16(x) && !is_bf16(y)) return std::nullopt;
  if (is_dual(x) || is_dual(y)) return std::nullopt;
  if (gate && (is_dual(*gate) || gate->sizes() != x.sizes() || gate->scalar_type() != y.scalar_type())) return std::nullopt;
  for (const Tensor* w : {&weight, post_weight ? &*post_weight : nullptr, scale ? &*scale : nullptr})
    if (w && (is_dual(*w) || w->dim() != 1 || w->size(0) != D || !w->is_contiguous() || !is_float(*w) ||
              w->scalar_type() != weight.scalar_type() || w->device() != x.device()))
      return std::nullopt;
  for (const Tensor* t : {&x, &y, gate ? &*gate : nullptr})
    if (t && (t->device() != x.device() || (t->dim() == 2 ? !apart(*t) : !t->is_contiguous()))) return std::nullopt;
  const bool flat = x.dim() == 2;
  const Tensor x2 = flat ? x : x.view({-1, D}), y2 = flat ? y : y.view({-1, D});
  const Optional g2 = !gate || flat ? gate : Optional(gate->view({-1, D}));
  auto wants = [](const Tensor& t) { return t.requires_grad(); };
  const bool grad = at::GradMode::is_enabled() &&
                    (wants(x) || wants(y) || wants(weight) || (gate && wants(*gate)) ||
                     (post_weight && wants(*post_weight)) || (scale && wants(*scale)));
  Tensor z, h;
  if (grad) {
    auto out = BlockNorm::apply(x2, y2, g2, weight, post_weight, scale, alpha, swish, eps);
    z = out[0];
    h = out[1];
  } else {
    std::tie(z, h, std::ignore) = norm_forward(x2, y2, g2, weight, post_weight, scale, alpha, swish, eps, false);
  }
  if (!flat) {
    z = z.view(x.sizes());
    h = h.view(x.sizes());
  }
  return std::make_tuple(z, h);
}

// ---- sampling (sampling.py) ----
// a filter's value: a tensor [rows] of one of two types, a number, or None (`none`)
template <class V>
bool option(const py::object& value, int64_t rows, const Tensor& like, at::ScalarType first, at::ScalarType second,
            V none, const void*& at, V& all, bool* is_second) {
  if (value.is_none()) {
    all = none;
  } else if (THPVariable_Check(value.ptr())) {
    const Tensor& t = THPVariable_Unpack(value.ptr());
    if (t.dim() != 1 || t.size(0) != rows || !t.is_contiguous() || t.device() != like.device() ||
        (t.scalar_type() != first && t.scalar_type() != second))
      return false;
    at = t.const_data_ptr();
    if (is_second) *is_second = t.scalar_type() == second;
  } else if (PyFloat_Check(value.ptr()) && !is_second) {
    all = (V)PyFloat_AS_DOUBLE(value.ptr());
  } else if (PyLong_CheckExact(value.ptr())) {
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(value.ptr(), &overflow);
    if (overflow) return false;
    all = (V)v;
  } else {
    return false;
  }
  return true;
}

std::optional<std::tuple<Tensor, Tensor>> sample(const Tensor& logits, const Tensor& noise, const py::object& temperature,
                                                 const py::object& top_k, const py::object& top_p,
                                                 const py::object& min_p, int64_t most) {
  if (logits.dim() != 2 || !logits.is_cuda() || !is_float(logits) || logits.size(1) < 1 || logits.size(1) > most)
    return std::nullopt;
  if (noise.sizes() != logits.sizes() || noise.scalar_type() != at::kFloat || noise.device() != logits.device())
    return std::nullopt;
  if (logits.size(1) > 1 && (logits.stride(1) != 1 || noise.stride(1) != 1)) return std::nullopt;
  KdnSampleArgs a{};
  a.rows = logits.size(0);
  a.V = logits.size(1);
  const void *t = nullptr, *p = nullptr, *m = nullptr;
  bool k64 = false;
  if (temperature.is_none() ||
      !option(temperature, a.rows, logits, at::kFloat, at::kFloat, 1.f, t, a.temperature_all, nullptr) ||
      !option(top_k, a.rows, logits, at::kInt, at::kLong, (int64_t)0, a.top_k, a.top_k_all, &k64) ||
      !option(top_p, a.rows, logits, at::kFloat, at::kFloat, 1.f, p, a.top_p_all, nullptr) ||
      !option(min_p, a.rows, logits, at::kFloat, at::kFloat, 0.f, m, a.min_p_all, nullptr))
    return std::nullopt;
  a.temperature = static_cast<const float*>(t);
  a.top_p = static_cast<const float*>(p);
  a.min_p = static_cast<const float*>(m);
  a.top_k_i64 = k64;
  a.logits_bf16 = is_bf16(logits);
  a.logits = logits.const_data_ptr();
  a.noise = static_cast<const float*>(noise.const_data_ptr());
  a.logits_stride = logits.stride(0);
  a.noise_stride = noise.stride(0);
  Tensor token = at::empty({a.rows}, noise.options().dtype(at::kLong)), prob = at::empty({a.rows}, noise.options());
  a.token = static_cast<int64_t*>(token.data_ptr());
  a.prob = static_cast<float*>(prob.data_ptr());
  launch(entry.sample, a, logits, "kdn_sample");
  return std::make_tuple(token, prob);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("step", &step);
  m.def("block_norm", &block_norm);
  m.def("sample", &sample);
}
