// Python bindings of the fused causal attention kernels.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <array>
#include <climits>
#include <cmath>

#include "kernels/api.h"

namespace {
using at::Tensor;

// [B, T, H, hd] view whose head dim is dense and whose batch stride is T * token stride,
// i.e. a column slice of a [B*T, W] row-major buffer.
bool is_token_major(const Tensor& t) {
  return t.dim() == 4 && t.stride(3) == 1 && t.stride(2) == t.size(3) && t.stride(0) == t.size(1) * t.stride(1) &&
         (t.stride(1) % 8) == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) == 0;
}
Tensor token_major(const Tensor& t) { return is_token_major(t) ? t : t.contiguous(); }

void check(int rc, const char* what) {
  TORCH_CHECK(rc != TITB_ERR_SHAPE, "titb200: ", what, ": head_dim must be 64 or 128 and Hq % Hkv == 0");
  TORCH_CHECK(rc != TITB_ERR_ALIGNMENT, "titb200: ", what, ": operands must be 16-byte aligned");
  TORCH_CHECK(rc != TITB_ERR_TENSOR_MAP, "titb200: ", what, ": TMA tensor map could not be encoded");
  TORCH_CHECK(rc == 0, "titb200: ", what, " failed: ", cudaGetErrorString(static_cast<cudaError_t>(rc)));
}

std::vector<Tensor> attn_fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, double scale) {
  TORCH_CHECK(q_.is_cuda() && q_.scalar_type() == at::kBFloat16, "titb200 attention: bf16 CUDA tensors");
  c10::cuda::CUDAGuard guard(q_.device());
  Tensor q = token_major(q_), k = token_major(k_), v = token_major(v_);
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), hd = q.size(3), Hkv = k.size(2);
  Tensor o = at::empty({B, T, Hq, hd}, q.options());
  Tensor lse = at::empty({B, Hq, T}, q.options().dtype(at::kFloat));
  TitbAttnDesc d{};
  d.q = q.data_ptr(); d.k = k.data_ptr(); d.v = v.data_ptr(); d.o = o.data_ptr(); d.lse = lse.data_ptr<float>();
  d.B = (int)B; d.T = (int)T; d.Hq = (int)Hq; d.Hkv = (int)Hkv; d.hd = (int)hd;
  d.q_stride_t = q.stride(1); d.k_stride_t = k.stride(1); d.v_stride_t = v.stride(1); d.o_stride_t = Hq * hd;
  d.scale = (float)scale;
  check(titb_attn_fwd(&d, at::cuda::getCurrentCUDAStream().stream()), "attn_fwd");
  return {o, lse};
}

// Gradients are written into dq/dk/dv when given (token-major views, e.g. slices of one fused
// dQKV buffer); otherwise fresh contiguous tensors are returned.
std::vector<Tensor> attn_bwd(const Tensor& d_o_, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o,
                             const Tensor& lse, double scale, const c10::optional<Tensor>& dq_,
                             const c10::optional<Tensor>& dk_, const c10::optional<Tensor>& dv_) {
  c10::cuda::CUDAGuard guard(q_.device());
  Tensor q = token_major(q_), k = token_major(k_), v = token_major(v_), d_o = token_major(d_o_);
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), hd = q.size(3), Hkv = k.size(2);
  Tensor dq = dq_.has_value() && dq_->defined() ? *dq_ : at::empty({B, T, Hq, hd}, q.options());
  Tensor dk = dk_.has_value() && dk_->defined() ? *dk_ : at::empty({B, T, Hkv, hd}, q.options());
  Tensor dv = dv_.has_value() && dv_->defined() ? *dv_ : at::empty({B, T, Hkv, hd}, q.options());
  TORCH_CHECK(is_token_major(dq) && is_token_major(dk) && is_token_major(dv), "titb200 attention: bad gradient views");
  Tensor delta = at::empty({B, Hq, T}, q.options().dtype(at::kFloat));
  Tensor acc = at::empty({B, T, Hq, hd}, q.options().dtype(at::kFloat));
  TitbAttnDesc d{};
  d.q = q.data_ptr(); d.k = k.data_ptr(); d.v = v.data_ptr(); d.o = o.data_ptr(); d.lse = lse.data_ptr<float>();
  d.d_o = d_o.data_ptr(); d.dq = dq.data_ptr(); d.dk = dk.data_ptr(); d.dv = dv.data_ptr();
  d.delta = delta.data_ptr<float>(); d.dq_accum = acc.data_ptr<float>();
  d.B = (int)B; d.T = (int)T; d.Hq = (int)Hq; d.Hkv = (int)Hkv; d.hd = (int)hd;
  d.q_stride_t = q.stride(1); d.k_stride_t = k.stride(1); d.v_stride_t = v.stride(1); d.o_stride_t = o.stride(1);
  d.do_stride_t = d_o.stride(1); d.dq_stride_t = dq.stride(1); d.dk_stride_t = dk.stride(1); d.dv_stride_t = dv.stride(1);
  d.scale = (float)scale;
  check(titb_attn_bwd(&d, at::cuda::getCurrentCUDAStream().stream()), "attn_bwd");
  return {dq, dk, dv};
}

// ---- window and sinks
void limits_check(const Tensor& t, int64_t B, int64_t T, int64_t Hq, int64_t hd, int64_t window, int64_t sinks, double scale) {
  const float scale32 = static_cast<float>(scale);   // what the kernels take
  TORCH_CHECK(scale32 > 0.f && std::isfinite(scale32), "titb200 window_attention: scale must be positive, got ", scale);
  TORCH_CHECK(window >= 1, "titb200 window_attention: window must be at least 1, got ", window);
  TORCH_CHECK(sinks >= 0, "titb200 window_attention: sinks must not be negative, got ", sinks);
  if (!t.is_cuda()) return;
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat,
              "titb200 window_attention: only float32 and bfloat16 tensors are supported, got ", t.scalar_type());
  TORCH_CHECK(hd > 0 && hd <= 128 && hd % 8 == 0, "titb200 window_attention: head_dim must be a multiple of 8 up to 128, got ", hd);
  TORCH_CHECK(T <= 32 * 32767LL && B * Hq < (1LL << 31), "titb200 window_attention: too many tokens or heads");
}
void window_check(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, double scale) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "titb200 window_attention: q [B, T, Hq, hd], k and v [B, T, Hkv, hd]");
  TORCH_CHECK(k.sizes() == v.sizes(), "titb200 window_attention: k and v must have the same shape");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
              "titb200 window_attention: q and k must agree in batch, length and head_dim");
  TORCH_CHECK(k.size(2) > 0 && q.size(2) % k.size(2) == 0, "titb200 window_attention: Hq must be a multiple of Hkv");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() && q.device() == k.device() &&
                  q.device() == v.device(), "titb200 window_attention: q, k and v must share dtype and device");
  limits_check(q, q.size(0), q.size(1), q.size(2), q.size(3), window, sinks, scale);
}

// Elements between the tokens of a [B, T, H, hd] view, taken from a dimension that has more than one entry.
int64_t token_stride(const Tensor& t) {
  return t.size(1) > 1 ? t.stride(1) : t.size(0) > 1 ? t.stride(0) : t.size(2) * t.size(3);
}
// A view is used in place when its heads are dense, its sequences T tokens apart and its rows 16-byte aligned; any other is
// copied.
bool addressable(const Tensor& t) {
  if (t.numel() == 0) return true;
  const int64_t st = token_stride(t);
  return (t.size(3) == 1 || t.stride(3) == 1) && (t.size(2) == 1 || t.stride(2) == t.size(3)) &&
         (t.size(0) == 1 || t.stride(0) == t.size(1) * st) && st >= t.size(2) * t.size(3) && st % (16 / t.element_size()) == 0 &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) == 0;
}
Tensor in_place_or_copy(const Tensor& t) { return addressable(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// A [B, T, H, hd] operand of the kernels: a tensor of its own, or a slice of a fused projection.
struct Rows {
  void* ptr;
  int64_t stride;   // elements between tokens
};
Rows rows_of(const Tensor& t) { return {t.data_ptr(), token_stride(t)}; }
struct Shape {
  int64_t B, T, Hq, Hkv, hd;
};

TitbWindowDesc window_desc(const Shape& s, Rows q, Rows k, Rows v, at::ScalarType type, int64_t window, int64_t sinks, double scale) {
  TitbWindowDesc w{};
  TitbAttnDesc& d = w.attn;
  d.q = q.ptr; d.k = k.ptr; d.v = v.ptr;
  d.B = (int)s.B; d.T = (int)s.T; d.Hq = (int)s.Hq; d.Hkv = (int)s.Hkv; d.hd = (int)s.hd;
  d.q_stride_t = q.stride; d.k_stride_t = k.stride; d.v_stride_t = v.stride;
  d.o_stride_t = s.Hq * s.hd;
  d.scale = (float)scale;
  w.window = (int)std::min<int64_t>(window, INT_MAX);
  w.sinks = (int)std::min<int64_t>(sinks, INT_MAX);
  w.dtype = type == at::kBFloat16 ? 1 : 0;
  return w;
}

// {o [B, T, Hq, hd], lse fp32 [B, Hq, T], what the rounding of o left (bf16, when a backward pass may follow)}
std::array<Tensor, 3> window_forward(const Shape& s, Rows q, Rows k, Rows v, const at::TensorOptions& opt, int64_t window,
                                     int64_t sinks, double scale, bool training) {
  Tensor o = at::empty({s.B, s.T, s.Hq, s.hd}, opt);
  Tensor lse = at::empty({s.B, s.Hq, s.T}, opt.dtype(at::kFloat));
  TitbWindowDesc w = window_desc(s, q, k, v, o.scalar_type(), window, sinks, scale);
  w.attn.o = o.data_ptr(); w.attn.lse = lse.data_ptr<float>();
  Tensor o_lo;
  if (training && w.dtype == 1) {
    o_lo = at::empty_like(o);
    w.o_lo = o_lo.data_ptr();
  }
  check(titb_window_attn_fwd(&w, at::cuda::getCurrentCUDAStream().stream()), "window_attention");
  return {o, lse, o_lo};
}

void window_backward(const Shape& s, const Tensor& d_o_, Rows q, Rows k, Rows v, const Tensor& o, const Tensor& lse, const Tensor& o_lo,
                     Rows dq, Rows dk, Rows dv, int64_t window, int64_t sinks, double scale) {
  TORCH_CHECK(d_o_.sizes() == o.sizes() && d_o_.scalar_type() == o.scalar_type() && d_o_.device() == o.device(),
              "titb200 window_attention: the gradient must look like the output");
  const Tensor d_o = in_place_or_copy(d_o_);
  TitbWindowDesc w = window_desc(s, q, k, v, o.scalar_type(), window, sinks, scale);
  TitbAttnDesc& d = w.attn;
  d.o = o.data_ptr(); d.lse = lse.data_ptr<float>();
  w.o_lo = o_lo.defined() ? o_lo.data_ptr() : nullptr;
  d.d_o = d_o.data_ptr(); d.do_stride_t = token_stride(d_o);
  d.dq = dq.ptr; d.dk = dk.ptr; d.dv = dv.ptr;
  d.dq_stride_t = dq.stride; d.dk_stride_t = dk.stride; d.dv_stride_t = dv.stride;
  // one scratch buffer: delta, to a multiple of four floats, and the kernels' workspace
  const int64_t n_delta = (s.B * s.Hq * s.T + 3) / 4 * 4;
  Tensor scratch = at::empty({n_delta + titb_window_attn_bwd_workspace(&w)}, o.options().dtype(at::kFloat));
  d.delta = scratch.data_ptr<float>();
  w.workspace = d.delta + n_delta;
  check(titb_window_attn_bwd(&w, at::cuda::getCurrentCUDAStream().stream()), "window_attention backward");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients of a backward pass that is itself recorded: usable as values, an error where they are differentiated.
variable_list first_order_only(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads) g = g.detach().set_requires_grad(true);   // the error node is attached to inputs that require one
  auto error = std::make_shared<torch::autograd::DelayedError>("titb200 window_attention has no second derivative",
                                                               static_cast<int64_t>(grads.size()));
  return (*error)(std::move(grads));
}

// The autograd functions are C++ ones: forward and backward through a Python one took 97 us of host time, which is more than
// the kernels run on a few hundred tokens; 75 us now, most of it the autograd engine.
struct WindowAttention : public torch::autograd::Function<WindowAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t window, int64_t sinks,
                        double scale, bool training) {
    c10::cuda::CUDAGuard guard(q_.device());
    const Tensor q = in_place_or_copy(q_), k = in_place_or_copy(k_), v = in_place_or_copy(v_);
    const Shape s{q.size(0), q.size(1), q.size(2), k.size(2), q.size(3)};
    auto [o, lse, o_lo] = window_forward(s, rows_of(q), rows_of(k), rows_of(v), q.options(), window, sinks, scale, training);
    ctx->save_for_backward({q, k, v, o, lse, o_lo});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2];
    c10::cuda::CUDAGuard guard(q.device());
    const Shape s{q.size(0), q.size(1), q.size(2), k.size(2), q.size(3)};
    at::AutoDispatchBelowADInplaceOrView below;
    // no query heads: no kernel runs, and no query sees a key
    const auto gradient = [&](int64_t heads) {
      return s.Hq > 0 ? at::empty({s.B, s.T, heads, s.hd}, q.options()) : at::zeros({s.B, s.T, heads, s.hd}, q.options());
    };
    Tensor dq = gradient(s.Hq), dk = gradient(s.Hkv), dv = gradient(s.Hkv);
    window_backward(s, grads[0], rows_of(q), rows_of(k), rows_of(v), saved[3], saved[4], saved[5], rows_of(dq), rows_of(dk), rows_of(dv),
                    ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble());
    grads = first_order_only({dq, dk, dv});
    return {grads[0], grads[1], grads[2], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// Over a fused projection buffer [B, T, (Hq + 2 Hkv) * hd]: q, k and v are read in place, the gradient has the same layout.
struct WindowAttentionQKV : public torch::autograd::Function<WindowAttentionQKV> {
  static std::array<Rows, 3> parts(const Tensor& qkv, const Shape& s) {
    char* p = static_cast<char*>(qkv.data_ptr());
    const int64_t row = s.hd * qkv.element_size(), stride = (s.Hq + 2 * s.Hkv) * s.hd;
    return {Rows{p, stride}, Rows{p + s.Hq * row, stride}, Rows{p + (s.Hq + s.Hkv) * row, stride}};
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv_, int64_t Hq, int64_t Hkv, int64_t window, int64_t sinks, double scale,
                        bool training) {
    c10::cuda::CUDAGuard guard(qkv_.device());
    Tensor qkv = qkv_.contiguous();
    if (reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16) qkv = qkv.clone();
    const Shape s{qkv.size(0), qkv.size(1), Hq, Hkv, qkv.size(2) / (Hq + 2 * Hkv)};
    const auto in = parts(qkv, s);
    auto [o, lse, o_lo] = window_forward(s, in[0], in[1], in[2], qkv.options(), window, sinks, scale, training);
    ctx->save_for_backward({qkv, o, lse, o_lo});
    ctx->saved_data["Hq"] = Hq;
    ctx->saved_data["Hkv"] = Hkv;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& qkv = saved[0];
    c10::cuda::CUDAGuard guard(qkv.device());
    const int64_t Hq = ctx->saved_data["Hq"].toInt(), Hkv = ctx->saved_data["Hkv"].toInt();
    const Shape s{qkv.size(0), qkv.size(1), Hq, Hkv, qkv.size(2) / (Hq + 2 * Hkv)};
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor dqkv = at::empty_like(qkv);
    const auto in = parts(qkv, s), out = parts(dqkv, s);
    window_backward(s, grads[0], in[0], in[1], in[2], saved[1], saved[2], saved[3], out[0], out[1], out[2], ctx->saved_data["window"].toInt(),
                    ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble());
    grads = first_order_only({dqkv});
    return {grads[0], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, double scale) {
  window_check(q, k, v, window, sinks, scale);
  TORCH_CHECK(q.is_cuda(), "titb200 window_attention: CUDA tensors");
  const bool training = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  return WindowAttention::apply(q, k, v, window, sinks, scale, training);
}

void qkv_check(const Tensor& qkv, int64_t Hq, int64_t Hkv) {
  TORCH_CHECK(qkv.dim() == 3 && Hq > 0 && Hkv > 0 && qkv.size(2) > 0 && qkv.size(2) % (Hq + 2 * Hkv) == 0,
              "titb200 window_attention: a projection of shape ", qkv.sizes(), " does not hold ", Hq, " + 2 * ", Hkv, " heads");
}
Tensor window_attention_qkv(const Tensor& qkv, int64_t Hq, int64_t Hkv, int64_t window, int64_t sinks, double scale) {
  qkv_check(qkv, Hq, Hkv);
  TORCH_CHECK(qkv.is_cuda(), "titb200 window_attention: CUDA tensors");
  TORCH_CHECK(Hq % Hkv == 0, "titb200 window_attention: Hq must be a multiple of Hkv");
  limits_check(qkv, qkv.size(0), qkv.size(1), Hq, qkv.size(2) / (Hq + 2 * Hkv), window, sinks, scale);
  return WindowAttentionQKV::apply(qkv, Hq, Hkv, window, sinks, scale, at::GradMode::is_enabled() && qkv.requires_grad());
}
}  // namespace

void bind_attention(pybind11::module_& m) {
  m.def("attn_fwd", &attn_fwd);
  m.def("attn_bwd", &attn_bwd, py::arg("d_o"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"), py::arg("lse"),
        py::arg("scale"), py::arg("dq") = py::none(), py::arg("dk") = py::none(), py::arg("dv") = py::none());
  m.def("window_check", &window_check);
  m.def("window_qkv_check", &qkv_check);
  m.def("window_attention", &window_attention);
  m.def("window_attention_qkv", &window_attention_qkv);
}
