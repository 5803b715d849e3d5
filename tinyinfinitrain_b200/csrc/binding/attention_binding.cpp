// Python bindings of the fused causal attention kernels.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>

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
void window_check(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "titb200 window_attention: q [B, T, Hq, hd], k and v [B, T, Hkv, hd]");
  TORCH_CHECK(k.sizes() == v.sizes(), "titb200 window_attention: k and v must have the same shape");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
              "titb200 window_attention: q and k must agree in batch, length and head_dim");
  TORCH_CHECK(k.size(2) > 0 && q.size(2) % k.size(2) == 0, "titb200 window_attention: Hq must be a multiple of Hkv");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type() && q.device() == k.device() &&
                  q.device() == v.device(), "titb200 window_attention: q, k and v must share dtype and device");
  TORCH_CHECK(window >= 1, "titb200 window_attention: window must be at least 1, got ", window);
  TORCH_CHECK(sinks >= 0, "titb200 window_attention: sinks must not be negative, got ", sinks);
  if (!q.is_cuda()) return;
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kFloat,
              "titb200 window_attention: only float32 and bfloat16 tensors are supported, got ", q.scalar_type());
  TORCH_CHECK(q.size(3) > 0 && q.size(3) <= 128 && q.size(3) % 8 == 0,
              "titb200 window_attention: head_dim must be a multiple of 8 up to 128, got ", q.size(3));
  TORCH_CHECK(q.size(1) <= 32 * 32767LL && q.size(0) * q.size(2) < (1LL << 31), "titb200 window_attention: too many tokens or heads");
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

TitbWindowDesc window_desc(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, double scale) {
  TitbWindowDesc w{};
  TitbAttnDesc& d = w.attn;
  d.q = q.data_ptr(); d.k = k.data_ptr(); d.v = v.data_ptr();
  d.B = (int)q.size(0); d.T = (int)q.size(1); d.Hq = (int)q.size(2); d.Hkv = (int)k.size(2); d.hd = (int)q.size(3);
  d.q_stride_t = token_stride(q); d.k_stride_t = token_stride(k); d.v_stride_t = token_stride(v);
  d.scale = (float)scale;
  w.window = (int)std::min<int64_t>(window, INT_MAX);
  w.sinks = (int)std::min<int64_t>(sinks, INT_MAX);
  w.dtype = q.scalar_type() == at::kBFloat16 ? 1 : 0;
  return w;
}

std::vector<Tensor> window_attn_fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t window, int64_t sinks,
                                    double scale) {
  TORCH_CHECK(q_.is_cuda(), "titb200 window_attention: CUDA tensors");
  window_check(q_, k_, v_, window, sinks);
  c10::cuda::CUDAGuard guard(q_.device());
  Tensor q = in_place_or_copy(q_), k = in_place_or_copy(k_), v = in_place_or_copy(v_);
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), hd = q.size(3);
  Tensor o = at::empty({B, T, Hq, hd}, q.options());
  Tensor lse = at::empty({B, Hq, T}, q.options().dtype(at::kFloat));
  TitbWindowDesc w = window_desc(q, k, v, window, sinks, scale);
  w.attn.o = o.data_ptr(); w.attn.lse = lse.data_ptr<float>(); w.attn.o_stride_t = Hq * hd;
  check(titb_window_attn_fwd(&w, at::cuda::getCurrentCUDAStream().stream()), "window_attention");
  return {o, lse};
}

// Gradients are written into dq / dk / dv, views of the layouts that attn_bwd takes, or into fresh tensors.
std::vector<Tensor> window_attn_bwd(const Tensor& d_o_, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& o,
                                    const Tensor& lse, int64_t window, int64_t sinks, double scale,
                                    const c10::optional<Tensor>& dq_, const c10::optional<Tensor>& dk_,
                                    const c10::optional<Tensor>& dv_) {
  window_check(q_, k_, v_, window, sinks);
  TORCH_CHECK(d_o_.sizes() == q_.sizes() && d_o_.scalar_type() == q_.scalar_type() && d_o_.device() == q_.device(),
              "titb200 window_attention: the gradient must look like the output");
  c10::cuda::CUDAGuard guard(q_.device());
  Tensor q = in_place_or_copy(q_), k = in_place_or_copy(k_), v = in_place_or_copy(v_), d_o = in_place_or_copy(d_o_);
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), hd = q.size(3), Hkv = k.size(2);
  Tensor dq = dq_.has_value() && dq_->defined() ? *dq_ : at::empty({B, T, Hq, hd}, q.options());
  Tensor dk = dk_.has_value() && dk_->defined() ? *dk_ : at::empty({B, T, Hkv, hd}, q.options());
  Tensor dv = dv_.has_value() && dv_->defined() ? *dv_ : at::empty({B, T, Hkv, hd}, q.options());
  TORCH_CHECK(addressable(dq) && addressable(dk) && addressable(dv), "titb200 window_attention: bad gradient views");
  Tensor delta = at::empty({B, Hq, T}, q.options().dtype(at::kFloat));
  TitbWindowDesc w = window_desc(q, k, v, window, sinks, scale);
  TitbAttnDesc& d = w.attn;
  d.o = o.data_ptr(); d.lse = lse.data_ptr<float>(); d.o_stride_t = token_stride(o);
  d.d_o = d_o.data_ptr(); d.dq = dq.data_ptr(); d.dk = dk.data_ptr(); d.dv = dv.data_ptr();
  d.delta = delta.data_ptr<float>();
  d.do_stride_t = token_stride(d_o); d.dq_stride_t = token_stride(dq); d.dk_stride_t = token_stride(dk); d.dv_stride_t = token_stride(dv);
  Tensor work = at::empty({titb_window_attn_bwd_workspace(&w)}, q.options().dtype(at::kFloat));
  w.workspace = work.data_ptr<float>();
  check(titb_window_attn_bwd(&w, at::cuda::getCurrentCUDAStream().stream()), "window_attention backward");
  return {dq, dk, dv};
}
}  // namespace

void bind_attention(pybind11::module_& m) {
  m.def("attn_fwd", &attn_fwd);
  m.def("attn_bwd", &attn_bwd, py::arg("d_o"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"), py::arg("lse"),
        py::arg("scale"), py::arg("dq") = py::none(), py::arg("dk") = py::none(), py::arg("dv") = py::none());
  m.def("window_check", &window_check);
  m.def("window_attn_fwd", &window_attn_fwd);
  m.def("window_attn_bwd", &window_attn_bwd, py::arg("d_o"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"),
        py::arg("lse"), py::arg("window"), py::arg("sinks"), py::arg("scale"), py::arg("dq") = py::none(),
        py::arg("dk") = py::none(), py::arg("dv") = py::none());
}
