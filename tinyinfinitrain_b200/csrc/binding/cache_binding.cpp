// Python bindings of the paged key-value cache: appending tokens and the attention of one new token per sequence.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "kernels/api.h"

namespace {
using at::Tensor;
using c10::optional;

void check(int rc, const char* what) {
  TORCH_CHECK(rc != TITB_ERR_SHAPE, "titb200: ", what, ": unsupported shape");
  TORCH_CHECK(rc != TITB_ERR_ALIGNMENT, "titb200: ", what, ": operands must be 16-byte aligned");
  TORCH_CHECK(rc == 0, "titb200: ", what, " failed: ", cudaGetErrorString(static_cast<cudaError_t>(rc)));
}

void forward_only(const char* what, std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t->requires_grad(), "titb200 ", what, " has no gradient: call it under torch.no_grad()");
}

// What both operators ask of the cache, on any device.
void cache_check(const char* what, const Tensor& x, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table,
                 const Tensor& per_seq, int64_t B, int64_t Hq, int64_t Hkv, int64_t hd, int64_t window, int64_t sinks) {
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(), "titb200 ", what,
              ": k_cache and v_cache must both be [pages, Hkv, page_size, head_dim]");
  TORCH_CHECK(k_cache.size(1) == Hkv && k_cache.size(3) == hd && k_cache.size(2) > 0, "titb200 ", what, ": a cache of ", Hkv,
              " heads of ", hd, " expected, got ", k_cache.sizes());
  TORCH_CHECK(k_cache.is_contiguous() && v_cache.is_contiguous(), "titb200 ", what, ": the cache must be contiguous");
  TORCH_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "titb200 ", what, ": n_head must be a multiple of n_kv_head");
  TORCH_CHECK(hd > 0 && hd <= 128 && hd % 8 == 0, "titb200 ", what, ": head_dim must be a multiple of 8 up to 128, got ", hd);
  TORCH_CHECK(table.dim() == 2 && table.size(0) == B && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1),
              "titb200 ", what, ": page_table must be an int32 [", B, ", pages of a sequence] tensor with dense rows");
  TORCH_CHECK(per_seq.dim() == 1 && per_seq.size(0) == B && per_seq.scalar_type() == at::kInt && per_seq.is_contiguous(), "titb200 ",
              what, ": positions and counts must be contiguous int32 tensors of ", B, " elements");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, "titb200 ", what,
              ": only float32 and bfloat16 tensors are supported, got ", x.scalar_type());
  TORCH_CHECK(x.scalar_type() == k_cache.scalar_type() && x.scalar_type() == v_cache.scalar_type(), "titb200 ", what,
              ": the cache must have the dtype of the new tokens");
  for (const Tensor* t : {&k_cache, &v_cache, &table, &per_seq})
    TORCH_CHECK(t->device() == x.device(), "titb200 ", what, ": all tensors must be on one device");
  TORCH_CHECK(window >= 1, "titb200 ", what, ": window must be at least 1, got ", window);
  TORCH_CHECK(sinks >= 0, "titb200 ", what, ": sinks must not be negative, got ", sinks);
  TORCH_CHECK(k_cache.size(0) < INT_MAX && k_cache.size(2) < INT_MAX && table.size(1) < INT_MAX && B < INT_MAX, "titb200 ", what,
              ": the cache is too large");
}

TitbCacheDesc cache_desc(const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, int64_t Hq, int64_t window,
                         int64_t sinks) {
  TitbCacheDesc d{};
  d.k_cache = k_cache.data_ptr(); d.v_cache = v_cache.data_ptr();
  d.page_table = table.data_ptr<int>(); d.table_stride = table.stride(0); d.table_width = (int)table.size(1);
  d.n_pages = (int)k_cache.size(0); d.page_size = (int)k_cache.size(2);
  d.B = (int)table.size(0); d.Hq = (int)Hq; d.Hkv = (int)k_cache.size(1); d.hd = (int)k_cache.size(3);
  d.window = (int)std::min<int64_t>(window, INT_MAX);
  d.sinks = (int)std::min<int64_t>(sinks, INT_MAX);
  d.dtype = k_cache.scalar_type() == at::kBFloat16 ? 1 : 0;
  return d;
}

void append_check(const Tensor& qkv, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& starts,
                  int64_t n_head, int64_t n_kv_head, double theta, const optional<Tensor>& counts, int64_t window, int64_t sinks) {
  forward_only("cache_append", {&qkv, &k_cache, &v_cache});
  TORCH_CHECK(qkv.dim() == 3, "titb200 cache_append: expects a projection [B, T, (n_head + 2 n_kv_head) * head_dim]");
  TORCH_CHECK(n_head > 0 && n_kv_head > 0 && k_cache.dim() == 4 && qkv.size(2) == (n_head + 2 * n_kv_head) * k_cache.size(3),
              "titb200 cache_append: a projection of width ", qkv.size(2), " does not hold ", n_head, " + 2 * ", n_kv_head,
              " heads of the cache's size");
  cache_check("cache_append", qkv, k_cache, v_cache, table, starts, qkv.size(0), n_head, n_kv_head, k_cache.size(3), window, sinks);
  const char *ck = static_cast<const char*>(k_cache.data_ptr()), *cv = static_cast<const char*>(v_cache.data_ptr());
  const int64_t held = k_cache.numel() * k_cache.element_size();
  TORCH_CHECK(held == 0 || ck + held <= cv || cv + held <= ck, "titb200 cache_append: k_cache and v_cache share memory");
  if (counts.has_value())
    TORCH_CHECK(counts->dim() == 1 && counts->size(0) == qkv.size(0) && counts->scalar_type() == at::kInt && counts->is_contiguous() &&
                    counts->device() == qkv.device(),
                "titb200 cache_append: counts must be a contiguous int32 tensor of ", qkv.size(0), " elements on the same device");
  TORCH_CHECK(theta >= 0.0 && std::isfinite(theta), "titb200 cache_append: theta must be positive, got ", theta);
  TORCH_CHECK(qkv.size(1) < INT_MAX, "titb200 cache_append: too many tokens");
}

// theta == 0: no rotation.  Returns q [B, T, Hq, hd], or with return_k the pair of q and k; without rotation views of qkv.
py::object cache_append(const Tensor& qkv_, Tensor& k_cache, Tensor& v_cache, const Tensor& table, const Tensor& starts,
                                 int64_t n_head, int64_t n_kv_head, double theta, const optional<Tensor>& counts, int64_t window,
                                 int64_t sinks, bool return_k) {
  TORCH_CHECK(qkv_.is_cuda(), "titb200 cache_append: CUDA tensors");
  append_check(qkv_, k_cache, v_cache, table, starts, n_head, n_kv_head, theta, counts, window, sinks);
  c10::cuda::CUDAGuard guard(qkv_.device());
  const int64_t align = 16 / qkv_.element_size();
  const bool usable = qkv_.stride(2) == 1 && qkv_.stride(0) % align == 0 && qkv_.stride(1) % align == 0 &&
                      (reinterpret_cast<uintptr_t>(qkv_.data_ptr()) % 16) == 0;
  const Tensor qkv = usable ? qkv_ : qkv_.clone(at::MemoryFormat::Contiguous);
  const int64_t B = qkv.size(0), T = qkv.size(1), hd = k_cache.size(3);
  Tensor q, k;
  if (theta > 0.0) {
    q = at::empty({B, T, n_head, hd}, qkv.options());
    if (return_k) k = at::empty({B, T, n_kv_head, hd}, qkv.options());
  }
  const TitbCacheDesc d = cache_desc(k_cache, v_cache, table, n_head, window, sinks);
  check(titb_cache_append(&d, qkv.data_ptr(), qkv.stride(0), qkv.stride(1), (int)T, starts.data_ptr<int>(),
                          counts.has_value() ? counts->data_ptr<int>() : nullptr, theta, q.defined() ? q.data_ptr() : nullptr,
                          k.defined() ? k.data_ptr() : nullptr, at::cuda::getCurrentCUDAStream().stream()),
        "cache_append");
  for (const Tensor* c : {&k_cache, &v_cache})   // so that autograd sees the write where it has kept the cache
    if (!c->is_inference()) c->unsafeGetTensorImpl()->bump_version();
  if (theta == 0.0) {
    const auto view = [&](int64_t first, int64_t heads) {
      return qkv_.as_strided({B, T, heads, hd}, {qkv_.stride(0), qkv_.stride(1), hd * qkv_.stride(2), qkv_.stride(2)},
                             qkv_.storage_offset() + first * hd * qkv_.stride(2));
    };
    q = view(0, n_head);
    if (return_k) k = view(n_head, n_kv_head);
  }
  if (return_k) return py::make_tuple(q, k);
  return py::cast(q);
}

void paged_check(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& lengths,
                 int64_t window, int64_t sinks, double scale) {
  const float scale32 = static_cast<float>(scale);   // what the kernels take
  TORCH_CHECK(scale32 > 0.f && std::isfinite(scale32), "titb200 paged_attention: scale must be positive, got ", scale);
  forward_only("paged_attention", {&q, &k_cache, &v_cache});
  TORCH_CHECK(q.dim() == 3 && k_cache.dim() == 4, "titb200 paged_attention: q [B, Hq, hd], caches [pages, Hkv, page_size, hd]");
  cache_check("paged_attention", q, k_cache, v_cache, table, lengths, q.size(0), q.size(1), k_cache.size(1), q.size(2), window,
              sinks);
}

Tensor paged_attention(const Tensor& q_, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& lengths,
                       int64_t window, int64_t sinks, double scale) {
  TORCH_CHECK(q_.is_cuda(), "titb200 paged_attention: CUDA tensors");
  paged_check(q_, k_cache, v_cache, table, lengths, window, sinks, scale);
  c10::cuda::CUDAGuard guard(q_.device());
  const int64_t align = 16 / q_.element_size();
  const bool usable = q_.stride(2) == 1 && q_.stride(1) == q_.size(2) && q_.stride(0) % align == 0 &&
                      (reinterpret_cast<uintptr_t>(q_.data_ptr()) % 16) == 0;
  const Tensor q = usable ? q_ : q_.clone(at::MemoryFormat::Contiguous);
  Tensor o = at::empty(q_.sizes(), q.options());
  const TitbCacheDesc d = cache_desc(k_cache, v_cache, table, q.size(1), window, sinks);
  const int64_t bytes = titb_paged_attention_workspace(&d);
  Tensor work;
  if (bytes > 0) work = at::empty({bytes}, q.options().dtype(at::kByte));
  check(titb_paged_attention(&d, q.data_ptr(), q.stride(0), lengths.data_ptr<int>(), (float)scale, o.data_ptr(),
                             bytes > 0 ? work.data_ptr() : nullptr, at::cuda::getCurrentCUDAStream().stream()),
        "paged_attention");
  return o;
}
}  // namespace

void bind_cache(pybind11::module_& m) {
  m.def("cache_append_check", &append_check);
  m.def("cache_append", &cache_append);
  m.def("paged_attention_check", &paged_check);
  m.def("paged_attention", &paged_attention);
}
