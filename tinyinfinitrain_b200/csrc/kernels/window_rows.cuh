// Window attention, some elements of one row at a time and over its visible pairs only.
//
// Inside a tile a pair that is masked has a probability of zero, but its values still take part in the products, and zero times
// NaN or infinity is NaN.  So the kernels look at what they are about to store, and elements that are not finite are taken
// again here, where masked pairs do not appear.  That costs nothing as long as all inputs are finite.  What is not finite by
// right (a visible NaN) stays so: a score that is NaN ends the row at once, so a step that has diverged does not crawl.
#pragma once
#include "api.h"
#include "common.cuh"

namespace titb {

struct WinRows {
  const void *q, *k, *v, *d_o;
  long long q_st, k_st, v_st, do_st;   // elements between tokens
  const float *lse, *delta;            // [B, Hq, T]
  int T, Hq, Hkv, hd, window, sinks;
  float scale;
  template <typename T_>
  __device__ const T_* row(const void* base, long long stride, int b, int t, int h) const {
    return static_cast<const T_*>(base) + (static_cast<long long>(b) * T + t) * stride + static_cast<long long>(h) * hd;
  }
  __device__ long long stat(int b, int h, int t) const { return (static_cast<long long>(b) * Hq + h) * T + t; }
};

inline WinRows window_rows(const TitbAttnDesc& d, int window, int sinks) {
  return {d.q, d.k, d.v, d.d_o, d.q_stride_t, d.k_stride_t, d.v_stride_t, d.do_stride_t, d.lse, d.delta, d.T, d.Hq, d.Hkv, d.hd,
          window, sinks, d.scale};
}

// 0 while everything that was put in is finite, else NaN.
__device__ __forceinline__ void probe_finite(float& probe, float x) { probe = fmaf(x, 0.f, probe); }
__device__ __forceinline__ void probe_finite(uint32_t& probe, uint32_t bf16x2) {
  asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(probe) : "r"(bf16x2), "r"(0u));
}

// The rows start on 16 bytes and n is a multiple of 8.
template <typename T>
__device__ inline float row_dot(const T* a, const T* b, int n) {
  constexpr int V = 16 / sizeof(T);
  float s = 0.f;
#pragma unroll 2
  for (int i = 0; i < n; i += V) {
    const uint4 ua = *reinterpret_cast<const uint4*>(a + i), ub = *reinterpret_cast<const uint4*>(b + i);
    const T *x = reinterpret_cast<const T*>(&ua), *y = reinterpret_cast<const T*>(&ub);
#pragma unroll
    for (int e = 0; e < V; ++e) s = fmaf(to_f32(x[e]), to_f32(y[e]), s);
  }
  return s;
}
template <typename T, int N>
__device__ inline void row_store(T* out, const float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = from_f32<T>(x[e]);
}

// Elements [d0, d0 + N) of output row i; `lo` (may be null) receives what their rounding left.
template <typename T, int N>
__device__ __forceinline__ void window_o_again(const WinRows& w, int b, int h, int i, float lse, int d0, T* out, bf16* lo) {
  const int hk = h / (w.Hq / w.Hkv), first = max(0, i - w.window + 1);
  const T* q = w.row<T>(w.q, w.q_st, b, i, h);
  float acc[N] = {};
#pragma unroll 1
  for (int j = min(w.sinks, first) > 0 ? 0 : first; j <= i; j = j + 1 == min(w.sinks, first) ? first : j + 1) {
    const float s = row_dot(q, w.row<T>(w.k, w.k_st, b, j, hk), w.hd), p = expf(s * w.scale - lse);
    const T* v = w.row<T>(w.v, w.v_st, b, j, hk) + d0;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = fmaf(p, to_f32(v[e]), acc[e]);
    if (p != p) break;
  }
  row_store(out, acc);
  if (lo) {
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] -= to_f32(from_f32<T>(acc[e]));
    row_store(lo, acc);
  }
}

// Elements [d0, d0 + N) of dQ's row i.
template <typename T, int N>
__device__ __noinline__ void window_dq_again(const WinRows& w, int b, int h, int i, int d0, T* out) {
  const int hk = h / (w.Hq / w.Hkv), first = max(0, i - w.window + 1);
  const T *q = w.row<T>(w.q, w.q_st, b, i, h), *g = w.row<T>(w.d_o, w.do_st, b, i, h);
  const float lse = w.lse[w.stat(b, h, i)], delta = w.delta[w.stat(b, h, i)];
  float acc[N] = {};
  for (int j = min(w.sinks, first) > 0 ? 0 : first; j <= i; j = j + 1 == min(w.sinks, first) ? first : j + 1) {
    const T* k = w.row<T>(w.k, w.k_st, b, j, hk);
    const float s = row_dot(q, k, w.hd), p = expf(s * w.scale - lse);
    const float ds = p * (row_dot(g, w.row<T>(w.v, w.v_st, b, j, hk), w.hd) - delta) * w.scale;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = fmaf(ds, to_f32(k[d0 + e]), acc[e]);
    if (ds != ds) break;
  }
  row_store(out, acc);
}

// Elements [d0, d0 + N) of row j of dK (or dV), from queries [i0, i1).
template <typename T, typename Out, int N>
__device__ __noinline__ void window_dkv_again(const WinRows& w, int b, int hk, int j, int i0, int i1, bool value, int d0, Out* out) {
  const int G = w.Hq / w.Hkv;
  const T *k = w.row<T>(w.k, w.k_st, b, j, hk), *v = w.row<T>(w.v, w.v_st, b, j, hk);
  const long long reach = static_cast<long long>(j) + w.window;
  i0 = max(i0, j);
  i1 = min(i1, w.T);
  if (j >= w.sinks && reach < i1) i1 = static_cast<int>(reach);
  float acc[N] = {};
  for (int h = hk * G; h < hk * G + G; ++h)
    for (int i = i0; i < i1; ++i) {
      const T *q = w.row<T>(w.q, w.q_st, b, i, h), *g = w.row<T>(w.d_o, w.do_st, b, i, h);
      float f = expf(row_dot(q, k, w.hd) * w.scale - w.lse[w.stat(b, h, i)]);
      if (!value) f *= (row_dot(g, v, w.hd) - w.delta[w.stat(b, h, i)]) * w.scale;
      const T* x = (value ? g : q) + d0;
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] = fmaf(f, to_f32(x[e]), acc[e]);
      if (f != f) {
        row_store(out, acc);
        return;
      }
    }
  row_store(out, acc);
}

}  // namespace titb
