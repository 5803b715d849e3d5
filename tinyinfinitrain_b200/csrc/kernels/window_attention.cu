// Causal attention over a window of the last positions and a few first ones (sinks), on the CUDA cores: fp32 tensors, and bf16
// tensors whose head size the tensor-core kernels (attention_tcgen05.cu) do not take.
//
//   visible(i, j) = j <= i and (i - j < window or j < sinks)
//   forward   S = scale Q K^T, O = softmax over the visible j of S times V, lse = log of the softmax's denominator
//   backward  P = exp(S - lse), dV = P^T dO, dS = P (dO V^T - delta), dQ = scale dS K, dK = scale dS^T Q, with
//             delta = rowsum(dO O)
//
// Tiles of the score matrix that hold no visible pair are not visited: a tile of queries meets the key tiles of the sinks
// and those from its first query's window to its own; a tile of keys meets the query tiles up to its last key's window, or
// all later ones when a sink lies in it.  All arithmetic is fp32.  The backward pass takes the scores twice, once per key tile
// (dK, dV) and once per query tile (delta, dQ), so that every sum has one owner and a fixed order: no atomics.
#include <cuda_runtime.h>

#include "api.h"
#include "common.cuh"

namespace titb {

// bf16 heads of 64 and 128 (attention_tcgen05.cu)
int window_tc_fwd(const TitbAttnDesc* d, int window, int sinks, cudaStream_t st);
int window_tc_bwd(const TitbAttnDesc* d, int window, int sinks, float* sink_part, cudaStream_t st);
long long window_tc_sink_floats(const TitbAttnDesc* d, int window, int sinks);

constexpr int kWinThreads = 256;   // 16 x 16 threads over a tile
constexpr int kWinRows = 64;       // rows of the tile that a CTA owns
constexpr int kWinPitch = kWinRows + 4;

struct WinArgs {
  const void *q, *k, *v, *d_o;
  void *o, *dq, *dk, *dv;
  float *lse, *delta;
  int T, Hq, Hkv, hd, window, sinks;
  float scale;
  long long q_st, k_st, v_st, o_st, do_st, dq_st, dk_st, dv_st;   // elements between tokens
};

__device__ __forceinline__ bool win_visible(int i, int j, int window, int sinks) {
  return j <= i && (i - j < window || j < sinks);
}

// Four values of row `t` of a [T, stride] matrix from column d on; zeros past the sequence and past the head.
template <typename T>
__device__ __forceinline__ float4 load4(const T* base, long long t, long long stride, int d, int n_rows, int hd) {
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (t < n_rows && d < hd) {
    const T* p = base + t * stride + d;
    if constexpr (sizeof(T) == 4) {
      r = *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
      r = make_float4(a.x, a.y, b.x, b.y);
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 r) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = r;
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(r.x, r.y), pack_bf16x2(r.z, r.w));
  }
}

// ROWS rows from row t0 on into shared memory: transposed ([HD][pitch], one row's element d at tr[d * pitch + row]) and / or
// as they are ([ROWS][HD + 4]).
template <typename T, int HD, int ROWS, bool TR, bool RM>
__device__ __forceinline__ void load_tile(const T* base, long long stride, int t0, int n_rows, int hd, float* tr, int pitch,
                                          float* rm) {
  constexpr int kVecs = HD / 4;
  for (int i = threadIdx.x; i < ROWS * kVecs; i += kWinThreads) {
    // eight lanes along the head, four rows: whole 128-byte segments of fp32 rows
    const int lane = i & 31, grp = i >> 5;
    const int d = ((grp % (kVecs / 8)) * 8 + (lane & 7)) * 4, r = (grp / (kVecs / 8)) * 4 + (lane >> 3);
    const float4 x = load4(base, t0 + r, stride, d, n_rows, hd);
    if (TR) {
      tr[d * pitch + r] = x.x;
      tr[(d + 1) * pitch + r] = x.y;
      tr[(d + 2) * pitch + r] = x.z;
      tr[(d + 3) * pitch + r] = x.w;
    }
    if (RM) *reinterpret_cast<float4*>(rm + r * (HD + 4) + d) = x;
  }
}

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ void fma4(float (&acc)[4], float a, float4 b) {
  acc[0] = fmaf(a, b.x, acc[0]);
  acc[1] = fmaf(a, b.y, acc[1]);
  acc[2] = fmaf(a, b.z, acc[2]);
  acc[3] = fmaf(a, b.w, acc[3]);
}

template <int HD>
struct WinFwdSmem {
  static constexpr int kQ = 0, kK = kQ + HD * kWinPitch, kV = kK + HD * kWinPitch, kP = kV + 64 * (HD + 4);
  static constexpr int kBytes = (kP + 64 * kWinPitch) * 4;
};

// One CTA per 64 queries of a head.  A thread holds 4 x 4 scores and 4 rows x HD / 16 columns of the output.
template <typename T, int HD>
__global__ void __launch_bounds__(kWinThreads) window_fwd_kernel(const WinArgs p) {
  using Sm = WinFwdSmem<HD>;
  extern __shared__ __align__(16) float sm[];
  float *Qt = sm + Sm::kQ, *Kt = sm + Sm::kK, *V = sm + Sm::kV, *Pt = sm + Sm::kP;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int h = blockIdx.x % p.Hq, b = blockIdx.x / p.Hq, hk = h / (p.Hq / p.Hkv);
  const int q0 = (gridDim.y - 1 - blockIdx.y) * kWinRows;
  const long long row0 = static_cast<long long>(b) * p.T;
  const T* q = static_cast<const T*>(p.q) + row0 * p.q_st + h * p.hd;
  const T* k = static_cast<const T*>(p.k) + row0 * p.k_st + hk * p.hd;
  const T* v = static_cast<const T*>(p.v) + row0 * p.v_st + hk * p.hd;

  load_tile<T, HD, kWinRows, true, false>(q, p.q_st, q0, p.T, p.hd, Qt, kWinPitch, nullptr);
  float acc[4][HD / 16] = {};
  float m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) { m[r] = -INFINITY; l[r] = 0.f; }

  const int first = max(0, q0 - p.window + 1) / 64, last = min(q0 + kWinRows, p.T) - 1;
  const int sink_tiles = min((p.sinks + 63) / 64, first);
  const int n_tiles = sink_tiles + last / 64 - first + 1;
  for (int it = 0; it < n_tiles; ++it) {
    const int k0 = (it < sink_tiles ? it : first + it - sink_tiles) * 64;
    __syncthreads();
    load_tile<T, HD, 64, true, false>(k, p.k_st, k0, p.T, p.hd, Kt, kWinPitch, nullptr);
    load_tile<T, HD, 64, false, true>(v, p.v_st, k0, p.T, p.hd, nullptr, 0, V);
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 8
    for (int d = 0; d < HD; ++d) {
      const float4 a = *reinterpret_cast<const float4*>(Qt + d * kWinPitch + ty * 4);
      const float4 c = *reinterpret_cast<const float4*>(Kt + d * kWinPitch + tx * 4);
      fma4(s[0], a.x, c); fma4(s[1], a.y, c); fma4(s[2], a.z, c); fma4(s[3], a.w, c);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = q0 + ty * 4 + r;
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = win_visible(i, k0 + tx * 4 + c, p.window, p.sinks) ? s[r][c] * p.scale : -INFINITY;
        top = fmaxf(top, s[r][c]);
      }
      top = fmaxf(m[r], half_warp_max(top));
      const float ref = top == -INFINITY ? 0.f : top;       // a row may see nothing of its first tiles
      const float keep = expf(m[r] - ref);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = expf(s[r][c] - ref);
        sum += s[r][c];
      }
      l[r] = l[r] * keep + half_warp_sum(sum);
      m[r] = top;
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) acc[r][c] *= keep;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<float4*>(Pt + (tx * 4 + c) * kWinPitch + ty * 4) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
    __syncthreads();
#pragma unroll 4
    for (int n = 0; n < 64; ++n) {
      const float4 a = *reinterpret_cast<const float4*>(Pt + n * kWinPitch + ty * 4);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const float4 x = *reinterpret_cast<const float4*>(V + n * (HD + 4) + c * 64 + tx * 4);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[0][c * 4]), a.x, x);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[1][c * 4]), a.y, x);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[2][c * 4]), a.z, x);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[3][c * 4]), a.w, x);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = q0 + ty * 4 + r;
    if (i >= p.T) continue;
    const float inv = 1.f / l[r];
    T* o = static_cast<T*>(p.o) + (row0 + i) * p.o_st + h * p.hd;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const int d = c * 64 + tx * 4;
      if (d < p.hd)
        store4(o + d, make_float4(acc[r][c * 4] * inv, acc[r][c * 4 + 1] * inv, acc[r][c * 4 + 2] * inv, acc[r][c * 4 + 3] * inv));
    }
    if (tx == 0) p.lse[(static_cast<long long>(b) * p.Hq + h) * p.T + i] = m[r] + logf(l[r]);
  }
}

// The other operand's rows arrive 32 at a time in the backward kernels.
constexpr int kWinStep = 32;
constexpr int kWinStepPitch = kWinStep + 4;

template <int HD>
struct WinDqSmem {
  static constexpr int kQ = 0, kDO = kQ + HD * kWinPitch, kK = kDO + HD * kWinPitch, kV = kK + HD * kWinStepPitch,
                       kKr = kV + HD * kWinStepPitch, kDS = kKr + kWinStep * (HD + 4);
  static constexpr int kBytes = (kDS + kWinStep * kWinPitch) * 4;
};

// One CTA per 64 queries of a head: delta, then dQ.
template <typename T, int HD>
__global__ void __launch_bounds__(kWinThreads) window_dq_kernel(const WinArgs p) {
  using Sm = WinDqSmem<HD>;
  extern __shared__ __align__(16) float sm[];
  float *Qt = sm + Sm::kQ, *Dt = sm + Sm::kDO, *Kt = sm + Sm::kK, *Vt = sm + Sm::kV, *Kr = sm + Sm::kKr, *St = sm + Sm::kDS;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int h = blockIdx.x % p.Hq, b = blockIdx.x / p.Hq, hk = h / (p.Hq / p.Hkv);
  const int q0 = (gridDim.y - 1 - blockIdx.y) * kWinRows;
  const long long row0 = static_cast<long long>(b) * p.T;
  const T* q = static_cast<const T*>(p.q) + row0 * p.q_st + h * p.hd;
  const T* k = static_cast<const T*>(p.k) + row0 * p.k_st + hk * p.hd;
  const T* v = static_cast<const T*>(p.v) + row0 * p.v_st + hk * p.hd;
  const T* d_o = static_cast<const T*>(p.d_o) + row0 * p.do_st + h * p.hd;
  const T* o = static_cast<const T*>(p.o) + row0 * p.o_st + h * p.hd;
  const long long stat0 = (static_cast<long long>(b) * p.Hq + h) * p.T;

  load_tile<T, HD, kWinRows, true, false>(q, p.q_st, q0, p.T, p.hd, Qt, kWinPitch, nullptr);
  load_tile<T, HD, kWinRows, true, false>(d_o, p.do_st, q0, p.T, p.hd, Dt, kWinPitch, nullptr);
  float lse[4], delta[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = q0 + ty * 4 + r;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const float4 a = load4(d_o, i, p.do_st, c * 64 + tx * 4, p.T, p.hd), x = load4(o, i, p.o_st, c * 64 + tx * 4, p.T, p.hd);
      s += a.x * x.x + a.y * x.y + a.z * x.z + a.w * x.w;
    }
    delta[r] = half_warp_sum(s);
    lse[r] = i < p.T ? p.lse[stat0 + i] : 0.f;
    if (tx == 0 && i < p.T) p.delta[stat0 + i] = delta[r];
  }
  float acc[4][HD / 16] = {};
  const int first = max(0, q0 - p.window + 1) / kWinStep, last = min(q0 + kWinRows, p.T) - 1;
  const int sink_tiles = min((p.sinks + kWinStep - 1) / kWinStep, first);
  const int n_tiles = sink_tiles + last / kWinStep - first + 1;
  for (int it = 0; it < n_tiles; ++it) {
    const int k0 = (it < sink_tiles ? it : first + it - sink_tiles) * kWinStep;
    __syncthreads();
    load_tile<T, HD, kWinStep, true, true>(k, p.k_st, k0, p.T, p.hd, Kt, kWinStepPitch, Kr);
    load_tile<T, HD, kWinStep, true, false>(v, p.v_st, k0, p.T, p.hd, Vt, kWinStepPitch, nullptr);
    __syncthreads();
    float s[4][2] = {}, dp[4][2] = {};
#pragma unroll 8
    for (int d = 0; d < HD; ++d) {
      const float4 a = *reinterpret_cast<const float4*>(Qt + d * kWinPitch + ty * 4);
      const float4 g = *reinterpret_cast<const float4*>(Dt + d * kWinPitch + ty * 4);
      const float2 x = *reinterpret_cast<const float2*>(Kt + d * kWinStepPitch + tx * 2);
      const float2 y = *reinterpret_cast<const float2*>(Vt + d * kWinStepPitch + tx * 2);
      const float ar[4] = {a.x, a.y, a.z, a.w}, gr[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[r][0] = fmaf(ar[r], x.x, s[r][0]);
        s[r][1] = fmaf(ar[r], x.y, s[r][1]);
        dp[r][0] = fmaf(gr[r], y.x, dp[r][0]);
        dp[r][1] = fmaf(gr[r], y.y, dp[r][1]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = q0 + ty * 4 + r;
        const bool see = i < p.T && win_visible(i, k0 + tx * 2 + c, p.window, p.sinks);
        s[r][c] = see ? expf(s[r][c] * p.scale - lse[r]) * (dp[r][c] - delta[r]) * p.scale : 0.f;
      }
#pragma unroll
    for (int c = 0; c < 2; ++c)
      *reinterpret_cast<float4*>(St + (tx * 2 + c) * kWinPitch + ty * 4) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
    __syncthreads();
#pragma unroll 4
    for (int n = 0; n < kWinStep; ++n) {
      const float4 a = *reinterpret_cast<const float4*>(St + n * kWinPitch + ty * 4);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const float4 x = *reinterpret_cast<const float4*>(Kr + n * (HD + 4) + c * 64 + tx * 4);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[0][c * 4]), a.x, x);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[1][c * 4]), a.y, x);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[2][c * 4]), a.z, x);
        fma4(*reinterpret_cast<float(*)[4]>(&acc[3][c * 4]), a.w, x);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = q0 + ty * 4 + r;
    if (i >= p.T) continue;
    T* dq = static_cast<T*>(p.dq) + (row0 + i) * p.dq_st + h * p.hd;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const int d = c * 64 + tx * 4;
      if (d < p.hd) store4(dq + d, make_float4(acc[r][c * 4], acc[r][c * 4 + 1], acc[r][c * 4 + 2], acc[r][c * 4 + 3]));
    }
  }
}

template <int HD>
struct WinDkvSmem {
  static constexpr int kK = 0, kV = kK + HD * kWinPitch, kQ = kV + HD * kWinPitch, kDO = kQ + HD * kWinStepPitch,
                       kQr = kDO + HD * kWinStepPitch, kDr = kQr + kWinStep * (HD + 4), kP = kDr + kWinStep * (HD + 4),
                       kDS = kP + kWinStep * kWinPitch;
  static constexpr int kBytes = (kDS + kWinStep * kWinPitch) * 4;
};

// One CTA per 64 keys of a kv head, over the query heads that share it; reads the delta that window_dq_kernel wrote.
template <typename T, int HD>
__global__ void __launch_bounds__(kWinThreads) window_dkv_kernel(const WinArgs p) {
  using Sm = WinDkvSmem<HD>;
  extern __shared__ __align__(16) float sm[];
  float *Kt = sm + Sm::kK, *Vt = sm + Sm::kV, *Qt = sm + Sm::kQ, *Dt = sm + Sm::kDO, *Qr = sm + Sm::kQr, *Dr = sm + Sm::kDr,
        *Pt = sm + Sm::kP, *St = sm + Sm::kDS;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int hk = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv, G = p.Hq / p.Hkv;
  const int k0 = blockIdx.y * kWinRows;
  const long long row0 = static_cast<long long>(b) * p.T;
  load_tile<T, HD, kWinRows, true, false>(static_cast<const T*>(p.k) + row0 * p.k_st + hk * p.hd, p.k_st, k0, p.T, p.hd, Kt,
                                          kWinPitch, nullptr);
  load_tile<T, HD, kWinRows, true, false>(static_cast<const T*>(p.v) + row0 * p.v_st + hk * p.hd, p.v_st, k0, p.T, p.hd, Vt,
                                          kWinPitch, nullptr);
  float dk[4][HD / 16] = {}, dv[4][HD / 16] = {};
  // the last query that sees a key of this tile
  const long long reach = static_cast<long long>(min(k0 + kWinRows, p.T)) - 1 + p.window - 1;
  const int last = k0 < p.sinks || reach > p.T - 1 ? p.T - 1 : static_cast<int>(reach);
  const int first = k0 / kWinStep, n_steps = last / kWinStep - first + 1;
  for (int it = 0; it < G * n_steps; ++it) {
    const int h = hk * G + it / n_steps, q0 = (first + it % n_steps) * kWinStep;
    const long long stat0 = (static_cast<long long>(b) * p.Hq + h) * p.T;
    __syncthreads();
    load_tile<T, HD, kWinStep, true, true>(static_cast<const T*>(p.q) + row0 * p.q_st + h * p.hd, p.q_st, q0, p.T, p.hd, Qt,
                                           kWinStepPitch, Qr);
    load_tile<T, HD, kWinStep, true, true>(static_cast<const T*>(p.d_o) + row0 * p.do_st + h * p.hd, p.do_st, q0, p.T, p.hd, Dt,
                                           kWinStepPitch, Dr);
    float lse[2], delta[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i = q0 + tx * 2 + c;
      lse[c] = i < p.T ? p.lse[stat0 + i] : 0.f;
      delta[c] = i < p.T ? p.delta[stat0 + i] : 0.f;
    }
    __syncthreads();
    float s[4][2] = {}, dp[4][2] = {};
#pragma unroll 8
    for (int d = 0; d < HD; ++d) {
      const float4 a = *reinterpret_cast<const float4*>(Kt + d * kWinPitch + ty * 4);
      const float4 g = *reinterpret_cast<const float4*>(Vt + d * kWinPitch + ty * 4);
      const float2 x = *reinterpret_cast<const float2*>(Qt + d * kWinStepPitch + tx * 2);
      const float2 y = *reinterpret_cast<const float2*>(Dt + d * kWinStepPitch + tx * 2);
      const float ar[4] = {a.x, a.y, a.z, a.w}, gr[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[r][0] = fmaf(ar[r], x.x, s[r][0]);
        s[r][1] = fmaf(ar[r], x.y, s[r][1]);
        dp[r][0] = fmaf(gr[r], y.x, dp[r][0]);
        dp[r][1] = fmaf(gr[r], y.y, dp[r][1]);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = q0 + tx * 2 + c, j = k0 + ty * 4 + r;
        const bool see = i < p.T && win_visible(i, j, p.window, p.sinks);
        const float prob = see ? expf(s[r][c] * p.scale - lse[c]) : 0.f;
        s[r][c] = prob;
        dp[r][c] = see ? prob * (dp[r][c] - delta[c]) * p.scale : 0.f;
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      *reinterpret_cast<float4*>(Pt + (tx * 2 + c) * kWinPitch + ty * 4) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
      *reinterpret_cast<float4*>(St + (tx * 2 + c) * kWinPitch + ty * 4) = make_float4(dp[0][c], dp[1][c], dp[2][c], dp[3][c]);
    }
    __syncthreads();
#pragma unroll 2
    for (int n = 0; n < kWinStep; ++n) {
      const float4 a = *reinterpret_cast<const float4*>(Pt + n * kWinPitch + ty * 4);
      const float4 g = *reinterpret_cast<const float4*>(St + n * kWinPitch + ty * 4);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const float4 x = *reinterpret_cast<const float4*>(Dr + n * (HD + 4) + c * 64 + tx * 4);
        const float4 y = *reinterpret_cast<const float4*>(Qr + n * (HD + 4) + c * 64 + tx * 4);
        fma4(*reinterpret_cast<float(*)[4]>(&dv[0][c * 4]), a.x, x);
        fma4(*reinterpret_cast<float(*)[4]>(&dv[1][c * 4]), a.y, x);
        fma4(*reinterpret_cast<float(*)[4]>(&dv[2][c * 4]), a.z, x);
        fma4(*reinterpret_cast<float(*)[4]>(&dv[3][c * 4]), a.w, x);
        fma4(*reinterpret_cast<float(*)[4]>(&dk[0][c * 4]), g.x, y);
        fma4(*reinterpret_cast<float(*)[4]>(&dk[1][c * 4]), g.y, y);
        fma4(*reinterpret_cast<float(*)[4]>(&dk[2][c * 4]), g.z, y);
        fma4(*reinterpret_cast<float(*)[4]>(&dk[3][c * 4]), g.w, y);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = k0 + ty * 4 + r;
    if (j >= p.T) continue;
    T* ok = static_cast<T*>(p.dk) + (row0 + j) * p.dk_st + hk * p.hd;
    T* ov = static_cast<T*>(p.dv) + (row0 + j) * p.dv_st + hk * p.hd;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const int d = c * 64 + tx * 4;
      if (d < p.hd) {
        store4(ok + d, make_float4(dk[r][c * 4], dk[r][c * 4 + 1], dk[r][c * 4 + 2], dk[r][c * 4 + 3]));
        store4(ov + d, make_float4(dv[r][c * 4], dv[r][c * 4 + 1], dv[r][c * 4 + 2], dv[r][c * 4 + 3]));
      }
    }
  }
}

// more than the sequence changes nothing
static int window_of(const TitbWindowDesc* w) { return w->window < w->attn.T ? w->window : w->attn.T; }
static int sinks_of(const TitbWindowDesc* w) { return w->sinks < w->attn.T ? w->sinks : w->attn.T; }
static bool on_tensor_cores(const TitbWindowDesc* w) { return w->dtype == 1 && (w->attn.hd == 64 || w->attn.hd == 128); }

static WinArgs win_args(const TitbWindowDesc* w) {
  const TitbAttnDesc& d = w->attn;
  WinArgs a{};
  a.q = d.q; a.k = d.k; a.v = d.v; a.o = d.o; a.lse = d.lse;
  a.d_o = d.d_o; a.dq = d.dq; a.dk = d.dk; a.dv = d.dv; a.delta = d.delta;
  a.T = d.T; a.Hq = d.Hq; a.Hkv = d.Hkv; a.hd = d.hd; a.scale = d.scale;
  a.window = window_of(w); a.sinks = sinks_of(w);
  a.q_st = d.q_stride_t; a.k_st = d.k_stride_t; a.v_st = d.v_stride_t; a.o_st = d.o_stride_t;
  a.do_st = d.do_stride_t; a.dq_st = d.dq_stride_t; a.dk_st = d.dk_stride_t; a.dv_st = d.dv_stride_t;
  return a;
}

template <typename K>
static cudaError_t win_launch(K kernel, const WinArgs& a, int heads, int B, int smem, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>(heads) * B, (a.T + kWinRows - 1) / kWinRows);
  kernel<<<grid, kWinThreads, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int HD>
static int win_fwd(const TitbWindowDesc* w, cudaStream_t st) {
  return static_cast<int>(win_launch(window_fwd_kernel<T, HD>, win_args(w), w->attn.Hq, w->attn.B, WinFwdSmem<HD>::kBytes, st));
}
template <typename T, int HD>
static int win_bwd(const TitbWindowDesc* w, cudaStream_t st) {
  const WinArgs a = win_args(w);
  const cudaError_t e = win_launch(window_dq_kernel<T, HD>, a, w->attn.Hq, w->attn.B, WinDqSmem<HD>::kBytes, st);
  if (e != cudaSuccess) return static_cast<int>(e);
  return static_cast<int>(win_launch(window_dkv_kernel<T, HD>, a, w->attn.Hkv, w->attn.B, WinDkvSmem<HD>::kBytes, st));
}

static int win_check(const TitbWindowDesc* w, bool backward) {
  const TitbAttnDesc& d = w->attn;
  if (d.hd <= 0 || d.hd > 128 || d.hd % 8 || d.Hkv <= 0 || d.Hq % d.Hkv || w->window < 1 || w->sinks < 0) return TITB_ERR_SHAPE;
  // grid: heads x batch along x, tiles along y
  if (static_cast<long long>(d.Hq) * d.B > 0x7fffffffLL || (d.T + kWinRows - 1LL) / kWinRows > 65535) return TITB_ERR_SHAPE;
  const int mask = w->dtype == 1 ? 7 : 3;
  auto bad = [&](const void* p, long long st) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0 || (st & mask) != 0; };
  if (bad(d.q, d.q_stride_t) || bad(d.k, d.k_stride_t) || bad(d.v, d.v_stride_t) || bad(d.o, d.o_stride_t))
    return TITB_ERR_ALIGNMENT;
  if (backward && (bad(d.d_o, d.do_stride_t) || bad(d.dq, d.dq_stride_t) || bad(d.dk, d.dk_stride_t) || bad(d.dv, d.dv_stride_t)))
    return TITB_ERR_ALIGNMENT;
  return 0;
}

}  // namespace titb

using namespace titb;

TITB_API int titb_window_attn_fwd(const TitbWindowDesc* w, cudaStream_t st) {
  (void)cudaGetLastError();
  if (w->attn.B <= 0 || w->attn.T <= 0 || w->attn.Hq <= 0) return 0;
  if (const int rc = win_check(w, false)) return rc;
  if (on_tensor_cores(w)) return window_tc_fwd(&w->attn, window_of(w), sinks_of(w), st);
  if (w->dtype == 1) return w->attn.hd <= 64 ? win_fwd<bf16, 64>(w, st) : win_fwd<bf16, 128>(w, st);
  return w->attn.hd <= 64 ? win_fwd<float, 64>(w, st) : win_fwd<float, 128>(w, st);
}

TITB_API int titb_window_attn_bwd(const TitbWindowDesc* w, cudaStream_t st) {
  (void)cudaGetLastError();
  if (w->attn.B <= 0 || w->attn.T <= 0 || w->attn.Hq <= 0) return 0;
  if (const int rc = win_check(w, true)) return rc;
  if (on_tensor_cores(w)) {
    TitbAttnDesc d = w->attn;
    d.dq_accum = w->workspace;
    float* sink_part = w->workspace + static_cast<long long>(d.B) * d.T * d.Hq * d.hd;
    return window_tc_bwd(&d, window_of(w), sinks_of(w), sink_part, st);
  }
  if (w->dtype == 1) return w->attn.hd <= 64 ? win_bwd<bf16, 64>(w, st) : win_bwd<bf16, 128>(w, st);
  return w->attn.hd <= 64 ? win_bwd<float, 64>(w, st) : win_bwd<float, 128>(w, st);
}

TITB_API long long titb_window_attn_bwd_workspace(const TitbWindowDesc* w) {
  const TitbAttnDesc& d = w->attn;
  if (d.B <= 0 || d.T <= 0 || d.Hq <= 0 || win_check(w, false) || !on_tensor_cores(w)) return 0;
  return static_cast<long long>(d.B) * d.T * d.Hq * d.hd + window_tc_sink_floats(&d, window_of(w), sinks_of(w));
}
