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
// Bound by the reads of shared memory: two 16-byte reads feed eight packed multiply-adds (70 % of what the SM can read; a layout
// with half as many distinct words a read changed nothing), and by tiles that are half masked where the window is short.
// Measured (B200), 2 x 512 tokens, 12 heads of 64, window 128, sinks 2, forward and backward of one pass: 64 x 64 tiles 230 us, 32
// rows a CTA 156, packed products 130, 32 x 32 tiles in two buffers 114 us, with the look for what is not
// finite 115 (27 + 37 + 42 us and the join of 3).
#include <cuda_runtime.h>

#include "api.h"
#include "common.cuh"
#include "window_rows.cuh"

namespace titb {

// bf16 heads of 64 and 128 (attention_tcgen05.cu)
int window_tc_fwd(const TitbAttnDesc* d, int window, int sinks, void* o_lo, cudaStream_t st);
int window_tc_bwd(const TitbAttnDesc* d, int window, int sinks, float* sink_part, const void* o_lo, cudaStream_t st);
long long window_tc_sink_floats(const TitbAttnDesc* d, int window, int sinks);

constexpr int kWinThreads = 128;   // 8 x 16 threads of 4 x 2 scores
constexpr int kWinRows = 32;       // rows of the tile that a CTA owns
constexpr int kWinStep = 32;       // rows of the other operand that arrive at a time, while those before are multiplied
constexpr int kCols = kWinStep / 16;
// Tiles are [rows][HD + 4], weights [step row][kWeightPitch]: odd numbers of 16-byte units, so that rows that neighbouring lanes
// read or write lie in different banks.
constexpr int kWeightPitch = kWinRows + 4;

struct WinArgs {
  const void *q, *k, *v, *d_o;
  void *o, *dq, *dk, *dv;
  bf16* o_lo;   // what the rounding of a bf16 o left, or null
  float *lse, *delta;
  int B, T, Hq, Hkv, hd, window, sinks;
  float scale;
  long long q_st, k_st, v_st, o_st, do_st, dq_st, dk_st, dv_st;   // elements between tokens
  // key tiles that hold sinks, the query steps that one of their CTAs takes, the CTAs of a tile, and their sums, fp32
  // [parts][B][sink_tiles][Hkv][dK, dV][kWinRows][hd]
  int sink_tiles, sink_step, sink_parts;
  float* sink_part;
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

// ROWS rows from row t0 on into shared memory.
template <typename T, int HD, int ROWS>
__device__ __forceinline__ void load_tile(const T* base, long long stride, int t0, int n_rows, int hd, float* tile) {
#pragma unroll 8
  for (int i = threadIdx.x; i < ROWS * HD / 4; i += kWinThreads) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    *reinterpret_cast<float4*>(tile + r * (HD + 4) + d) = load4(base, t0 + r, stride, d, n_rows, hd);
  }
}

// The same while the CTA computes on: fp32 rows are copied asynchronously (wait_tiles ends the wait for all but the copies that
// were issued last), bf16 rows have to be converted on their way.
template <typename T, int HD>
__device__ __forceinline__ void fetch_tile(const T* base, long long stride, int t0, int n_rows, int hd, float* tile) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll 8
    for (int i = threadIdx.x; i < kWinStep * HD / 4; i += kWinThreads) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4;
      const bool real = t0 + r < n_rows && d < hd;
      const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(tile + r * (HD + 4) + d));
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
                   "l"(base + (real ? (t0 + r) * stride + d : 0LL)), "r"(real ? 16 : 0)
                   : "memory");
    }
  } else {
    load_tile<T, HD, kWinStep>(base, stride, t0, n_rows, hd, tile);
  }
}
// 32 floats from element t0 on; zeros past the sequence.
__device__ __forceinline__ void fetch_row(const float* base, int t0, int n, float* row, int lane) {
  const bool real = t0 + lane < n;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(row + lane))),
               "l"(base + (real ? t0 + lane : 0)), "r"(real ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void commit_tiles() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_tiles() {
  asm volatile("cp.async.wait_group 1;" ::: "memory");
  __syncthreads();
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

// acc[r][c] = own row ty * 4 + r times step row tx + 16 c.  Even and odd elements of the head are summed apart, two to an
// instruction.
template <int HD>
__device__ __forceinline__ void scores(float (&acc)[4][kCols], const float* own, const float* step, int ty, int tx) {
  float even[4][kCols] = {}, odd[4][kCols] = {};
#pragma unroll 4
  for (int d = 0; d < HD; d += 4) {
    float4 a[4], b[kCols];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const float4*>(own + (ty * 4 + r) * (HD + 4) + d);
#pragma unroll
    for (int c = 0; c < kCols; ++c) b[c] = *reinterpret_cast<const float4*>(step + (tx + 16 * c) * (HD + 4) + d);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        fma2(even[r][c], odd[r][c], a[r].x, a[r].y, b[c].x, b[c].y, even[r][c], odd[r][c]);
        fma2(even[r][c], odd[r][c], a[r].z, a[r].w, b[c].z, b[c].w, even[r][c], odd[r][c]);
      }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[r][c] = even[r][c] + odd[r][c];
}
// w ([step row][own row]) <- s
__device__ __forceinline__ void store_weights(float* w, const float (&s)[4][kCols], int ty, int tx) {
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    *reinterpret_cast<float4*>(w + (tx + 16 * c) * kWeightPitch + ty * 4) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
}
// acc[r] += sum over the step's rows n of w[n][own row ty * 4 + r] times elements 64 c + 4 tx .. of row n; two rows to an
// instruction (acc[c][e][r] with e the element).
template <int HD>
__device__ __forceinline__ void accumulate(float (&acc)[HD / 64][4][4], const float* w, const float* step, int ty, int tx) {
#pragma unroll 4
  for (int n = 0; n < kWinStep; ++n) {
    const float4 a = *reinterpret_cast<const float4*>(w + n * kWeightPitch + ty * 4);
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const float4 x = *reinterpret_cast<const float4*>(step + n * (HD + 4) + c * 64 + tx * 4);
      const float xe[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float(&s)[4] = acc[c][e];
        fma2(s[0], s[1], a.x, a.y, xe[e], xe[e], s[0], s[1]);
        fma2(s[2], s[3], a.z, a.w, xe[e], xe[e], s[2], s[3]);
      }
    }
  }
}
template <typename T, int HD>
__device__ __forceinline__ void store_rows(T* base, long long stride, int t0, int n_rows, int hd, const float (&acc)[HD / 64][4][4],
                                           int ty, int tx) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (t0 + ty * 4 + r < n_rows)
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const int d = c * 64 + tx * 4;
        if (d >= hd) continue;
        Pack<T, 4> x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = from_f32<T>(acc[c][e][r]);
        *reinterpret_cast<Pack<T, 4>*>(base + (t0 + ty * 4 + r) * stride + d) = x;
      }
}

template <int HD>
__device__ __forceinline__ bool piece_finite(const float (&acc)[HD / 64][4][4], int c, int r) {
  float probe = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) probe_finite(probe, acc[c][e][r]);
  return probe == 0.f;
}

// The warp's eight rows of a tile (the first is that of its lane 0) that are not finite.
template <int HD>
__device__ __forceinline__ uint32_t bad_rows(const float (&acc)[HD / 64][4][4], int hd, int n_rows, int row, int tx) {
  uint32_t bad = 0u;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    bool mine = false;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) mine = mine || (c * 64 + tx * 4 < hd && !piece_finite<HD>(acc, c, r));
    const uint32_t votes = __ballot_sync(0xffffffffu, mine && row + r < n_rows);
    bad |= (votes & 0xffffu ? 1u << r : 0u) | (votes >> 16 ? 1u << (4 + r) : 0u);
  }
  return bad;
}

template <int HD>
struct WinFwdSmem {
  static constexpr int kTile = kWinStep * (HD + 4);   // K and V in two buffers each
  static constexpr int kQ = 0, kK = kQ + kWinRows * (HD + 4), kV = kK + 2 * kTile, kP = kV + 2 * kTile;
  static constexpr int kBytes = (kP + kWinStep * kWeightPitch) * 4;
};

// One CTA per 32 queries of a head.
template <typename T, int HD>
__global__ void __launch_bounds__(kWinThreads) window_fwd_kernel(const WinArgs p, const __grid_constant__ WinRows rows) {
  using Sm = WinFwdSmem<HD>;
  extern __shared__ __align__(16) float sm[];
  float *Qs = sm + Sm::kQ, *Ks = sm + Sm::kK, *Vs = sm + Sm::kV, *Ps = sm + Sm::kP;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int h = blockIdx.x % p.Hq, b = blockIdx.x / p.Hq, hk = h / (p.Hq / p.Hkv);
  const int q0 = (gridDim.y - 1 - blockIdx.y) * kWinRows;
  const long long row0 = static_cast<long long>(b) * p.T;
  const T* q = static_cast<const T*>(p.q) + row0 * p.q_st + h * p.hd;
  const T* k = static_cast<const T*>(p.k) + row0 * p.k_st + hk * p.hd;
  const T* v = static_cast<const T*>(p.v) + row0 * p.v_st + hk * p.hd;

  load_tile<T, HD, kWinRows>(q, p.q_st, q0, p.T, p.hd, Qs);
  float acc[HD / 64][4][4] = {};
  float m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) { m[r] = -INFINITY; l[r] = 0.f; }

  const int first = max(0, q0 - p.window + 1) / kWinStep, last = min(q0 + kWinRows, p.T) - 1;
  const int sink_steps = min((p.sinks + kWinStep - 1) / kWinStep, first);
  const int n_steps = sink_steps + last / kWinStep - first + 1;
  const auto key0 = [&](int it) { return (it < sink_steps ? it : first + it - sink_steps) * kWinStep; };
  const auto fetch = [&](int it) {
    if (it < n_steps) {
      fetch_tile<T, HD>(k, p.k_st, key0(it), p.T, p.hd, Ks + (it & 1) * Sm::kTile);
      fetch_tile<T, HD>(v, p.v_st, key0(it), p.T, p.hd, Vs + (it & 1) * Sm::kTile);
    }
    commit_tiles();
  };
  fetch(0);
  for (int it = 0; it < n_steps; ++it) {
    const int k0 = key0(it);
    fetch(it + 1);
    wait_tiles();
    float s[4][kCols];
    scores<HD>(s, Qs, Ks + (it & 1) * Sm::kTile, ty, tx);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = q0 + ty * 4 + r;
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        s[r][c] = win_visible(i, k0 + tx + 16 * c, p.window, p.sinks) ? s[r][c] * p.scale : -INFINITY;
        top = fmaxf(top, s[r][c]);
      }
      top = fmaxf(m[r], half_warp_max(top));
      const float ref = top == -INFINITY ? 0.f : top;       // a row may see nothing of its first steps
      const float keep = expf(m[r] - ref);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        s[r][c] = expf(s[r][c] - ref);
        sum += s[r][c];
      }
      l[r] = l[r] * keep + half_warp_sum(sum);
      m[r] = top;
#pragma unroll
      for (int e = 0; e < HD / 16; ++e) acc[e / 4][e % 4][r] *= keep;
    }
    store_weights(Ps, s, ty, tx);
    __syncthreads();
    accumulate<HD>(acc, Ps, Vs + (it & 1) * Sm::kTile, ty, tx);
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = q0 + ty * 4 + r;
    const float inv = 1.f / l[r];
#pragma unroll
    for (int e = 0; e < HD / 16; ++e) acc[e / 4][e % 4][r] *= inv;
    if (tx == 0 && i < p.T) p.lse[(static_cast<long long>(b) * p.Hq + h) * p.T + i] = m[r] + logf(l[r]);
  }
  store_rows<T, HD>(static_cast<T*>(p.o) + row0 * p.o_st + h * p.hd, p.o_st, q0, p.T, p.hd, acc, ty, tx);
  if (sizeof(T) == 2 && p.o_lo) {
#pragma unroll
    for (int e = 0; e < HD / 16; ++e)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[e / 4][e % 4][r] -= to_f32(from_f32<T>(acc[e / 4][e % 4][r]));
    store_rows<bf16, HD>(p.o_lo + row0 * p.o_st + h * p.hd, p.o_st, q0, p.T, p.hd, acc, ty, tx);
  }
  if (const uint32_t bad = bad_rows<HD>(acc, p.hd, p.T, q0 + ty * 4, tx)) {
    __syncwarp();   // rows and log-sum-exp are read again by other lanes
    const int i0 = q0 + static_cast<int>(threadIdx.x >> 5) * 8;
    const long long at = (row0 + i0) * p.o_st + h * p.hd;
    query_rows_again<T, false>(rows, b, h, i0, bad, static_cast<T*>(p.o) + at, p.o_st,
                               sizeof(T) == 2 && p.o_lo ? p.o_lo + at : nullptr);
  }
}

template <int HD>
struct WinDqSmem {
  static constexpr int kTile = kWinStep * (HD + 4);
  static constexpr int kQ = 0, kDO = kQ + kWinRows * (HD + 4), kK = kDO + kWinRows * (HD + 4), kV = kK + 2 * kTile, kDS = kV + 2 * kTile;
  static constexpr int kBytes = (kDS + kWinStep * kWeightPitch) * 4;
};

// One CTA per 32 queries of a head: delta, then dQ.
template <typename T, int HD>
__global__ void __launch_bounds__(kWinThreads) window_dq_kernel(const WinArgs p, const __grid_constant__ WinRows rows) {
  using Sm = WinDqSmem<HD>;
  extern __shared__ __align__(16) float sm[];
  float *Qs = sm + Sm::kQ, *Ds = sm + Sm::kDO, *Ks = sm + Sm::kK, *Vs = sm + Sm::kV, *Ss = sm + Sm::kDS;
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

  load_tile<T, HD, kWinRows>(q, p.q_st, q0, p.T, p.hd, Qs);
  load_tile<T, HD, kWinRows>(d_o, p.do_st, q0, p.T, p.hd, Ds);
  float lse[4], delta[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = q0 + ty * 4 + r;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      const float4 a = load4(d_o, i, p.do_st, c * 64 + tx * 4, p.T, p.hd);
      float4 x = load4(o, i, p.o_st, c * 64 + tx * 4, p.T, p.hd);
      if (sizeof(T) == 2 && p.o_lo) {   // added to o first: the product with an infinite dO has the sign of their sum
        const float4 y = load4(static_cast<const bf16*>(p.o_lo) + row0 * p.o_st + h * p.hd, i, p.o_st, c * 64 + tx * 4, p.T, p.hd);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      s += a.x * x.x + a.y * x.y + a.z * x.z + a.w * x.w;
    }
    delta[r] = half_warp_sum(s);
    lse[r] = i < p.T ? p.lse[stat0 + i] : 0.f;
    if (tx == 0 && i < p.T) p.delta[stat0 + i] = delta[r];
  }
  float acc[HD / 64][4][4] = {};
  const int first = max(0, q0 - p.window + 1) / kWinStep, last = min(q0 + kWinRows, p.T) - 1;
  const int sink_steps = min((p.sinks + kWinStep - 1) / kWinStep, first);
  const int n_steps = sink_steps + last / kWinStep - first + 1;
  const auto key0 = [&](int it) { return (it < sink_steps ? it : first + it - sink_steps) * kWinStep; };
  const auto fetch = [&](int it) {
    if (it < n_steps) {
      fetch_tile<T, HD>(k, p.k_st, key0(it), p.T, p.hd, Ks + (it & 1) * Sm::kTile);
      fetch_tile<T, HD>(v, p.v_st, key0(it), p.T, p.hd, Vs + (it & 1) * Sm::kTile);
    }
    commit_tiles();
  };
  fetch(0);
  for (int it = 0; it < n_steps; ++it) {
    const int k0 = key0(it);
    fetch(it + 1);
    wait_tiles();
    float s[4][kCols], dp[4][kCols];
    scores<HD>(s, Qs, Ks + (it & 1) * Sm::kTile, ty, tx);
    scores<HD>(dp, Ds, Vs + (it & 1) * Sm::kTile, ty, tx);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int i = q0 + ty * 4 + r;
        const bool see = i < p.T && win_visible(i, k0 + tx + 16 * c, p.window, p.sinks);
        s[r][c] = see ? expf(s[r][c] * p.scale - lse[r]) * (dp[r][c] - delta[r]) * p.scale : 0.f;
      }
    store_weights(Ss, s, ty, tx);
    __syncthreads();
    accumulate<HD>(acc, Ss, Ks + (it & 1) * Sm::kTile, ty, tx);
    __syncthreads();
  }
  store_rows<T, HD>(static_cast<T*>(p.dq) + row0 * p.dq_st + h * p.hd, p.dq_st, q0, p.T, p.hd, acc, ty, tx);
  if (const uint32_t bad = bad_rows<HD>(acc, p.hd, p.T, q0 + ty * 4, tx)) {
    __syncwarp();   // rows and delta are read again by other lanes
    const int i0 = q0 + static_cast<int>(threadIdx.x >> 5) * 8;
    query_rows_again<T, true>(rows, b, h, i0, bad, static_cast<T*>(p.dq) + (row0 + i0) * p.dq_st + h * p.hd, p.dq_st, nullptr);
  }
}

template <int HD>
struct WinDkvSmem {
  static constexpr int kTile = kWinStep * (HD + 4);
  static constexpr int kK = 0, kV = kK + kWinRows * (HD + 4), kQ = kV + kWinRows * (HD + 4), kDO = kQ + 2 * kTile, kP = kDO + 2 * kTile,
                       kDS = kP + kWinStep * kWeightPitch, kStat = kDS + kWinStep * kWeightPitch;   // lse and delta, two buffers
  static constexpr int kBytes = (kStat + 4 * kWinStep) * 4;
};

// One CTA per 32 keys of a kv head, over the query heads that share it; reads the delta that window_dq_kernel wrote.  The
// query steps of a tile that holds sinks reach to the end of the sequence and are split over sink_parts CTAs.
template <typename T, int HD>
__global__ void __launch_bounds__(kWinThreads) window_dkv_kernel(const WinArgs p, const __grid_constant__ WinRows rows) {
  using Sm = WinDkvSmem<HD>;
  extern __shared__ __align__(16) float sm[];
  float *Ks = sm + Sm::kK, *Vs = sm + Sm::kV, *Qs = sm + Sm::kQ, *Ds = sm + Sm::kDO, *Ps = sm + Sm::kP, *Ss = sm + Sm::kDS, *stat = sm + Sm::kStat;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int hk = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv, G = p.Hq / p.Hkv;
  const int n_sink_ctas = p.sink_tiles * p.sink_parts, y = blockIdx.y;
  const bool sink_cta = y < n_sink_ctas;
  const int part = sink_cta ? y % p.sink_parts : 0;
  const int tile = sink_cta ? y / p.sink_parts : y - n_sink_ctas + p.sink_tiles;
  const int k0 = tile * kWinRows;
  const long long row0 = static_cast<long long>(b) * p.T;
  // query steps, up to the last query that sees a key of this tile
  const long long reach = static_cast<long long>(min(k0 + kWinRows, p.T)) - 1 + p.window - 1;
  const int last = (sink_cta || reach > p.T - 1 ? p.T - 1 : static_cast<int>(reach)) / kWinStep;
  const int first = k0 / kWinStep + part * p.sink_step;
  const int n_steps = min(last - first + 1, sink_cta ? p.sink_step : last - first + 1);
  if (n_steps <= 0) return;   // a later tile has fewer parts
  load_tile<T, HD, kWinRows>(static_cast<const T*>(p.k) + row0 * p.k_st + hk * p.hd, p.k_st, k0, p.T, p.hd, Ks);
  load_tile<T, HD, kWinRows>(static_cast<const T*>(p.v) + row0 * p.v_st + hk * p.hd, p.v_st, k0, p.T, p.hd, Vs);
  float dk[HD / 64][4][4] = {}, dv[HD / 64][4][4] = {};
  const int n_all = G * n_steps;
  const auto fetch = [&](int it) {
    if (it < n_all) {
      const int h = hk * G + it / n_steps, q0 = (first + it % n_steps) * kWinStep, buf = it & 1;
      const long long stat0 = (static_cast<long long>(b) * p.Hq + h) * p.T;
      fetch_tile<T, HD>(static_cast<const T*>(p.q) + row0 * p.q_st + h * p.hd, p.q_st, q0, p.T, p.hd, Qs + buf * Sm::kTile);
      fetch_tile<T, HD>(static_cast<const T*>(p.d_o) + row0 * p.do_st + h * p.hd, p.do_st, q0, p.T, p.hd, Ds + buf * Sm::kTile);
      if (threadIdx.x < 32) fetch_row(p.lse + stat0, q0, p.T, stat + buf * 2 * kWinStep, threadIdx.x);
      else if (threadIdx.x < 64) fetch_row(p.delta + stat0, q0, p.T, stat + buf * 2 * kWinStep + kWinStep, threadIdx.x - 32);
    }
    commit_tiles();
  };
  fetch(0);
  for (int it = 0; it < n_all; ++it) {
    const int q0 = (first + it % n_steps) * kWinStep, buf = it & 1;
    fetch(it + 1);
    wait_tiles();
    float s[4][kCols], dp[4][kCols], lse[kCols], delta[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      lse[c] = stat[buf * 2 * kWinStep + tx + 16 * c];
      delta[c] = stat[buf * 2 * kWinStep + kWinStep + tx + 16 * c];
    }
    scores<HD>(s, Ks, Qs + buf * Sm::kTile, ty, tx);
    scores<HD>(dp, Vs, Ds + buf * Sm::kTile, ty, tx);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int i = q0 + tx + 16 * c, j = k0 + ty * 4 + r;
        const bool see = i < p.T && win_visible(i, j, p.window, p.sinks);
        const float prob = see ? expf(s[r][c] * p.scale - lse[c]) : 0.f;
        s[r][c] = prob;
        dp[r][c] = see ? prob * (dp[r][c] - delta[c]) * p.scale : 0.f;
      }
    store_weights(Ps, s, ty, tx);
    store_weights(Ss, dp, ty, tx);
    __syncthreads();
    accumulate<HD>(dv, Ps, Ds + buf * Sm::kTile, ty, tx);
    accumulate<HD>(dk, Ss, Qs + buf * Sm::kTile, ty, tx);
    __syncthreads();
  }
  if (part == 0) {   // holds all queries that see keys of the tile that are no sinks
    store_rows<T, HD>(static_cast<T*>(p.dk) + row0 * p.dk_st + hk * p.hd, p.dk_st, k0, p.T, p.hd, dk, ty, tx);
    store_rows<T, HD>(static_cast<T*>(p.dv) + row0 * p.dv_st + hk * p.hd, p.dv_st, k0, p.T, p.hd, dv, ty, tx);
  }
  const bool parts = sink_cta && p.sink_parts > 1;
  const long long block = ((static_cast<long long>(part) * p.B + b) * p.sink_tiles + tile) * p.Hkv + hk;
  float* sum = p.sink_part + block * 2 * kWinRows * p.hd;
  if (parts) {
    store_rows<float, HD>(sum, p.hd, 0, p.sinks - k0, p.hd, dk, ty, tx);
    store_rows<float, HD>(sum + kWinRows * p.hd, p.hd, 0, p.sinks - k0, p.hd, dv, ty, tx);
  }
  const uint32_t bad_k = bad_rows<HD>(dk, p.hd, p.T, k0 + ty * 4, tx);
  const uint32_t bad_v = bad_rows<HD>(dv, p.hd, p.T, k0 + ty * 4, tx);
  if (bad_k | bad_v) {
    __syncwarp();   // the rows are read again by other lanes
    const int r0 = static_cast<int>(threadIdx.x >> 5) * 8, j0 = k0 + r0;
    const int i0 = first * kWinStep, i1 = (first + n_steps) * kWinStep;
    const uint32_t in_part = parts ? bit_range(0, p.sinks - j0) : 0u, whole = part == 0 ? ~in_part : 0u;
    float *sum_k = sum + r0 * p.hd, *sum_v = sum + (kWinRows + r0) * p.hd;
    T* dk0 = static_cast<T*>(p.dk) + (row0 + j0) * p.dk_st + hk * p.hd;
    T* dv0 = static_cast<T*>(p.dv) + (row0 + j0) * p.dv_st + hk * p.hd;
    if (bad_k & in_part) key_rows_again<T, float, false>(rows, b, hk, j0, bad_k & in_part, i0, i1, sum_k, p.hd);
    if (bad_v & in_part) key_rows_again<T, float, true>(rows, b, hk, j0, bad_v & in_part, i0, i1, sum_v, p.hd);
    if (bad_k & whole) key_rows_again<T, T, false>(rows, b, hk, j0, bad_k & whole, i0, i1, dk0, p.dk_st);
    if (bad_v & whole) key_rows_again<T, T, true>(rows, b, hk, j0, bad_v & whole, i0, i1, dv0, p.dv_st);
  }
}

// dK and dV of the sinks: the sums of their parts, in order, over what part 0 left.
template <typename T>
__global__ void window_join_kernel(const WinArgs p) {
  const int rows = p.sinks, steps = (p.T + kWinStep - 1) / kWinStep;
  const long long n = static_cast<long long>(p.B) * rows * p.Hkv * 2 * p.hd;
  const long long part_size = static_cast<long long>(p.B) * p.sink_tiles * p.Hkv * 2 * kWinRows * p.hd;
  for (long long x = blockIdx.x * (long long)blockDim.x + threadIdx.x; x < n; x += (long long)gridDim.x * blockDim.x) {
    const int d = static_cast<int>(x % p.hd);
    long long r = x / p.hd;
    const int which = static_cast<int>(r % 2), hk = static_cast<int>(r / 2 % p.Hkv);
    r = r / 2 / p.Hkv;
    const int t = static_cast<int>(r % rows), b = static_cast<int>(r / rows), tile = t / kWinRows;
    const float* src = p.sink_part + (((static_cast<long long>(b) * p.sink_tiles + tile) * p.Hkv + hk) * 2 + which) * kWinRows * p.hd + (t % kWinRows) * p.hd + d;
    const int parts = (steps - tile * kWinRows / kWinStep + p.sink_step - 1) / p.sink_step;
    float sum = 0.f;
    for (int c = 0; c < parts; ++c) sum += src[c * part_size];
    const long long bt = static_cast<long long>(b) * p.T + t;
    T* dst = which == 0 ? static_cast<T*>(p.dk) + bt * p.dk_st : static_cast<T*>(p.dv) + bt * p.dv_st;
    dst[hk * p.hd + d] = from_f32<T>(sum);
  }
}

// Parts of a sink tile no longer than what another tile of keys takes, or than a CTA's share of all work.
struct WinSplit {
  int tiles, step, parts;
};
static WinSplit win_split(const TitbAttnDesc& d, int window, int sinks) {
  const long long steps = (d.T + kWinStep - 1) / kWinStep, near = (window + kWinRows + kWinStep - 2LL) / kWinStep + 1;
  const long long tiles = (sinks + kWinRows - 1) / kWinRows, all = (d.T + kWinRows - 1) / kWinRows;
  if (tiles == 0) return {0, 1, 1};
  const long long work = static_cast<long long>(d.Hkv) * d.B * (tiles * steps + (all - tiles) * near), share = work / (device_sm_count() * 8LL);
  const long long step = near > share ? near : share;
  return {static_cast<int>(tiles), static_cast<int>(step < steps ? step : steps), static_cast<int>((steps + step - 1) / step)};
}
static long long win_part_floats(const TitbAttnDesc& d, const WinSplit& s) {
  return s.parts > 1 ? static_cast<long long>(s.parts) * d.B * s.tiles * d.Hkv * 2 * kWinRows * d.hd : 0;
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
  a.B = d.B; a.T = d.T; a.Hq = d.Hq; a.Hkv = d.Hkv; a.hd = d.hd; a.scale = d.scale;
  a.window = window_of(w); a.sinks = sinks_of(w); a.o_lo = static_cast<bf16*>(w->o_lo);
  a.q_st = d.q_stride_t; a.k_st = d.k_stride_t; a.v_st = d.v_stride_t; a.o_st = d.o_stride_t;
  a.do_st = d.do_stride_t; a.dq_st = d.dq_stride_t; a.dk_st = d.dk_stride_t; a.dv_st = d.dv_stride_t;
  return a;
}

template <typename K>
static cudaError_t win_launch(K kernel, const WinArgs& a, const WinRows& rows, int heads, int jobs, int smem, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<dim3(static_cast<unsigned>(heads) * a.B, jobs), kWinThreads, smem, st>>>(a, rows);
  return cudaGetLastError();
}

template <typename T, int HD>
static int win_fwd(const TitbWindowDesc* w, cudaStream_t st) {
  const WinArgs a = win_args(w);
  return static_cast<int>(win_launch(window_fwd_kernel<T, HD>, a, window_rows(w->attn, a.window, a.sinks), a.Hq,
                                     (a.T + kWinRows - 1) / kWinRows, WinFwdSmem<HD>::kBytes, st));
}
template <typename T, int HD>
static int win_bwd(const TitbWindowDesc* w, cudaStream_t st) {
  WinArgs a = win_args(w);
  const WinRows rows = window_rows(w->attn, a.window, a.sinks);
  const WinSplit split = win_split(w->attn, a.window, a.sinks);
  a.sink_tiles = split.tiles; a.sink_step = split.step; a.sink_parts = split.parts;
  a.sink_part = w->workspace;
  const int tiles = (a.T + kWinRows - 1) / kWinRows;
  cudaError_t e = win_launch(window_dq_kernel<T, HD>, a, rows, a.Hq, tiles, WinDqSmem<HD>::kBytes, st);
  if (e != cudaSuccess) return static_cast<int>(e);
  e = win_launch(window_dkv_kernel<T, HD>, a, rows, a.Hkv, tiles + split.tiles * (split.parts - 1), WinDkvSmem<HD>::kBytes, st);
  if (e != cudaSuccess || split.tiles == 0 || split.parts == 1) return static_cast<int>(e);
  const long long n = win_part_floats(w->attn, split) / split.parts, most = device_sm_count() * 8LL;
  window_join_kernel<T><<<static_cast<int>((n + 255) / 256 < most ? (n + 255) / 256 : most), 256, 0, st>>>(a);
  return static_cast<int>(cudaGetLastError());
}

static int win_check(const TitbWindowDesc* w, bool backward) {
  const TitbAttnDesc& d = w->attn;
  if (d.hd <= 0 || d.hd > 128 || d.hd % 8 || d.Hkv <= 0 || d.Hq % d.Hkv || w->window < 1 || w->sinks < 0) return TITB_ERR_SHAPE;
  // grid: heads x batch along x, tiles along y
  if (static_cast<long long>(d.Hq) * d.B > 0x7fffffffLL || (d.T + kWinRows - 1LL) / kWinRows > 32767) return TITB_ERR_SHAPE;
  const int mask = w->dtype == 1 ? 7 : 3;
  auto bad = [&](const void* p, long long st) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0 || (st & mask) != 0; };
  if (reinterpret_cast<uintptr_t>(w->o_lo) & 15) return TITB_ERR_ALIGNMENT;
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
  if (on_tensor_cores(w)) return window_tc_fwd(&w->attn, window_of(w), sinks_of(w), w->o_lo, st);
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
    return window_tc_bwd(&d, window_of(w), sinks_of(w), sink_part, w->o_lo, st);
  }
  if (w->dtype == 1) return w->attn.hd <= 64 ? win_bwd<bf16, 64>(w, st) : win_bwd<bf16, 128>(w, st);
  return w->attn.hd <= 64 ? win_bwd<float, 64>(w, st) : win_bwd<float, 128>(w, st);
}

TITB_API long long titb_window_attn_bwd_workspace(const TitbWindowDesc* w) {
  const TitbAttnDesc& d = w->attn;
  if (d.B <= 0 || d.T <= 0 || d.Hq <= 0 || win_check(w, false)) return 0;
  if (!on_tensor_cores(w)) return win_part_floats(d, win_split(d, window_of(w), sinks_of(w)));
  return static_cast<long long>(d.B) * d.T * d.Hq * d.hd + window_tc_sink_floats(&d, window_of(w), sinks_of(w));
}
