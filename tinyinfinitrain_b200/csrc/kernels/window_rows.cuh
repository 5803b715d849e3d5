// Window attention, the rows that came out not finite, over their visible pairs only.
//
// Inside a tile a pair that is masked has a probability of zero, but its values still take part in the products, and
// zero times NaN or infinity is NaN.  So the kernels look at what they store, and a warp takes rows that are not finite
// again here, where masked pairs do not appear.
//
// Every output is a sum over pairs of a weight f (one number a pair) times a vector x that all rows of a warp share:
//   O  = sum_j P_ij V_j      dQ = sum_j dS_ij K_j      dV = sum_i P_ij dO_i      dK = sum_i dS_ij Q_i
// What is not finite by right is told from the few terms that are not, without the products of the others:
//   - a log-sum-exp that is not finite means undefined probabilities: the row, and the keys that it sees, are NaN;
//   - a finite score has a positive weight, so an infinity of V or dO is an infinity of the sum (NaN where both signs
//     meet, or a score of -inf has weight zero), and a K that is not finite beside a finite log-sum-exp has a score of
//     -inf: zero times K;
//   - an infinite delta makes dS infinite or NaN for the whole row.
// Finding them takes one pass over the vectors for 32 rows, which ends when nothing can be added.  Only columns that
// are finite by right are summed again: those that a masked neighbour within the tiles' borders has spoilt, and sums
// that overflow on their way; two neighbours at a time, a lane holding columns, so that vectors are read whole and once for
// both.
// Measured (B200), 1 x 1024, 8 / 2 heads of 64 and 128, window 256 or none, forward and backward: 0.13 ms when all is
// finite, 0.2 ms with all gradients or values NaN, 0.2 to 5 ms with single infinities or NaN rows.  As a thread's work,
// 16 columns at a time and without an end but at an undefined weight, 30 to 110 ms.  Asking for the next vectors under
// the sums of those at hand was slower: the registers are those that the tile kernels leave.
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
  __device__ bool visible(int i, int j) const { return j <= i && (i - j < window || j < sinks); }
  // the last query that sees key j
  __device__ int last_query(int j) const {
    const long long reach = static_cast<long long>(j) + window - 1;
    return j < sinks || reach > T - 1 ? T - 1 : static_cast<int>(reach);
  }
};

inline WinRows window_rows(const TitbAttnDesc& d, int window, int sinks) {
  return {d.q,   d.k,     d.v, d.d_o, d.q_stride_t, d.k_stride_t, d.v_stride_t, d.do_stride_t,
          d.lse, d.delta, d.T, d.Hq,  d.Hkv,        d.hd,         window,       sinks,         d.scale};
}

// 0 while everything that was put in is finite, else NaN.
__device__ __forceinline__ void probe_finite(float& probe, float x) { probe = fmaf(x, 0.f, probe); }
__device__ __forceinline__ void probe_finite(uint32_t& probe, uint32_t bf16x2) {
  asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(probe) : "r"(bf16x2), "r"(0u));
}

// Bits [lo, hi) of a 32-bit word; lo and hi may lie outside it.
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi <= lo ? 0u : (0xffffffffu >> (32 - (hi - lo))) << lo;
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

// Columns of a row of up to 128 elements, two neighbours and two 64 further on to a lane; a set of columns is a bit per
// lane in four words.
constexpr int kRowWords = 4;
__device__ __forceinline__ int column_of(int e, int lane) { return (e >> 1) * 64 + lane * 2 + (e & 1); }
// word e of the set of a whole row's
__device__ __forceinline__ uint32_t columns_of(int e, int hd) { return bit_range(0, (hd - (e >> 1) * 64) / 2); }
template <typename T>
struct RowPart {
  Pack<T, 2> half[2];
  __device__ __forceinline__ void load(const T* row, int hd, int lane) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      half[c].v[0] = half[c].v[1] = from_f32<T>(0.f);
      if (c * 64 + lane * 2 < hd) half[c] = *reinterpret_cast<const Pack<T, 2>*>(row + c * 64 + lane * 2);
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return to_f32(half[e >> 1].v[e & 1]); }
};
template <typename T>
__device__ __forceinline__ void row_columns(const T* row, int hd, int lane, float (&x)[kRowWords]) {
  RowPart<T> part;
  part.load(row, hd, lane);
#pragma unroll
  for (int e = 0; e < kRowWords; ++e) x[e] = part[e];
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

// What is known of a lane's row: columns whose sum holds +inf, -inf or NaN.
struct RowKinds {
  uint32_t pos[kRowWords], neg[kRowWords], nan[kRowWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) pos[e] = neg[e] = nan[e] = 0u;
  }
  __device__ __forceinline__ void undefined() {
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) nan[e] = 0xffffffffu;
  }
  // every column of the row is NaN
  __device__ __forceinline__ bool settled(int hd) const {
    bool all = true;
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) all = all && (~(nan[e] | (pos[e] & neg[e])) & columns_of(e, hd)) == 0u;
    return all;
  }
};

// The infinite and undefined columns of a vector that the warp shares, as sets.
struct VectorKinds {
  uint32_t pos[kRowWords], neg[kRowWords], nan[kRowWords];
  __device__ __forceinline__ bool take(const float (&x)[kRowWords]) {
    uint32_t any = 0u;
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) {
      pos[e] = __ballot_sync(0xffffffffu, x[e] == INFINITY);
      neg[e] = __ballot_sync(0xffffffffu, x[e] == -INFINITY);
      nan[e] = __ballot_sync(0xffffffffu, x[e] != x[e]);
      any |= pos[e] | neg[e] | nan[e];
    }
    return any != 0u;
  }
  __device__ __forceinline__ bool news_to(const RowKinds& k) const {
    uint32_t any = 0u;
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) any |= ((pos[e] & ~k.pos[e]) | (neg[e] & ~k.neg[e]) | nan[e]) & ~k.nan[e];
    return any != 0u;
  }
  // times a positive weight, or (`zero`) one of zero
  __device__ __forceinline__ void add_to(RowKinds& k, bool zero) const {
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) {
      k.nan[e] |= zero ? pos[e] | neg[e] | nan[e] : nan[e];
      if (!zero) {
        k.pos[e] |= pos[e];
        k.neg[e] |= neg[e];
      }
    }
  }
};

// Row r of the warp: x becomes what its columns are by right where that is not finite, else what the kernel stored.
// Returns the columns of this lane (a bit each) that have to be summed again: those stored that should be finite and
// are not, or `all` others.
template <typename Out>
__device__ __forceinline__ uint32_t row_verdict(const RowKinds& kinds, int r, bool all, const Out* stored, int hd,
                                                int lane, float (&x)[kRowWords]) {
  uint32_t want = 0u;
#pragma unroll
  for (int e = 0; e < kRowWords; ++e) {
    const uint32_t p = __shfl_sync(0xffffffffu, kinds.pos[e], r), n = __shfl_sync(0xffffffffu, kinds.neg[e], r);
    const uint32_t u = __shfl_sync(0xffffffffu, kinds.nan[e], r) | (p & n);
    const int d = column_of(e, lane);
    x[e] = d < hd ? to_f32(stored[d]) : 0.f;
    if (u >> lane & 1u) x[e] = __int_as_float(0x7fffffff);
    else if (p >> lane & 1u) x[e] = INFINITY;
    else if (n >> lane & 1u) x[e] = -INFINITY;
    else if (d < hd && (all || !is_finite(x[e]))) want |= 1u << e;
  }
  return want;
}

// Every value's sum over the warp, in all lanes.  With each exchange a lane keeps half of the values, so that N of them
// take N - 1 + log2(32 / N) exchanges, and N to hand the sums out.
template <int N>
__device__ __forceinline__ void sum_lanes(float (&a)[N], int lane) {
  int d = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2, d /= 2) {
    const bool high = lane & d;
#pragma unroll
    for (int m = 0; m < n / 2; ++m) {
      const float mine = high ? a[m + n / 2] : a[m], other = high ? a[m] : a[m + n / 2];
      a[m] = mine + __shfl_xor_sync(0xffffffffu, other, d);
    }
  }
#pragma unroll
  for (int e = 16 / N; e > 0; e /= 2) a[0] += __shfl_xor_sync(0xffffffffu, a[0], e);
  const float own = a[0];
#pragma unroll
  for (int m = 0; m < N; ++m) a[m] = __shfl_sync(0xffffffffu, own, m * (32 / N));
}

// Rows that are summed again, A at a time over the same vectors: neighbours see much the same ones.
constexpr int kPairs = 4;
template <int A>
struct RowsAgain {
  uint32_t want[A];                           // as row_verdict returns them
  float own[A][kRowWords], pair[A][kRowWords], acc[A][kRowWords];
  // No wanted column is anything but NaN: more terms change nothing.
  __device__ __forceinline__ bool settled() const {
    bool open = false;
#pragma unroll
    for (int k = 0; k < A; ++k)
#pragma unroll
      for (int e = 0; e < kRowWords; ++e) open = open || ((want[k] >> e & 1u) && acc[k][e] == acc[k][e]);
    return !__any_sync(0xffffffffu, open);
  }
};

// Some vectors and what belongs to them: x is what the rows' own vectors are scored with, y the other one, which takes
// part in dP (DS) or is the one that is added (else).
template <typename T, bool DS>
struct VectorsAgain {
  RowPart<T> x[kPairs], y[kPairs];
  float lse[kPairs], delta[kPairs];
};

// The terms of the first n of them; see(k, u): row k sees vector u.  lse and delta are the vectors' (KEYS) or the rows'
// own.
template <typename T, bool DS, bool KEYS, int A, typename S>
__device__ __forceinline__ void add_pairs(RowsAgain<A>& r, const VectorsAgain<T, DS>& v, const float (&lse)[A],
                                          const float (&delta)[A], float scale, int n, int lane, S see) {
  constexpr int N = A * kPairs;
  float sums[DS ? 2 * N : N];
#pragma unroll
  for (int m = 0; m < N; ++m) {
    const int k = m / kPairs, u = m % kPairs;
    float s = 0.f, dp = 0.f;
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) {
      s = fmaf(r.own[k][e], v.x[u][e], s);
      if (DS) dp = fmaf(r.pair[k][e], v.y[u][e], dp);
    }
    sums[m] = s;
    if (DS) sums[N + m] = dp;
  }
  sum_lanes(sums, lane);
#pragma unroll
  for (int m = 0; m < N; ++m) {
    const int k = m / kPairs, u = m % kPairs;
    if (u >= n || !see(k, u)) continue;
    float f = expf(sums[m] * scale - (KEYS ? v.lse[u] : lse[k]));
    if (DS) f *= (sums[N + m] - (KEYS ? v.delta[u] : delta[k])) * scale;
#pragma unroll
    for (int e = 0; e < kRowWords; ++e) r.acc[k][e] = fmaf(f, DS ? v.x[u][e] : v.y[u][e], r.acc[k][e]);
  }
}

// Rows i0 + r of O (or dQ) of head h, for the bits r of `bad`.  out: row i0, `stride` elements between tokens; lo (may
// be null): what the rounding of O left, laid out the same.  A: rows that are summed at a time.  A whole warp, which
// sees the rows, the log-sum-exp and delta as stored.
template <typename T, bool DQ, int A = 2>
__device__ __noinline__ void query_rows_again(const WinRows& w, int b, int h, int i0, uint32_t bad, T* out,
                                              long long stride, bf16* lo) {
  const int lane = threadIdx.x & 31, hk = h / (w.Hq / w.Hkv), i = i0 + lane;
  const bool mine = bad >> lane & 1u;
  RowKinds kinds;
  kinds.clear();
  bool sum_all = false, done = !mine;
  if (mine) {
    done = !is_finite(w.lse[w.stat(b, h, i)]);
    if (DQ) {
      const float delta = w.delta[w.stat(b, h, i)];
      done = done || delta != delta;
      sum_all = !done && !is_finite(delta);
    }
    if (done) kinds.undefined();
    done = done || sum_all;
  }
  const uint32_t open = __ballot_sync(0xffffffffu, !done);
  if (open) {
    const int first = max(0, i0 + __ffs(open) - 1 - w.window + 1), last = i0 + 31 - __clz(open);
    const int sinks = min(w.sinks, first), n = sinks + last - first + 1;
    const auto key = [&](int v) { return v < sinks ? v : first + v - sinks; };
    const auto columns = [&](int j, float (&x)[kRowWords]) {
      row_columns(DQ ? w.row<T>(w.k, w.k_st, b, j, hk) : w.row<T>(w.v, w.v_st, b, j, hk), w.hd, lane, x);
    };
    constexpr int kBatch = 8;
    for (int v0 = 0; v0 < n; v0 += kBatch) {
      float probe = 0.f, x[kRowWords];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        columns(key(min(v0 + u, n - 1)), x);
#pragma unroll
        for (int e = 0; e < kRowWords; ++e) probe_finite(probe, x[e]);
      }
      if (!__any_sync(0xffffffffu, probe != 0.f)) continue;
#pragma unroll 1
      for (int u = v0; u < min(v0 + kBatch, n); ++u) {
        const int j = key(u);
        if (!__any_sync(0xffffffffu, !done && w.visible(i, j))) continue;
        columns(j, x);
        VectorKinds vec;
        if (!vec.take(x)) continue;
        // a weight of zero, which makes an infinity NaN that is known already, takes a K that is not finite
        bool odd = false;
        if (!DQ) {
          probe = 0.f;
          row_columns(w.row<T>(w.k, w.k_st, b, j, hk), w.hd, lane, x);
#pragma unroll
          for (int e = 0; e < kRowWords; ++e) probe_finite(probe, x[e]);
          odd = __any_sync(0xffffffffu, probe != 0.f);
        }
        if (!done && w.visible(i, j) && (odd || vec.news_to(kinds))) {
          bool zero = DQ;
          if (!DQ) {
            const T *q = w.row<T>(w.q, w.q_st, b, i, h), *k = w.row<T>(w.k, w.k_st, b, j, hk);
            zero = row_dot(q, k, w.hd) * w.scale == -INFINITY;
          }
          vec.add_to(kinds, zero);
          done = kinds.settled(w.hd);
        }
      }
      if (__all_sync(0xffffffffu, done)) break;
    }
  }
#pragma unroll 1
  while (bad) {
    int t[A];
    float x[A][kRowWords], lse[A], delta[A];
    RowsAgain<A> rows{};
    uint32_t any = 0u;
#pragma unroll
    for (int k = 0; k < A; ++k) {
      t[k] = -1;
      lse[k] = delta[k] = 0.f;
      if (!bad) continue;
      const int r = __ffs(bad) - 1;
      bad &= bad - 1;
      t[k] = i0 + r;
      rows.want[k] = row_verdict(kinds, r, __shfl_sync(0xffffffffu, sum_all, r), out + r * stride, w.hd, lane, x[k]);
      any |= rows.want[k];
      lse[k] = w.lse[w.stat(b, h, t[k])];
      row_columns(w.row<T>(w.q, w.q_st, b, t[k], h), w.hd, lane, rows.own[k]);
      if (DQ) {
        delta[k] = w.delta[w.stat(b, h, t[k])];
        row_columns(w.row<T>(w.d_o, w.do_st, b, t[k], h), w.hd, lane, rows.pair[k]);
      }
    }
    if (__any_sync(0xffffffffu, any)) {
      const int last = t[A - 1] < 0 ? t[0] : t[A - 1];
      const int first = max(0, t[0] - w.window + 1), sinks = min(w.sinks, first), n = sinks + last - first + 1;
      const auto key = [&](int v) { return v < sinks ? v : first + v - sinks; };
#pragma unroll 1
      for (int v0 = 0; v0 < n; v0 += kPairs) {
        VectorsAgain<T, DQ> now;
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
          const int j = key(min(v0 + u, n - 1));
          now.x[u].load(w.row<T>(w.k, w.k_st, b, j, hk), w.hd, lane);
          now.y[u].load(w.row<T>(w.v, w.v_st, b, j, hk), w.hd, lane);
        }
        add_pairs<T, DQ, false>(rows, now, lse, delta, w.scale, min(kPairs, n - v0), lane,
                                [&](int k, int u) { return w.visible(t[k], key(v0 + u)); });
        if (rows.settled()) break;
      }
    }
#pragma unroll
    for (int k = 0; k < A; ++k)
#pragma unroll
      for (int e = 0; e < kRowWords; ++e) {
        const int d = column_of(e, lane);
        if (t[k] < 0 || d >= w.hd) continue;
        const float sum = rows.want[k] >> e & 1u ? rows.acc[k][e] : x[k][e];
        const T rounded = from_f32<T>(sum);
        const long long at = (t[k] - i0) * stride + d;
        out[at] = rounded;
        if (lo) lo[at] = from_f32<bf16>(is_finite(to_f32(rounded)) ? sum - to_f32(rounded) : 0.f);
      }
  }
}

// Rows j0 + r of dV (VALUE) or dK of kv head hk, for the bits r of `bad`: their sums over queries [ia, ib).  out: row
// j0, `stride` elements between rows.  A whole warp, as above.
template <typename T, typename Out, bool VALUE>
__device__ __noinline__ void key_rows_again(const WinRows& w, int b, int hk, int j0, uint32_t bad, int ia, int ib,
                                            Out* out, long long stride) {
  constexpr int A = 2;
  const int lane = threadIdx.x & 31, G = w.Hq / w.Hkv, j = j0 + lane;
  const bool mine = bad >> lane & 1u;
  RowKinds kinds;
  kinds.clear();
  bool done = !mine;
  const int last = mine ? w.last_query(j) : -1;   // of this row
  const int i_lo = max(ia, j0 + __ffs(bad) - 1), i_hi = min(min(ib, w.T), __reduce_max_sync(0xffffffffu, last) + 1);
  const auto columns = [&](int i, int h, float (&x)[kRowWords]) {
    row_columns(VALUE ? w.row<T>(w.d_o, w.do_st, b, i, h) : w.row<T>(w.q, w.q_st, b, i, h), w.hd, lane, x);
  };
  const auto score = [&](int i, int h) {
    return row_dot(w.row<T>(w.q, w.q_st, b, i, h), w.row<T>(w.k, w.k_st, b, j, hk), w.hd) * w.scale;
  };
  // a K whose scores may be -inf: a weight of zero makes NaN of an infinity that is known already
  const T* own = w.row<T>(w.k, w.k_st, b, mine ? j : j0 + __ffs(bad) - 1, hk);
  const bool odd = VALUE && !is_finite(row_dot(own, own, w.hd));
  bool settled = false;
#pragma unroll 1
  for (int h = hk * G; h < hk * G + G && !settled; ++h) {
#pragma unroll 1
    for (int i32 = i_lo; i32 < i_hi && !settled; i32 += 32) {
      const bool real = i32 + lane < i_hi;
      const float lse = real ? w.lse[w.stat(b, h, i32 + lane)] : 0.f;
      const float delta = !VALUE && real ? w.delta[w.stat(b, h, i32 + lane)] : 0.f;
      const bool undefined = !is_finite(lse) || delta != delta;
      const uint32_t no = __ballot_sync(0xffffffffu, undefined);
      if (mine && (no & bit_range(j - i32, last + 1 - i32))) {
        kinds.undefined();
        done = true;
      }
      if (VALUE) {
        constexpr int kBatch = 8;
#pragma unroll 1
        for (int i0 = i32; i0 < min(i32 + 32, i_hi); i0 += kBatch) {
          float probe = 0.f, x[kRowWords];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            columns(min(i0 + u, i_hi - 1), h, x);
#pragma unroll
            for (int e = 0; e < kRowWords; ++e) probe_finite(probe, x[e]);
          }
          if (!__any_sync(0xffffffffu, probe != 0.f)) continue;
#pragma unroll 1
          for (int i = i0; i < min(i0 + kBatch, i_hi); ++i) {
            if (!__any_sync(0xffffffffu, !done && i >= j && i <= last)) continue;
            columns(i, h, x);
            VectorKinds vec;
            if (!vec.take(x)) continue;
            if (!done && i >= j && i <= last && (odd || vec.news_to(kinds))) {
              vec.add_to(kinds, score(i, h) == -INFINITY);
              done = kinds.settled(w.hd);
            }
          }
        }
      } else {
        uint32_t inf = __ballot_sync(0xffffffffu, !undefined && !is_finite(delta));
#pragma unroll 1
        for (; inf; inf &= inf - 1) {
          const int t = __ffs(inf) - 1, i = i32 + t;
          const float lse_i = __shfl_sync(0xffffffffu, lse, t), delta_i = __shfl_sync(0xffffffffu, delta, t);
          const bool concerned = !done && i >= j && i <= last;
          if (!__any_sync(0xffffffffu, concerned)) continue;
          float x[kRowWords];
          columns(i, h, x);
          uint32_t up[kRowWords], down[kRowWords];
#pragma unroll
          for (int e = 0; e < kRowWords; ++e) {
            up[e] = __ballot_sync(0xffffffffu, x[e] > 0.f);
            down[e] = __ballot_sync(0xffffffffu, x[e] < 0.f);
          }
          if (concerned) {
            const float dp = row_dot(w.row<T>(w.d_o, w.do_st, b, i, h), w.row<T>(w.v, w.v_st, b, j, hk), w.hd);
            const float f = expf(score(i, h) - lse_i) * (dp - delta_i) * w.scale;
            if (f != f) {
              kinds.undefined();
            } else if (!is_finite(f)) {
#pragma unroll
              for (int e = 0; e < kRowWords; ++e) {
                kinds.pos[e] |= f > 0.f ? up[e] : down[e];
                kinds.neg[e] |= f > 0.f ? down[e] : up[e];
                kinds.nan[e] |= ~(up[e] | down[e]);
              }
            }
            done = kinds.settled(w.hd);
          }
        }
      }
      settled = __all_sync(0xffffffffu, done);
    }
  }
#pragma unroll 1
  while (bad) {
    int t[A], until[A];
    const float unused[A] = {};
    float x[A][kRowWords];
    RowsAgain<A> rows{};
    uint32_t any = 0u;
#pragma unroll
    for (int k = 0; k < A; ++k) {
      t[k] = w.T;
      until[k] = -1;
      if (!bad) continue;
      const int r = __ffs(bad) - 1;
      bad &= bad - 1;
      t[k] = j0 + r;
      until[k] = w.last_query(t[k]);
      rows.want[k] = row_verdict(kinds, r, false, out + r * stride, w.hd, lane, x[k]);
      any |= rows.want[k];
      row_columns(w.row<T>(w.k, w.k_st, b, t[k], hk), w.hd, lane, rows.own[k]);
      if (!VALUE) row_columns(w.row<T>(w.v, w.v_st, b, t[k], hk), w.hd, lane, rows.pair[k]);
    }
    if (__any_sync(0xffffffffu, any)) {
      const int from = max(ia, t[0]);
      int to = 0;
#pragma unroll
      for (int k = 0; k < A; ++k) to = max(to, min(min(ib, w.T), until[k] + 1));
      bool open = from < to;
#pragma unroll 1
      for (int h = hk * G; h < hk * G + G && open; ++h) {
#pragma unroll 1
        for (int i = from; i < to && open; i += kPairs) {
          VectorsAgain<T, !VALUE> now;
#pragma unroll
          for (int u = 0; u < kPairs; ++u) {
            const int iu = min(i + u, to - 1);
            now.x[u].load(w.row<T>(w.q, w.q_st, b, iu, h), w.hd, lane);
            now.y[u].load(w.row<T>(w.d_o, w.do_st, b, iu, h), w.hd, lane);
            now.lse[u] = w.lse[w.stat(b, h, iu)];
            if (!VALUE) now.delta[u] = w.delta[w.stat(b, h, iu)];
          }
          add_pairs<T, !VALUE, true>(rows, now, unused, unused, w.scale, min(kPairs, to - i), lane,
                                     [&](int k, int u) { return i + u >= t[k] && i + u <= until[k]; });
          open = !rows.settled();
        }
      }
    }
#pragma unroll
    for (int k = 0; k < A; ++k)
#pragma unroll
      for (int e = 0; e < kRowWords; ++e) {
        const int d = column_of(e, lane);
        if (until[k] < 0 || d >= w.hd) continue;
        out[(t[k] - j0) * stride + d] = from_f32<Out>(rows.want[k] >> e & 1u ? rows.acc[k][e] : x[k][e]);
      }
  }
}

}  // namespace titb
