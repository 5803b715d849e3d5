// Paged key-value cache: appending tokens (with the rotary embedding) and the attention of one new token per sequence.
#include <cuda_runtime.h>

#include <cmath>

#include "api.h"
#include "common.cuh"

namespace titb {

// Where a sequence's positions lie in the cache.
struct PageMap {
  const int* table;   // this sequence's row of the page table
  int width, n_pages, page_size;
  // Row of `pos` (in rows of a head's [page_size, hd] block), or -1 when the table does not lead into the cache.
  __device__ __forceinline__ long long row(int pos, int Hkv, int hk) const {
    const int slot = pos / page_size;
    if (pos < 0 || slot >= width) return -1;
    const int page = table[slot];
    if (page < 0 || page >= n_pages) return -1;
    return (static_cast<long long>(page) * Hkv + hk) * page_size + (pos - slot * page_size);
  }
};

struct CacheArgs {
  void *k_cache, *v_cache;
  const int* page_table;
  long long table_stride;
  int table_width, n_pages, page_size, B, Hq, Hkv, hd, window, sinks;
  int* status;
  __device__ __forceinline__ PageMap map(int b) const {
    return {page_table + b * table_stride, table_width, n_pages, page_size};
  }
};

static CacheArgs cache_args(const TitbCacheDesc* d) {
  CacheArgs a{};
  a.k_cache = d->k_cache; a.v_cache = d->v_cache;
  a.page_table = d->page_table; a.table_stride = d->table_stride; a.table_width = d->table_width;
  a.n_pages = d->n_pages; a.page_size = d->page_size;
  a.B = d->B; a.Hq = d->Hq; a.Hkv = d->Hkv; a.hd = d->hd;
  a.window = d->window; a.sinks = d->sinks;
  a.status = titb_status_ptr();
  return a;
}

// --------------------------------------------------------------------------------------------------- append
constexpr int kMaxHalf = 64;   // angles of a head of up to 128

struct AppendArgs {
  CacheArgs c;
  const void* qkv;
  long long stride_b, stride_t;
  int T;
  const int *starts, *counts;
  void *q_out, *k_out;
  int rotate;
  double turns[kMaxHalf];   // theta^(-2 i / hd) / (2 pi): turns of pair i per position
};

// Sine and cosine of pos * theta^(-2 i / hd).  The number of turns is taken in 64 bits (at position 131072 an fp32 angle
// would be off by up to 0.004), its fraction in two fp32 parts.
__device__ __forceinline__ void rope_sincos(int pos, double turns, float& sn, float& cs) {
  const double t = pos * turns;
  const double x = 2.0 * (t - rint(t));
  const float hi = static_cast<float>(x), lo = static_cast<float>(x - hi) * 3.14159265f;
  float s, c;
  sincospif(hi, &s, &c);
  sn = fmaf(lo, c, s);
  cs = fmaf(-lo, s, c);
}

// V neighbouring elements of both halves of a head per thread.
template <typename T, int V>
__global__ void __launch_bounds__(256) cache_append_kernel(const __grid_constant__ AppendArgs p) {
  __shared__ double turns[kMaxHalf];
  if (threadIdx.x < kMaxHalf) turns[threadIdx.x] = p.turns[threadIdx.x];
  __syncthreads();
  const CacheArgs& c = p.c;
  const int half = c.hd / 2, chunks = half / V, heads = c.Hq + 2 * c.Hkv;
  const long long n = static_cast<long long>(c.B) * p.T * heads * chunks;
  for (long long x = blockIdx.x * 256LL + threadIdx.x; x < n; x += gridDim.x * 256LL) {
    const int i = static_cast<int>(x % chunks) * V;
    const int h = static_cast<int>(x / chunks % heads);
    const long long bt = x / chunks / heads;
    const int b = static_cast<int>(bt / p.T), t = static_cast<int>(bt - static_cast<long long>(b) * p.T);
    const int start = p.starts[b], count = p.counts ? min(p.counts[b], p.T) : p.T;
    const long long pos = static_cast<long long>(start) + t;
    const T* src = static_cast<const T*>(p.qkv) + b * p.stride_b + t * p.stride_t + static_cast<long long>(h) * c.hd + i;
    const Pack<T, V> lo = *reinterpret_cast<const Pack<T, V>*>(src);
    const Pack<T, V> hi = *reinterpret_cast<const Pack<T, V>*>(src + half);
    Pack<T, V> a = lo, d = hi;
    if (p.rotate && h < c.Hq + c.Hkv) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float sn, cs;
        rope_sincos(static_cast<int>(pos), turns[i + e], sn, cs);
        const float u = to_f32(lo.v[e]), w = to_f32(hi.v[e]);
        a.v[e] = from_f32<T>(u * cs - w * sn);
        d.v[e] = from_f32<T>(w * cs + u * sn);
      }
    }
    auto put = [&](void* base, long long row) {
      T* dst = static_cast<T*>(base) + row * c.hd + i;
      *reinterpret_cast<Pack<T, V>*>(dst) = a;
      *reinterpret_cast<Pack<T, V>*>(dst + half) = d;
    };
    if (h < c.Hq) {
      if (p.q_out) put(p.q_out, bt * c.Hq + h);
      continue;
    }
    const int hk = (h - c.Hq) % c.Hkv;
    const bool key = h < c.Hq + c.Hkv;
    if (key && p.k_out) put(p.k_out, bt * c.Hkv + hk);
    const long long end = static_cast<long long>(start) + count;
    if (t < count && (pos >= end - c.window || pos < c.sinks)) {
      const long long row = pos <= 0x7fffffffLL ? c.map(b).row(static_cast<int>(pos), c.Hkv, hk) : -1;
      if (row >= 0) put(key ? c.k_cache : c.v_cache, row);
      else atomicExch(c.status, kStatusBadPage);
    }
  }
}

// --------------------------------------------------------------------------------------------------- attention
// Of a sequence with n cached positions a query sees the first s and the last ones: position v of that list is v < s ? v :
// v + gap.
struct Seen {
  int n, s, gap;
  __device__ __forceinline__ int pos(int v) const { return v < s ? v : v + gap; }
};
__device__ __forceinline__ Seen seen_of(int length, int limit, int window, int sinks) {
  const int n = min(max(length, 0), limit);
  if (n <= window) return {n, 0, 0};
  const int s = min(sinks, n - window);
  return {s + window, s, n - window - s};
}

struct PagedArgs {
  CacheArgs c;
  const void* q;
  long long q_stride_b;
  const int* lengths;
  void* o;
  float scale;
};

constexpr int kPagedWarps = 4;
constexpr int kPagedHeads = 4;   // query heads that share the loads of a pass over the cache

// One CTA per (sequence, kv head, group of query heads).  L lanes hold a row (16 bytes each); every group of L lanes takes
// rows of its own and keeps its own running maximum, sum and output, which meet at the end.
template <typename T, int L>
__global__ void __launch_bounds__(kPagedWarps * 32) paged_attention_kernel(const PagedArgs p) {
  constexpr int VN = 16 / sizeof(T), kRows = 32 / L, kGroups = kPagedWarps * kRows;
  __shared__ float sm_m[kPagedHeads][kGroups], sm_l[kPagedHeads][kGroups];
  __shared__ float sm_o[kPagedHeads][kGroups][L * VN];
  const CacheArgs& c = p.c;
  const int lane = threadIdx.x & 31, grp = (threadIdx.x >> 5) * kRows + lane / L, d0 = (lane % L) * VN;
  const int G = c.Hq / c.Hkv, hgroups = (G + kPagedHeads - 1) / kPagedHeads;
  const int hk = blockIdx.x / hgroups, g0 = (blockIdx.x % hgroups) * kPagedHeads, b = blockIdx.y;
  const int ng = min(kPagedHeads, G - g0);
  const bool in_head = d0 < c.hd;
  const int limit = static_cast<int>(min(static_cast<long long>(c.table_width) * c.page_size, 0x7fffffffLL));
  const int length = p.lengths[b];
  if ((length < 0 || length > limit) && threadIdx.x == 0) atomicExch(c.status, kStatusBadPage);
  const Seen seen = seen_of(length, limit, c.window, c.sinks);
  const PageMap map = c.map(b);

  float q[kPagedHeads][VN], o[kPagedHeads][VN] = {}, m[kPagedHeads], l[kPagedHeads];
#pragma unroll
  for (int g = 0; g < kPagedHeads; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < VN; ++e) q[g][e] = 0.f;
    if (g < ng && in_head) {
      const Pack<T, VN> x = ld128(static_cast<const T*>(p.q) + b * p.q_stride_b + (hk * G + g0 + g) * c.hd + d0);
#pragma unroll
      for (int e = 0; e < VN; ++e) q[g][e] = to_f32(x.v[e]) * p.scale;
    }
  }
  for (int v = grp; v - grp < seen.n; v += kGroups) {   // all lanes take part in every round's shuffles
    const long long row = v < seen.n ? map.row(seen.pos(v), c.Hkv, hk) : -1;
    if (v < seen.n && row < 0 && lane % L == 0) atomicExch(c.status, kStatusBadPage);
    Pack<T, VN> kx{}, vx{};
    if (row >= 0 && in_head) {
      kx = ld128(static_cast<const T*>(c.k_cache) + row * c.hd + d0);
      vx = ld128(static_cast<const T*>(c.v_cache) + row * c.hd + d0);
    }
#pragma unroll
    for (int g = 0; g < kPagedHeads; ++g) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < VN; ++e) s = fmaf(q[g][e], to_f32(kx.v[e]), s);
#pragma unroll
      for (int w = 1; w < L; w <<= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      if (row < 0) continue;
      const float top = fmaxf(m[g], s), ref = top == -INFINITY ? 0.f : top;   // a score may be -inf
      const float keep = expf(m[g] - ref), x = expf(s - ref);
      m[g] = top;
      l[g] = fmaf(l[g], keep, x);
#pragma unroll
      for (int e = 0; e < VN; ++e) o[g][e] = fmaf(o[g][e], keep, x * to_f32(vx.v[e]));
    }
  }
#pragma unroll
  for (int g = 0; g < kPagedHeads; ++g) {
    if (lane % L == 0) {
      sm_m[g][grp] = m[g];
      sm_l[g][grp] = l[g];
    }
#pragma unroll
    for (int e = 0; e < VN; ++e) sm_o[g][grp][d0 + e] = o[g][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ng * c.hd; i += kPagedWarps * 32) {
    const int g = i / c.hd, d = i % c.hd;
    float top = -INFINITY, sum = 0.f, acc = 0.f;
    for (int w = 0; w < kGroups; ++w) top = fmaxf(top, sm_m[g][w]);
    for (int w = 0; w < kGroups; ++w) {
      if (sm_l[g][w] == 0.f) continue;
      const float f = expf(sm_m[g][w] - top);
      sum = fmaf(sm_l[g][w], f, sum);
      acc = fmaf(sm_o[g][w][d], f, acc);
    }
    static_cast<T*>(p.o)[(static_cast<long long>(b) * c.Hq + hk * G + g0 + g) * c.hd + d] = from_f32<T>(sum > 0.f ? acc / sum : 0.f);
  }
}

static int cache_check(const TitbCacheDesc* d) {
  if (d->hd <= 0 || d->hd > 128 || d->hd % 8 || d->Hkv <= 0 || d->Hq % d->Hkv || d->page_size <= 0 || d->table_width < 0 ||
      d->n_pages < 0 || d->sinks < 0 || d->window < 1 || (d->dtype != 0 && d->dtype != 1))
    return TITB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(d->k_cache) & 15) || (reinterpret_cast<uintptr_t>(d->v_cache) & 15)) return TITB_ERR_ALIGNMENT;
  return 0;
}

template <typename T>
static int append_launch(const AppendArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int half = a.c.hd / 2;
  const bool wide = half % V == 0;   // hd is a multiple of 8, so quarters of a row's half are always whole
  const long long n = static_cast<long long>(a.c.B) * a.T * (a.c.Hq + 2 * a.c.Hkv) * (half / (wide ? V : 4));
  const long long blocks = (n + 255) / 256, most = device_sm_count() * 16LL;
  const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
  if (wide) cache_append_kernel<T, V><<<grid, 256, 0, st>>>(a);
  else cache_append_kernel<T, 4><<<grid, 256, 0, st>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int L>
static int paged_launch(const PagedArgs& a, cudaStream_t st) {
  const int G = a.c.Hq / a.c.Hkv;
  const dim3 grid(a.c.Hkv * ((G + kPagedHeads - 1) / kPagedHeads), a.c.B);
  paged_attention_kernel<T, L><<<grid, kPagedWarps * 32, 0, st>>>(a);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace titb

using namespace titb;

TITB_API int titb_cache_append(const TitbCacheDesc* d, const void* qkv, long long qkv_stride_b, long long qkv_stride_t, int T,
                               const int* starts, const int* counts, double theta, void* q_out, void* k_out, cudaStream_t st) {
  (void)cudaGetLastError();
  if (d->B <= 0 || T <= 0) return 0;
  if (const int rc = cache_check(d)) return rc;
  auto bad = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  const int mask = d->dtype == 1 ? 7 : 3;
  if (bad(qkv) || bad(q_out) || bad(k_out) || (qkv_stride_b & mask) || (qkv_stride_t & mask)) return TITB_ERR_ALIGNMENT;
  AppendArgs a{};
  a.c = cache_args(d);
  a.qkv = qkv; a.stride_b = qkv_stride_b; a.stride_t = qkv_stride_t; a.T = T;
  a.starts = starts; a.counts = counts; a.q_out = q_out; a.k_out = k_out;
  a.rotate = theta > 0.0;
  if (a.rotate) {
    // in extended precision, so that 64 rounded products do not show in the 53 bits that are kept
    const long double step = std::pow(static_cast<long double>(theta), -2.0L / d->hd);
    long double f = 0.159154943091895335768883763372514362L;   // 1 / (2 pi)
    for (int i = 0; i < d->hd / 2; ++i, f *= step) a.turns[i] = static_cast<double>(f);
  }
  return d->dtype == 1 ? append_launch<bf16>(a, st) : append_launch<float>(a, st);
}

TITB_API int titb_paged_attention(const TitbCacheDesc* d, const void* q, long long q_stride_b, const int* lengths, float scale,
                                  void* o, cudaStream_t st) {
  (void)cudaGetLastError();
  if (d->B <= 0 || d->Hq <= 0) return 0;
  if (const int rc = cache_check(d)) return rc;
  if (d->B > 65535) return TITB_ERR_SHAPE;
  auto bad = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (bad(q) || bad(o) || (q_stride_b & (d->dtype == 1 ? 7 : 3))) return TITB_ERR_ALIGNMENT;
  PagedArgs a{};
  a.c = cache_args(d);
  a.q = q; a.q_stride_b = q_stride_b; a.lengths = lengths; a.o = o; a.scale = scale;
  if (d->dtype == 1) return d->hd <= 64 ? paged_launch<bf16, 8>(a, st) : paged_launch<bf16, 16>(a, st);
  return d->hd <= 64 ? paged_launch<float, 16>(a, st) : paged_launch<float, 32>(a, st);
}
