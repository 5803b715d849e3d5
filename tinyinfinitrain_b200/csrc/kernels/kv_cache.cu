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
  a.page_table = d->page_table; a.table_stride = d->table_stride;
  a.table_width = d->n_pages > 0 ? d->table_width : 0;   // without pages no entry leads anywhere
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
  int rotate, tokens, per;   // tokens and heads of a CTA
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

// A CTA takes up to kAppendTokens tokens and `per` of their heads.  The sines and cosines of its tokens go to shared memory once
// (their 64-bit reduction costs more than a head's bytes), then a thread moves V neighbouring elements of both halves of a
// head at a time, two of them in flight.  Before, every thread took the angles of eight heads of its own:
// 112 registers, 13 warps on an SM, 31 us for 2 x 1999 tokens, 32 / 8 heads of 128 (106 MB); now 23.5 us (4.5 TB/s).  Bound by
// the latency of the reads: of 43000 cycles an SM works 33000, the others being the launch, the first reads and the end of the
// one wave; there 28 warps (63 registers a thread) wait for their reads two fifths of the time and issue in half of the cycles.
// Neither memory (DRAM 33 %, L2 26 %: what is written stays in the L2) nor issue is full.  Asking for the rows ahead of the
// angles (prefetch to the L2) did not help.  64 single tokens: 5 us, of which the launch, positions,
// page table and angles one behind the other are most.
constexpr int kAppendTokens = 8, kAppendThreads = 256, kAppendCtas = 4;   // the last: CTAs of an SM

template <typename T, int V>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) cache_append_kernel(const __grid_constant__ AppendArgs p) {
  constexpr int U = 2;
  __shared__ __align__(16) float sin_of[kAppendTokens][kMaxHalf], cos_of[kAppendTokens][kMaxHalf];
  __shared__ long long row_of[kAppendTokens];   // of the cache, of kv head 0 (the others follow page_size rows apart); -1: none
  __shared__ long long src_of[kAppendTokens];   // of the projection
  dependency_wait();
  dependents_launch();
  const CacheArgs& c = p.c;
  const int half = c.hd / 2, chunks = half / V, heads = c.Hq + 2 * c.Hkv, rotated = p.rotate ? c.Hq + c.Hkv : 0;
  const int h0 = blockIdx.y * p.per, nh = min(p.per, heads - h0);
  const int bt0 = blockIdx.x * p.tokens, nt = min(p.tokens, c.B * p.T - bt0);
  if (threadIdx.x < kAppendTokens) {
    const int kk = threadIdx.x;
    if (kk < nt) {
      const int b = (bt0 + kk) / p.T, t = bt0 + kk - b * p.T;
      src_of[kk] = b * p.stride_b + t * p.stride_t;
      const int start = p.starts[b], count = p.counts ? min(p.counts[b], p.T) : p.T;
      const long long pos = static_cast<long long>(start) + t;
      long long row = -1;
      if (h0 + nh > c.Hq && t < count && (pos >= static_cast<long long>(start) + count - c.window || pos < c.sinks)) {
        if (pos <= 0x7fffffffLL) row = c.map(b).row(static_cast<int>(pos), c.Hkv, 0);
        if (row < 0) atomicExch(c.status, kStatusBadPage);
      }
      row_of[kk] = row;
    }
  }
  if (h0 < rotated)
    for (int x = threadIdx.x; x < nt * half; x += kAppendThreads) {
      const int kk = x / half, e = x - kk * half, b = (bt0 + kk) / p.T, t = bt0 + kk - b * p.T;
      rope_sincos(static_cast<int>(static_cast<long long>(p.starts[b]) + t), p.turns[e], sin_of[kk][e], cos_of[kk][e]);
    }
  __syncthreads();
  // a thread stays at its place in the heads and steps from head to head: (token, head) pairs in a row, `lanes` at a time
  const int lanes = kAppendThreads / chunks, i = static_cast<int>(threadIdx.x) % chunks * V;
  int h = static_cast<int>(threadIdx.x) / chunks, k = 0;
  if (h >= lanes) return;   // what does not fill a row of chunks
  const auto settle = [&]() {
    while (h >= nh) {
      h -= nh;
      ++k;
    }
  };
  settle();
  while (k < nt) {
    Pack<T, V> lo[U], hi[U];
    int ku[U], hu[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ku[u] = k < nt && (h0 + h >= c.Hq || p.q_out) ? k : -1;
      hu[u] = h0 + h;
      if (ku[u] >= 0) {
        const T* src = static_cast<const T*>(p.qkv) + src_of[k] + static_cast<long long>(hu[u]) * c.hd + i;
        lo[u] = *reinterpret_cast<const Pack<T, V>*>(src);
        hi[u] = *reinterpret_cast<const Pack<T, V>*>(src + half);
      }
      h += lanes;
      settle();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ku[u] < 0) continue;
      if (hu[u] < rotated) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          const float4 sn = *reinterpret_cast<const float4*>(&sin_of[ku[u]][i + e]);
          const float4 cs = *reinterpret_cast<const float4*>(&cos_of[ku[u]][i + e]);
          const float s4[4] = {sn.x, sn.y, sn.z, sn.w}, c4[4] = {cs.x, cs.y, cs.z, cs.w};
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const float a = to_f32(lo[u].v[e + f]), w = to_f32(hi[u].v[e + f]);
            lo[u].v[e + f] = from_f32<T>(a * c4[f] - w * s4[f]);
            hi[u].v[e + f] = from_f32<T>(w * c4[f] + a * s4[f]);
          }
        }
      }
      auto put = [&](void* base, long long r) {
        T* dst = static_cast<T*>(base) + r * c.hd + i;
        *reinterpret_cast<Pack<T, V>*>(dst) = lo[u];
        *reinterpret_cast<Pack<T, V>*>(dst + half) = hi[u];
      };
      if (hu[u] < c.Hq) {
        put(p.q_out, static_cast<long long>(bt0 + ku[u]) * c.Hq + hu[u]);
        continue;
      }
      const bool key = hu[u] < c.Hq + c.Hkv;
      const int hk = hu[u] - c.Hq - (key ? 0 : c.Hkv);
      if (key && p.k_out) put(p.k_out, static_cast<long long>(bt0 + ku[u]) * c.Hkv + hk);
      if (row_of[ku[u]] >= 0) put(key ? c.k_cache : c.v_cache, row_of[ku[u]] + static_cast<long long>(hk) * c.page_size);
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
  float* parts;   // per CTA two slots of partial results, [heads][hd] sums, [heads] maxima, [heads] denominators
  int4* joins;    // per CTA the item whose first tiles it took, when others took the rest
};

// The work is cut into tiles of TILE positions of one item, an item being a sequence, one of its kv heads and up to HG of
// the query heads that share it.  All tiles in a row (by sequence, then item, then position) are dealt to the CTAs in equal
// runs, whatever the lengths, which only the device knows: a long sequence is split over as many CTAs as its share of the work,
// and short ones share a CTA.  An item that a CTA holds from end to end is finished there.  Of any other the CTA leaves the
// sums, their maximum and denominator in its slots (0: the item began before its run, 1: it goes on behind it), and
// paged_join_kernel adds the slots up in order.
__device__ __forceinline__ int paged_limit(const CacheArgs& c) {
  return static_cast<int>(min(static_cast<long long>(c.table_width) * c.page_size, 0x7fffffffLL));
}
template <int HG>
__device__ __forceinline__ int items_of(const CacheArgs& c) {
  return c.Hkv * ((c.Hq / c.Hkv + HG - 1) / HG);
}

// A run of tiles.
template <int TILE, int HG>
struct TileWalk {
  int b, item, t, n_tiles;
  Seen seen;
  __device__ __forceinline__ void enter(const PagedArgs& p, int limit) {
    seen = seen_of(p.lengths[b], limit, p.c.window, p.c.sinks);
    n_tiles = (seen.n + TILE - 1) / TILE;
  }
  __device__ __forceinline__ void next(const PagedArgs& p, int limit) {
    if (++t < n_tiles) return;
    t = 0;
    if (++item < items_of<HG>(p.c)) return;
    item = 0;
    do {
      if (++b >= p.c.B) return;   // behind the last tile
      enter(p, limit);
    } while (n_tiles == 0);
  }
};

struct Run {
  int n;          // tiles of this CTA
  long long per;  // tiles of every CTA but the last ones
  long long first;
};

// This CTA's run, and the walk at its first tile.  Threads count the tiles of neighbouring sequences; a scan over the block
// gives the sequence in which the run begins.  All threads of the CTA.
template <int TILE, int HG, int THREADS>
__device__ __forceinline__ Run begin_run(const PagedArgs& p, TileWalk<TILE, HG>& walk) {
  __shared__ long long warp_sum[THREADS / 32];
  __shared__ int at_b;
  __shared__ long long at_rem;
  const int limit = paged_limit(p.c), items = items_of<HG>(p.c), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = (p.c.B + THREADS - 1) / THREADS, b0 = min(p.c.B, static_cast<int>(threadIdx.x) * chunk), b1 = min(p.c.B, b0 + chunk);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int length = p.lengths[b];
    if (blockIdx.x == 0 && (length < 0 || length > limit)) atomicExch(p.c.status, kStatusBadPage);
    mine += static_cast<long long>((seen_of(length, limit, p.c.window, p.c.sinks).n + TILE - 1) / TILE) * items;
  }
  long long scan = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += x;
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  long long before = scan - mine, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  Run run;
  run.per = (total + gridDim.x - 1) / gridDim.x;
  run.first = blockIdx.x * run.per;
  run.n = static_cast<int>(max(0LL, min(run.per, total - run.first)));
  if (run.n > 0 && run.first >= before && run.first < before + mine) {
    long long rem = run.first - before;
    int b = b0;
    for (;; ++b) {
      const long long here = static_cast<long long>((seen_of(p.lengths[b], limit, p.c.window, p.c.sinks).n + TILE - 1) / TILE) * items;
      if (rem < here) break;
      rem -= here;
    }
    at_b = b;
    at_rem = rem;
  }
  __syncthreads();
  if (run.n > 0) {
    walk.b = at_b;
    walk.enter(p, limit);
    walk.item = static_cast<int>(at_rem / walk.n_tiles);
    walk.t = static_cast<int>(at_rem % walk.n_tiles);
  }
  return run;
}

// Zeros for the sequences that see nothing.
template <typename T>
__device__ __forceinline__ void clear_empty(const PagedArgs& p) {
  const int limit = paged_limit(p.c), n = p.c.Hq * p.c.hd;
  for (int b = blockIdx.x; b < p.c.B; b += gridDim.x)
    if (min(p.lengths[b], limit) <= 0)
      for (int i = threadIdx.x; i < n; i += blockDim.x) static_cast<T*>(p.o)[static_cast<long long>(b) * n + i] = from_f32<T>(0.f);
}

template <int HG>
__device__ __forceinline__ long long slot_floats(const CacheArgs& c) { return HG * (c.hd + 2); }

// The end of an item, or of this CTA's run inside one: the sums of `W` workers (o: [W][HG][pitch], m, l: [W][HG], base-2 maxima)
// become the output or a partial result.  All threads; begins and ends with a barrier of the CTA.
template <typename T, int HG, int W>
__device__ __forceinline__ void finish_item(const PagedArgs& p, int b, int item, bool whole, bool began_before, const float* o,
                                            int worker_stride, int pitch, const float (*m)[HG], const float (*l)[HG]) {
  const CacheArgs& c = p.c;
  const int G = c.Hq / c.Hkv, hgroups = (G + HG - 1) / HG, hk = item / hgroups, g0 = item % hgroups * HG, ng = min(HG, G - g0);
  float* slot = p.parts + (blockIdx.x * 2LL + (began_before ? 0 : 1)) * slot_floats<HG>(c);
  __syncthreads();
  for (int i = threadIdx.x; i < ng * (c.hd / 4); i += blockDim.x) {
    const int g = i / (c.hd / 4), d = i % (c.hd / 4) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, m[w][g]);
    const float ref = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (m[w][g] == -INFINITY && l[w][g] == 0.f) continue;   // saw nothing
      const float f = exp2f(m[w][g] - ref);
      const float4 x = *reinterpret_cast<const float4*>(o + w * worker_stride + g * pitch + d);
      sum = fmaf(l[w][g], f, sum);
      acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    }
    if (whole) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T* dst = static_cast<T*>(p.o) + (static_cast<long long>(b) * c.Hq + hk * G + g0 + g) * c.hd + d;
      Pack<T, 4> r;
      r.v[0] = from_f32<T>(acc.x * inv); r.v[1] = from_f32<T>(acc.y * inv);
      r.v[2] = from_f32<T>(acc.z * inv); r.v[3] = from_f32<T>(acc.w * inv);
      *reinterpret_cast<Pack<T, 4>*>(dst) = r;
    } else {
      *reinterpret_cast<float4*>(slot + g * c.hd + d) = acc;
      if (d == 0) {
        slot[HG * c.hd + g] = top;
        slot[HG * (c.hd + 1) + g] = sum;
      }
    }
  }
  __syncthreads();
}

// One CTA per CTA of the main kernel: the item that began in that one's run and went on behind it.  A warp takes a head's maxima
// and denominators, a lane a part's, and leaves the parts' weights in shared memory; then a thread adds four elements of the
// parts, eight loads in flight (a sequence alone on the card, 8 items on 296 CTAs, has 37 parts to a head: the join and its launch
// take 9 of 95 us, and 14 of 99 with two dependent passes over the parts).
template <typename T, int HG>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs p) {
  extern __shared__ float weight[];   // [HG][parts]
  __shared__ float inv[HG];
  dependency_wait();
  const CacheArgs& c = p.c;
  const int4 join = p.joins[blockIdx.x];   // sequence, item, last CTA, in use
  if (!join.w) return;
  const int G = c.Hq / c.Hkv, hgroups = (G + HG - 1) / HG, hk = join.y / hgroups, g0 = join.y % hgroups * HG, ng = min(HG, G - g0);
  const long long size = slot_floats<HG>(c);
  const int parts = join.z - blockIdx.x + 1, lane = threadIdx.x & 31;
  const auto part = [&](int r) { return p.parts + ((blockIdx.x + r) * 2LL + (r == 0 ? 1 : 0)) * size; };
  for (int g = threadIdx.x >> 5; g < ng; g += 4) {
    float top = -INFINITY, sum = 0.f;
    for (int r = lane; r < parts; r += 32) {
      const float m = part(r)[HG * c.hd + g];
      weight[g * parts + r] = m;
      top = fmaxf(top, m);
    }
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int r = lane; r < parts; r += 32) {
      const float f = exp2f(weight[g * parts + r] - ref);
      weight[g * parts + r] = f;
      sum = fmaf(part(r)[HG * (c.hd + 1) + g], f, sum);
    }
    sum = warp_sum(sum);
    if (lane == 0) inv[g] = sum == 0.f ? 0.f : 1.f / sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ng * (c.hd / 4); i += blockDim.x) {
    const int g = i / (c.hd / 4), d = i % (c.hd / 4) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int r = 0; r < parts; ++r) {
      const float f = weight[g * parts + r];
      const float4 x = *reinterpret_cast<const float4*>(part(r) + g * c.hd + d);
      acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    }
    T* dst = static_cast<T*>(p.o) + (static_cast<long long>(join.x) * c.Hq + hk * G + g0 + g) * c.hd + d;
    Pack<T, 4> o;
    o.v[0] = from_f32<T>(acc.x * inv[g]); o.v[1] = from_f32<T>(acc.y * inv[g]);
    o.v[2] = from_f32<T>(acc.z * inv[g]); o.v[3] = from_f32<T>(acc.w * inv[g]);
    *reinterpret_cast<Pack<T, 4>*>(dst) = o;
  }
}

constexpr int kPagedThreads = 128;

// At the last tile of a CTA's run, for the join: whether its item began in the run and goes on behind it, and up to which CTA.
template <int TILE, int HG>
__device__ __forceinline__ void note_join(const PagedArgs& p, const Run& run, const TileWalk<TILE, HG>& at) {
  if (threadIdx.x != 0 || p.joins == nullptr) return;
  const long long last = run.first + run.n - 1 + (at.n_tiles - 1 - at.t);   // the item's last tile
  const bool use = at.t < run.n && at.t + 1 < at.n_tiles;
  p.joins[blockIdx.x] = make_int4(at.b, at.item, static_cast<int>(last / run.per), use);
}

// ---- any head size, fp32 arithmetic on the CUDA cores.  L lanes hold a row (16 bytes each); every group of L lanes takes rows
// of its own, kBatch at a time, and keeps its own running maximum, sum and output.  Serves fp32 caches, whose products the
// matrix instructions would round, and head sizes that those do not take.  Four query heads share a row's loads: more would
// cost the registers that keep 16 warps on an SM.  Bound by the latency of page table and rows on short caches: 4 sequences of 777
// positions, 12 heads of 64: 12 us with the join (90 us as one CTA an item).
constexpr int kPagedHeads = 4;   // query heads that share the loads of a pass over the cache
constexpr int kPagedTile = 64;

template <typename T, int L>
__global__ void __launch_bounds__(kPagedThreads) paged_attention_kernel(const PagedArgs p) {
  constexpr int VN = 16 / sizeof(T), kRows = 32 / L, kGroups = kPagedThreads / L, kBatch = 4, HG = kPagedHeads;
  static_assert(kPagedTile % kGroups == 0 && kPagedTile / kGroups % kBatch == 0, "tile rows per group");
  __shared__ float sm_m[kGroups][HG], sm_l[kGroups][HG];
  __shared__ __align__(16) float sm_o[kGroups][HG][L * VN];
  dependency_wait();
  dependents_launch();
  const CacheArgs& c = p.c;
  const int lane = threadIdx.x & 31, grp = (threadIdx.x >> 5) * kRows + lane / L, d0 = (lane % L) * VN;
  const int G = c.Hq / c.Hkv, hgroups = (G + HG - 1) / HG, limit = paged_limit(c);
  const bool in_head = d0 < c.hd;
  TileWalk<kPagedTile, HG> walk;
  const Run run = begin_run<kPagedTile, HG, kPagedThreads>(p, walk);
  clear_empty<T>(p);
  if (run.n == 0) {
    if (threadIdx.x == 0 && p.joins) p.joins[blockIdx.x].w = 0;
    return;
  }
  const float sc = p.scale * 1.4426950408889634f;

  float q[HG][VN], o[HG][VN], m[HG], l[HG];
  bool began_before = walk.t > 0, fresh = true;
  for (int it = 0; it < run.n; ++it) {
    const int hk = walk.item / hgroups, g0 = walk.item % hgroups * HG;
    if (fresh) {
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int e = 0; e < VN; ++e) q[g][e] = o[g][e] = 0.f;
        if (g0 + g < G && in_head) {
          const Pack<T, VN> x = ld128(static_cast<const T*>(p.q) + walk.b * p.q_stride_b + static_cast<long long>(hk * G + g0 + g) * c.hd + d0);
#pragma unroll
          for (int e = 0; e < VN; ++e) q[g][e] = to_f32(x.v[e]) * sc;
        }
      }
      fresh = false;
    }
    const PageMap map = c.map(walk.b);
    // the rows of a batch are looked up under the loads of the batch before
    int next[kBatch];
    auto look_up = [&](int r) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int v = walk.t * kPagedTile + (r + u) * kGroups + grp;
        next[u] = v < walk.seen.n ? static_cast<int>(map.row(walk.seen.pos(v), c.Hkv, hk)) : -1;
        if (v < walk.seen.n && next[u] < 0) atomicExch(c.status, kStatusBadPage);
      }
    };
    look_up(0);
    for (int r = 0; r < kPagedTile / kGroups; r += kBatch) {
      int row[kBatch];
      Pack<T, VN> kx[kBatch], vx[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        row[u] = next[u];
        kx[u] = vx[u] = Pack<T, VN>{};
        if (row[u] >= 0 && in_head) {
          kx[u] = ld128(static_cast<const T*>(c.k_cache) + static_cast<long long>(row[u]) * c.hd + d0);
          vx[u] = ld128(static_cast<const T*>(c.v_cache) + static_cast<long long>(row[u]) * c.hd + d0);
        }
      }
      if (r + kBatch < kPagedTile / kGroups) look_up(r + kBatch);
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        if (g0 + g >= G) break;
        float s[kBatch], top = m[g];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          s[u] = 0.f;
#pragma unroll
          for (int e = 0; e < VN; ++e) s[u] = fmaf(q[g][e], to_f32(kx[u].v[e]), s[u]);
#pragma unroll
          for (int w = 1; w < L; w <<= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], w);
          if (row[u] < 0) s[u] = -INFINITY;
          top = fmaxf(top, s[u]);
        }
        const float ref = top == -INFINITY ? 0.f : top;   // nothing seen yet, or scores of -inf
        const float keep = exp2f(m[g] - ref);
        m[g] = top;
        l[g] *= keep;
#pragma unroll
        for (int e = 0; e < VN; ++e) o[g][e] *= keep;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const float x = exp2f(s[u] - ref);
          l[g] += x;
#pragma unroll
          for (int e = 0; e < VN; ++e) o[g][e] = fmaf(x, to_f32(vx[u].v[e]), o[g][e]);
        }
      }
    }
    const bool item_ends = walk.t + 1 == walk.n_tiles;
    if (item_ends || it + 1 == run.n) {
#pragma unroll
      for (int g = 0; g < HG; ++g) {
        if (lane % L == 0) {
          sm_m[grp][g] = m[g];
          sm_l[grp][g] = l[g];
        }
#pragma unroll
        for (int e = 0; e < VN; ++e) sm_o[grp][g][d0 + e] = o[g][e];
      }
      if (it + 1 == run.n) note_join(p, run, walk);
      finish_item<T, HG, kGroups>(p, walk.b, walk.item, item_ends && !began_before, began_before, &sm_o[0][0][0], HG * L * VN, L * VN,
                                  sm_m, sm_l);
      began_before = false;
      fresh = true;
    }
    if (it + 1 < run.n) walk.next(p, limit);
  }
}

// ---- bf16 heads of 64 and 128: matrix instructions on rows that arrive asynchronously
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 16 bytes into shared memory, or 16 zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void load_matrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// C[16 x 8] += A[16 x 16] B[16 x 8]
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kMmaHeads = 16;    // rows of the matrix instructions: the query heads of an item

template <int HD>
struct PagedMma {
  static constexpr int kKeys = 2048 / HD;              // rows of a warp's step: 4 KB of keys and 4 KB of values
  static constexpr int kTile = 4 * kKeys;              // of a CTA's
  static constexpr int kCtas = HD == 64 ? 3 : 2;        // that share an SM
  static constexpr int kStages = HD == 64 ? 2 : 3;
  static constexpr int kStepBytes = 2 * kKeys * HD * 2;
  static constexpr int kMeta = 4 * kStages * kStepBytes;
  static constexpr int kStat = kMeta + 4 * kStages * 16;
  static constexpr int kSmem = kStat + 2 * 4 * kMmaHeads * 4;
};

// Each of the four warps takes its quarter of every tile: it copies the rows into a ring of its own (no barrier of the CTA
// inside an item), multiplies them with the item's queries, keeps its own maximum, sum and output, and meets the others at
// the item's end.  The rows are swizzled (16-byte unit u of row r at u ^ (r & 7)), so that both the plain and the transposing
// matrix loads are free of bank conflicts.  UPPER: more than eight query heads in an item.
// Bound by memory: the cache is read once, and mma.sync, which pads the heads to 16 rows, needs a fifth of its rate for it.  Next
// to that counts the latency of a step's instructions, with eight to twelve warps on an SM: hd 64 is better off with three CTAs
// and two stages (192 sequences, window 1024 of up to 32768, 32 / 8 heads: 69 us, 5.6 TB/s; two CTAs and three stages 79 us),
// hd 128 the other way round (131071 positions, 32 / 8 heads: 94 us, 5.7 TB/s; 102 us).  64 sequences of up to 8192 positions, 32 / 8
// heads of 128: 97 us, 6.0 TB/s.  The first kernel, one CTA an item on the CUDA cores: 293 us, 21 ms, 1.35 ms.
// V is multiplied by P rounded to bf16 and by what that rounding left: without the second the output was off by 0.177 %, 0.165 %
// being its own rounding.  Up to eight heads leave half of the product's rows empty, which take the remainder for nothing; more
// heads take a second product (64 x 8192 positions, 32 / 2 heads of 128: 101 -> 105 us).
template <int HD, bool UPPER>
__global__ void __launch_bounds__(kPagedThreads, PagedMma<HD>::kCtas) paged_mma_kernel(const PagedArgs p) {
  using Cfg = PagedMma<HD>;
  constexpr int KEYS = Cfg::kKeys, STAGES = Cfg::kStages, HG = kMmaHeads;
  constexpr int kUnits = HD / 8, kRowsPerCopy = 32 / kUnits, kCopies = KEYS / kRowsPerCopy;
  extern __shared__ __align__(128) uint8_t smem[];
  dependency_wait();
  dependents_launch();
  const CacheArgs& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = c.Hq / c.Hkv, hgroups = (G + HG - 1) / HG, limit = paged_limit(c);
  uint8_t* ring = smem + warp * STAGES * Cfg::kStepBytes;
  int4* meta = reinterpret_cast<int4*>(smem + Cfg::kMeta) + warp * STAGES;
  float(*sm_m)[HG] = reinterpret_cast<float(*)[HG]>(smem + Cfg::kStat);
  float(*sm_l)[HG] = sm_m + 4;

  TileWalk<Cfg::kTile, HG> ahead;   // runs ahead of the arithmetic
  const Run run = begin_run<Cfg::kTile, HG, kPagedThreads>(p, ahead);
  clear_empty<bf16>(p);
  if (run.n == 0) {
    if (threadIdx.x == 0 && p.joins) p.joins[blockIdx.x].w = 0;
    return;
  }
  bool began_before = ahead.t > 0;

  // The cache row of this lane's key of the step that is copied next (-1: none), looked up a step early.
  int row = -1;
  auto look_up = [&]() {
    row = -1;
    const int v = ahead.t * Cfg::kTile + warp * KEYS + lane;
    if (lane < KEYS && v < ahead.seen.n) {
      row = static_cast<int>(c.map(ahead.b).row(ahead.seen.pos(v), c.Hkv, ahead.item / hgroups));
      if (row < 0) atomicExch(c.status, kStatusBadPage);
    }
  };
  int issued = 0;
  auto copy_step = [&]() {
    if (issued < run.n) {
      const int st = issued % STAGES;
      const uint32_t base = smem_addr(ring + st * Cfg::kStepBytes);
      const uint32_t real = __ballot_sync(0xffffffffu, row >= 0);
      if (lane == 0)
        meta[st] = make_int4(static_cast<int>(real), ahead.b, ahead.item, (ahead.t + 1 == ahead.n_tiles ? 1 : 0) | (ahead.t == 0 ? 2 : 0));
      if (issued + 1 == run.n) note_join(p, run, ahead);
      const int u = lane % kUnits;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int r = i * kRowsPerCopy + lane / kUnits;
        const int src = __shfl_sync(0xffffffffu, row, r);
        const long long off = static_cast<long long>(max(src, 0)) * HD + u * 8;
        const uint32_t dst = base + r * HD * 2 + ((u ^ (r & 7)) << 4);
        copy16(dst, static_cast<const bf16*>(c.k_cache) + off, src >= 0);
        copy16(dst + KEYS * HD * 2, static_cast<const bf16*>(c.v_cache) + off, src >= 0);
      }
      if (++issued < run.n) {
        ahead.next(p, limit);
        look_up();
      }
    }
    copy_commit();
  };

  uint32_t q[HD / 16][4];
  // sums of V times P rounded to bf16, and times what that rounding left: with up to eight heads in rows 8 .. 15 of the same
  // product, which would be empty, else (UPPER) in a product and an accumulator of their own
  float o[HD / 8][4], rest[UPPER ? HD / 8 : 1][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const float sc = p.scale * 1.4426950408889634f;
  const int gr = lane >> 2, tq = lane & 3;

  // An item's queries, and nothing accumulated: before the wait for its first rows.
  auto begin_item = [&](int b, int item) {
    const int hk = item / hgroups, g0 = item % hgroups * HG;
    const bf16* src = static_cast<const bf16*>(p.q) + b * p.q_stride_b + static_cast<long long>(hk * G + g0) * HD + tq * 2;
    const bool lo = g0 + gr < G, hi = UPPER && g0 + gr + 8 < G;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      q[k][0] = lo ? *reinterpret_cast<const uint32_t*>(src + gr * HD + k * 16) : 0u;
      q[k][2] = lo ? *reinterpret_cast<const uint32_t*>(src + gr * HD + k * 16 + 8) : 0u;
      q[k][1] = hi ? *reinterpret_cast<const uint32_t*>(src + (gr + 8) * HD + k * 16) : 0u;
      q[k][3] = hi ? *reinterpret_cast<const uint32_t*>(src + (gr + 8) * HD + k * 16 + 8) : 0u;
    }
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
      o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
      if (UPPER) rest[d][0] = rest[d][1] = rest[d][2] = rest[d][3] = 0.f;
    }
    m0 = m1 = -INFINITY;
    l0 = l1 = 0.f;
  };

  look_up();
  begin_item(ahead.b, ahead.item);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) copy_step();
  for (int it = 0; it < run.n; ++it) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    copy_step();   // into the stage that the step before this one has read
    const int st = it % STAGES;
    const int4 info = meta[st];
    const uint32_t real = static_cast<uint32_t>(info.x);
    if (real != 0) {
      const uint32_t kb = smem_addr(ring + st * Cfg::kStepBytes), vb = kb + KEYS * HD * 2;
      float s[KEYS / 8][4];
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int n = 0; n < KEYS / 16; ++n) {
        const int r = n * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t f[4];
          load_matrix4(f, kb + r * HD * 2 + (((2 * k + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
          mma16(s[2 * n], q[k], f[0], f[1]);
          mma16(s[2 * n + 1], q[k], f[2], f[3]);
        }
      }
      // scores in units of log 2; lanes of a quad share a head
      float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool see = real & (1u << (n * 8 + e)) << (2 * tq);
          s[n][e] = see ? s[n][e] * sc : -INFINITY;
          t0 = fmaxf(t0, s[n][e]);
          if (UPPER) {
            s[n][2 + e] = see ? s[n][2 + e] * sc : -INFINITY;
            t1 = fmaxf(t1, s[n][2 + e]);
          }
        }
      }
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
      if (UPPER) {
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
      }
      if (__any_sync(0xffffffffu, t0 > m0 || (UPPER && t1 > m1))) {
        const float n0 = fmaxf(m0, t0), a0 = exp2_fast(m0 - (n0 == -INFINITY ? 0.f : n0));
        float a1 = 1.f;
        m0 = n0;
        l0 *= a0;
        if (UPPER) {
          const float n1 = fmaxf(m1, t1);
          a1 = exp2_fast(m1 - (n1 == -INFINITY ? 0.f : n1));
          m1 = n1;
          l1 *= a1;
        }
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) {
          o[d][0] *= a0;
          o[d][1] *= a0;
          o[d][2] *= UPPER ? a1 : a0;
          o[d][3] *= UPPER ? a1 : a0;
          if (UPPER) {
            rest[d][0] *= a0;
            rest[d][1] *= a0;
            rest[d][2] *= a1;
            rest[d][3] *= a1;
          }
        }
      }
      const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t pf[KEYS / 16][4], pr[UPPER ? KEYS / 16 : 1][4];
      const auto left = [](float x0, float x1, uint32_t rounded) {
        return pack_bf16x2(x0 - __uint_as_float(rounded << 16), x1 - __uint_as_float(rounded & 0xffff0000u));
      };
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n) {
        const float x0 = exp2_fast(s[n][0] - r0), x1 = exp2_fast(s[n][1] - r0);
        l0 += x0 + x1;
        const uint32_t p0 = pack_bf16x2(x0, x1);
        pf[n / 2][(n & 1) * 2] = p0;
        if (UPPER) {
          const float y0 = exp2_fast(s[n][2] - r1), y1 = exp2_fast(s[n][3] - r1);
          l1 += y0 + y1;
          const uint32_t p1 = pack_bf16x2(y0, y1);
          pf[n / 2][(n & 1) * 2 + 1] = p1;
          pr[n / 2][(n & 1) * 2] = left(x0, x1, p0);
          pr[n / 2][(n & 1) * 2 + 1] = left(y0, y1, p1);
        } else {
          pf[n / 2][(n & 1) * 2 + 1] = left(x0, x1, p0);
        }
      }
#pragma unroll
      for (int n = 0; n < KEYS / 16; ++n) {
        const int r = n * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          uint32_t f[4];
          load_matrix4_t(f, vb + r * HD * 2 + (((2 * d + (lane >> 4)) ^ (r & 7)) << 4));
          mma16(o[2 * d], pf[n], f[0], f[1]);
          mma16(o[2 * d + 1], pf[n], f[2], f[3]);
          if (UPPER) {
            mma16(rest[2 * d], pr[n], f[0], f[1]);
            mma16(rest[2 * d + 1], pr[n], f[2], f[3]);
          }
        }
      }
    }
    const bool item_ends = info.w & 1;
    if (item_ends || it + 1 == run.n) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      if (tq == 0) {
        sm_m[warp][gr] = m0;
        sm_l[warp][gr] = l0;
        sm_m[warp][gr + 8] = m1;
        sm_l[warp][gr + 8] = l1;
      }
      // this warp's sums go where the step's rows were, which it has read; nothing is copied there before the next step
      __syncwarp();
      float* sum = reinterpret_cast<float*>(ring + st * Cfg::kStepBytes);
      // an infinite V is infinite in the first sum; what it makes of the second, whose weights have any sign, does not count
      const auto whole = [](float x, float r) { return fabsf(r) < INFINITY ? x + r : x; };
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        const float(&r)[4] = rest[UPPER ? d : 0];
        *reinterpret_cast<float2*>(sum + gr * HD + d * 8 + tq * 2) =
            make_float2(whole(o[d][0], UPPER ? r[0] : o[d][2]), whole(o[d][1], UPPER ? r[1] : o[d][3]));
        if (UPPER)
          *reinterpret_cast<float2*>(sum + (gr + 8) * HD + d * 8 + tq * 2) = make_float2(whole(o[d][2], r[2]), whole(o[d][3], r[3]));
      }
      finish_item<bf16, HG, 4>(p, info.y, info.z, item_ends && !began_before, began_before,
                               reinterpret_cast<const float*>(smem + st * Cfg::kStepBytes), STAGES * Cfg::kStepBytes / 4, HD, sm_m, sm_l);
      began_before = false;
      if (it + 1 < run.n) {   // whose rows are on their way
        const int4 next = meta[(it + 1) % STAGES];
        begin_item(next.y, next.z);
      }
    }
  }
}

static int cache_check(const TitbCacheDesc* d) {
  if (d->hd <= 0 || d->hd > 128 || d->hd % 8 || d->Hkv <= 0 || d->Hq % d->Hkv || d->page_size <= 0 || d->table_width < 0 ||
      d->n_pages < 0 || static_cast<long long>(d->n_pages) * d->Hkv > 0x7fffffffLL / d->page_size || d->sinks < 0 || d->window < 1 || (d->dtype != 0 && d->dtype != 1))
    return TITB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(d->k_cache) & 15) || (reinterpret_cast<uintptr_t>(d->v_cache) & 15)) return TITB_ERR_ALIGNMENT;
  return 0;
}

template <typename T>
static int append_launch(AppendArgs a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int half = a.c.hd / 2, heads = a.c.Hq + 2 * a.c.Hkv;
  const bool wide = half % V == 0;   // hd is a multiple of 8, so quarters of a row's half are always whole
  // whole tokens, as many to a CTA as make one wave (or several, of the most); few tokens: the heads are split over CTAs
  const long long tokens = static_cast<long long>(a.c.B) * a.T, want = device_sm_count() * 2LL, wave = device_sm_count() * static_cast<long long>(kAppendCtas);
  if (tokens * heads * (half / 4) > 0x7fffffffLL) return TITB_ERR_SHAPE;
  const long long each = (tokens + wave - 1) / wave;
  a.tokens = static_cast<int>(each < kAppendTokens ? each : kAppendTokens);
  long long splits = tokens >= want ? 1 : want / tokens;
  const int least = (kAppendThreads + half / (wide ? V : 4) - 1) / (half / (wide ? V : 4));   // heads that give each thread something to do
  a.per = static_cast<int>((heads + splits - 1) / splits);
  if (a.per < least) a.per = least < heads ? least : heads;
  const dim3 grid(static_cast<unsigned>((tokens + a.tokens - 1) / a.tokens), (heads + a.per - 1) / a.per);
  if (grid.y > 65535) return TITB_ERR_SHAPE;
  return static_cast<int>(wide ? launch_dependent(cache_append_kernel<T, V>, grid, dim3(kAppendThreads), 0, st, a)
                               : launch_dependent(cache_append_kernel<T, 4>, grid, dim3(kAppendThreads), 0, st, a));
}

// The grid of the attention over the cache follows what the page table could hold; the work is dealt on the device.
struct PagedPlan {
  bool mma, join;
  int heads, ctas;
};
static PagedPlan paged_plan(const TitbCacheDesc* d) {
  PagedPlan plan{};
  plan.mma = d->dtype == 1 && (d->hd == 64 || d->hd == 128);
  plan.heads = plan.mma ? kMmaHeads : kPagedHeads;
  const int tile = !plan.mma ? kPagedTile : d->hd == 64 ? PagedMma<64>::kTile : PagedMma<128>::kTile;
  const long long held = static_cast<long long>(d->table_width) * d->page_size, seen = static_cast<long long>(d->window) + d->sinks;
  const long long tiles = ((held < seen ? held : seen) + tile - 1) / tile;
  const int G = d->Hq / d->Hkv;
  const long long items = static_cast<long long>(d->B) * d->Hkv * ((G + plan.heads - 1) / plan.heads);
  // what fits on an SM: shared memory decides for the matrix kernel, registers for the other
  const long long most = device_sm_count() * static_cast<long long>(!plan.mma ? 4 : d->hd == 64 ? PagedMma<64>::kCtas : PagedMma<128>::kCtas);
  plan.ctas = static_cast<int>(tiles == 0 ? 1 : items > most / tiles ? most : items * tiles);
  plan.join = tiles > 1;   // otherwise every item is one tile
  return plan;
}
static long long plan_slot_floats(const TitbCacheDesc* d, const PagedPlan& plan) { return static_cast<long long>(plan.heads) * (d->hd + 2); }

template <typename K>
static int paged_launch(K kernel, const PagedArgs& a, const PagedPlan& plan, int smem, cudaStream_t st) {
  if (smem > 0) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return static_cast<int>(launch_dependent(kernel, dim3(plan.ctas), dim3(kPagedThreads), smem, st, a));
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

TITB_API long long titb_paged_attention_workspace(const TitbCacheDesc* d) {
  if (d->B <= 0 || d->Hq <= 0 || cache_check(d)) return 0;
  const PagedPlan plan = paged_plan(d);
  return plan.join ? plan.ctas * (2 * plan_slot_floats(d, plan) * 4 + static_cast<long long>(sizeof(int4))) : 0;
}

TITB_API int titb_paged_attention(const TitbCacheDesc* d, const void* q, long long q_stride_b, const int* lengths, float scale,
                                  void* o, void* workspace, cudaStream_t st) {
  (void)cudaGetLastError();
  if (d->B <= 0 || d->Hq <= 0) return 0;
  if (const int rc = cache_check(d)) return rc;
  auto bad = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (bad(q) || bad(o) || bad(workspace) || (q_stride_b & (d->dtype == 1 ? 7 : 3))) return TITB_ERR_ALIGNMENT;
  const PagedPlan plan = paged_plan(d);
  PagedArgs a{};
  a.c = cache_args(d);
  a.q = q; a.q_stride_b = q_stride_b; a.lengths = lengths; a.o = o; a.scale = scale;
  if (plan.join) {
    a.joins = static_cast<int4*>(workspace);
    a.parts = reinterpret_cast<float*>(a.joins + plan.ctas);
  }
  int rc;
  if (plan.mma) {
    const bool upper = d->Hq / d->Hkv > 8;
    if (d->hd == 64)
      rc = upper ? paged_launch(paged_mma_kernel<64, true>, a, plan, PagedMma<64>::kSmem, st)
                 : paged_launch(paged_mma_kernel<64, false>, a, plan, PagedMma<64>::kSmem, st);
    else
      rc = upper ? paged_launch(paged_mma_kernel<128, true>, a, plan, PagedMma<128>::kSmem, st)
                 : paged_launch(paged_mma_kernel<128, false>, a, plan, PagedMma<128>::kSmem, st);
  } else if (d->dtype == 1) {
    rc = d->hd <= 64 ? paged_launch(paged_attention_kernel<bf16, 8>, a, plan, 0, st)
                     : paged_launch(paged_attention_kernel<bf16, 16>, a, plan, 0, st);
  } else {
    rc = d->hd <= 64 ? paged_launch(paged_attention_kernel<float, 16>, a, plan, 0, st)
                     : paged_launch(paged_attention_kernel<float, 32>, a, plan, 0, st);
  }
  if (rc != 0 || !plan.join) return rc;
  auto join = d->dtype == 0 ? paged_join_kernel<float, kPagedHeads> : plan.mma ? paged_join_kernel<bf16, kMmaHeads> : paged_join_kernel<bf16, kPagedHeads>;
  return static_cast<int>(launch_dependent(join, dim3(plan.ctas), dim3(128), plan.heads * plan.ctas * 4, st, a));
}
