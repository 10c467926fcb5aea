// Log probability of a given token for each row of logits, the entropy of the
// row and its top alternatives; and the gradient of the logits.
//
//   m = max_j x_j,  c_j = x_j - m,  S = sum_j e^c_j
//   logprob_j = c_j - log S                (m and log S apart: m + log S would
//                                           round away a logprob near 0)
//   entropy   = log S - sum_j e^c_j c_j / S
//   dx_j = gl (d_jt - p_j) + sum_i gk_i (d_{j,id_i} - p_j) - gH p_j (logprob_j + entropy)
//
// One pass over the row: every thread keeps (m, S, Q = sum e^c c) of what it
// has read, and two such triples join as
//   m' = max(m1, m2), S' = S1 f1 + S2 f2, Q' = f1 (Q1 + S1 (m1 - m')) + f2 (...),
//   fi = e^(mi - m').
// The running max starts at the lowest finite value, not -inf, so that m - m
// is never inf - inf: a masked column (-inf) adds e^-inf = 0 to S, and its
// product with c is dropped.  A row with no column left (S = 0) gives logprob
// -inf, entropy 0 and no gradient; a row with a NaN or +inf gives NaN.
//
// Alternatives are the top_k largest logits, ties to the lowest index; in a
// NaN row every column ties.  They come out of the same pass: a thread's own
// maximum is at hand when it is over, the top_k-th largest of 128 maxima (of
// groups of threads) is a bound that at least top_k columns reach and about
// top_k more do not pass, and only the threads whose maximum reaches it read
// their columns again (from L2).
//
// A row is read by one CTA, or, where there are fewer rows than SMs, by a
// cluster of up to 8 whose parts are joined over distributed shared memory.
// Rows may start at any alignment: a thread works on whole 16-byte chunks of
// the address space, and the first and the last chunk of a row element by
// element.

// Memory bounds it, the exponentials close behind: at the copy rate the forward
// would use 0.7 of the SFUs' rate for bf16.  Products and sums go two to an
// instruction, rescaling by a new maximum is a branch that few chunks take, and
// a warp's threads meet over one common maximum.  Measured (B200): 16376 x 32000
// bf16 with entropy 183 us (0.88 of the 6536 GB/s copy rate), its gradient 358
// us (0.90); 4 x 32000 fp32 with 20 alternatives 8 us, 24 x 256000 with 64 17 us;
// 4096 x 32000 with 20 alternatives 81 us against 53 without any.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>

#include "common.cuh"
#include "step_ops.h"

namespace gmdn {
namespace {

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;

constexpr int kSms = 148;
constexpr int kMaxThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int kGroups = 128;   // maxima the bound is taken from
constexpr int kList = 1024;    // columns above the bound, or at it, that are kept
static_assert(kList >= kMaxCluster * kMaxTopK, "rank 0 joins the cluster's lists in one");
// Logarithms are clamped here where they multiply a factor e^c: that is 0 long
// before, and 0 * -inf, or a sum of S times a mask's -3e38, is not a number.
constexpr float kFar = -1000.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = 1.925962991e-08f;   // what fp32 leaves of log2 e

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 pair(float a) { return make_float2(a, a); }

struct Stat {
  float m, s, q;
};
// A warp's threads joined: one maximum, every thread's sums brought to it, plain sums.  `kWidth`
// lanes in all (a power of two); every lane gets the result.
template <int kWidth>
__device__ __forceinline__ Stat join_lanes(Stat a) {
  float m = a.m;
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  const float d = fmaxf(a.m - m, kFar), f = ex2(d * kLog2e);
  a.q = f * fmaf(a.s, d, a.q);
  a.s *= f;
  a.m = m;
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(~0u, a.s, o);
    a.q += __shfl_xor_sync(~0u, a.q, o);
  }
  return a;
}

// 16 bytes of a row
template <typename T>
struct Chunk;
template <>
struct Chunk<bf16> {
  static constexpr int E = 8;
  uint32_t w[4];
  __device__ __forceinline__ float2 get(int k) const {
    return make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
  }
  __device__ __forceinline__ void set(int i, float v) {   // i constant after unrolling
    const uint32_t b = f32_to_bf16(v);
    w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | (b << 16) : (w[i / 2] & 0xffff0000u) | b;
  }
  __device__ __forceinline__ float largest() const {   // NaN left out
    __nv_bfloat162 h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = *reinterpret_cast<const __nv_bfloat162*>(&w[k]);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <>
struct Chunk<float> {
  static constexpr int E = 4;
  uint32_t w[4];
  __device__ __forceinline__ float2 get(int k) const {
    return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
  }
  __device__ __forceinline__ void set(int i, float v) { w[i] = __float_as_uint(v); }
  __device__ __forceinline__ float largest() const {
    return fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])),
                 fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
  }
};
template <typename T>
__device__ __forceinline__ float value(const Chunk<T>& c, int i) {
  const float2 v = c.get(i / 2);
  return i & 1 ? v.y : v.x;
}
template <typename T>
__device__ __forceinline__ float element(const T* p) {
  return static_cast<float>(*p);
}

// A row as chunks: chunk j holds elements first(j) .. first(j) + E - 1, those
// outside the row read as -inf.
template <typename T>
struct Row {
  static constexpr int E = Chunk<T>::E;
  const T* x;
  int V, off, chunks, full0, full1;   // chunks full0 .. full1 - 1 lie wholly in the row
  __device__ __forceinline__ Row(const T* row, int vocab) : x(row), V(vocab) {
    off = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    chunks = (off + V - 1) / E + 1;
    full0 = off ? 1 : 0;
    full1 = (off + V) / E;
  }
  __device__ __forceinline__ Chunk<T> load_full(int j) const {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(x - off) + j);
    Chunk<T> c;
    c.w[0] = r.x;
    c.w[1] = r.y;
    c.w[2] = r.z;
    c.w[3] = r.w;
    return c;
  }
  __device__ __forceinline__ int first(int j) const { return j * E - off; }
  __device__ __forceinline__ Chunk<T> load(int j) const {
    if (j >= full0 && j < full1) return load_full(j);
    const int i0 = first(j);
    Chunk<T> c;
#pragma unroll
    for (int k = 0; k < E; ++k)
      c.set(k, i0 + k >= 0 && i0 + k < V ? element(x + i0 + k) : -INFINITY);
    return c;
  }
};

// (value, index) in one key: larger value first, then the lower index.
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
  uint32_t u = __float_as_uint(v + 0.f);   // -0 is 0
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<unsigned long long>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int key_index(unsigned long long k) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct __align__(16) TopShared {
  unsigned long long above[kList], at[kList];
  unsigned long long best[kMaxTopK];
  float thread_max[kMaxThreads], group_max[kGroups];
  unsigned long long warp_best[kMaxThreads / 32];
  int warp_count[kMaxThreads / 32];
  int hot[kMaxThreads];   // threads whose maximum reaches the bound
  int n_hot, n_above, n_at;
  uint32_t bound;         // ordered()
};

// The place of key k among n keys, largest first.  The keys' storage may be read up to the
// next multiple of 8 (what lies there is not counted).
__device__ __forceinline__ int place(const unsigned long long* keys, int n, unsigned long long k) {
  int r = 0;
  for (int i = 0; i < n; i += 8) {
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(keys + i + u);
      r += (v.x > k && i + u < n) + (v.y > k && i + u + 1 < n);
    }
  }
  return r;
}

// The largest columns of chunks [c0, c1) into sh.best, falling: k of them, or all and then 0
// (no column's key).  `mine`: the thread's largest value (at least -FLT_MAX) over chunks
// c0 + tid, + blockDim, ....  In a row with NaN the result means nothing.
template <typename T>
__device__ void top_columns(TopShared& sh, const Row<T>& row, int c0, int c1, int k, float mine) {
  constexpr int E = Chunk<T>::E;
  const int tid = threadIdx.x, n = blockDim.x, lane = tid & 31, w = tid >> 5;
  sh.thread_max[tid] = mine;
  if (tid < k) sh.best[tid] = 0;
  if (tid == 0) {
    sh.n_hot = sh.n_above = sh.n_at = 0;
    sh.bound = 0;
  }
  __syncthreads();
  if (tid < kGroups) {
    // groups of threads far apart: chunks that lie together fall into different groups
    float g = mine;
    for (int t = tid + kGroups; t < n; t += kGroups) g = fmaxf(g, sh.thread_max[t]);
    sh.group_max[tid] = g;
  }
  __syncthreads();
  if (tid < kGroups) {   // the largest maximum that k of them reach
    const float g = sh.group_max[tid];
    int reach = 0;
#pragma unroll 8
    for (int t = 0; t < kGroups; t += 4) {
      const float4 o = *reinterpret_cast<const float4*>(sh.group_max + t);
      reach += (o.x >= g) + (o.y >= g) + (o.z >= g) + (o.w >= g);
    }
    const uint32_t top = __reduce_max_sync(~0u, reach >= k ? ordered(g) : 0u);
    if (lane == 0) atomicMax(&sh.bound, top);
  }
  __syncthreads();
  const uint32_t ub = sh.bound;
  const float bound = __uint_as_float((ub & 0x80000000u) ? (ub & 0x7fffffffu) : ~ub);
  const int lo = max(row.first(c0), 0), hi = min(row.first(c1), row.V);
  const int want = max(min(k, hi - lo), 0);
  if (mine >= bound) sh.hot[atomicAdd(&sh.n_hot, 1)] = tid;
  __syncthreads();
  // the hot threads' chunks, 16 lanes a thread: read again, from L1 or L2
  const int each = (c1 - c0 + n - 1) / n, n_hot = sh.n_hot;
  auto keep = [&](const Chunk<T>& c, int j) {
    if (!(c.largest() >= bound)) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = value(c, e);
      const int col = row.first(j) + e;
      if (v >= bound && col >= 0 && col < row.V) {
        int* count = v > bound ? &sh.n_above : &sh.n_at;
        unsigned long long* list = v > bound ? sh.above : sh.at;
        const int slot = atomicAdd(count, 1);
        if (slot < kList) list[slot] = key_of(v, col);
      }
    }
  };
  for (int h = tid / 16; h < n_hot; h += n / 8) {
    const int h2 = h + n / 16;
    const int j0 = c0 + sh.hot[h], j1 = h2 < n_hot ? c0 + sh.hot[h2] : c1;
    for (int i = (tid & 15) * n; i < each * n; i += 16 * n) {
      Chunk<T> a, b;
      if (j0 + i < c1) a = row.load(j0 + i);
      if (j1 + i < c1) b = row.load(j1 + i);
      if (j0 + i < c1) keep(a, j0 + i);
      if (j1 + i < c1) keep(b, j1 + i);
    }
  }
  __syncthreads();
  const int na = sh.n_above, nt = sh.n_at;
  if (na > kList) {
    // more columns above the bound than the list holds (they all lie in few threads): one
    // column a round, the largest below the last
    unsigned long long last = ~0ull;
    for (int r = 0; r < want; ++r) {
      unsigned long long b = 0;
      for (int j = c0 + tid; j < c1; j += n) {
        const Chunk<T> c = row.load(j);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = row.first(j) + e;
          const unsigned long long q = key_of(value(c, e), i);
          if (i >= 0 && i < row.V && q < last && q > b) b = q;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(~0u, b, o);
        if (q > b) b = q;
      }
      __syncthreads();
      if (lane == 0) sh.warp_best[w] = b;
      __syncthreads();
      for (int i = 0; i < n / 32; ++i)
        if (sh.warp_best[i] > b) b = sh.warp_best[i];
      last = b;
      if (tid == 0) sh.best[r] = b;
    }
    __syncthreads();
    return;
  }
  for (int i = tid; i < na; i += n) {
    const int r = place(sh.above, na, sh.above[i]);
    if (r < want) sh.best[r] = sh.above[i];
  }
  int have = min(na, want);
  if (have < want && nt <= kList) {
    for (int i = tid; i < nt; i += n) {
      const int r = na + place(sh.at, nt, sh.at[i]);
      if (r < want) sh.best[r] = sh.at[i];
    }
    have = min(na + nt, want);
  }
  // Too many columns at the bound to list, or (bound -FLT_MAX) columns at -inf are needed too:
  // the first ones in order, tile by tile.
  float tie = nt <= kList ? -INFINITY : bound;
  for (int pass = 0; pass < 2 && have < want; ++pass) {
    int found = 0;
    for (int base = c0; base < c1 && have + found < want; base += n) {
      const int j = base + tid;
      uint32_t hits = 0;
      if (j < c1) {
        const Chunk<T> c = row.load(j);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = row.first(j) + e;
          if (value(c, e) == tie && i >= 0 && i < row.V) hits |= 1u << e;
        }
      }
      const int mine_n = __popc(hits);
      int before = mine_n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, before, o);
        if (lane >= o) before += v;
      }
      __syncthreads();
      if (lane == 31) sh.warp_count[w] = before;
      __syncthreads();
      before -= mine_n;
      int total = 0;
      for (int i = 0; i < n / 32; ++i) {
        if (i < w) before += sh.warp_count[i];
        total += sh.warp_count[i];
      }
      for (int e = 0; e < E; ++e)
        if (hits >> e & 1) {
          const int r = have + found + before++;
          if (r < want) sh.best[r] = key_of(tie, row.first(j) + e);
        }
      found += total;
    }
    have = min(have + found, want);
    tie = -INFINITY;   // below the lowest finite value there is nothing else
  }
  __syncthreads();
}

// Max, sum and (kEnt) entropy sum of U chunks.
template <typename T, bool kEnt, int U>
__device__ __forceinline__ void absorb(const Chunk<T>* c, float& m, float2& s, float2& q) {
  constexpr int P = Chunk<T>::E / 2;
  float top = c[0].largest();
#pragma unroll
  for (int u = 1; u < U; ++u) top = fmaxf(top, c[u].largest());
  if (top > m) {
    const float d = fmaxf(m - top, kFar), f = ex2(d * kLog2e);
    if constexpr (kEnt) {
      q.x = f * fmaf(s.x, d, q.x);
      q.y = f * fmaf(s.y, d, q.y);
    }
    s = __fmul2_rn(s, pair(f));
    m = top;
  }
  const float2 nm = pair(-m);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float2 d = __fadd2_rn(c[u].get(k), nm);
      const float2 y = __fmul2_rn(d, pair(kLog2e));
      const float2 e = make_float2(ex2(y.x), ex2(y.y));   // NaN stays
      s = __fadd2_rn(s, e);
      if constexpr (kEnt) {
        d = make_float2(fmaxf(d.x, kFar), fmaxf(d.y, kFar));
        q = __ffma2_rn(e, d, q);
      }
    }
}

constexpr int kUnroll = 4;

template <typename T, bool kEnt, bool kTop, bool kCluster>
__global__ void __launch_bounds__(kMaxThreads) logprobs_fwd_kernel(LogprobArgs p) {
  extern __shared__ __align__(16) char dyn[];   // kTop: TopShared
  __shared__ Stat warp_stat[kMaxThreads / 32];
  __shared__ Stat cta_stat;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, n = blockDim.x;
  int parts = 1, rank = 0;
  if constexpr (kCluster) {
    parts = cg::this_cluster().num_blocks();
    rank = cg::this_cluster().block_rank();
  }
  const long long r = blockIdx.x / parts;
  const long long b = r / p.length;
  const T* x = static_cast<const T*>(p.logits) + b * p.stride_b + (r - b * p.length) * p.stride_t;
  const Row<T> row(x, p.vocab);
  // the given token's logit, on its way while the row is read
  const bool writer = rank == 0 && tid == 0;
  int64_t t = 0;
  float xt = 0.f;
  if (writer && p.logprobs) {
    t = p.targets[r];
    if (t >= 0 && t < p.vocab) xt = element(x + t);
  }
  const int per = (row.chunks + parts - 1) / parts;
  const int c0 = min(rank * per, row.chunks), c1 = min(c0 + per, row.chunks);
  float m = -FLT_MAX;
  float2 s = pair(0.f), q = pair(0.f);
  int j = c0 + tid;
  const int c1f = min(c1, row.full1);
  if (j < row.full0) {   // a row's first chunk, if short
    const Chunk<T> c = row.load(j);
    absorb<T, kEnt, 1>(&c, m, s, q);
    j += n;
  }
  // kUnroll chunks at a time, the next ones on their way while these are summed
  auto fetch = [&](int at, Chunk<T>* c) {
    if (at + (kUnroll - 1) * n < c1f) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) c[u] = row.load_full(at + u * n);
      return;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (at + u * n < c1) {
        c[u] = row.load(at + u * n);
      } else {
#pragma unroll
        for (int k = 0; k < Chunk<T>::E; ++k) c[u].set(k, -INFINITY);
      }
    }
  };
  Chunk<T> now[kUnroll], next[kUnroll];
  if (j < c1) fetch(j, now);
  for (; j < c1; j += kUnroll * n) {
    if (j + kUnroll * n < c1) fetch(j + kUnroll * n, next);
    absorb<T, kEnt, kUnroll>(now, m, s, q);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) now[u] = next[u];
  }
  const float mine = m;
  Stat a = join_lanes<32>(Stat{m, s.x + s.y, q.x + q.y});
  if (lane == 0) warp_stat[w] = a;
  __syncthreads();
  if (kTop || w == 0) {   // the warps whose results are used
    const int warps = n / 32;
    a = lane % 16 < warps ? warp_stat[lane % 16] : Stat{-FLT_MAX, 0.f, 0.f};
    a = join_lanes<16>(a);
  }
  TopShared& sh = *reinterpret_cast<TopShared*>(dyn);
  if constexpr (kTop) top_columns(sh, row, c0, c1, p.top_k, mine);
  if constexpr (kCluster) {
    // rank 0 takes the parts together: the stats, and the lists of alternatives
    auto cluster = cg::this_cluster();
    if (tid == 0) cta_stat = a;
    cluster.sync();
    if (rank == 0) {
      a = lane % 8 < parts ? *cluster.map_shared_rank(&cta_stat, lane % 8)
                           : Stat{-FLT_MAX, 0.f, 0.f};
      a = join_lanes<8>(a);
      if constexpr (kTop) {
        const int all = parts * p.top_k;
        for (int i = tid; i < all; i += n)
          sh.above[i] = cluster.map_shared_rank(&sh, i / p.top_k)->best[i % p.top_k];
        __syncthreads();
        // a column's place: its rank in every part's falling list, found by halving, all the
        // lists a step at a time
        for (int i = tid; i < all; i += n) {
          const unsigned long long key = sh.above[i];
          int ahead[kMaxCluster] = {};
          for (int step = kMaxTopK; step > 0; step >>= 1) {
            if (step > p.top_k) continue;
#pragma unroll
            for (int l = 0; l < kMaxCluster; ++l) {
              const int to = ahead[l] + step;
              if (l < parts && to <= p.top_k && sh.above[l * p.top_k + to - 1] > key) ahead[l] = to;
            }
          }
          int at = 0;
#pragma unroll
          for (int l = 0; l < kMaxCluster; ++l) at += ahead[l];
          if (key && at < p.top_k) sh.best[at] = key;
        }
        __syncthreads();
      }
    }
    cluster.sync();   // the others' shared memory is read until here
    if (rank != 0) return;
  }
  const bool empty = a.s == 0.f, bad = !(a.s >= 0.f) || a.m == INFINITY;
  const float ls = logf(a.s), nan = __int_as_float(0x7fffffff);
  auto logprob = [&](float v) { return bad ? nan : (empty ? -INFINITY : (v - a.m) - ls); };
  if (writer) {
    const float H = bad ? nan : (empty ? 0.f : ls - a.q / a.s);
    if (p.stats)
      reinterpret_cast<float4*>(p.stats)[r] = make_float4(a.m, bad ? nan : ls, kEnt ? H : nan,
                                                            bad ? nan : a.s);
    if (p.entropy) p.entropy[r] = H;
    if (p.logprobs)
      p.logprobs[r] = t == p.ignore_index ? 0.f : (t >= 0 && t < p.vocab ? logprob(xt) : nan);
  }
  if constexpr (kTop) {
    if (tid < p.top_k) {
      const long long o = r * p.top_k + tid;
      p.top_ids[o] = bad ? tid : key_index(sh.best[tid]);
      p.top_logprobs[o] = bad ? nan : logprob(key_value(sh.best[tid]));
    }
  }
}

// ---------------------------------------------------------------------------
// gradient
// ---------------------------------------------------------------------------

constexpr int kBwdThreads = 256;   // at most; at least kMaxTopK
constexpr int kBwdUnroll = 4;

// Elements i0 .. i0 + E - 1 of a row that lies `shift` elements above a 16-byte
// boundary there: the two aligned chunks that hold them, shifted together.
template <typename T>
__device__ __forceinline__ Chunk<T> load_shifted(const T* x, int i0, int shift) {
  Chunk<T> c;
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(x + i0 - shift));
  if (shift == 0) {
    c.w[0] = a.x;
    c.w[1] = a.y;
    c.w[2] = a.z;
    c.w[3] = a.w;
    return c;
  }
  const uint4 b = __ldg(reinterpret_cast<const uint4*>(x + i0 - shift) + 1);
  uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const int bytes = shift * static_cast<int>(sizeof(T));
  if (bytes & 8) {
#pragma unroll
    for (int k = 0; k < 6; ++k) v[k] = v[k + 2];
  }
  if (bytes & 4) {
#pragma unroll
    for (int k = 0; k < 5; ++k) v[k] = v[k + 1];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) c.w[k] = bytes & 2 ? __funnelshift_r(v[k], v[k + 1], 16) : v[k];
  return c;
}

// Grid: `parts` CTAs a row.  The gradient of a column is p (A + B logprob),
// A = -(w + gH H), B = -gH, w = gl + sum gk; the given token's column has gl
// on top where it is computed, the alternatives' columns are written again at
// the end, each by one thread.
template <typename T, bool kEnt, bool kTop>
__global__ void __launch_bounds__(kBwdThreads) logprobs_bwd_kernel(LogprobArgs p, int parts) {
  constexpr int E = Chunk<T>::E, U = kBwdUnroll;
  // 32-bit divisions: the grid has fewer than 2^31 CTAs, so there are fewer rows than that
  const uint32_t ru = blockIdx.x / static_cast<uint32_t>(parts);
  const uint32_t b = ru / static_cast<uint32_t>(p.length);
  const long long r = ru;
  const int part = static_cast<int>(blockIdx.x - ru * parts), tid = threadIdx.x, n = blockDim.x;
  const T* x = static_cast<const T*>(p.logits) + b * p.stride_b + (r - b * p.length) * p.stride_t;
  T* out = static_cast<T*>(p.dlogits) + r * p.vocab;
  const int V = p.vocab;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T));
  const int chunks = (off + V - 1) / E + 1;
  // every chunk of `out` starts `shift` elements above a boundary of the logits
  const int shift =
      static_cast<int>((reinterpret_cast<uintptr_t>(x) / sizeof(T) + E - off) % E);
  const int c0 = part * n * U;
  // chunks of `out` that lie wholly in the row; with shift 0 those of the logits too
  const int full0 = off ? 1 : 0, full1 = (off + V) / E;
  uint4* out16 = reinterpret_cast<uint4*>(out - off);
  auto load_edge = [&](int j) {
    const int i0 = j * E - off;
    if (i0 - shift >= 0 && i0 - shift + (shift ? 2 * E : E) <= V) return load_shifted(x, i0, shift);
    Chunk<T> c;
#pragma unroll
    for (int k = 0; k < E; ++k)
      c.set(k, i0 + k >= 0 && i0 + k < V ? element(x + i0 + k) : -INFINITY);
    return c;
  };
  Chunk<T> c[U];
  if (shift == 0) {
    const uint4* in16 = reinterpret_cast<const uint4*>(x - off);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = c0 + u * n + tid;
      if (j >= full0 && j < full1) {
        const uint4 v = __ldcs(in16 + j);
        c[u].w[0] = v.x;
        c[u].w[1] = v.y;
        c[u].w[2] = v.z;
        c[u].w[3] = v.w;
      } else if (j < chunks) {
        c[u] = load_edge(j);
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * n + tid < chunks) c[u] = load_edge(c0 + u * n + tid);
  }
  const float4 st = __ldg(reinterpret_cast<const float4*>(p.stats) + r);
  const float m = st.x, ls = st.y, nan = __int_as_float(0x7fffffff);
  const float gh = kEnt && p.g_entropy ? p.g_entropy[r] : 0.f;
  int t = -1;
  float gl = 0.f;
  if (p.g_logprobs) {
    const int64_t tt = p.targets[r];
    if (tt != p.ignore_index) {
      const bool ok = tt >= 0 && tt < V;
      gl = p.g_logprobs[r];
      if (!ok && gl != 0.f) gl = nan;
      t = ok ? static_cast<int>(tt) : -1;
    }
  }
  float wsum = gl;
  // alternative `tid`, on its way while the row is worked on
  int64_t top_i = -1;
  float top_g = 0.f;
  bool any_top = false;
  if constexpr (kTop) {
    const int lane = tid & 31;
    const float* gk = p.g_top + r * p.top_k;
    if (tid < p.top_k) {
      top_i = p.top_ids[r * p.top_k + tid];
      top_g = gk[tid];
    }
    const float g0 = lane < p.top_k ? gk[lane] : 0.f;
    const float g1 = lane + 32 < p.top_k ? gk[lane + 32] : 0.f;
    any_top = g0 != 0.f || g1 != 0.f;   // NaN too
    wsum += warp_sum(g0 + g1);
  }
  // No gradient: a row without columns, and one whose cotangents are all 0 (an ignored target),
  // whatever it holds.
  const bool zero = ls == -INFINITY ||
                    (gl == 0.f && gh == 0.f && !(kTop && __any_sync(~0u, any_top)));
  const float A = kEnt ? -fmaf(gh, st.z, wsum) : -wsum, B = -gh;
  // 1 / S where a gradient's fp32 digits need it (stats made by hand may leave S at 0)
  const float inv = sizeof(T) == 4 ? (st.w > 0.f ? __fdiv_rn(1.f, st.w) : expf(-ls)) : 0.f;
  auto grad2 = [&](float2 v) {
    float2 c = __fadd2_rn(v, pair(-m)), e, lp;
    if constexpr (sizeof(T) == 4) {
      // p = e^c / S: e^(c - log S) would round its exponent twice, |logprob| 2^-24 each, and the
      // product with log2 e once more; here its rounding, and that of log2 e, goes into the
      // exponential as 1 + l log 2.  A NaN row has NaN in S.
      c = make_float2(fmaxf(c.x, kFar), fmaxf(c.y, kFar));
      const float2 y = __fmul2_rn(c, pair(kLog2e));
      float2 l = __ffma2_rn(c, pair(kLog2e), make_float2(-y.x, -y.y));
      l = __ffma2_rn(c, pair(kLog2eLow), l);
      e = make_float2(ex2(y.x), ex2(y.y));
      e = __fmul2_rn(e, __ffma2_rn(l, pair(inv * 0.6931471805599453f), pair(inv)));
      lp = __fadd2_rn(c, pair(-ls));   // at least kFar - log S
    } else {
      lp = __fadd2_rn(c, pair(-ls));
      const float2 y = __fmul2_rn(lp, pair(kLog2e));
      e = make_float2(ex2(y.x), ex2(y.y));
    }
    if constexpr (kEnt) {
      if constexpr (sizeof(T) == 2) lp = make_float2(fmaxf(lp.x, kFar), fmaxf(lp.y, kFar));
      return __fmul2_rn(e, __ffma2_rn(lp, pair(B), pair(A)));
    }
    return __fmul2_rn(e, pair(A));
  };
  const int tj = t >= 0 ? (t + off) / E : -1;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int j = c0 + u * n + tid;
    if (j >= chunks) break;
    float2 g[E / 2];
#pragma unroll
    for (int k = 0; k < E / 2; ++k) g[k] = pair(0.f);
    if (!zero) {
#pragma unroll
      for (int k = 0; k < E / 2; ++k) g[k] = grad2(c[u].get(k));
      if (j == tj) {
        const int at = t + off - j * E;
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          if (2 * k == at) g[k].x += gl;
          if (2 * k + 1 == at) g[k].y += gl;
        }
      }
    }
    if (j >= full0 && j < full1) {
      uint4 o;
      if constexpr (sizeof(T) == 2) {
        __nv_bfloat162 h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(g[k].x, g[k].y);
        o = *reinterpret_cast<uint4*>(h);
      } else {
        o = make_uint4(__float_as_uint(g[0].x), __float_as_uint(g[0].y), __float_as_uint(g[1].x),
                       __float_as_uint(g[1].y));
      }
      out16[j] = o;
    } else {
      const int i0 = j * E - off;
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (i0 + k >= 0 && i0 + k < V)
          out[i0 + k] = static_cast<T>(k & 1 ? g[k / 2].y : g[k / 2].x);
    }
  }
  if constexpr (kTop) {
    const bool here = top_i >= max(c0 * E - off, 0) && top_i < min((c0 + n * U) * E - off, V);
    const float v = here ? grad2(pair(element(x + top_i))).x + top_g + (top_i == t ? gl : 0.f) : 0.f;
    __syncthreads();
    if (here && !zero) out[top_i] = static_cast<T>(v);
  }
}

template <typename T, bool kEnt, bool kTop>
cudaError_t launch_fwd(const LogprobArgs& p, cudaStream_t st) {
  const long long rows = p.batch * p.length;
  const int chunks = (p.vocab * static_cast<long long>(sizeof(T)) + 15) / 16;
  // fewer rows than SMs: a cluster a row, as long as a part keeps a thread of the smallest CTA
  // busy
  int parts = 1;
  while (parts < kMaxCluster && rows * parts < kSms && chunks / (2 * parts) >= 128) parts *= 2;
  const int per = chunks / parts;
  // Threads a CTA by how many CTAs an SM gets: one is bound by latency and takes as many as have
  // a chunk; with four or more, 128 threads make the most of what a CTA does once (16376 x 32000
  // bf16: 183 us against 203 with 256; 300 x 256000: 45 us with 256, 64 with 128).
  const long long ctas = rows * parts;
  int threads = ctas <= kSms ? 512 : (ctas < 4 * kSms ? 256 : 128);
  while (threads > 128 && per < threads) threads /= 2;
  if (rows * parts > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const size_t smem = kTop ? sizeof(TopShared) : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return parts > 1 ? cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, kEnt, kTop, true>, p)
                   : cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, kEnt, kTop, false>, p);
}
template <typename T>
cudaError_t fwd_typed(const LogprobArgs& p, cudaStream_t st) {
  // the entropy is also what a backward through it reads from the stats
  if (p.entropy)
    return p.top_k ? launch_fwd<T, true, true>(p, st) : launch_fwd<T, true, false>(p, st);
  return p.top_k ? launch_fwd<T, false, true>(p, st) : launch_fwd<T, false, false>(p, st);
}

template <typename T, bool kEnt, bool kTop>
cudaError_t launch_bwd(const LogprobArgs& p, cudaStream_t st) {
  const long long rows = p.batch * p.length;
  const int chunks = (p.vocab * static_cast<long long>(sizeof(T)) + 15) / 16 + 1;
  constexpr int U = kBwdUnroll;
  const int threads = chunks >= U * 256 ? 256 : (chunks >= U * 128 ? 128 : 64);
  const int parts = (chunks + threads * U - 1) / (threads * U);
  if (rows * parts > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  logprobs_bwd_kernel<T, kEnt, kTop>
      <<<static_cast<unsigned>(rows * parts), threads, 0, st>>>(p, parts);
  return cudaGetLastError();
}
template <typename T>
cudaError_t bwd_typed(const LogprobArgs& p, cudaStream_t st) {
  if (p.g_entropy)
    return p.g_top ? launch_bwd<T, true, true>(p, st) : launch_bwd<T, true, false>(p, st);
  return p.g_top ? launch_bwd<T, false, true>(p, st) : launch_bwd<T, false, false>(p, st);
}

}  // namespace

cudaError_t token_logprobs_fwd(const LogprobArgs& p, cudaStream_t st) {
  return p.f32 ? fwd_typed<float>(p, st) : fwd_typed<bf16>(p, st);
}
cudaError_t token_logprobs_bwd(const LogprobArgs& p, cudaStream_t st) {
  return p.f32 ? bwd_typed<float>(p, st) : bwd_typed<bf16>(p, st);
}

}  // namespace gmdn
