// Layer norm and RMS norm over the model width, with an optional residual add
// in front, forward and backward.
//
//   s  = x + res, rounded to its stored type (no res: s = x)
//   layer: mean = sum(s) / D, xh = (s - mean) / sqrt(sum((s - mean)^2) / D + eps)
//   rms:   xh = s / sqrt(sum(s^2) / D + eps)
//   y  = xh w + b
//   backward, with g = dy w:
//   ds = (g - xh sum(g xh) / D [layer: - sum(g) / D]) rstd + dh
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Every sum is held in fp32; s, y and ds are rounded once, to their stored
// types (the norm reads the rounded s, so the backward sees what the forward
// saw).
//
// Memory bounds it: ~10 operations an element forward and ~14 backward against
// 8 to 16 bytes.  So a row is read once and held in registers from its first
// sum to its last output, and dw, db are summed in registers over all of a
// thread's rows.  Measured (B200, copy rate 6536 GB/s): 16384 x 768, fp32 stream
// and bf16 branch: forward 26 us (0.89 of the copy rate), backward 42 us (0.73,
// with the 5 us join of the CTAs' column sums); 8192 x 8192 bf16 layer norm 96
// and 114 us (0.86, 0.72); RMS norm of fp32 rows of 4096 and 8192 elements 0.85 to
// 0.91 both ways.  A layer norm of such rows waits for two sums a row: fp32 8192 x
// 8192 119 and 148 us (0.69, 0.83), 4897 x 13704 154 and 231 (0.53, 0.53).  The
// backward is lowest at 1024, where it writes the most partials: 16384 rows of
// fp32 42 us (0.61).

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "common.cuh"
#include "step_ops.h"

namespace cg = cooperative_groups;

namespace gmdn {
namespace {

// ---------------------------------------------------------------------------
// Rows in registers.  A row is held by part of a warp, a warp (short rows, no
// barrier) or a CTA; each thread has NV groups of 8 consecutive elements of it,
// group v * threads + thread, each one or two 16-byte accesses a tensor.  A
// thread walks rows grid apart: the next row's loads are issued as soon as the
// current one's registers are converted, before its reductions, so memory is
// busy while the row is summed.
//
// Where the width is no multiple of 8, rows start at any place of the groups
// of 8 elements that the memory falls into.  The grid's step is then a multiple
// of 8 rows, so a thread sees one such place, `off` elements into its first
// group, in all its rows: it loads the groups of the row whole (the first and
// the last hold elements of the rows beside, which it masks out), keeps the same
// columns throughout, and finds the weights in a copy in shared memory that is
// shifted by `off`.
// ---------------------------------------------------------------------------

constexpr int kSms = 148;
constexpr int kRowThreads = 128; // CTA of warp rows
constexpr int kMaxCta = 512;     // threads of a CTA row: 128 registers each
constexpr int kPair = -2;        // LPR: a row lies over a cluster of two CTAs
constexpr int kBuf = 256;        // floats a CTA's sums go through: two buffers of 128
using bf16 = __nv_bfloat16;

template <typename T>
struct Raw {   // 8 consecutive elements as loaded
  uint4 r[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k)
      r[k] = __ldcs(reinterpret_cast<const uint4*>(p) + k);
  }
  // the first n of them (the tensor ends there)
  __device__ __forceinline__ void load_some(const T* p, int n) {
    T v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < n ? p[k] : static_cast<T>(0.f);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k)
      r[k] = reinterpret_cast<const uint4*>(v)[k];
  }
  __device__ __forceinline__ float get(int k) const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w = k < 4 ? (k < 2 ? r[0].x : r[0].y) : (k < 6 ? r[0].z : r[0].w);
      return __uint_as_float(k & 1 ? w & 0xffff0000u : w << 16);
    } else {
      const uint4& q = r[k / 4];
      return __uint_as_float((k & 3) < 2 ? ((k & 1) ? q.y : q.x) : ((k & 1) ? q.w : q.z));
    }
  }
};

// 8 elements at i, those of `mask` (0xff: all, one or two 16-byte stores)
__device__ __forceinline__ void store_group(void* base, size_t i, const float* v, bool f32,
                                            uint32_t mask) {
  if (mask != 0xffu) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (mask >> k & 1) store_act(base, i + k, v[k], f32);
  } else if (f32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
    *reinterpret_cast<uint4*>(static_cast<bf16*>(base) + i) = *reinterpret_cast<uint4*>(h);
  }
}

// Sums over a row's threads; every thread gets them.  LPR lanes of a warp a row,
// or (0) a CTA: one barrier for N sums (at most 4), `red` alternating between
// two buffers of 128 floats, so that a warp that is ahead writes the other one.
template <int LPR>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int o = (LPR > 0 ? LPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
template <int LPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float*& red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum<LPR>(v[i]);
  if constexpr (LPR == 0) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[32 * i + w] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < n ? red[32 * i + lane] : 0.f);
    red = reinterpret_cast<float*>(reinterpret_cast<uintptr_t>(red) ^ 512);
  }
}
// The same over the two CTAs of a row, in two steps: each warp writes its sums to both CTAs'
// buffers and arrives at the cluster's barrier; then they wait and add.  The barrier's release
// waits for a thread's outstanding accesses, so the next row is fetched between the steps
// (2048 x 16384: 117 us against 141 with the loads before them).
template <int N>
__device__ __forceinline__ void pair_arrive(float (&v)[N], float* red) {
  auto cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, at = (threadIdx.x >> 5) + 16 * cluster.block_rank();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (lane < 2) {
    float* to = cluster.map_shared_rank(red, lane);
#pragma unroll
    for (int i = 0; i < N; ++i) to[32 * i + at] = v[i];
  }
  cluster.barrier_arrive();
}
template <int N>
__device__ __forceinline__ void pair_wait(float (&v)[N], float*& red) {
  const int lane = threadIdx.x & 31, n = blockDim.x >> 5;
  cg::this_cluster().barrier_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane % 16 < n ? red[32 * i + lane] : 0.f);
  red = reinterpret_cast<float*>(reinterpret_cast<uintptr_t>(red) ^ 512);
}

// 8 values rounded to bf16, in place, pairs at a time
__device__ __forceinline__ void round_bf16(float* v) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[k], v[k + 1]);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
    v[k] = __uint_as_float(w << 16);
    v[k + 1] = __uint_as_float(w & 0xffff0000u);
  }
}

__device__ __forceinline__ void load_param8(const float* p, float* q) {
  *reinterpret_cast<float4*>(q) = __ldg(reinterpret_cast<const float4*>(p));
  *reinterpret_cast<float4*>(q + 4) = __ldg(reinterpret_cast<const float4*>(p) + 1);
}

struct None {};

// Where a thread's part of its rows lies.
template <int NV, int LPR, bool kOdd>
struct Place {
  static constexpr bool kWarp = LPR > 0;
  static constexpr int L = kWarp ? LPR : 1, kCtas = LPR == kPair ? 2 : 1;   // CTAs a row
  static constexpr int kSlots = kWarp ? kRowThreads / L : 1;   // rows a CTA has at a time
  int tid, tpr, slot, lead, off, width;
  long long row, step;        // the thread's first row; `lead` more than its warp's first
  uint32_t mask[kOdd ? NV : 1];   // kOdd: the row's elements of each group
  __device__ __forceinline__ Place(int D) : width(D) {
    tid = kWarp ? threadIdx.x % L : threadIdx.x + blockIdx.x % kCtas * blockDim.x;
    tpr = kWarp ? L : kCtas * blockDim.x;
    slot = kWarp ? threadIdx.x / L : 0;
    lead = kWarp ? slot % (32 / (kWarp ? L : 32)) : 0;
    row = static_cast<long long>(blockIdx.x / kCtas) * kSlots + slot;
    step = static_cast<long long>(gridDim.x / kCtas) * kSlots;
    off = 0;
    if constexpr (kOdd) {
      off = static_cast<int>((row % 8 * (D % 8)) % 8);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = group(v) * 8 - off;   // the group's first column
        mask[v] = 0;
        if (c < D)
          mask[v] = (c < 0 ? 0xffu << -c & 0xffu : 0xffu) &
                    (D - c < 8 ? 0xffu >> (8 - (D - c)) : 0xffu);
      }
    }
  }
  // whether the row reaches into group v, and its elements there
  __device__ __forceinline__ bool has(int v) const {
    return kOdd ? mask[kOdd ? v : 0] != 0 : group(v) * 8 < width;
  }
  __device__ __forceinline__ uint32_t bits(int v) const { return kOdd ? mask[kOdd ? v : 0] : 0xffu; }
  __device__ __forceinline__ int group(int v) const { return v * tpr + tid; }
  // the row's first group as an element of the tensor
  __device__ __forceinline__ size_t base(long long r, int D) const {
    return static_cast<size_t>(r) * D - off;
  }
  template <typename T>
  __device__ __forceinline__ void load(Raw<T>& raw, const T* p, size_t i, size_t total) const {
    if (!kOdd || i + 8 <= total)
      raw.load(p + i);
    else
      raw.load_some(p + i, static_cast<int>(total - i));
  }
  // a (width) parameter's shared copy for this thread's slot: column c at off + c, 0 around
  static __host__ __device__ int copy_floats(int D) { return (D + 14) / 8 * 8; }
  __device__ __forceinline__ void copy(float* dst, const float* src, int D) const {
    for (int i = kWarp ? tid : threadIdx.x; i < copy_floats(D); i += kWarp ? tpr : blockDim.x) {
      const int c = i - off;
      dst[i] = c >= 0 && c < D ? src[c] : 0.f;
    }
  }
  // 8 values of a parameter for group v
  __device__ __forceinline__ void param(const float* global, const float* shared, int v,
                                        float* q) const {
    if constexpr (kOdd) {
      const float4* p = reinterpret_cast<const float4*>(shared + group(v) * 8);
      *reinterpret_cast<float4*>(q) = p[0];
      *reinterpret_cast<float4*>(q + 4) = p[1];
    } else {
      load_param8(global + group(v) * 8, q);
    }
  }
};

// R rows a step: their sums share barriers and their loads of the weights.  CTA
// rows with two groups a thread take two (8192 x 8192 bf16 layer norm: 96 us
// against 109 one row a step, two CTAs an SM instead of one).
template <typename TX, typename TR, int NV, int LPR, bool kOdd, int R>
__global__ void __launch_bounds__(LPR > 0 ? kRowThreads : kMaxCta) norm_fwd_regs(NormFwdArgs p) {
  constexpr bool kRes = !std::is_same<TR, None>::value;
  using TL = typename std::conditional<kRes, TR, TX>::type;   // the residual's loads
  constexpr bool kHf32 = std::is_same<TX, float>::value || std::is_same<TR, float>::value;
  __shared__ __align__(1024) float buf[kBuf];
  extern __shared__ __align__(16) float params[];   // kOdd: weight, bias, a copy a slot
  float* red = buf;
  const int D = p.width;
  const float inv = 1.f / static_cast<float>(D);
  const size_t total = static_cast<size_t>(p.rows) * D;
  const Place<NV, LPR, kOdd> at(D);
  float *sw = nullptr, *sb = nullptr;
  if constexpr (kOdd) {
    const int n = at.copy_floats(D);
    sw = params + at.slot * n;
    sb = sw + (p.weight ? at.kSlots * n : 0);
    if (p.weight) at.copy(sw, p.weight, D);
    if (p.bias) at.copy(sb, p.bias, D);
    __syncthreads();
  }
  const TX* x = static_cast<const TX*>(p.x);
  const TL* res = static_cast<const TL*>(p.res);
  Raw<TX> rx[R][NV];
  Raw<TL> rr[R][NV];
  auto fetch = [&](long long first) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const long long row = first + q * at.step;
      if (row < p.rows) {
        const size_t base = at.base(row, D);
#pragma unroll
        for (int v = 0; v < NV; ++v)
          if (at.has(v)) {
            at.load(rx[q][v], x, base + at.group(v) * 8, total);
            if constexpr (kRes) at.load(rr[q][v], res, base + at.group(v) * 8, total);
          }
      }
    }
  };
  fetch(at.row);
  // a warp's rows go together: its lanes meet in the sums whether they have a row or not
  for (long long r = at.row; r - at.lead < p.rows; r += R * at.step) {
    float s[R][NV][8], sum[R], mean[R], d12[2 * R], rstd[R];
    auto live = [&](int q) {
      return (q == 0 && (LPR == 0 || LPR == 32)) || r + q * at.step < p.rows;
    };
#pragma unroll
    for (int q = 0; q < R; ++q) {
      sum[q] = mean[q] = d12[2 * q] = d12[2 * q + 1] = 0.f;
      const size_t base = at.base(r + q * at.step, D);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const bool in = at.has(v) && live(q);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          s[q][v][k] = 0.f;
          if (in && (!kOdd || at.bits(v) >> k & 1)) {
            s[q][v][k] = rx[q][v].get(k);
            if constexpr (kRes) s[q][v][k] += rr[q][v].get(k);
          }
        }
        if constexpr (kRes && !kHf32) round_bf16(s[q][v]);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[q] += s[q][v][k];
        if constexpr (kRes)
          if (in) store_group(p.h, base + at.group(v) * 8, s[q][v], kHf32, at.bits(v));
      }
    }
    fetch(r + R * at.step);
    if (p.center) {
      row_sums<LPR>(sum, red);
#pragma unroll
      for (int q = 0; q < R; ++q) mean[q] = sum[q] * inv;
    }
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (at.has(v)) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float d = !kOdd || at.bits(v) >> k & 1 ? s[q][v][k] - mean[q] : 0.f;
            d12[2 * q] += d;
            d12[2 * q + 1] = fmaf(d, d, d12[2 * q + 1]);
          }
        }
    row_sums<LPR>(d12, red);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      float d1 = d12[2 * q], d2 = d12[2 * q + 1] * inv;
      if (p.center) {   // what the rounding of the mean left, taken out of both
        d1 *= inv;
        mean[q] += d1;
        d2 = fmaxf(d2 - d1 * d1, 0.f);
      }
      rstd[q] = rsqrtf(d2 + p.eps);
      if (at.tid == 0 && live(q)) {
        p.rstd[r + q * at.step] = rstd[q];
        if (p.center) p.mean[r + q * at.step] = mean[q];
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (at.has(v)) {
        float w[8], b[8];
        if (p.weight) at.param(p.weight, sw, v, w);
        if (p.bias) at.param(p.bias, sb, v, b);
#pragma unroll
        for (int q = 0; q < R; ++q) {
          if (!live(q)) continue;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float y = (s[q][v][k] - mean[q]) * rstd[q];
            if (p.weight) y *= w[k];
            if (p.bias) y += b[k];
            s[q][v][k] = y;
          }
          store_group(p.y, at.base(r + q * at.step, D) + at.group(v) * 8, s[q][v], p.y_f32,
                      at.bits(v));
        }
      }
  }
}

// TS: the type of s and dh.  dw and db are summed over a thread's rows in
// registers; a CTA's sums are one partial (norm_bwd_join adds the partials).
// kMaxThreads: an odd width's masks do not fit the 128 registers of 512 threads; up to 256
// they have 255.
template <typename TS, typename TG, int NV, int LPR, bool kOdd, bool kDb, int kMaxThreads>
__global__ void __launch_bounds__(LPR > 0 ? kRowThreads : kMaxThreads)
norm_bwd_regs(NormBwdArgs p) {
  __shared__ __align__(1024) float buf[kBuf];
  extern __shared__ __align__(16) float dyn[];   // kOdd: weight copies; then a warp row's sums
  float* red = buf;
  const int D = p.width;
  const float inv = 1.f / static_cast<float>(D);
  const size_t total = static_cast<size_t>(p.rows) * D;
  const Place<NV, LPR, kOdd> at(D);
  float* sw = nullptr;
  if constexpr (kOdd) {
    sw = dyn + at.slot * at.copy_floats(D);
    if (p.weight) at.copy(sw, p.weight, D);
    __syncthreads();
  }
  const TS *sp = static_cast<const TS*>(p.s), *dhp = static_cast<const TS*>(p.dh);
  const TG* gp = static_cast<const TG*>(p.dy);
  Raw<TS> rs[NV], rh[NV];
  Raw<TG> rg[NV];
  float rstd_next = 0.f, mean_next = 0.f;
  auto fetch = [&](long long row) {
    if (row >= p.rows) return;
    rstd_next = p.rstd[row];
    mean_next = p.center ? p.mean[row] : 0.f;
    const size_t base = at.base(row, D);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (at.has(v)) {
        at.load(rs[v], sp, base + at.group(v) * 8, total);
        at.load(rg[v], gp, base + at.group(v) * 8, total);
      }
  };
  float dw[NV][8], db[kDb ? NV : 1][8];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      dw[v][k] = 0.f;
      if constexpr (kDb) db[v][k] = 0.f;
    }
  if constexpr (LPR == kPair) cg::this_cluster().sync();   // the other CTA's memory is there
  fetch(at.row);
  for (long long r = at.row; r - at.lead < p.rows; r += at.step) {
    const bool live = LPR <= 0 || LPR == 32 || r < p.rows;
    const size_t base = at.base(r, D);
    const float rstd = rstd_next, mean = mean_next;
    float xh[NV][8], g[NV][8];
    float sums[2] = {0.f, 0.f};   // of g, of g xh
    float &a = sums[0], &b = sums[1];
    auto fetch_dh = [&] {   // needed last: in flight over the reduction, not a row ahead
      if (dhp && live) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
          if (at.has(v)) at.load(rh[v], dhp, base + at.group(v) * 8, total);
      }
    };
    if constexpr (LPR != kPair) fetch_dh();
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (at.has(v) && live) {
        float w[8];
        if (p.weight) at.param(p.weight, sw, v, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          xh[v][k] = (rs[v].get(k) - mean) * rstd;
          g[v][k] = rg[v].get(k);
          if (kOdd && !(at.bits(v) >> k & 1)) xh[v][k] = g[v][k] = 0.f;
          dw[v][k] = fmaf(g[v][k], xh[v][k], dw[v][k]);
          if constexpr (kDb) db[v][k] += g[v][k];
          if (p.weight) g[v][k] *= w[k];
          a += g[v][k];
          b = fmaf(g[v][k], xh[v][k], b);
        }
      }
    if constexpr (LPR == kPair) {
      pair_arrive(sums, red);
      fetch_dh();
    }
    fetch(r + at.step);
    if constexpr (LPR == kPair)
      pair_wait(sums, red);
    else
      row_sums<LPR>(sums, red);
    a = p.center ? a * inv : 0.f;
    b *= inv;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (at.has(v) && live) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          g[v][k] = fmaf(fmaf(xh[v][k], -b, g[v][k] - a), rstd, dhp ? rh[v].get(k) : 0.f);
        if (p.ds_a) store_group(p.ds_a, base + at.group(v) * 8, g[v], p.a_f32, at.bits(v));
        if (p.ds_b) store_group(p.ds_b, base + at.group(v) * 8, g[v], p.b_f32, at.bits(v));
      }
  }
  if (!p.dw && !p.db) return;
  float* out = p.partial + static_cast<size_t>(blockIdx.x / at.kCtas) * 2 * D;
#pragma unroll
  for (int which = 0; which < (kDb ? 2 : 1); ++which) {
    // CTA rows write the partial; warp rows their slot of `dyn` (over the weight copies)
    float* dst = LPR > 0 ? dyn + at.slot * D : out + which * D;
    if constexpr (LPR > 0) __syncthreads();
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (at.has(v)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float t = dw[v][k];
          if constexpr (kDb) t = which ? db[v][k] : t;
          if (at.bits(v) >> k & 1) dst[at.group(v) * 8 - at.off + k] = t;
        }
      }
    if constexpr (LPR > 0) {
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += kRowThreads) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < at.kSlots; ++w) t += dyn[w * D + c];
        out[which * D + c] = t;
      }
    }
  }
}

// How a width is held: by the most groups of 8 a row can touch.  Rows of up to
// 96 groups by 8, 16 or 32 lanes (three groups a lane are as many as the
// backward's five arrays of them leave registers for); CTA rows with two groups
// a thread up to 1024 groups; up to 2048 the forward with four (whose registers the
// backward does not have), the backward by a cluster of two CTAs.  Two CTAs a row
// pay for their barrier only where one cannot hold it: 2048 x 16384 (bf16, fp32
// stream) backward 117 us, against 279 for rows read again from L2 and 68 us forward
// (89 with two CTAs); 8192 x 8192 bf16 backward 111 us by one CTA, 171 by two.
// Other wide rows are read again for each pass (nv 0).
struct Shape {
  int nv, lanes, threads;   // lanes 0: CTA rows, kPair: two CTAs a row
  bool odd;
};
Shape shape_of(int D, bool fwd) {
  const bool odd = D % 8 != 0;
  const int groups = odd ? (D + 14) / 8 : D / 8;
  auto up = [&](int per) { return (groups + per * 32 - 1) / (per * 32) * 32; };
  if (groups <= 8) return {1, 8, kRowThreads, odd};
  if (groups <= 16) return {1, 16, kRowThreads, odd};
  if (groups <= 96) return {(groups + 31) / 32, 32, kRowThreads, odd};
  if (groups <= 2 * kMaxCta) return {2, 0, up(2), odd};
  if (groups <= 4 * kMaxCta) return fwd ? Shape{4, 0, up(4), odd} : Shape{2, kPair, up(4), odd};
  return {0, -1, 0, odd};
}
// A launch of clusters of two CTAs.
struct ClusterLaunch {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  ClusterLaunch(int ctas, int threads, size_t smem, cudaStream_t st) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {2, 1, 1};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
};
int slots_of(Shape sh) { return sh.lanes > 0 ? kRowThreads / sh.lanes : 1; }

// One wave of CTAs (kPair: of clusters, two CTAs each), each walking rows a grid apart;
// for odd widths the step is a multiple of 8 rows.
template <typename K>
cudaError_t wave(K kernel, long long rows, Shape sh, size_t smem, int* out) {
  const int slots = slots_of(sh);
  const long long want = (rows + slots - 1) / slots;
  long long grid = want;
  if (sh.lanes == kPair) {
    int n = 0;
    ClusterLaunch at(2 * kSms, sh.threads, smem, nullptr);
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &at.cfg);
    if (e != cudaSuccess) return e;
    if (n < 8) n = 8;   // an odd width's step is a multiple of 8 rows
    if (n < grid) grid = n;
  } else if (want > kSms) {
    int n = 1;
    const cudaError_t e =
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, sh.threads, smem);
    if (e != cudaSuccess) return e;
    const long long cap = static_cast<long long>(kSms) * (n < 1 ? 1 : n);
    if (cap < grid) grid = cap;
  }
  if (sh.odd && grid < want && slots % 8) {
    const int per = 8 / slots > 0 ? 8 / slots : 1;
    grid = grid / per * per;
  }
  *out = static_cast<int>(grid);
  return cudaSuccess;
}

// 48 KB, the kernel's own `buf` counted, is what a launch may use without being asked for more.
template <typename K>
cudaError_t allow(K kernel, size_t smem) {
  return smem + kBuf * sizeof(float) <= 48 * 1024
             ? cudaSuccess
             : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(smem));
}

// ---------------------------------------------------------------------------
// Rows of any width, read again for each pass
// ---------------------------------------------------------------------------

constexpr int kColThreads = 256;
constexpr int kColRows = 8;      // warps of a column block, each on every 8th row

// One CTA a row, any width: the row is read again for each pass (from L1 / L2).
__global__ void __launch_bounds__(kThreads) norm_fwd_rows(NormFwdArgs p) {
  __shared__ float red[32];
  const int D = p.width;
  const float inv = 1.f / static_cast<float>(D);
  const bool s_f32 = p.res ? (p.x_f32 || p.res_f32) : p.x_f32;
  const void* s = p.res ? p.h : p.x;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const size_t base = static_cast<size_t>(r) * D;
    float sum = 0.f;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      float v = load_act(p.x, base + i, p.x_f32);
      if (p.res) {
        v += load_act(p.res, base + i, p.res_f32);
        store_act(p.h, base + i, v, s_f32);
        v = load_act(p.h, base + i, s_f32);   // as rounded
      }
      sum += v;
    }
    float mean = p.center ? block_sum(sum, red) * inv : 0.f;
    float d1 = 0.f, d2 = 0.f;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float d = load_act(s, base + i, s_f32) - mean;
      d1 += d;
      d2 = fmaf(d, d, d2);
    }
    d2 = block_sum(d2, red) * inv;
    if (p.center) {   // what the rounding of the mean left, taken out of both
      const float c = block_sum(d1, red) * inv;
      mean += c;
      d2 = fmaxf(d2 - c * c, 0.f);
    }
    const float rstd = rsqrtf(d2 + p.eps);
    if (threadIdx.x == 0) {
      p.rstd[r] = rstd;
      if (p.center) p.mean[r] = mean;
    }
    for (int i = threadIdx.x; i < D; i += kThreads) {
      float v = (load_act(s, base + i, s_f32) - mean) * rstd;
      if (p.weight) v *= p.weight[i];
      if (p.bias) v += p.bias[i];
      store_act(p.y, base + i, v, p.y_f32);
    }
  }
}

__global__ void __launch_bounds__(kThreads) norm_bwd_rows(NormBwdArgs p) {
  __shared__ float red[32];
  const int D = p.width;
  const float inv = 1.f / static_cast<float>(D);
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const size_t base = static_cast<size_t>(r) * D;
    const float rstd = p.rstd[r], mean = p.center ? p.mean[r] : 0.f;
    float a = 0.f, b = 0.f;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float xh = (load_act(p.s, base + i, p.s_f32) - mean) * rstd;
      float g = load_act(p.dy, base + i, p.dy_f32);
      if (p.weight) g *= p.weight[i];
      a += g;
      b = fmaf(g, xh, b);
    }
    a = p.center ? block_sum(a, red) * inv : 0.f;
    b = block_sum(b, red) * inv;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float xh = (load_act(p.s, base + i, p.s_f32) - mean) * rstd;
      float g = load_act(p.dy, base + i, p.dy_f32);
      if (p.weight) g *= p.weight[i];
      float d = (g - a - xh * b) * rstd;
      if (p.dh) d += load_act(p.dh, base + i, p.s_f32);
      if (p.ds_a) store_act(p.ds_a, base + i, d, p.a_f32);
      if (p.ds_b) store_act(p.ds_b, base + i, d, p.b_f32);
    }
  }
}

// Column sums of a run of rows: block (column block, part), one partial each.
__global__ void __launch_bounds__(kColThreads) norm_bwd_cols(NormBwdArgs p, int parts) {
  __shared__ float red[2][kColRows][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const long long per = (p.rows + parts - 1) / parts;
  const long long r0 = per * blockIdx.y, r1 = min(r0 + per, p.rows);
  float dw = 0.f, db = 0.f;
  if (col < p.width) {
    for (long long r = r0 + w; r < r1; r += kColRows) {
      const size_t i = static_cast<size_t>(r) * p.width + col;
      const float g = load_act(p.dy, i, p.dy_f32);
      const float m = p.center ? p.mean[r] : 0.f;
      dw = fmaf(g, (load_act(p.s, i, p.s_f32) - m) * p.rstd[r], dw);
      db += g;
    }
  }
  red[0][w][lane] = dw;
  red[1][w][lane] = db;
  __syncthreads();
  if (w < 2 && col < p.width) {
    float t = 0.f;
    for (int k = 0; k < kColRows; ++k) t += red[w][k][lane];
    p.partial[(static_cast<size_t>(blockIdx.y) * 2 + w) * p.width + col] = t;
  }
}

// dw, db from the partials, in a fixed order (bit-reproducible): 32 columns a
// CTA, each warp every 32nd partial, blockIdx.y 0: dw, 1: db.
constexpr int kJoinWarps = 32, kJoinFly = 5;
__global__ void __launch_bounds__(kJoinWarps * 32, 1024 / (kJoinWarps * 16)) norm_bwd_join(const float* partial, float* dw,
                                                                 float* db, int D, int parts) {
  __shared__ float red[kJoinWarps][33];
  float* out = blockIdx.y == 0 ? dw : db;
  if (!out) return;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (col < D) {
    const float* src = partial + static_cast<size_t>(blockIdx.y) * D + col;
    for (int k0 = w; k0 < parts; k0 += kJoinWarps * kJoinFly) {
      float v[kJoinFly];   // all in flight: the kernel is nothing but their latency
#pragma unroll
      for (int u = 0; u < kJoinFly; ++u) {
        const int k = k0 + u * kJoinWarps;
        v[u] = k < parts ? __ldcg(src + static_cast<size_t>(k) * 2 * D) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kJoinFly; ++u) a += v[u];
    }
  }
  red[w][lane] = a;
  __syncthreads();
  if (w == 0 && col < D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kJoinWarps; ++k) t += red[k][lane];
    out[col] = t;
  }
}

int row_grid(long long rows) {
  return static_cast<int>(rows < kSms * 8 ? rows : kSms * 8);
}

template <typename TX, typename TR, int NV, int LPR, bool kOdd>
cudaError_t fwd_go(const NormFwdArgs& p, Shape sh, cudaStream_t st) {
  constexpr int R = LPR == 0 && NV == 2 && !kOdd ? 2 : 1;
  auto k = norm_fwd_regs<TX, TR, NV, LPR, kOdd, R>;
  const size_t copy = Place<NV, LPR, kOdd>::copy_floats(p.width) * sizeof(float) * slots_of(sh);
  const size_t smem = kOdd ? copy * ((p.weight ? 1 : 0) + (p.bias ? 1 : 0)) : 0;
  int grid = 0;
  cudaError_t e = allow(k, smem);
  if (e == cudaSuccess) e = wave(k, p.rows, sh, smem, &grid);
  if (e != cudaSuccess) return e;
  k<<<grid, sh.threads, smem, st>>>(p);
  return cudaGetLastError();
}
template <typename TX, typename TR, bool kOdd>
cudaError_t fwd_shaped(const NormFwdArgs& p, Shape sh, cudaStream_t st) {
  if (sh.lanes == 8) return fwd_go<TX, TR, 1, 8, kOdd>(p, sh, st);
  if (sh.lanes == 16) return fwd_go<TX, TR, 1, 16, kOdd>(p, sh, st);
  if (sh.lanes == 32) {
    if (sh.nv == 1) return fwd_go<TX, TR, 1, 32, kOdd>(p, sh, st);
    if (sh.nv == 2) return fwd_go<TX, TR, 2, 32, kOdd>(p, sh, st);
    return fwd_go<TX, TR, 3, 32, kOdd>(p, sh, st);
  }
  if (sh.nv == 2) return fwd_go<TX, TR, 2, 0, kOdd>(p, sh, st);
  return fwd_go<TX, TR, 4, 0, kOdd>(p, sh, st);
}
template <typename TX, typename TR>
cudaError_t fwd_typed(const NormFwdArgs& p, Shape sh, cudaStream_t st) {
  return sh.odd ? fwd_shaped<TX, TR, true>(p, sh, st) : fwd_shaped<TX, TR, false>(p, sh, st);
}

// Launches the rows' kernel with at most `most` CTAs (kPair: clusters); *parts: how many there are.
template <typename TS, typename TG, bool kDb, bool kOdd, int NV, int LPR, int kMaxThreads = kMaxCta>
cudaError_t bwd_go(const NormBwdArgs& p, Shape sh, int most, int* parts, cudaStream_t st) {
  auto k = norm_bwd_regs<TS, TG, NV, LPR, kOdd, kDb, kMaxThreads>;
  const int slots = slots_of(sh);
  const size_t copies = kOdd && p.weight ? Place<NV, LPR, kOdd>::copy_floats(p.width) * slots : 0;
  const size_t sums = LPR > 0 && (p.dw || p.db) ? static_cast<size_t>(p.width) * slots : 0;
  const size_t smem = sizeof(float) * (copies > sums ? copies : sums);
  int grid = 0;
  cudaError_t e = allow(k, smem);
  if (e == cudaSuccess) e = wave(k, p.rows, sh, smem, &grid);
  if (e != cudaSuccess) return e;
  if (grid > most) grid = most;   // a multiple of 8
  *parts = grid;
  if constexpr (LPR == kPair) {
    ClusterLaunch at(2 * grid, sh.threads, smem, st);
    return cudaLaunchKernelEx(&at.cfg, k, p);
  } else {
    k<<<grid, sh.threads, smem, st>>>(p);
    return cudaGetLastError();
  }
}
template <typename TS, typename TG, bool kDb, bool kOdd>
cudaError_t bwd_shaped(const NormBwdArgs& p, Shape sh, int most, int* parts, cudaStream_t st) {
  if (sh.lanes == 8) return bwd_go<TS, TG, kDb, kOdd, 1, 8>(p, sh, most, parts, st);
  if (sh.lanes == 16) return bwd_go<TS, TG, kDb, kOdd, 1, 16>(p, sh, most, parts, st);
  if (sh.lanes == 32) {
    if (sh.nv == 1) return bwd_go<TS, TG, kDb, kOdd, 1, 32>(p, sh, most, parts, st);
    if (sh.nv == 2) return bwd_go<TS, TG, kDb, kOdd, 2, 32>(p, sh, most, parts, st);
    return bwd_go<TS, TG, kDb, kOdd, 3, 32>(p, sh, most, parts, st);
  }
  if (sh.lanes == kPair) return bwd_go<TS, TG, kDb, kOdd, 2, kPair>(p, sh, most, parts, st);
  if (kOdd && sh.threads <= 256)
    return bwd_go<TS, TG, kDb, kOdd, 2, 0, 256>(p, sh, most, parts, st);
  return bwd_go<TS, TG, kDb, kOdd, 2, 0>(p, sh, most, parts, st);
}
template <typename TS, typename TG>
cudaError_t bwd_typed(const NormBwdArgs& p, Shape sh, int most, int* parts, cudaStream_t st) {
  if (sh.odd)
    return p.db ? bwd_shaped<TS, TG, true, true>(p, sh, most, parts, st)
                : bwd_shaped<TS, TG, false, true>(p, sh, most, parts, st);
  return p.db ? bwd_shaped<TS, TG, true, false>(p, sh, most, parts, st)
              : bwd_shaped<TS, TG, false, false>(p, sh, most, parts, st);
}

}  // namespace

cudaError_t norm_fwd(const NormFwdArgs& p, cudaStream_t st) {
  const Shape sh = shape_of(p.width, true);
  if (sh.nv == 0) {
    norm_fwd_rows<<<row_grid(p.rows), kThreads, 0, st>>>(p);
    return cudaGetLastError();
  }
  if (p.x_f32) {
    if (!p.res) return fwd_typed<float, None>(p, sh, st);
    return p.res_f32 ? fwd_typed<float, float>(p, sh, st) : fwd_typed<float, bf16>(p, sh, st);
  }
  if (!p.res) return fwd_typed<bf16, None>(p, sh, st);
  return p.res_f32 ? fwd_typed<bf16, float>(p, sh, st) : fwd_typed<bf16, bf16>(p, sh, st);
}

// The most partials of dw and db that a backward writes, one a CTA: 16 warps an
// SM (an odd width's rounded to its grid's multiple of 8).
int norm_bwd_partials(long long rows, int width) {
  const Shape sh = shape_of(width, false);
  const int all = sh.nv == 0 ? 2 * kSms : sh.lanes == kPair ? kSms / 2 : kSms * (512 / sh.threads);
  const int cap = sh.odd ? all / 8 * 8 : all;
  return static_cast<int>(rows < cap ? rows : cap);
}

cudaError_t norm_bwd(const NormBwdArgs& p, cudaStream_t st) {
  const Shape sh = shape_of(p.width, false);
  const int most = norm_bwd_partials(p.rows, p.width);
  int parts = most;
  cudaError_t e;
  if (sh.nv > 0) {
    if (p.s_f32)
      e = p.dy_f32 ? bwd_typed<float, float>(p, sh, most, &parts, st)
                   : bwd_typed<float, bf16>(p, sh, most, &parts, st);
    else
      e = p.dy_f32 ? bwd_typed<bf16, float>(p, sh, most, &parts, st)
                   : bwd_typed<bf16, bf16>(p, sh, most, &parts, st);
  } else {
    const long long want = (p.rows + 31) / 32;
    parts = static_cast<int>(want < most ? want : most);
    if (p.ds_a || p.ds_b) norm_bwd_rows<<<row_grid(p.rows), kThreads, 0, st>>>(p);
    if (p.dw || p.db)
      norm_bwd_cols<<<dim3((p.width + 31) / 32, parts), kColThreads, 0, st>>>(p, parts);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && (p.dw || p.db)) {
    norm_bwd_join<<<dim3((p.width + 31) / 32, p.db ? 2 : 1), kJoinWarps * 32, 0, st>>>(
        p.partial, p.dw, p.db, p.width, parts);
    e = cudaGetLastError();
  }
  return e;
}

}  // namespace gmdn
