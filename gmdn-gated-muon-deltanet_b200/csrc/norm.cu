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

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "common.cuh"
#include "cp_async.cuh"
#include "step_ops.h"

namespace gmdn {
namespace {

// ---------------------------------------------------------------------------
// Rows in registers.  A row is held by one warp (short rows, four a CTA, no
// barrier) or by one CTA; each thread has NV groups of VEC
// consecutive elements of it, group v * threads + thread.  VEC is 8 where the
// width is a multiple of 8, so that every row starts 16-byte aligned and a
// group is one or two 16-byte accesses; short rows of other widths go element
// by element (VEC 1), longer ones through shared memory (below).
// A thread walks rows grid apart: the next row's loads are issued as soon as
// the current one's registers are converted, before its reductions, so memory
// is busy while the row is summed.
// ---------------------------------------------------------------------------

constexpr int kSms = 148;
constexpr int kRowWarps = 4;     // warp rows of a CTA
constexpr int kMaxCta = 512;     // threads of a CTA row: 128 registers each
constexpr int kMaxResident = 4;  // CTAs an SM, at most: each writes a partial of dw and db
using bf16 = __nv_bfloat16;

template <typename T, int VEC>
struct Raw {   // VEC 8
  uint4 r[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k)
      r[k] = __ldcs(reinterpret_cast<const uint4*>(p) + k);
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
template <typename T>
struct Raw<T, 1> {
  T r;
  __device__ __forceinline__ void load(const T* p) { r = __ldcs(p); }
  __device__ __forceinline__ float get(int) const { return static_cast<float>(r); }
};
template <>
struct Raw<bf16, 1> {
  uint16_t r;
  __device__ __forceinline__ void load(const bf16* p) {
    r = __ldcs(reinterpret_cast<const unsigned short*>(p));
  }
  __device__ __forceinline__ float get(int) const { return bf16_to_f32(r); }
};

template <int VEC>
__device__ __forceinline__ void store_group(void* base, size_t i, const float* v, bool f32) {
  if constexpr (VEC == 1) {
    store_act(base, i, v[0], f32);
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
template <int VEC>
__device__ __forceinline__ void load_param(const float* p, int i, float* v) {
  if constexpr (VEC == 1) {
    v[0] = __ldg(p + i);
  } else {
    *reinterpret_cast<float4*>(v) = __ldg(reinterpret_cast<const float4*>(p + i));
    *reinterpret_cast<float4*>(v + 4) = __ldg(reinterpret_cast<const float4*>(p + i) + 1);
  }
}

// Sums of one value or two over a row's threads; every thread gets them.  A
// CTA's row takes one barrier: `red` alternates between two buffers of 64
// floats, so a warp that is ahead writes the other one.
template <bool kCta>
__device__ __forceinline__ void row_sum(float& a, float*& red) {
  a = warp_sum(a);
  if constexpr (kCta) {
    const int lane = threadIdx.x & 31, n = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
    a = (lane & 15) < n ? red[lane & 15] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
    red = reinterpret_cast<float*>(reinterpret_cast<uintptr_t>(red) ^ 256);
  }
}
template <bool kCta>
__device__ __forceinline__ void row_sums(float& a, float& b, float*& red) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (kCta) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockDim.x >> 5;
    if (lane == 0) {
      red[w] = a;
      red[32 + w] = b;
    }
    __syncthreads();
    a = warp_sum(lane < n ? red[lane] : 0.f);
    b = warp_sum(lane < n ? red[32 + lane] : 0.f);
    red = reinterpret_cast<float*>(reinterpret_cast<uintptr_t>(red) ^ 256);
  }
}

// v rounded to bf16, in place, pairs at a time
template <int VEC>
__device__ __forceinline__ void round_bf16(float* v) {
  if constexpr (VEC == 1) {
    v[0] = __bfloat162float(__float2bfloat16_rn(v[0]));
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[k], v[k + 1]);
      const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
      v[k] = __uint_as_float(w << 16);
      v[k + 1] = __uint_as_float(w & 0xffff0000u);
    }
  }
}

struct None {};

template <typename TX, typename TR, int VEC, int NV, bool kCta>
__global__ void __launch_bounds__(kCta ? kMaxCta : kRowWarps * 32, kCta && NV == 2 ? 2 : 1)
norm_fwd_regs(NormFwdArgs p) {
  constexpr bool kRes = !std::is_same<TR, None>::value;
  using TL = typename std::conditional<kRes, TR, TX>::type;   // the residual's loads
  constexpr bool kHf32 = std::is_same<TX, float>::value || std::is_same<TR, float>::value;
  __shared__ __align__(512) float buf[128];
  float* red = buf;
  const int tid = kCta ? threadIdx.x : threadIdx.x & 31, tpr = kCta ? blockDim.x : 32;
  const int D = p.width, groups = D / VEC;
  const float inv = 1.f / static_cast<float>(D);
  const long long step = static_cast<long long>(gridDim.x) * (kCta ? 1 : kRowWarps);
  long long r = kCta ? blockIdx.x
                     : static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
  const TX* x = static_cast<const TX*>(p.x);
  const TL* res = static_cast<const TL*>(p.res);
  Raw<TX, VEC> rx[NV];
  Raw<TL, VEC> rr[NV];
  auto fetch = [&](long long row) {
    if (row >= p.rows) return;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int g = v * tpr + tid;
      if (g < groups) {
        rx[v].load(x + row * D + g * VEC);
        if constexpr (kRes) rr[v].load(res + row * D + g * VEC);
      }
    }
  };
  fetch(r);
  for (; r < p.rows; r += step) {
    const size_t base = static_cast<size_t>(r) * D;
    float s[NV][VEC], sum = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int g = v * tpr + tid;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        s[v][k] = 0.f;
        if (g < groups) {
          s[v][k] = rx[v].get(k);
          if constexpr (kRes) s[v][k] += rr[v].get(k);
        }
      }
      if constexpr (kRes && !kHf32) round_bf16<VEC>(s[v]);
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum += s[v][k];
      if constexpr (kRes)
        if (g < groups) store_group<VEC>(p.h, base + g * VEC, s[v], kHf32);
    }
    fetch(r + step);
    float mean = 0.f;
    if (p.center) {
      row_sum<kCta>(sum, red);
      mean = sum * inv;
    }
    float d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v * tpr + tid < groups) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float d = s[v][k] - mean;
          d1 += d;
          d2 = fmaf(d, d, d2);
        }
      }
    row_sums<kCta>(d1, d2, red);
    d2 *= inv;
    if (p.center) {   // what the rounding of the mean left, taken out of both
      d1 *= inv;
      mean += d1;
      d2 = fmaxf(d2 - d1 * d1, 0.f);
    }
    const float rstd = rsqrtf(d2 + p.eps);
    if (tid == 0) {
      p.rstd[r] = rstd;
      if (p.center) p.mean[r] = mean;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int g = v * tpr + tid;
      if (g < groups) {
        float q[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[v][k] = (s[v][k] - mean) * rstd;
        if (p.weight) {
          load_param<VEC>(p.weight, g * VEC, q);
#pragma unroll
          for (int k = 0; k < VEC; ++k) s[v][k] *= q[k];
        }
        if (p.bias) {
          load_param<VEC>(p.bias, g * VEC, q);
#pragma unroll
          for (int k = 0; k < VEC; ++k) s[v][k] += q[k];
        }
        store_group<VEC>(p.y, base + g * VEC, s[v], p.y_f32);
      }
    }
  }
}

// TS: the type of s and dh.  dw and db are summed over a thread's rows in
// registers; a CTA's sums are one partial (norm_bwd_join adds the partials).
template <typename TS, typename TG, int VEC, int NV, bool kCta, bool kDb>
__global__ void __launch_bounds__(kCta ? kMaxCta : kRowWarps * 32)
norm_bwd_regs(NormBwdArgs p) {
  __shared__ __align__(512) float buf[128];
  extern __shared__ float cols[];   // warp rows: kRowWarps x D
  float* red = buf;
  const int tid = kCta ? threadIdx.x : threadIdx.x & 31, tpr = kCta ? blockDim.x : 32;
  const int D = p.width, groups = D / VEC;
  const float inv = 1.f / static_cast<float>(D);
  const long long step = static_cast<long long>(gridDim.x) * (kCta ? 1 : kRowWarps);
  long long r = kCta ? blockIdx.x
                     : static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
  const TS *sp = static_cast<const TS*>(p.s), *dhp = static_cast<const TS*>(p.dh);
  const TG* gp = static_cast<const TG*>(p.dy);
  Raw<TS, VEC> rs[NV], rh[NV];
  Raw<TG, VEC> rg[NV];
  float rstd_next = 0.f, mean_next = 0.f;
  auto fetch = [&](long long row) {
    if (row >= p.rows) return;
    rstd_next = p.rstd[row];
    mean_next = p.center ? p.mean[row] : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int g = v * tpr + tid;
      if (g < groups) {
        rs[v].load(sp + row * D + g * VEC);
        rg[v].load(gp + row * D + g * VEC);
      }
    }
  };
  float dw[NV][VEC], db[kDb ? NV : 1][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      dw[v][k] = 0.f;
      if constexpr (kDb) db[v][k] = 0.f;
    }
  fetch(r);
  for (; r < p.rows; r += step) {
    const size_t base = static_cast<size_t>(r) * D;
    const float rstd = rstd_next, mean = mean_next;
    float xh[NV][VEC], g[NV][VEC];
    float a = 0.f, b = 0.f;
    if (dhp) {   // needed last: in flight over the reduction, not a row ahead
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (v * tpr + tid < groups) rh[v].load(dhp + base + (v * tpr + tid) * VEC);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = v * tpr + tid;
      if (i < groups) {
        float w[VEC];
        if (p.weight) load_param<VEC>(p.weight, i * VEC, w);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          xh[v][k] = (rs[v].get(k) - mean) * rstd;
          g[v][k] = rg[v].get(k);
          dw[v][k] = fmaf(g[v][k], xh[v][k], dw[v][k]);
          if constexpr (kDb) db[v][k] += g[v][k];
          if (p.weight) g[v][k] *= w[k];
          a += g[v][k];
          b = fmaf(g[v][k], xh[v][k], b);
        }
      }
    }
    fetch(r + step);
    row_sums<kCta>(a, b, red);
    a = p.center ? a * inv : 0.f;
    b *= inv;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = v * tpr + tid;
      if (i < groups) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          g[v][k] = fmaf(fmaf(xh[v][k], -b, g[v][k] - a), rstd, dhp ? rh[v].get(k) : 0.f);
        if (p.ds_a) store_group<VEC>(p.ds_a, base + i * VEC, g[v], p.a_f32);
        if (p.ds_b) store_group<VEC>(p.ds_b, base + i * VEC, g[v], p.b_f32);
      }
    }
  }
  if (!p.dw && !p.db) return;
  float* out = p.partial + static_cast<size_t>(blockIdx.x) * 2 * D;
#pragma unroll
  for (int which = 0; which < (kDb ? 2 : 1); ++which) {
    float* dst = kCta ? out + which * D : cols + (threadIdx.x >> 5) * D;
    if (!kCta && which == 1) __syncthreads();   // cols is read below
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = v * tpr + tid;
      if (i < groups) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          float t = dw[v][k];
          if constexpr (kDb) t = which ? db[v][k] : t;
          dst[i * VEC + k] = t;
        }
      }
    }
    if constexpr (!kCta) {
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += kRowWarps * 32) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) t += cols[w * D + c];
        out[which * D + c] = t;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Rows whose width is no multiple of 8 start at any alignment.  One CTA a row:
// the row's 16-byte chunks, whole ones from the boundary below its start to the
// one above its end, come into a ring in shared memory by cp.async kStages - 1
// rows ahead (the last chunk of the tensor is cut to its end), and a thread
// reads its elements, v * threads + thread, from there.  With element-wise loads
// from global memory instead there are too few bytes in flight.  Every read of a
// stage is before the row's first sum, whose barrier lets the next issue
// overwrite it.
// ---------------------------------------------------------------------------

constexpr int kStages = 4;

__host__ __device__ inline int stage_bytes(int D, int es) { return (D * es + 46) / 16 * 16; }

template <typename T>
__device__ __forceinline__ void issue_row(char* dst, const void* base, size_t e0, int D,
                                          size_t total) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  const size_t a0 = e0 / E * E;
  const int chunks = (static_cast<int>(e0 - a0) + D + E - 1) / E;
  const T* src = static_cast<const T*>(base) + a0;
  const size_t left = total - a0;
  for (int c = threadIdx.x; c < chunks; c += blockDim.x) {
    const size_t rest = left - static_cast<size_t>(c) * E;
    cp_async_cg16(dst + 16 * c, src + static_cast<size_t>(c) * E,
                  rest < E ? static_cast<uint32_t>(rest) * sizeof(T) : 16u);
  }
}
// the row's element i
template <typename T>
__device__ __forceinline__ float stage_at(const char* src, size_t e0, int i) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  const int at = static_cast<int>(e0 % E) + i;
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(src)[at]);
  else
    return reinterpret_cast<const float*>(src)[at];
}

template <typename TX, typename TR, int NV>
__global__ void __launch_bounds__(kMaxCta, NV == 8 ? 2 : 1) norm_fwd_ring(NormFwdArgs p) {
  constexpr bool kRes = !std::is_same<TR, None>::value;
  using TL = typename std::conditional<kRes, TR, TX>::type;
  constexpr bool kHf32 = std::is_same<TX, float>::value || std::is_same<TR, float>::value;
  __shared__ __align__(512) float buf[128];
  extern __shared__ __align__(16) char ring[];
  float* red = buf;
  const int tid = threadIdx.x, tpr = blockDim.x, D = p.width;
  const float inv = 1.f / static_cast<float>(D);
  const size_t total = static_cast<size_t>(p.rows) * D;
  const int bx = stage_bytes(D, sizeof(TX)), stage = bx + (kRes ? stage_bytes(D, sizeof(TL)) : 0);
  auto issue = [&](long long row, int k) {
    if (row < p.rows) {
      const size_t e0 = static_cast<size_t>(row) * D;
      issue_row<TX>(ring + k * stage, p.x, e0, D, total);
      if constexpr (kRes) issue_row<TL>(ring + k * stage + bx, p.res, e0, D, total);
    }
    cp_async_commit();
  };
  for (int k = 0; k < kStages - 1; ++k)
    issue(blockIdx.x + static_cast<long long>(k) * gridDim.x, k);
  int at = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    issue(r + static_cast<long long>(kStages - 1) * gridDim.x, (at + kStages - 1) % kStages);
    cp_async_wait<kStages - 1>();
    __syncthreads();
    const size_t base = static_cast<size_t>(r) * D;
    const char* src = ring + at * stage;
    at = (at + 1) % kStages;
    float s[NV], sum = 0.f, d2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = v * tpr + tid;
      s[v] = 0.f;
      if (i < D) {
        s[v] = stage_at<TX>(src, base, i);
        if constexpr (kRes) {
          s[v] += stage_at<TL>(src + bx, base, i);
          if constexpr (!kHf32) s[v] = __bfloat162float(__float2bfloat16_rn(s[v]));
          store_act(p.h, base + i, s[v], kHf32);
        }
      }
      sum += s[v];
    }
    // here whatever `center` is: the barrier also frees the stage
    row_sum<true>(sum, red);
    float mean = p.center ? sum * inv : 0.f;
    float d1 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v * tpr + tid < D) {
        const float d = s[v] - mean;
        d1 += d;
        d2 = fmaf(d, d, d2);
      }
    row_sums<true>(d1, d2, red);
    d2 *= inv;
    if (p.center) {
      d1 *= inv;
      mean += d1;
      d2 = fmaxf(d2 - d1 * d1, 0.f);
    }
    const float rstd = rsqrtf(d2 + p.eps);
    if (tid == 0) {
      p.rstd[r] = rstd;
      if (p.center) p.mean[r] = mean;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = v * tpr + tid;
      if (i < D) {
        float y = (s[v] - mean) * rstd;
        if (p.weight) y *= __ldg(p.weight + i);
        if (p.bias) y += __ldg(p.bias + i);
        store_act(p.y, base + i, y, p.y_f32);
      }
    }
  }
  cp_async_wait<0>();
}

template <typename TS, typename TG, int NV>
__global__ void __launch_bounds__(kMaxCta, 1) norm_bwd_ring(NormBwdArgs p) {
  __shared__ __align__(512) float buf[128];
  extern __shared__ __align__(16) char ring[];
  float* red = buf;
  const int tid = threadIdx.x, tpr = blockDim.x, D = p.width;
  const float inv = 1.f / static_cast<float>(D);
  const size_t total = static_cast<size_t>(p.rows) * D;
  const int bs = stage_bytes(D, sizeof(TS)), bg = stage_bytes(D, sizeof(TG));
  const int stage = bs + bg + (p.dh ? bs : 0);
  auto issue = [&](long long row, int k) {
    if (row < p.rows) {
      const size_t e0 = static_cast<size_t>(row) * D;
      issue_row<TS>(ring + k * stage, p.s, e0, D, total);
      issue_row<TG>(ring + k * stage + bs, p.dy, e0, D, total);
      if (p.dh) issue_row<TS>(ring + k * stage + bs + bg, p.dh, e0, D, total);
    }
    cp_async_commit();
  };
  for (int k = 0; k < kStages - 1; ++k)
    issue(blockIdx.x + static_cast<long long>(k) * gridDim.x, k);
  float dw[NV], db[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) dw[v] = db[v] = 0.f;
  int at = 0;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    issue(r + static_cast<long long>(kStages - 1) * gridDim.x, (at + kStages - 1) % kStages);
    const float rstd = p.rstd[r], mean = p.center ? p.mean[r] : 0.f;
    cp_async_wait<kStages - 1>();
    __syncthreads();
    const size_t base = static_cast<size_t>(r) * D;
    const char* src = ring + at * stage;
    at = (at + 1) % kStages;
    float xh[NV], g[NV], dh[NV], a = 0.f, b = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = v * tpr + tid;
      if (i < D) {
        xh[v] = (stage_at<TS>(src, base, i) - mean) * rstd;
        g[v] = stage_at<TG>(src + bs, base, i);
        dh[v] = p.dh ? stage_at<TS>(src + bs + bg, base, i) : 0.f;
        dw[v] = fmaf(g[v], xh[v], dw[v]);
        db[v] += g[v];
        if (p.weight) g[v] *= __ldg(p.weight + i);
        a += g[v];
        b = fmaf(g[v], xh[v], b);
      }
    }
    row_sums<true>(a, b, red);
    a = p.center ? a * inv : 0.f;
    b *= inv;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = v * tpr + tid;
      if (i < D) {
        const float d = fmaf(fmaf(xh[v], -b, g[v] - a), rstd, dh[v]);
        if (p.ds_a) store_act(p.ds_a, base + i, d, p.a_f32);
        if (p.ds_b) store_act(p.ds_b, base + i, d, p.b_f32);
      }
    }
  }
  cp_async_wait<0>();
  if (!p.dw && !p.db) return;
  float* out = p.partial + static_cast<size_t>(blockIdx.x) * 2 * D;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int i = v * tpr + tid;
    if (i < D) {
      out[i] = dw[v];
      out[D + i] = db[v];
    }
  }
}

// How a width is held.  VEC 8: warp rows up to 768 elements (three groups a
// lane are as many as the backward's five arrays of them leave registers for),
// CTA rows with two groups a thread up to 8192, in the forward with four up to
// 16384.  VEC 1: warp rows up to 256, then the ring with 8 elements a thread up
// to 4096, 16 up to 8192 (as far as its stages fit).  Wider rows are read again
// for each pass (threads 0).
struct Shape {
  int vec, nv, threads;   // threads 32: warp rows
};
Shape shape_of(int D, bool fwd) {
  auto up = [](int n, int per) { return (n + per * 32 - 1) / (per * 32) * 32; };
  if (D % 8 == 0) {
    if (D <= 768) return {8, (D + 255) / 256, 32};
    if (D <= 16 * kMaxCta) return {8, 2, up(D, 16)};
    if (fwd && D <= 32 * kMaxCta) return {8, 4, up(D, 32)};
  } else if (D <= 256) {
    return {1, 8, 32};
  } else if (D <= 8 * kMaxCta) {
    return {1, 8, up(D, 8)};
  } else if (D <= 16 * kMaxCta) {
    return {1, 16, up(D, 16)};
  }
  return {0, 0, 0};
}
constexpr size_t kMaxRing = 220 * 1024;   // shared memory the ring's stages may take

// One wave of CTAs, each walking rows a grid apart.
template <typename K>
int wave(K kernel, long long rows, int threads, size_t smem) {
  const long long want = threads == 32 ? (rows + kRowWarps - 1) / kRowWarps : rows;
  if (want <= kSms) return static_cast<int>(want);
  int n = 1;
  cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads == 32 ? kRowWarps * 32 : threads,
                                                smem);
  const long long cap = static_cast<long long>(kSms) * (n < 1 ? 1 : n);
  return static_cast<int>(want < cap ? want : cap);
}

// ---------------------------------------------------------------------------
// Rows of any width, read again for each pass
// ---------------------------------------------------------------------------

constexpr int kColThreads = 256;
constexpr int kColRows = 8;      // warps of a column block, each on every 8th row
constexpr int kMaxPartials = 296;

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
      if (p.dh) d += load_act(p.dh, base + i, p.dh_f32);
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

template <typename TX, typename TR, int VEC, int NV, bool kCta>
void fwd_go(const NormFwdArgs& p, Shape sh, cudaStream_t st) {
  auto k = norm_fwd_regs<TX, TR, VEC, NV, kCta>;
  k<<<wave(k, p.rows, sh.threads, 0), kCta ? sh.threads : kRowWarps * 32, 0, st>>>(p);
}
// A ring kernel of this much shared memory, one wave; the stages of up to 8192
// elements of three fp32 tensors do not fit four times, so such rows are refused
// here and read again for each pass.
template <typename K>
cudaError_t allow(K kernel, size_t smem) {
  return smem <= 48 * 1024 ? cudaSuccess
                           : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  static_cast<int>(smem));
}
size_t ring_fwd(const NormFwdArgs& p) {
  return kStages * (stage_bytes(p.width, p.x_f32 ? 4 : 2) +
                    (p.res ? stage_bytes(p.width, p.res_f32 ? 4 : 2) : 0));
}
size_t ring_bwd(const NormBwdArgs& p) {
  return kStages * (stage_bytes(p.width, p.s_f32 ? 4 : 2) * (p.dh ? 2 : 1) +
                    stage_bytes(p.width, p.dy_f32 ? 4 : 2));
}
template <typename TX, typename TR, int NV>
cudaError_t fwd_ring(const NormFwdArgs& p, Shape sh, cudaStream_t st) {
  auto k = norm_fwd_ring<TX, TR, NV>;
  const size_t smem = ring_fwd(p);
  cudaError_t e = allow(k, smem);
  if (e != cudaSuccess) return e;
  k<<<wave(k, p.rows, sh.threads, smem), sh.threads, smem, st>>>(p);
  return cudaGetLastError();
}
template <typename TX, typename TR>
cudaError_t fwd_typed(const NormFwdArgs& p, Shape sh, cudaStream_t st) {
  if (sh.threads == 32) {
    if (sh.vec == 1) fwd_go<TX, TR, 1, 8, false>(p, sh, st);
    else if (sh.nv == 1) fwd_go<TX, TR, 8, 1, false>(p, sh, st);
    else if (sh.nv == 2) fwd_go<TX, TR, 8, 2, false>(p, sh, st);
    else fwd_go<TX, TR, 8, 3, false>(p, sh, st);
  } else {
    if (sh.vec == 1) return sh.nv == 8 ? fwd_ring<TX, TR, 8>(p, sh, st) : fwd_ring<TX, TR, 16>(p, sh, st);
    if (sh.nv == 2) fwd_go<TX, TR, 8, 2, true>(p, sh, st);
    else fwd_go<TX, TR, 8, 4, true>(p, sh, st);
  }
  return cudaGetLastError();
}

template <typename TS, typename TG, bool kDb, int VEC, int NV, bool kCta>
int bwd_go(const NormBwdArgs& p, Shape sh, int most, cudaStream_t st) {
  auto k = norm_bwd_regs<TS, TG, VEC, NV, kCta, kDb>;
  const size_t smem = !kCta && (p.dw || p.db) ? sizeof(float) * kRowWarps * p.width : 0;
  int grid = wave(k, p.rows, sh.threads, smem);
  if (grid > most) grid = most;
  k<<<grid, kCta ? sh.threads : kRowWarps * 32, smem, st>>>(p);
  return grid;
}
template <typename TS, typename TG, int NV>
int bwd_ring(const NormBwdArgs& p, Shape sh, int most, cudaStream_t st) {
  auto k = norm_bwd_ring<TS, TG, NV>;
  const size_t smem = ring_bwd(p);
  if (allow(k, smem) != cudaSuccess) return 0;
  int grid = wave(k, p.rows, sh.threads, smem);
  if (grid > most) grid = most;
  k<<<grid, sh.threads, smem, st>>>(p);
  return grid;
}
template <typename TS, typename TG, bool kDb>
int bwd_typed(const NormBwdArgs& p, Shape sh, int most, cudaStream_t st) {
  if (sh.threads == 32) {
    if (sh.vec == 1) return bwd_go<TS, TG, kDb, 1, 8, false>(p, sh, most, st);
    if (sh.nv == 1) return bwd_go<TS, TG, kDb, 8, 1, false>(p, sh, most, st);
    if (sh.nv == 2) return bwd_go<TS, TG, kDb, 8, 2, false>(p, sh, most, st);
    return bwd_go<TS, TG, kDb, 8, 3, false>(p, sh, most, st);
  }
  if (sh.vec == 1)
    return sh.nv == 8 ? bwd_ring<TS, TG, 8>(p, sh, most, st) : bwd_ring<TS, TG, 16>(p, sh, most, st);
  return bwd_go<TS, TG, kDb, 8, 2, true>(p, sh, most, st);
}

}  // namespace

cudaError_t norm_fwd(const NormFwdArgs& p, cudaStream_t st) {
  const Shape sh = shape_of(p.width, true);
  if (sh.threads == 0 || (sh.vec == 1 && sh.threads > 32 && ring_fwd(p) > kMaxRing)) {
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

// The most partials of dw and db that a backward writes, whichever way it takes.
int norm_bwd_partials(long long rows, int width) {
  (void)width;
  return static_cast<int>(rows < kSms * kMaxResident ? rows : kSms * kMaxResident);
}

cudaError_t norm_bwd(const NormBwdArgs& p, cudaStream_t st) {
  const Shape sh = shape_of(p.width, false);
  int parts = norm_bwd_partials(p.rows, p.width);
  if (sh.threads && !(sh.vec == 1 && sh.threads > 32 && ring_bwd(p) > kMaxRing)) {
    auto go = [&](auto ts, auto tg) {
      parts = p.db ? bwd_typed<decltype(ts), decltype(tg), true>(p, sh, parts, st)
                   : bwd_typed<decltype(ts), decltype(tg), false>(p, sh, parts, st);
    };
    if (p.s_f32) p.dy_f32 ? go(float{}, float{}) : go(float{}, bf16{});
    else p.dy_f32 ? go(bf16{}, float{}) : go(bf16{}, bf16{});
  } else {
    const int want = static_cast<int>((p.rows + 31) / 32 < kMaxPartials ? (p.rows + 31) / 32
                                                                        : kMaxPartials);
    if (want < parts) parts = want;
    if (p.ds_a || p.ds_b) norm_bwd_rows<<<row_grid(p.rows), kThreads, 0, st>>>(p);
    if (p.dw || p.db)
      norm_bwd_cols<<<dim3((p.width + 31) / 32, parts), kColThreads, 0, st>>>(p, parts);
  }
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && (p.dw || p.db)) {
    norm_bwd_join<<<dim3((p.width + 31) / 32, p.db ? 2 : 1), kJoinWarps * 32, 0, st>>>(
        p.partial, p.dw, p.db, p.width, parts);
    e = cudaGetLastError();
  }
  return e;
}

}  // namespace gmdn
