// Activations in 8 bits: packing and restoring a tensor, and GELU / SwiGLU
// whose backward reads the 8-bit checkpoint of their inputs.
//
// A block of 128 consecutive elements of the contiguous tensor shares a scale:
//   a = max |x|,  r = fl(127 / a),  q = round_even(x r),  restored q s, s = fl(a fl(1/127))
// |x| r <= 127 (1 + 2^-24), so q never leaves [-127, 127].  The product x r is
// rounded once, to the integer, by adding 1.5 * 2^23 in one fma, so the codes
// are exactly those of the formula.  A block whose largest magnitude is below
// 2^-100 is kept as zeros (r would leave the normal range); a block that holds
// a NaN or an infinity comes back as NaN.
//
//   GELU:   y = x P(x);  dx = dy (P(x) + x phi(x)), P the normal distribution
//   SwiGLU: y = a sig(a) u;  du = dy a sig(a),  da = dy u sig(a) (1 + a (1 - sig(a)))
// with the restored x, (u, a) in the backward, which also writes the restored
// y: the weight gradient of the projection that read y needs it.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "step_ops.h"

namespace gmdn {
namespace {

constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100
constexpr float kMagic = 12582912.f;              // 1.5 * 2^23
constexpr int kWarpsA = 8;
constexpr int kUnroll = 4;   // blocks (forward) / vectors (backward) a thread has in flight
constexpr int kCtas = 148 * 8;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tail = P(-|x|) and e = e^(-x^2 / 2) for the type of the tensors.
//
// bf16: Abramowitz & Stegun 7.1.26, P(-|x|) = poly(t) e / 2 with
// t = 1 / (1 + 0.3275911 |x| / sqrt 2): within 0.75e-7 of P (their bound on
// erf, halved), a 2^-15th of the rounding to bf16 where P is of order 1, at
// two SFU operations and ten others.  fp32: CUDA's normcdff, whose error in
// ulp the rounding to fp32 needs; those tensors move twice the bytes, which
// hides its ~3x arithmetic.
template <typename T>
struct Normal;
template <>
struct Normal<__nv_bfloat16> {
  __device__ __forceinline__ static void at(float x, float& tail, float& e) {
    e = ex2(x * x * -0.72134752044448170f);   // -log2(e) / 2
    const float t = rcp(fmaf(fabsf(x), 0.23164189f, 1.f));
    float q = fmaf(t, 0.5307027145f, -0.7265760135f);
    q = fmaf(t, q, 0.7107068705f);
    q = fmaf(t, q, -0.142248368f);
    q = fmaf(t, q, 0.127414796f);
    tail = t * q * e;
  }
};
template <>
struct Normal<float> {
  __device__ __forceinline__ static void at(float x, float& tail, float& e) {
    tail = normcdff(-fabsf(x));
    e = expf(-0.5f * x * x);
  }
};

// P(x) from tail, and from it GELU = x P and its derivative P + x phi.
__device__ __forceinline__ float share(float x, float tail) { return x < 0.f ? tail : 1.f - tail; }

template <typename T>
__device__ __forceinline__ float sigmoid(float a);
template <>
__device__ __forceinline__ float sigmoid<__nv_bfloat16>(float a) {
  return rcp(1.f + ex2(a * -1.4426950408889634f));   // within 2^-21
}
template <>
__device__ __forceinline__ float sigmoid<float>(float a) {
  return __fdiv_rn(1.f, 1.f + expf(-a));
}

// N consecutive elements (4: 8 or 16 bytes; 8: 16 or 32), aligned
template <int N>
__device__ __forceinline__ void load_n(const __nv_bfloat16* p, float* v) {
  uint32_t r[N / 2];
  if constexpr (N == 4)
    *reinterpret_cast<uint2*>(r) = __ldcs(reinterpret_cast<const uint2*>(p));
  else
    *reinterpret_cast<uint4*>(r) = __ldcs(reinterpret_cast<const uint4*>(p));
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    v[2 * k] = __uint_as_float(r[k] << 16);
    v[2 * k + 1] = __uint_as_float(r[k] & 0xffff0000u);
  }
}
template <int N>
__device__ __forceinline__ void load_n(const float* p, float* v) {
#pragma unroll
  for (int k = 0; k < N; k += 4)
    *reinterpret_cast<float4*>(v + k) = __ldcs(reinterpret_cast<const float4*>(p + k));
}
template <int N>
__device__ __forceinline__ void store_n(__nv_bfloat16* p, const float* v) {
  __nv_bfloat162 r[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; ++k) r[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
  if constexpr (N == 4)
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(r);
  else
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(r);
}
template <int N>
__device__ __forceinline__ void store_n(float* p, const float* v) {
#pragma unroll
  for (int k = 0; k < N; k += 4)
    *reinterpret_cast<float4*>(p + k) = *reinterpret_cast<const float4*>(v + k);
}

// A block's scale and factor from the largest magnitude of the lane's values
// (as bits: NaN > inf > every number), one warp a block.
__device__ __forceinline__ float block_scale(uint32_t top, float& r) {
  top = __reduce_max_sync(~0u, top);
  const float a = __uint_as_float(top);
  const bool bad = top >= 0x7f800000u, tiny = a < kTiny;
  r = (bad || tiny) ? 0.f : __fdiv_rn(127.f, a);
  return bad ? __int_as_float(0x7fffffff) : (tiny ? 0.f : a * (1.f / 127.f));
}
template <int N>
__device__ __forceinline__ uint32_t magnitude(const float* v) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
  return top;
}
// one element's code in the low byte
__device__ __forceinline__ uint32_t code(float v, float r) {
  return __float_as_uint(fmaf(v, r, kMagic));
}
__device__ __forceinline__ uint32_t codes4(const float* v, float r) {
  const uint32_t lo = __byte_perm(code(v[0], r), code(v[1], r), 0x0040);
  const uint32_t hi = __byte_perm(code(v[2], r), code(v[3], r), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

template <typename T, int kKind>   // 0 pack, 1 GELU, 2 SwiGLU
__device__ __forceinline__ float act_of(float x, float a) {
  if constexpr (kKind == 1) {
    float tail, e;
    Normal<T>::at(x, tail, e);
    return x * share(x, tail);
  } else {
    return a * sigmoid<T>(a) * x;
  }
}

// One warp a block of 128 elements, 4 consecutive ones a lane; kUnroll blocks
// loaded before the first is worked on.  One redux gives the block's largest
// magnitude.
template <typename T, int kKind>
__global__ void __launch_bounds__(kWarpsA * 32) act8_fwd_kernel(Act8Args p) {
  const int lane = threadIdx.x & 31;
  const long long nw = static_cast<long long>(gridDim.x) * kWarpsA;
  const long long w = static_cast<long long>(blockIdx.x) * kWarpsA + (threadIdx.x >> 5);
  const T* x = static_cast<const T*>(p.x);
  const T* gate = static_cast<const T*>(p.gate);
  T* y = static_cast<T*>(p.y);
  const long long full = p.n / kAct8Block;
  for (long long b0 = w; b0 < full; b0 += nw * kUnroll) {
    float v[kUnroll][4], a[kKind == 2 ? kUnroll : 1][4];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long b = b0 + u * nw;
      if (b < full) {
        load_n<4>(x + b * kAct8Block + lane * 4, v[u]);
        if constexpr (kKind == 2) load_n<4>(gate + b * kAct8Block + lane * 4, a[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long b = b0 + u * nw;
      if (b >= full) break;
      const long long i = b * kAct8Block + lane * 4;
      if constexpr (kKind != 0) {
        float out[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          out[k] = act_of<T, kKind>(v[u][k], kKind == 2 ? a[kKind == 2 ? u : 0][k] : 0.f);
        store_n<4>(y + i, out);
      }
      float r;
      float s = block_scale(magnitude<4>(v[u]), r);
      *reinterpret_cast<uint32_t*>(p.codes + i) = codes4(v[u], r);
      if (lane == 0) p.scales[b] = s;
      if constexpr (kKind == 2) {
        s = block_scale(magnitude<4>(a[u]), r);
        *reinterpret_cast<uint32_t*>(p.gate_codes + i) = codes4(a[u], r);
        if (lane == 0) p.gate_scales[b] = s;
      }
    }
  }
  const int rest = static_cast<int>(p.n - full * kAct8Block);
  if (rest == 0 || w != full % nw) return;
  // the last, short block: element lane + 32 k
  const long long base = full * kAct8Block;
  float v[4], a[4], r;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = lane + 32 * k;
    v[k] = i < rest ? static_cast<float>(x[base + i]) : 0.f;
    a[k] = 0.f;
    if constexpr (kKind == 2)
      if (i < rest) a[k] = static_cast<float>(gate[base + i]);
    if constexpr (kKind != 0)
      if (i < rest) y[base + i] = static_cast<T>(act_of<T, kKind>(v[k], a[k]));
  }
  float s = block_scale(magnitude<4>(v), r);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 32 * k < rest) p.codes[base + lane + 32 * k] = static_cast<int8_t>(code(v[k], r));
  if (lane == 0) p.scales[full] = s;
  if constexpr (kKind == 2) {
    s = block_scale(magnitude<4>(a), r);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane + 32 * k < rest)
        p.gate_codes[base + lane + 32 * k] = static_cast<int8_t>(code(a[k], r));
    if (lane == 0) p.gate_scales[full] = s;
  }
}

// The backward of one element; kKind 0: the restored value alone.
template <typename T, int kKind>
__device__ __forceinline__ void back(float x, float a, float dy, float& dx, float& da, float& y) {
  if constexpr (kKind == 0) {
    y = x;
  } else if constexpr (kKind == 1) {
    float tail, e;
    Normal<T>::at(x, tail, e);
    const float P = share(x, tail);
    dx = dy * fmaf(x * 0.3989422804014327f, e, P);
    y = x * P;
  } else {
    const float sg = sigmoid<T>(a), silu = a * sg;
    dx = dy * silu;
    da = dy * x * sg * fmaf(a, 1.f - sg, 1.f);
    y = silu * x;
  }
}

// 8 consecutive elements a lane (a 16th of a block), kVecs vectors in flight.
template <typename T, int kKind>
__global__ void __launch_bounds__(kWarpsA * 32) act8_bwd_kernel(Act8Args p) {
  constexpr int kVecs = 2;
  const long long nt = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long t = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const T* dy = static_cast<const T*>(p.dy);
  T *dx = static_cast<T*>(p.dx), *dg = static_cast<T*>(p.dgate), *y = static_cast<T*>(p.y);
  const long long vecs = p.n / 8;
  for (long long j0 = t; j0 < vecs; j0 += nt * kVecs) {
    uint2 c[kVecs], gc[kKind == 2 ? kVecs : 1];
    float s[kVecs], gs[kKind == 2 ? kVecs : 1], d[kVecs][8];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const long long j = j0 + u * nt;
      if (j < vecs) {
        c[u] = __ldcs(reinterpret_cast<const uint2*>(p.codes) + j);
        s[u] = p.scales[j / (kAct8Block / 8)];
        if constexpr (kKind == 2) {
          gc[u] = __ldcs(reinterpret_cast<const uint2*>(p.gate_codes) + j);
          gs[u] = p.gate_scales[j / (kAct8Block / 8)];
        }
        if constexpr (kKind != 0) load_n<8>(dy + j * 8, d[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const long long j = j0 + u * nt;
      if (j >= vecs) break;
      float ox[8], og[8], oy[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int8_t q = static_cast<int8_t>((k < 4 ? c[u].x : c[u].y) >> (8 * (k & 3)));
        float a = 0.f;
        if constexpr (kKind == 2)
          a = static_cast<float>(static_cast<int8_t>((k < 4 ? gc[u].x : gc[u].y) >> (8 * (k & 3)))) *
              gs[u];
        back<T, kKind>(static_cast<float>(q) * s[u], a, kKind != 0 ? d[u][k] : 0.f, ox[k], og[k],
                       oy[k]);
      }
      if constexpr (kKind != 0) store_n<8>(dx + j * 8, ox);
      if constexpr (kKind == 2) store_n<8>(dg + j * 8, og);
      if (kKind == 0 || y) store_n<8>(y + j * 8, oy);
    }
  }
  const long long i = vecs * 8 + t;   // the last elements, one a thread
  if (i < p.n) {
    float a = 0.f, ox, og, oy;
    if constexpr (kKind == 2)
      a = static_cast<float>(p.gate_codes[i]) * p.gate_scales[i / kAct8Block];
    back<T, kKind>(static_cast<float>(p.codes[i]) * p.scales[i / kAct8Block], a,
                   kKind != 0 ? static_cast<float>(dy[i]) : 0.f, ox, og, oy);
    if constexpr (kKind != 0) dx[i] = static_cast<T>(ox);
    if constexpr (kKind == 2) dg[i] = static_cast<T>(og);
    if (kKind == 0 || y) y[i] = static_cast<T>(oy);
  }
}

int grid_for(long long units, int per_cta) {
  const long long want = (units + per_cta - 1) / per_cta;
  return static_cast<int>(want < 1 ? 1 : (want < kCtas ? want : kCtas));
}

template <int kKind>
cudaError_t fwd(const Act8Args& p, cudaStream_t st) {
  const int grid = grid_for((p.n + kAct8Block - 1) / kAct8Block, kWarpsA);
  if (p.f32)
    act8_fwd_kernel<float, kKind><<<grid, kWarpsA * 32, 0, st>>>(p);
  else
    act8_fwd_kernel<__nv_bfloat16, kKind><<<grid, kWarpsA * 32, 0, st>>>(p);
  return cudaGetLastError();
}
template <int kKind>
cudaError_t bwd(const Act8Args& p, cudaStream_t st) {
  const int grid = grid_for((p.n + 7) / 8, kWarpsA * 32);
  if (p.f32)
    act8_bwd_kernel<float, kKind><<<grid, kWarpsA * 32, 0, st>>>(p);
  else
    act8_bwd_kernel<__nv_bfloat16, kKind><<<grid, kWarpsA * 32, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t pack8(const Act8Args& p, cudaStream_t st) { return fwd<0>(p, st); }
cudaError_t unpack8(const Act8Args& p, cudaStream_t st) { return bwd<0>(p, st); }
cudaError_t act8_fwd(const Act8Args& p, cudaStream_t st) {
  return p.gated ? fwd<2>(p, st) : fwd<1>(p, st);
}
cudaError_t act8_bwd(const Act8Args& p, cudaStream_t st) {
  return p.gated ? bwd<2>(p, st) : bwd<1>(p, st);
}

}  // namespace gmdn
