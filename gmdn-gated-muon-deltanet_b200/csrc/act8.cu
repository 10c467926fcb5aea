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
constexpr int kEl = 4;   // elements a lane: a warp covers one block

__device__ __forceinline__ float gelu_share(float x) { return normcdff(x); }
__device__ __forceinline__ float sigmoid(float a) { return 1.f / (1.f + expf(-a)); }

// The warp's 128 elements (v[k] of element base + lane + 32 k) into codes and a scale.
__device__ __forceinline__ void quantise(const float* v, long long base, long long n,
                                         int8_t* codes, float* scales) {
  const int lane = threadIdx.x & 31;
  uint32_t top = 0;   // magnitude as bits: NaN > inf > every number
#pragma unroll
  for (int k = 0; k < kEl; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
  const bool bad = top >= 0x7f800000u;
  const float a = __uint_as_float(top);
  const float r = (bad || a < kTiny) ? 0.f : __fdiv_rn(127.f, a);
  const float s = bad ? __int_as_float(0x7fffffff) : (a < kTiny ? 0.f : a * (1.f / 127.f));
#pragma unroll
  for (int k = 0; k < kEl; ++k) {
    const long long i = base + lane + 32 * k;
    if (i < n) codes[i] = static_cast<int8_t>(__float_as_int(fmaf(v[k], r, kMagic)) & 0xff);
  }
  if (lane == 0) scales[base / kAct8Block] = s;
}

template <int kKind>   // 0 pack, 1 GELU, 2 SwiGLU
__global__ void __launch_bounds__(kWarpsA * 32) act8_fwd_kernel(Act8Args p) {
  const int lane = threadIdx.x & 31;
  const long long blocks = (p.n + kAct8Block - 1) / kAct8Block;
  for (long long b = static_cast<long long>(blockIdx.x) * kWarpsA + (threadIdx.x >> 5); b < blocks;
       b += static_cast<long long>(gridDim.x) * kWarpsA) {
    const long long base = b * kAct8Block;
    float x[kEl], a[kEl];
#pragma unroll
    for (int k = 0; k < kEl; ++k) {
      const long long i = base + lane + 32 * k;
      x[k] = i < p.n ? load_act(p.x, i, p.f32) : 0.f;
      if (kKind == 2) a[k] = i < p.n ? load_act(p.gate, i, p.f32) : 0.f;
      if (i < p.n && kKind == 1) store_act(p.y, i, x[k] * gelu_share(x[k]), p.f32);
      if (i < p.n && kKind == 2) store_act(p.y, i, a[k] * sigmoid(a[k]) * x[k], p.f32);
    }
    quantise(x, base, p.n, p.codes, p.scales);
    if (kKind == 2) quantise(a, base, p.n, p.gate_codes, p.gate_scales);
  }
}

template <int kKind>   // 0 unpack, 1 GELU, 2 SwiGLU
__global__ void __launch_bounds__(kWarpsA * 32) act8_bwd_kernel(Act8Args p) {
  const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < p.n;
       i += stride) {
    const long long b = i / kAct8Block;
    const float x = static_cast<float>(p.codes[i]) * p.scales[b];
    if (kKind == 0) {
      store_act(p.y, i, x, p.f32);
      continue;
    }
    const float dy = load_act(p.dy, i, p.f32);
    if (kKind == 1) {
      const float P = gelu_share(x);
      const float phi = 0.3989422804014327f * expf(-0.5f * x * x);
      store_act(p.dx, i, dy * fmaf(x, phi, P), p.f32);
      if (p.y) store_act(p.y, i, x * P, p.f32);
    } else {
      const float a = static_cast<float>(p.gate_codes[i]) * p.gate_scales[b];
      const float sg = sigmoid(a);
      store_act(p.dx, i, dy * a * sg, p.f32);
      store_act(p.dgate, i, dy * x * sg * (1.f + a * (1.f - sg)), p.f32);
      if (p.y) store_act(p.y, i, a * sg * x, p.f32);
    }
  }
}

int grid_of(long long blocks) {
  const long long want = (blocks + kWarpsA - 1) / kWarpsA;
  return static_cast<int>(want < 148 * 8 ? want : 148 * 8);
}
long long blocks_of(long long n) { return (n + kAct8Block - 1) / kAct8Block; }

}  // namespace

cudaError_t pack8(const Act8Args& p, cudaStream_t st) {
  act8_fwd_kernel<0><<<grid_of(blocks_of(p.n)), kWarpsA * 32, 0, st>>>(p);
  return cudaGetLastError();
}
cudaError_t unpack8(const Act8Args& p, cudaStream_t st) {
  act8_bwd_kernel<0><<<grid_of(blocks_of(p.n)), kWarpsA * 32, 0, st>>>(p);
  return cudaGetLastError();
}
cudaError_t act8_fwd(const Act8Args& p, cudaStream_t st) {
  if (p.gated)
    act8_fwd_kernel<2><<<grid_of(blocks_of(p.n)), kWarpsA * 32, 0, st>>>(p);
  else
    act8_fwd_kernel<1><<<grid_of(blocks_of(p.n)), kWarpsA * 32, 0, st>>>(p);
  return cudaGetLastError();
}
cudaError_t act8_bwd(const Act8Args& p, cudaStream_t st) {
  if (p.gated)
    act8_bwd_kernel<2><<<grid_of(blocks_of(p.n)), kWarpsA * 32, 0, st>>>(p);
  else
    act8_bwd_kernel<1><<<grid_of(blocks_of(p.n)), kWarpsA * 32, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace gmdn
