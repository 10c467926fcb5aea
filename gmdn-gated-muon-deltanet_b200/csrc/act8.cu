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
//
// Memory bounds it, with the instruction slots close: bf16 GELU moves 5 bytes an
// element forward and 7 backward, which leaves ~27 and ~38 instructions an
// element at the copy rate; the kernels take 19.  Measured (B200): 16384 x 4096
// bf16 GELU 59 us forward (0.86 of the 6536 GB/s copy rate) and 85 backward
// (0.84), SwiGLU at 0.85 and more, fp32 GELU at 0.87 and 0.84.

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "step_ops.h"

namespace gmdn {
namespace {

constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100
constexpr float kMagic = 12582912.f;              // 1.5 * 2^23
constexpr int kWarpsA = 8;
constexpr int kSms = 148;
// CTAs an SM holds (their registers bound it); the grid is one wave of them
template <typename T, int kKind>
constexpr int kResident =
    (kKind == 0 ? 6 : (kKind == 1 ? 4 : 3)) - (sizeof(T) == 4 ? 1 : 0);

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

// Pairs of elements: two fp32 operations an instruction.
__device__ __forceinline__ float2 pair(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }

// P(x) of the normal distribution and e = e^(-x^2 / 2), by the tensors' type.
//
// bf16: for x < 0, P = t q(t) e with t = 1 / (1 + 0.292 |x|) (the form of Abramowitz & Stegun
// 7.1.26), for the other side 1 less that.  q's six coefficients are a linear program's fit to
// the function in fp64 for |x| <= 14.2, towards the least of two bounds at once.  As fp32 numbers
// they give P within 6.8e-8, and within 5.4e-5 of its value where it is small; evaluated in fp32
// within 2.4e-7 and 5.7e-5 (in a model of the roundings), far below bf16's 2^-8 on either side.
// Two SFU operations and eleven others.
//
// fp32 needs more digits, on both sides: for |x| < 1, P = 1/2 + x R(x^2), where
// nothing cancels; beyond, the form above with more terms, in t = 1 / (1 + 0.3 |x|),
// and with e's exponent in two parts, since its rounding is a relative error of x^2 / 2
// half ulps.  R and the terms are weighted least-squares fits (reweighted towards
// the smallest largest error) to the functions in fp64: with the coefficients as fp32
// numbers 3.4e-8 and 2.4e-8 relative.
// P is within 8e-7 of its value relative (largest seen: 3.8e-7), rounding and the
// SFU's 2^-22 included, on the small side too (subnormal P is 0).  About 18
// instructions an element:
// 8192 x 4096 GELU 53 us forward and 81 backward, against 86 and 99 with
// CUDA's normcdff.
__device__ __forceinline__ void normal2(float2 x, float2& P, float2& e, __nv_bfloat16) {
  const float2 h = mul2(mul2(x, pair(-0.72134752044448170f)), x);   // -x^2 log2(e) / 2
  e = make_float2(ex2(h.x), ex2(h.y));
  const float2 t = make_float2(rcp(fmaf(fabsf(x.x), 0.2919999957084656f, 1.f)),
                               rcp(fmaf(fabsf(x.y), 0.2919999957084656f, 1.f)));
  float2 q = fma2(t, pair(-0.08656206727027893f), pair(0.27009639143943787f));
  q = fma2(t, q, pair(-0.07534580677747726f));
  q = fma2(t, q, pair(0.170305073261261f));
  q = fma2(t, q, pair(0.10408246517181396f));
  q = fma2(t, q, pair(0.11742392182350159f));
  const float2 tail = mul2(mul2(t, q), e);
  const float2 rest = fma2(tail, pair(-1.f), pair(1.f));
  P = make_float2(x.x < 0.f ? tail.x : rest.x, x.y < 0.f ? tail.y : rest.y);
}
__device__ __forceinline__ void normal2(float2 x, float2& P, float2& e, float) {
  // P(-15) is 0 in fp32; infinities stay out of the differences below
  const float2 a = make_float2(fminf(fabsf(x.x), 15.f), fminf(fabsf(x.y), 15.f));
  const float2 s = mul2(a, a), rest = fma2(a, a, neg2(s));   // a^2 = s + rest
  constexpr float kHi = 0.7213475108146667f, kLo = 9.629815e-9f;   // log2(e) / 2
  const float2 h = mul2(s, pair(-kHi));
  float2 l = fma2(s, pair(-kHi), neg2(h));
  l = fma2(rest, pair(-kHi), l);
  l = fma2(s, pair(-kLo), l);
  e = make_float2(ex2(h.x), ex2(h.y));
  e = fma2(e, mul2(l, pair(0.6931471805599453f)), e);   // 2^l = 1 + l log 2
  const float2 t = make_float2(rcp(fmaf(a.x, 0.3f, 1.f)), rcp(fmaf(a.y, 0.3f, 1.f)));
  float2 q = fma2(t, pair(0.028240492567420006f), pair(-0.08061183243989944f));
  q = fma2(t, q, pair(0.046382151544094086f));
  q = fma2(t, q, pair(0.009018266573548317f));
  q = fma2(t, q, pair(0.06179765984416008f));
  q = fma2(t, q, pair(0.08690078556537628f));
  q = fma2(t, q, pair(0.10893955081701279f));
  q = fma2(t, q, pair(0.11968203634023666f));
  q = fma2(t, q, pair(0.1196826919913292f));
  const float2 tail = mul2(mul2(t, q), e);
  float2 c = fma2(s, pair(-7.654207365703769e-06f), pair(0.00011348637053743005f));
  c = fma2(s, c, pair(-0.0011863299878314137f));
  c = fma2(s, c, pair(0.009973322972655296f));
  c = fma2(s, c, pair(-0.06649035960435867f));
  c = fma2(s, c, pair(0.3989422917366028f));
  c = fma2(x, c, pair(0.5f));
  P = make_float2(a.x < 1.f ? c.x : (x.x < 0.f ? tail.x : 1.f - tail.x),
                  a.y < 1.f ? c.y : (x.y < 0.f ? tail.y : 1.f - tail.y));
}

__device__ __forceinline__ float2 sigmoid2(float2 a, __nv_bfloat16) {   // within 2^-21 + |a| 2^-23
  const float2 h = mul2(a, pair(-1.4426950408889634f));
  return make_float2(rcp(1.f + ex2(h.x)), rcp(1.f + ex2(h.y)));
}
__device__ __forceinline__ float2 sigmoid2(float2 a, float) {
  return make_float2(__fdiv_rn(1.f, 1.f + expf(-a.x)), __fdiv_rn(1.f, 1.f + expf(-a.y)));
}

// 32 bytes (sm_100's widest access), streamed past L1
struct __align__(32) Wide {
  uint32_t w[8];
};
__device__ __forceinline__ Wide load32(const void* p) {
  Wide v;
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]),
                 "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p));
  return v;
}
__device__ __forceinline__ void store32(void* p, const Wide& v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]),
               "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]),
               "r"(v.w[7])
               : "memory");
}

// 16 consecutive elements as loaded; an 8th of a block of 128.
constexpr int kVec = 16;
constexpr int kLanes = kAct8Block / kVec;   // lanes that share a block
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  Wide r;
  __device__ __forceinline__ void load(const void* p, uint32_t j) {
    r = load32(static_cast<const Wide*>(p) + j);
  }
  __device__ __forceinline__ float2 get(int k) const {
    return make_float2(__uint_as_float(r.w[k] << 16), __uint_as_float(r.w[k] & 0xffff0000u));
  }
  // the largest magnitude, as fp32 bits: NaN > inf > every number
  __device__ __forceinline__ uint32_t magnitude() const {
    uint32_t m = r.w[0] & 0x7fff7fffu;
#pragma unroll
    for (int k = 1; k < 8; ++k) m = __vmaxu2(m, r.w[k] & 0x7fff7fffu);
    return max(m & 0xffff0000u, m << 16);
  }
  __device__ __forceinline__ static void store(void* p, uint32_t j, const float2* v) {
    Wide o;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[k].x, v[k].y);
      o.w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    store32(static_cast<Wide*>(p) + j, o);
  }
};
template <>
struct Vec<float> {
  Wide r[2];
  __device__ __forceinline__ void load(const void* p, uint32_t j) {
    r[0] = load32(static_cast<const Wide*>(p) + 2 * static_cast<size_t>(j));
    r[1] = load32(static_cast<const Wide*>(p) + 2 * static_cast<size_t>(j) + 1);
  }
  __device__ __forceinline__ float2 get(int k) const {
    return make_float2(__uint_as_float(r[k / 4].w[2 * k % 8]),
                       __uint_as_float(r[k / 4].w[2 * k % 8 + 1]));
  }
  __device__ __forceinline__ uint32_t magnitude() const {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) m = max(m, r[k / 8].w[k % 8] & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ static void store(void* p, uint32_t j, const float2* v) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Wide o;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o.w[2 * k] = __float_as_uint(v[4 * h + k].x);
        o.w[2 * k + 1] = __float_as_uint(v[4 * h + k].y);
      }
      store32(static_cast<Wide*>(p) + 2 * static_cast<size_t>(j) + h, o);
    }
  }
};

// A block's scale, and its factor r, from the largest magnitude's bits.
__device__ __forceinline__ float block_scale(uint32_t top, float& r) {
  const float a = __uint_as_float(top);
  const bool bad = top >= 0x7f800000u, tiny = a < kTiny;
  r = (bad || tiny) ? 0.f : __fdiv_rn(127.f, a);
  return bad ? __int_as_float(0x7fffffff) : (tiny ? 0.f : a * (1.f / 127.f));
}
// codes of a pair, each in the low byte of its word
__device__ __forceinline__ float2 code2(float2 v, float r) {
  return fma2(v, pair(r), pair(kMagic));
}
__device__ __forceinline__ uint32_t codes4(float2 v0, float2 v1, float r) {
  const float2 a = code2(v0, r), b = code2(v1, r);
  const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// the pair that two codes stand for
__device__ __forceinline__ float2 value2(uint32_t q, int k, float s) {
  const int a = static_cast<int8_t>(q >> (16 * k)), b = static_cast<int8_t>(q >> (16 * k + 8));
  return mul2(make_float2(static_cast<float>(a), static_cast<float>(b)), pair(s));
}

template <typename T, int kKind>   // 1 GELU of x, 2 SwiGLU of x and the gate a
__device__ __forceinline__ float2 act2(float2 x, float2 a) {
  if constexpr (kKind == 1) {
    float2 P, e;
    normal2(x, P, e, T{});
    return mul2(x, P);
  } else {
    return mul2(mul2(a, sigmoid2(a, T{})), x);
  }
}

// The codes and the scale of a lane's 16 elements; 8 lanes (`group`) share a block.
template <typename T>
__device__ __forceinline__ void pack_vec(const Vec<T>& v, uint32_t group, uint32_t j,
                                         int8_t* codes, float* scales) {
  const uint32_t top = __reduce_max_sync(group, v.magnitude());
  float r;
  const float s = block_scale(top, r);
  uint32_t c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k] = codes4(v.get(2 * k), v.get(2 * k + 1), r);
  reinterpret_cast<uint4*>(codes)[j] = make_uint4(c[0], c[1], c[2], c[3]);
  if (threadIdx.x % kLanes == 0) scales[j / kLanes] = s;
}

// 16 consecutive elements a lane, a quarter of a warp a block of 128: 32-byte
// accesses, and one redux and one division for every 16 elements of a lane.
// The next vector is loaded before the current one is worked on: the kernels
// are nearly out of instruction slots, so what hides the loads is not more
// warps.  Vector indexes are 32-bit (the caller splits longer tensors).
template <typename T, int kKind>   // 0 pack, 1 GELU, 2 SwiGLU
__global__ void __launch_bounds__(kWarpsA * 32, kResident<T, kKind>) act8_fwd_kernel(Act8Args p) {
  const uint32_t nt = gridDim.x * blockDim.x;
  const uint32_t t = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t group = 0xffu << (threadIdx.x & 24);
  const T* x = static_cast<const T*>(p.x);
  const T* gate = static_cast<const T*>(p.gate);
  T* y = static_cast<T*>(p.y);
  const long long full = p.n / kAct8Block;
  const uint32_t vecs = static_cast<uint32_t>(full * kLanes);
  Vec<T> now, next, gnow, gnext;
  auto fetch = [&](uint32_t j, Vec<T>& v, Vec<T>& g) {
    if (j < vecs) {
      v.load(x, j);
      if constexpr (kKind == 2) g.load(gate, j);
    }
  };
  fetch(t, now, gnow);
  for (uint32_t j = t; j < vecs; j += nt) {
    fetch(j + nt, next, gnext);
    if constexpr (kKind != 0) {
      float2 out[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        out[k] = act2<T, kKind>(now.get(k), kKind == 2 ? gnow.get(k) : now.get(k));
      Vec<T>::store(y, j, out);
    }
    pack_vec(now, group, j, p.codes, p.scales);
    if constexpr (kKind == 2) pack_vec(gnow, group, j, p.gate_codes, p.gate_scales);
    now = next;
    if constexpr (kKind == 2) gnow = gnext;
  }
  // the last, short block: one warp, element lane + 32 k
  const int rest = static_cast<int>(p.n - full * kAct8Block);
  if (rest == 0 || blockIdx.x != gridDim.x - 1 || threadIdx.x >= 32) return;
  const long long base = full * kAct8Block;
  const int lane = threadIdx.x;
  auto pack_rest = [&](const T* in, int8_t* codes, float* scales) {
    uint32_t top = 0;
    for (int i = lane; i < rest; i += 32)
      top = max(top, __float_as_uint(static_cast<float>(in[base + i])) & 0x7fffffffu);
    float r;
    const float s = block_scale(__reduce_max_sync(~0u, top), r);
    for (int i = lane; i < rest; i += 32)
      codes[base + i] = static_cast<int8_t>(
          __float_as_uint(fmaf(static_cast<float>(in[base + i]), r, kMagic)));
    if (lane == 0) scales[full] = s;
  };
  pack_rest(x, p.codes, p.scales);
  if constexpr (kKind == 2) pack_rest(gate, p.gate_codes, p.gate_scales);
  if constexpr (kKind != 0)
    for (int i = lane; i < rest; i += 32)
      y[base + i] = static_cast<T>(
          act2<T, kKind>(pair(static_cast<float>(x[base + i])),
                         pair(kKind == 2 ? static_cast<float>(gate[base + i]) : 0.f)).x);
}

// The backward of a pair; kKind 0: the restored value alone.
template <typename T, int kKind>
__device__ __forceinline__ void back2(float2 x, float2 a, float2 dy, float2& dx, float2& da,
                                      float2& y) {
  if constexpr (kKind == 0) {
    y = x;
  } else if constexpr (kKind == 1) {
    float2 P, e;
    normal2(x, P, e, T{});
    dx = mul2(dy, fma2(mul2(x, pair(0.3989422804014327f)), e, P));
    y = mul2(x, P);
  } else {
    const float2 sg = sigmoid2(a, T{}), silu = mul2(a, sg);
    dx = mul2(dy, silu);
    // sig (1 + a (1 - sig)) = sig + silu - silu sig
    const float2 slope = fma2(neg2(silu), sg, make_float2(sg.x + silu.x, sg.y + silu.y));
    da = mul2(mul2(dy, x), slope);
    y = mul2(silu, x);
  }
}

template <typename T, int kKind>   // 0 unpack, 1 GELU, 2 SwiGLU
__global__ void __launch_bounds__(kWarpsA * 32, kResident<T, kKind>) act8_bwd_kernel(Act8Args p) {
  const uint32_t nt = gridDim.x * blockDim.x;
  const uint32_t t = blockIdx.x * blockDim.x + threadIdx.x;
  const T* dy = static_cast<const T*>(p.dy);
  T *dx = static_cast<T*>(p.dx), *dg = static_cast<T*>(p.dgate), *y = static_cast<T*>(p.y);
  const uint32_t vecs = static_cast<uint32_t>(p.n / kVec);
  struct In {
    uint4 c, gc;
    float s, gs;
    Vec<T> d;
  } now, next;
  auto fetch = [&](uint32_t j, In& in) {
    if (j < vecs) {
      in.c = __ldcs(reinterpret_cast<const uint4*>(p.codes) + j);
      in.s = p.scales[j / kLanes];
      if constexpr (kKind == 2) {
        in.gc = __ldcs(reinterpret_cast<const uint4*>(p.gate_codes) + j);
        in.gs = p.gate_scales[j / kLanes];
      }
      if constexpr (kKind != 0) in.d.load(dy, j);
    }
  };
  auto word = [](const uint4& c, int k) {
    return k < 2 ? (k < 1 ? c.x : c.y) : (k < 3 ? c.z : c.w);
  };
  fetch(t, now);
  for (uint32_t j = t; j < vecs; j += nt) {
    fetch(j + nt, next);
    float2 ox[8], og[8], oy[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 v = value2(word(now.c, k / 2), k & 1, now.s);
      float2 a = v, d = v;
      if constexpr (kKind == 2) a = value2(word(now.gc, k / 2), k & 1, now.gs);
      if constexpr (kKind != 0) d = now.d.get(k);
      back2<T, kKind>(v, a, d, ox[k], og[k], oy[k]);
    }
    if constexpr (kKind != 0) Vec<T>::store(dx, j, ox);
    if constexpr (kKind == 2) Vec<T>::store(dg, j, og);
    if (kKind == 0 || y) Vec<T>::store(y, j, oy);
    now = next;
  }
  const long long i = static_cast<long long>(vecs) * kVec + t;   // the last elements, one a thread
  if (i < p.n) {
    float2 a = pair(0.f), ox, og, oy;
    if constexpr (kKind == 2)
      a = pair(static_cast<float>(p.gate_codes[i]) * p.gate_scales[i / kAct8Block]);
    back2<T, kKind>(pair(static_cast<float>(p.codes[i]) * p.scales[i / kAct8Block]), a,
                    pair(kKind != 0 ? static_cast<float>(dy[i]) : 0.f), ox, og, oy);
    if constexpr (kKind != 0) dx[i] = static_cast<T>(ox.x);
    if constexpr (kKind == 2) dg[i] = static_cast<T>(og.x);
    if (kKind == 0 || y) y[i] = static_cast<T>(oy.x);
  }
}

// Calls with more elements than the 32-bit vector indexes reach run in slabs.
constexpr long long kSlab = 1ll << 34;

template <typename T, int kKind, bool kFwd>
cudaError_t launch(const Act8Args& p, cudaStream_t st) {
  const long long n = p.n;
  constexpr size_t es = sizeof(T);
  constexpr int cap = kSms * kResident<T, kKind>;
  auto on = [](auto* ptr, size_t bytes) {
    using P = decltype(ptr);
    return ptr ? (P)((char*)ptr + bytes) : ptr;
  };
  for (long long at = 0; at < n; at += kSlab) {
    Act8Args q = p;
    q.n = n - at < kSlab ? n - at : kSlab;
    q.x = on(p.x, at * es);
    q.gate = on(p.gate, at * es);
    q.dy = on(p.dy, at * es);
    q.dx = on(p.dx, at * es);
    q.dgate = on(p.dgate, at * es);
    q.y = on(p.y, at * es);
    q.codes = on(p.codes, at);
    q.gate_codes = on(p.gate_codes, at);
    q.scales = on(p.scales, at / kAct8Block * sizeof(float));
    q.gate_scales = on(p.gate_scales, at / kAct8Block * sizeof(float));
    const long long ctas = (q.n + kVec * kWarpsA * 32 - 1) / (kVec * kWarpsA * 32);
    const int grid = static_cast<int>(ctas < cap ? ctas : cap);
    if constexpr (kFwd)
      act8_fwd_kernel<T, kKind><<<grid, kWarpsA * 32, 0, st>>>(q);
    else
      act8_bwd_kernel<T, kKind><<<grid, kWarpsA * 32, 0, st>>>(q);
  }
  return cudaGetLastError();
}

template <int kKind, bool kFwd>
cudaError_t launch_typed(const Act8Args& p, cudaStream_t st) {
  return p.f32 ? launch<float, kKind, kFwd>(p, st) : launch<__nv_bfloat16, kKind, kFwd>(p, st);
}

}  // namespace

cudaError_t pack8(const Act8Args& p, cudaStream_t st) { return launch_typed<0, true>(p, st); }
cudaError_t unpack8(const Act8Args& p, cudaStream_t st) { return launch_typed<0, false>(p, st); }
cudaError_t act8_fwd(const Act8Args& p, cudaStream_t st) {
  return p.gated ? launch_typed<2, true>(p, st) : launch_typed<1, true>(p, st);
}
cudaError_t act8_bwd(const Act8Args& p, cudaStream_t st) {
  return p.gated ? launch_typed<2, false>(p, st) : launch_typed<1, false>(p, st);
}

}  // namespace gmdn
