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
// NaN row every column ties.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>

#include "common.cuh"
#include "step_ops.h"

namespace gmdn {
namespace {

constexpr int kLpThreads = 512;
// Logarithms are clamped here where they multiply a factor e^c: that is 0 long
// before, and 0 * -inf, or a sum of S times a mask's -3e38, is not a number.
constexpr float kFar = -1000.f;

struct Stat {
  float m, s, q;
};

__device__ __forceinline__ void join(Stat& a, float m, float s, float q) {
  const float mn = fmaxf(a.m, m);
  const float da = fmaxf(a.m - mn, kFar), db = fmaxf(m - mn, kFar);
  const float fa = __expf(da), fb = __expf(db);
  a.q = fa * fmaf(a.s, da, a.q) + fb * fmaf(s, db, q);
  a.s = fa * a.s + fb * s;
  a.m = mn;
}

__device__ __forceinline__ void add(Stat& a, float x) {
  if (x > a.m) {
    const float d = fmaxf(a.m - x, kFar);
    const float f = __expf(d);
    a.q = f * fmaf(a.s, d, a.q);
    a.s *= f;
    a.m = x;
  }
  const float c = x - a.m;
  const float e = __expf(c);   // NaN stays NaN in s
  a.s += e;
  a.q = fmaf(e, fmaxf(c, kFar), a.q);
}

__device__ __forceinline__ const char* row_of(const LogprobArgs& p, long long r) {
  const long long b = r / p.length, t = r - b * p.length;
  return static_cast<const char*>(p.logits) + (b * p.stride_b + t * p.stride_t) * (p.f32 ? 4 : 2);
}

// (value, index) in one key: larger value first, then the lower index.
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
  uint32_t u = __float_as_uint(v + 0.f);   // -0 is 0
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<unsigned long long>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

__global__ void __launch_bounds__(kLpThreads) logprobs_fwd_rows(LogprobArgs p, long long rows) {
  __shared__ float sm[32], ss[32], sq[32];
  __shared__ unsigned long long best[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const char* row = row_of(p, r);
    Stat a{-FLT_MAX, 0.f, 0.f};
    for (int j = threadIdx.x; j < p.vocab; j += kLpThreads) add(a, load_act(row, j, p.f32));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      join(a, __shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o),
           __shfl_xor_sync(~0u, a.q, o));
    if (lane == 0) {
      sm[w] = a.m;
      ss[w] = a.s;
      sq[w] = a.q;
    }
    __syncthreads();
    a = Stat{sm[0], ss[0], sq[0]};
    for (int k = 1; k < kLpThreads / 32; ++k) join(a, sm[k], ss[k], sq[k]);
    const bool empty = a.s == 0.f, bad = !(a.s >= 0.f) || a.m == INFINITY;
    const float ls = logf(a.s);
    const float nan = __int_as_float(0x7fffffff);
    auto logprob = [&](float x) {
      return bad ? nan : (empty ? -INFINITY : (x - a.m) - ls);
    };
    if (threadIdx.x == 0) {
      const float H = bad ? nan : (empty ? 0.f : ls - a.q / a.s);
      if (p.stats) {
        float4 st = make_float4(a.m, ls, H, 0.f);
        if (bad) st.y = nan;
        reinterpret_cast<float4*>(p.stats)[r] = st;
      }
      if (p.entropy) p.entropy[r] = H;
      if (p.logprobs) {
        const int64_t t = p.targets[r];
        float lp = 0.f;
        if (t != p.ignore_index)
          lp = (t >= 0 && t < p.vocab) ? logprob(load_act(row, t, p.f32)) : nan;
        p.logprobs[r] = lp;
      }
    }
    // alternatives: k rounds, each the largest key below the last one taken
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top_k; ++k) {
      if (bad) {
        if (threadIdx.x == 0) {
          p.top_ids[r * p.top_k + k] = k;
          p.top_logprobs[r * p.top_k + k] = nan;
        }
        continue;
      }
      unsigned long long b = 0;
      for (int j = threadIdx.x; j < p.vocab; j += kLpThreads) {
        const unsigned long long q = key_of(load_act(row, j, p.f32), j);
        if (q < last && q > b) b = q;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(~0u, b, o);
        if (q > b) b = q;
      }
      __syncthreads();
      if (lane == 0) best[w] = b;
      __syncthreads();
      for (int i = 0; i < kLpThreads / 32; ++i)
        if (best[i] > b) b = best[i];
      last = b;
      if (threadIdx.x == 0) {
        const int id = static_cast<int>(0xffffffffu - static_cast<uint32_t>(b));
        p.top_ids[r * p.top_k + k] = id;
        p.top_logprobs[r * p.top_k + k] = logprob(load_act(row, id, p.f32));
      }
    }
    __syncthreads();
  }
}

// The gradient of column x of a row, without the terms of given columns.
struct RowGrad {
  float m, ls, H, w, gh;   // w = gl + sum gk
  bool empty;
  __device__ __forceinline__ float at(float x) const {
    if (empty) return 0.f;
    const float lp = fmaxf((x - m) - ls, kFar);
    // a masked column: p = 0, no gradient; NaN stays
    const float pr = __expf((x - m) - ls);
    return -pr * fmaf(gh, lp + H, w);
  }
};

__global__ void __launch_bounds__(kLpThreads) logprobs_bwd_rows(LogprobArgs p, long long rows) {
  const size_t es = p.f32 ? 4 : 2;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const char* row = row_of(p, r);
    char* out = static_cast<char*>(p.dlogits) + static_cast<size_t>(r) * p.vocab * es;
    const float4 st = reinterpret_cast<const float4*>(p.stats)[r];
    RowGrad g{st.x, st.y, st.z, 0.f, p.g_entropy ? p.g_entropy[r] : 0.f, st.y == -INFINITY};
    int64_t t = -1;
    float gl = 0.f;
    if (p.g_logprobs && p.targets[r] != p.ignore_index) {
      t = p.targets[r];
      gl = (t >= 0 && t < p.vocab) ? p.g_logprobs[r] : __int_as_float(0x7fffffff);
      if (t >= p.vocab) t = -1;
    }
    g.w = gl;
    if (p.g_top)
      for (int k = 0; k < p.top_k; ++k) g.w += p.g_top[r * p.top_k + k];
    for (int j = threadIdx.x; j < p.vocab; j += kLpThreads) {
      float v = g.at(load_act(row, j, p.f32));
      if (!g.empty) {
        if (j == t) v += gl;
        if (p.g_top)
          for (int k = 0; k < p.top_k; ++k)
            if (p.top_ids[r * p.top_k + k] == j) v += p.g_top[r * p.top_k + k];
      }
      store_act(out, j, v, p.f32);
    }
  }
}

}  // namespace

cudaError_t token_logprobs_fwd(const LogprobArgs& p, cudaStream_t st) {
  const long long rows = p.batch * p.length;
  const int grid = static_cast<int>(rows < 148 * 4 ? rows : 148 * 4);
  logprobs_fwd_rows<<<grid, kLpThreads, 0, st>>>(p, rows);
  return cudaGetLastError();
}

cudaError_t token_logprobs_bwd(const LogprobArgs& p, cudaStream_t st) {
  const long long rows = p.batch * p.length;
  const int grid = static_cast<int>(rows < 148 * 4 ? rows : 148 * 4);
  logprobs_bwd_rows<<<grid, kLpThreads, 0, st>>>(p, rows);
  return cudaGetLastError();
}

}  // namespace gmdn
