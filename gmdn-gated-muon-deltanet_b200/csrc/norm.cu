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

#include "common.cuh"
#include "step_ops.h"

namespace gmdn {
namespace {

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

// dw, db from the partials, in a fixed order (bit-reproducible).
__global__ void __launch_bounds__(kColThreads) norm_bwd_join(NormBwdArgs p, int parts) {
  __shared__ float red[2][kColRows][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float a = 0.f, b = 0.f;
  if (col < p.width) {
    for (int k = w; k < parts; k += kColRows) {
      a += p.partial[(static_cast<size_t>(k) * 2) * p.width + col];
      b += p.partial[(static_cast<size_t>(k) * 2 + 1) * p.width + col];
    }
  }
  red[0][w][lane] = a;
  red[1][w][lane] = b;
  __syncthreads();
  if (w < 2 && col < p.width) {
    float t = 0.f;
    for (int k = 0; k < kColRows; ++k) t += red[w][k][lane];
    float* out = w == 0 ? p.dw : p.db;
    if (out) out[col] = t;
  }
}

int row_grid(long long rows) { return static_cast<int>(rows < 148 * 8 ? rows : 148 * 8); }

}  // namespace

cudaError_t norm_fwd(const NormFwdArgs& p, cudaStream_t st) {
  norm_fwd_rows<<<row_grid(p.rows), kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

int norm_bwd_partials(long long rows, int width) {
  (void)width;
  const long long want = (rows + 31) / 32;
  return static_cast<int>(want < 1 ? 1 : (want < kMaxPartials ? want : kMaxPartials));
}

cudaError_t norm_bwd(const NormBwdArgs& p, cudaStream_t st) {
  if (p.ds_a || p.ds_b) norm_bwd_rows<<<row_grid(p.rows), kThreads, 0, st>>>(p);
  if (p.dw || p.db) {
    const int parts = norm_bwd_partials(p.rows, p.width);
    const int cb = (p.width + 31) / 32;
    norm_bwd_cols<<<dim3(cb, parts), kColThreads, 0, st>>>(p, parts);
    norm_bwd_join<<<cb, kColThreads, 0, st>>>(p, parts);
  }
  return cudaGetLastError();
}

}  // namespace gmdn
