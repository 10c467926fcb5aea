// Kernels of the training step around the mixer: the model-width norm, the
// token log probabilities and the 8-bit activation checkpoints.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace gmdn {

// ---- norm.cu: layer norm / RMS norm of x (+ residual) over the last axis ----
struct NormFwdArgs {
  const void *x, *res;           // (rows, width); res may be null
  const float *weight, *bias;    // (width), either may be null
  void *y, *h;                   // h = x + res in its stored type (res given)
  float *rstd, *mean;            // (rows); mean only with center
  long long rows;
  int width;
  float eps;
  bool center, x_f32, res_f32, y_f32;   // h is fp32 if x or res is
};
struct NormBwdArgs {
  const void* s;                 // what was normalised: x, or h
  const float *rstd, *mean, *weight;
  const void *dy, *dh;           // dh: in the type of s, may be null
  void *ds_a, *ds_b;             // the gradient of s in one or two types (either may be null)
  float *dw, *db;                // either may be null
  float* partial;                // norm_bwd_partials(...) x 2 x width floats
  long long rows;
  int width;
  bool center, s_f32, dy_f32, a_f32, b_f32;
};
cudaError_t norm_fwd(const NormFwdArgs& p, cudaStream_t st);
int norm_bwd_partials(long long rows, int width);
cudaError_t norm_bwd(const NormBwdArgs& p, cudaStream_t st);

// ---- logprobs.cu: log probabilities of given tokens --------------------------
struct LogprobArgs {
  const void* logits;            // row (b, t) at b * stride_b + t * stride_t elements
  long long batch, length, stride_b, stride_t;
  int vocab;
  bool f32;
  const int64_t* targets;        // (batch, length), may be null (forward)
  int64_t ignore_index;
  float* stats;                  // (rows, 4): max, log of the sum, entropy, the sum
  float *logprobs, *entropy, *top_logprobs;   // any may be null
  int64_t* top_ids;              // (rows, top_k)
  int top_k;
  // backward
  const float *g_logprobs, *g_entropy, *g_top;   // any may be null
  void* dlogits;                 // contiguous (batch, length, vocab)
};
constexpr int kMaxTopK = 64;
cudaError_t token_logprobs_fwd(const LogprobArgs& p, cudaStream_t st);
cudaError_t token_logprobs_bwd(const LogprobArgs& p, cudaStream_t st);

// ---- act8.cu: activations in 8 bits ------------------------------------------
constexpr int kAct8Block = 128;  // consecutive elements that share a scale
struct Act8Args {
  const void *x, *gate;          // forward inputs; gate: SwiGLU (null: GELU)
  int8_t *codes, *gate_codes;
  float *scales, *gate_scales;   // one for each 128 elements
  const void* dy;                // backward
  void *dx, *dgate, *y;          // y may be null in the backward
  long long n;
  bool f32, gated;
};
cudaError_t pack8(const Act8Args& p, cudaStream_t st);
cudaError_t unpack8(const Act8Args& p, cudaStream_t st);   // codes, scales -> y
cudaError_t act8_fwd(const Act8Args& p, cudaStream_t st);
cudaError_t act8_bwd(const Act8Args& p, cudaStream_t st);

}  // namespace gmdn
