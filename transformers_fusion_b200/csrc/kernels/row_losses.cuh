// What the losses on rows of logits (token_losses.cu) and the scoring of given tokens (linear_logprobs.cu) have in common.
#pragma once
#include "tfb_ptx.cuh"

namespace tfb {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ long long ld_idx(const void* p, long long i, int is64) {
  return is64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Log-probability of a target with the logit zy, and the row's logsumexp, from the other columns' maximum m and s = sum exp(z - m): lp = -log(1 + q), q = s exp(m - zy), so
// that a nearly certain token's lp (a small q) has the relative error of q, where zy - lse has the rounding of two numbers of the size of zy.  `in`: whether the
// target is in the vocabulary; m and s are those of the whole row where it is not.
__device__ __forceinline__ void score_of(float m, double s, float zy, bool in, float& lp, float& lse) {
  const double d = double(m) - double(zy);
  const bool far = !(d < 600.0);      // where exp(d) might overflow (or a value is not finite), 1 + q is q
  const double a = !in || far ? double(m) + log(s) : 0.0, l = far ? double(zy) - a : 0.0 - log1p(s * exp(d));
  const bool top = zy == INFINITY;
  lp = in && !top ? float(l) : NAN;
  lse = !in || zy == -INFINITY ? float(a) : top ? NAN : float(double(zy) - l);
}

}  // namespace tfb
