// The running softmax statistics shared by the log-probability kernels (logprobs.cu, head_logprobs.cu).
//
// A set of logits z is summarised by m = max z, s = sum exp(z - m) and t = sum exp(z - m) (z - m), all in fp32:
//   lse = m + ln s,   log p_i = (z_i - m) - ln s,   entropy = -sum p_i log p_i = ln s - t / s
// and two summaries merge into the summary of the union, so a row can be cut over threads, CTAs and vocabulary tiles.
// What the corner cases mean:
//   -inf          a masked token: probability 0, log probability -inf, never an alternative
//   all masked    lse -inf, every log probability -inf, entropy 0
//   NaN or +inf   the row has no distribution: lse, entropy and log probabilities are NaN, there are no alternatives
// m starts at -FLT_MAX instead of -inf, so that z - m is never inf - inf for a masked token, and takes part in a maximum
// that keeps NaN; differences are cut off below at kFar (their exponential is 0 long before, and its product with a sum of 2^30
// terms is finite), so that 0 * -inf never is.
#pragma once

#include <cfloat>

#include "common.cuh"

namespace rk {

#ifdef __CUDACC__

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e28f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct SoftStats {
  float m = -FLT_MAX, s = 0.f, t = 0.f;
};

// Moves the statistics to another maximum (>= the present one).
__device__ __forceinline__ void raise(SoftStats& a, float m) {
  const float d = fmaxf(a.m - m, kFar), c = exp2f(d * kLog2e);
  a.t = c * (a.t + d * a.s);
  a.s *= c;
  a.m = m;
}

// One logit at a maximum that is already in place.
__device__ __forceinline__ void add(SoftStats& a, float z) {
  const float d = fmaxf(z - a.m, kFar), e = exp2f(d * kLog2e);
  a.s += e;
  a.t = fmaf(e, d, a.t);
}

__device__ __forceinline__ SoftStats merge(SoftStats a, SoftStats b) {
  const float m = max_nan(a.m, b.m);
  raise(a, m);
  raise(b, m);
  a.s += b.s;
  a.t += b.t;
  return a;
}

__device__ __forceinline__ SoftStats shfl_xor(const SoftStats& a, int o) {
  SoftStats b;
  b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
  b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
  b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
  return b;
}

__device__ __forceinline__ SoftStats warp_merge(SoftStats a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = merge(a, shfl_xor(a, o));
  return a;
}

struct RowResult {
  float m, log_s, lse, entropy;
  bool poisoned, empty;  // NaN / +inf among the logits; nothing but masked tokens
  __device__ __forceinline__ float logprob(float z) const {
    if (poisoned) return __int_as_float(0x7fffffff);
    if (empty) return -INFINITY;
    return (z - m) - log_s;
  }
};

// ln x for x >= 1 to two half steps or so (the build's fast logf is off by 2^-22 near 1, and the 64-bit logarithm took a
// microsecond at the end of every row): x = 2^e f with f in [0.75, 1.5), ln f = 2 atanh((f - 1) / (f + 1)) by its series up to the
// ninth power, whose next term is below 2^-28 for |u| <= 0.2.
__device__ __forceinline__ float ln_from_one(float x) {
  const int bits = __float_as_int(x), e = (bits - 0x3f400000) >> 23;  // 0x3f400000: 0.75
  const float f = __int_as_float(bits - (e << 23)), d = f - 1.f, u = __fdiv_rn(d, f + 1.f), w = u * u;
  const float p = w * fmaf(w, fmaf(w, fmaf(w, 2.f / 9.f, 2.f / 7.f), 2.f / 5.f), 2.f / 3.f);
  return fmaf(static_cast<float>(e), 0.693147182464599609375f, fmaf(u, p, 2.f * u) + static_cast<float>(e) * -1.904654323148236e-9f);
}

__device__ __forceinline__ RowResult finish(const SoftStats& a) {
  RowResult r;
  r.m = a.m;
  r.poisoned = !(a.m <= FLT_MAX) || a.s != a.s;  // (a sum that is no number is not passed off as one)
  r.empty = !r.poisoned && a.s == 0.f;
  r.log_s = r.empty ? 0.f : ln_from_one(fmaxf(a.s, 1.f));  // (the largest logit alone is 1, but for the rounding of rescalings)
  const float nan = __int_as_float(0x7fffffff);
  r.lse = r.poisoned ? nan : r.empty ? -INFINITY : a.m + r.log_s;
  r.entropy = r.poisoned ? nan : r.empty ? 0.f : r.log_s - __fdiv_rn(a.t, a.s);
  if (r.entropy < 0.f) r.entropy = 0.f;  // (NaN stays)
  return r;
}

// The answer for a given token id: an id below 0 asks for nothing and gets 0; one beyond the vocabulary gets NaN.
template <typename Load>
__device__ __forceinline__ float given_logprob(const RowResult& r, int64_t id, int64_t V, Load&& load) {
  if (id < 0) return 0.f;
  if (id >= V) return __int_as_float(0x7fffffff);
  return r.logprob(load(id));
}

#endif  // __CUDACC__

}  // namespace rk
