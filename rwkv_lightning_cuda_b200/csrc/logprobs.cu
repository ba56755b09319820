// Log probabilities of given tokens over logits [rows, V], with the entropy, the log of the sum of exponentials and the
// likeliest alternatives of every row (definitions and corner cases: logprob.cuh).  One CTA per row: one pass for the
// statistics, then one pass per alternative, each taking the largest (value, lowest id) below the one before.
#include "common.cuh"
#include "kernels.h"
#include "logprob.cuh"

namespace rk {
namespace {

constexpr int kThreads = 512;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(half v) { return __half2float(v); }

// Orders (value, id) pairs as whole numbers: larger value first, then the lower id.  -0 counts as +0.
__device__ __forceinline__ unsigned long long rank_key(float v, int id) {
  const uint32_t u = __float_as_uint(v + 0.f);
  const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<unsigned long long>(o) << 32) | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ int key_id(unsigned long long k) { return static_cast<int>(~static_cast<uint32_t>(k)); }
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(TokenLogprobsArgs a) {
  __shared__ SoftStats part[kThreads / 32];
  __shared__ unsigned long long best_w[kThreads / 32];
  __shared__ RowResult row;
  const int r = blockIdx.x, t = threadIdx.x;
  const T* z = static_cast<const T*>(a.logits) + static_cast<long long>(r) * a.ld;
  SoftStats st;
  for (int i = t; i < a.V; i += kThreads) {
    const float v = to_float(z[i]);
    const float m = max_nan(st.m, v);
    if (m != st.m) raise(st, m);
    add(st, v);
  }
  st = warp_merge(st);
  if ((t & 31) == 0) part[t >> 5] = st;
  __syncthreads();
  if (t == 0) {
    for (int i = 1; i < kThreads / 32; ++i) st = merge(st, part[i]);
    row = finish(st);
    if (a.entropy) a.entropy[r] = row.entropy;
    if (a.lse) a.lse[r] = row.lse;
  }
  __syncthreads();
  const RowResult res = row;
  for (int i = t; i < a.n_tokens; i += kThreads) {
    const size_t o = static_cast<size_t>(r) * a.n_tokens + i;
    a.logprobs[o] = given_logprob(res, a.tokens[o], a.V, [&](int64_t id) { return to_float(z[id]); });
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    unsigned long long best = 0;
    if (!res.poisoned && !res.empty)
      for (int i = t; i < a.V; i += kThreads) {
        const float v = to_float(z[i]);
        const unsigned long long key = v > -INFINITY ? rank_key(v, i) : 0;
        if (key < last && key > best) best = key;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if ((t & 31) == 0) best_w[t >> 5] = best;
    __syncthreads();
    for (int i = 0; i < kThreads / 32; ++i) best = best_w[i] > best ? best_w[i] : best;
    last = best;
    if (t == 0) {
      const size_t o = static_cast<size_t>(r) * a.top_k + k;
      a.top_ids[o] = best ? key_id(best) : -1;
      a.top_logprobs[o] = best ? res.logprob(key_value(best)) : res.poisoned ? res.lse : -INFINITY;
    }
  }
}

}  // namespace

int token_logprobs(cudaStream_t stream, const TokenLogprobsArgs& a) {
  RK_REQUIRE(a.rows > 0 && a.V > 0 && a.logits, kBadArg, "token_logprobs: bad argument");
  RK_REQUIRE(a.ld >= a.V, kShape, "token_logprobs: row stride %lld below the vocabulary size %d", a.ld, a.V);
  RK_REQUIRE(a.n_tokens >= 0 && (a.n_tokens == 0 || (a.tokens && a.logprobs)), kBadArg, "token_logprobs: tokens without their output");
  RK_REQUIRE(a.top_k >= 0 && a.top_k <= kMaxTopLogprobs, kBadArg, "token_logprobs: top_k %d outside [0, %d]", a.top_k, kMaxTopLogprobs);
  RK_REQUIRE(a.top_k == 0 || (a.top_ids && a.top_logprobs), kBadArg, "token_logprobs: alternatives without their outputs");
  if (a.is_half) token_logprobs_kernel<half><<<a.rows, kThreads, 0, stream>>>(a);
  else token_logprobs_kernel<float><<<a.rows, kThreads, 0, stream>>>(a);
  RK_LAUNCH_CHECK("token_logprobs launch");
  return kOk;
}

}  // namespace rk
