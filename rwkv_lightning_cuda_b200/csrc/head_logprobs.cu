// The head product with its softmax statistics: for every row of x [rows, K] the log probability of a given token under
// softmax(x W^T), the entropy and the log of the sum of exponentials, W [V, K] being the head matrix in any of the
// models' weight formats.  The logits (rows * V fp32) are never written: a tile of them is reduced to (m, s, t) per row
// where it is computed, and a second kernel merges a row's tiles (logprob.cuh).  fp16 operands, fp32 sums; int8 weights
// are exact integers with the channel's scale on the sum, 4-bit weights half((q - zero) * scale).
// A CTA computes 64 rows x 64 tokens from fp32 tiles in shared memory, a thread 4 x 4 of them.
#include "common.cuh"
#include "kernels.h"
#include "logprob.cuh"

namespace rk {
namespace {

constexpr int kTile = 64, kStep = 32;

__device__ __forceinline__ float head_weight(const HeadLogprobsArgs& a, int groups, int n, int k) {
  const size_t o = static_cast<size_t>(n) * a.K + k;
  if (a.fmt == 0) return __half2float(static_cast<const half*>(a.w)[o]);
  if (a.fmt == 1) return static_cast<float>(static_cast<const int8_t*>(a.w)[o]);
  const uint8_t byte = static_cast<const uint8_t*>(a.w)[o >> 1];
  const size_t g = static_cast<size_t>(n) * groups + k / a.group;
  const float z = a.zero ? __half2float(a.zero[g]) : 8.f;
  return __half2float(__float2half_rn(((k & 1 ? byte >> 4 : byte & 15) - z) * __half2float(a.scale[g])));
}

__global__ void __launch_bounds__(256) head_tile_kernel(HeadLogprobsArgs a) {
  __shared__ float xs[kStep][kTile + 1], wsh[kStep][kTile + 1];
  const int n0 = blockIdx.x * kTile, r0 = blockIdx.y * kTile, t = threadIdx.x, tx = t & 15, ty = t >> 4;
  const int groups = a.fmt == 2 ? (a.K + a.group - 1) / a.group : 0;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += kStep) {
    for (int i = t; i < kTile * kStep; i += 256) {
      const int k = i % kStep, j = i / kStep;
      xs[k][j] = r0 + j < a.rows && k0 + k < a.K ? __half2float(a.x[static_cast<size_t>(r0 + j) * a.K + k0 + k]) : 0.f;
      wsh[k][j] = n0 + j < a.V && k0 + k < a.K ? head_weight(a, groups, n0 + j, k0 + k) : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty + 16 * i], wsh[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + ty + 16 * i;
    const int64_t id = a.tokens && r < a.rows ? a.tokens[r] : -1;
    SoftStats st;
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (n >= a.V) continue;
      const float z = acc[i][j] * (a.fmt == 1 ? __half2float(a.scale[n]) : 1.f);
      if (id == n) a.given[r] = z;
      const float m = max_nan(st.m, z);
      raise(st, m);
      add(st, z);
    }
    for (int o = 8; o > 0; o >>= 1) st = merge(st, shfl_xor(st, o));
    if (tx == 0 && r < a.rows) a.part[static_cast<size_t>(blockIdx.x) * a.rows + r] = make_float4(st.m, st.s, st.t, 0.f);
  }
}

// One warp per row merges the row's tiles.
__global__ void __launch_bounds__(256) head_merge_kernel(HeadLogprobsArgs a, int tiles) {
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= a.rows) return;
  SoftStats st;
  for (int i = lane; i < tiles; i += 32) {
    const float4 p = a.part[static_cast<size_t>(i) * a.rows + r];
    SoftStats b;
    b.m = p.x; b.s = p.y; b.t = p.z;
    st = merge(st, b);
  }
  st = warp_merge(st);
  if (lane != 0) return;
  const RowResult res = finish(st);
  if (a.entropy) a.entropy[r] = res.entropy;
  if (a.lse) a.lse[r] = res.lse;
  if (a.tokens) a.logprobs[r] = given_logprob(res, a.tokens[r], a.V, [&](int64_t) { return a.given[r]; });
}

}  // namespace

size_t head_logprobs_workspace(int rows, int V) {
  const size_t tiles = (static_cast<size_t>(V) + kTile - 1) / kTile;
  return static_cast<size_t>(rows) * (tiles * sizeof(float4) + sizeof(float));
}

int head_logprobs(cudaStream_t stream, HeadLogprobsArgs a, void* workspace, size_t workspace_bytes) {
  RK_REQUIRE(a.rows > 0 && a.K > 0 && a.V > 0 && a.x && a.w, kBadArg, "head_logprobs: bad argument");
  RK_REQUIRE(!a.tokens == !a.logprobs, kBadArg, "head_logprobs: tokens without their output");
  RK_REQUIRE(a.fmt >= 0 && a.fmt <= 2, kBadArg, "head_logprobs: unknown weight format %d", a.fmt);
  RK_REQUIRE(a.fmt == 0 || a.scale, kBadArg, "head_logprobs: quantised weights need scales");
  RK_REQUIRE(a.K % 32 == 0, kShape, "head_logprobs: K must be a multiple of 32 (got %d)", a.K);
  RK_REQUIRE(a.fmt != 2 || a.group == 32 || a.group == 64 || a.group == 128, kShape, "head_logprobs: groups of 32, 64 or 128 (got %d)", a.group);
  RK_REQUIRE(((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0, kBadArg,
             "head_logprobs: x, the weights and the workspace must be 16-byte aligned");
  RK_REQUIRE(workspace && workspace_bytes >= head_logprobs_workspace(a.rows, a.V), kBadArg, "head_logprobs: the workspace needs %zu bytes",
             head_logprobs_workspace(a.rows, a.V));
  const int tiles = (a.V + kTile - 1) / kTile;
  a.part = static_cast<float4*>(workspace);
  a.given = reinterpret_cast<float*>(a.part + static_cast<size_t>(tiles) * a.rows);
  RK_REQUIRE(a.rows <= 65535 * kTile, kShape, "head_logprobs: too many rows");
  head_tile_kernel<<<dim3(tiles, (a.rows + kTile - 1) / kTile), 256, 0, stream>>>(a);
  RK_LAUNCH_CHECK("head_logprobs launch");
  head_merge_kernel<<<(a.rows + 7) / 8, 256, 0, stream>>>(a, tiles);
  RK_LAUNCH_CHECK("head_logprobs merge launch");
  return kOk;
}

}  // namespace rk
