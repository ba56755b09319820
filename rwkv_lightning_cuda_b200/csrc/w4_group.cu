// 4-bit weights with group scales: y = epi(x W^T) with W[n,k] = (q[n,k] - zero[n,g]) * scale[n,g], g = k / group, for
// groups of 32, 64 or 128 input channels, the last of which may be short, and without zeros (then 8) or with them.
// Packing as the other 4-bit format: byte j of a row holds q[2j] (low nibble) and q[2j + 1] (high nibble).  The scale
// multiplies the group's sum in fp32: a weight is never rounded to half, unlike in the format of groups of 128 that the
// models' matrices use.
// One warp per output channel and row; lane i takes the words (8 weights) i, i + 32, ...
#include "common.cuh"
#include "kernels.h"

namespace rk {
namespace {

__global__ void __launch_bounds__(256) w4_group_simple_kernel(W4GroupArgs a) {
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5), m = blockIdx.y, lane = threadIdx.x & 31;
  if (n >= a.N) return;
  const int groups = (a.K + a.group - 1) / a.group, shift = 31 - __clz(a.group);
  const uint32_t* qw = reinterpret_cast<const uint32_t*>(a.q + static_cast<size_t>(n) * (a.K >> 1));
  const half* x = a.x + static_cast<size_t>(m) * a.K;
  float acc = 0.f;
  for (int w = lane; w < (a.K >> 3); w += 32) {
    const size_t g = static_cast<size_t>(n) * groups + ((w << 3) >> shift);
    const float s = __half2float(a.scale[g]), z = a.zero ? __half2float(a.zero[g]) : 8.f;
    const uint32_t u = qw[w];
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) part += (static_cast<float>((u >> (4 * i)) & 15u) - z) * __half2float(x[(w << 3) + i]);
    acc += part * s;
  }
  acc = warp_sum(acc);
  if (lane != 0) return;
  const size_t o = static_cast<size_t>(m) * a.N + n;
  const half hy = __float2half_rn(acc);
  if (a.epi == kEpiF32) {
    static_cast<float*>(a.y)[o] = __half2float(hy);
  } else if (a.epi == kEpiRelu2) {
    const float u = fmaxf(__half2float(hy), 0.f);
    static_cast<half*>(a.y)[o] = __float2half_rn(u * u);
  } else {
    static_cast<half*>(a.y)[o] = hy;
  }
}

// One warp per group: lane i handles the byte(s) i, i + 32 of it (a group of 128 is 64 bytes).
__global__ void __launch_bounds__(128) pack_w4_group_kernel(int K, int group, int groups, long long n_groups, const half* __restrict__ W,
                                                            uint8_t* __restrict__ q, half* __restrict__ scale, half* __restrict__ zero) {
  const long long gi = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (gi >= n_groups) return;
  const int lane = threadIdx.x & 31;
  const long long n = gi / groups;
  const int k0 = static_cast<int>(gi - n * groups) * group, len = min(group, K - k0);
  const half* w = W + n * K + k0;
  float mn = 0.f, mx = 0.f;
  for (int i = lane; i < len; i += 32) {
    const float v = __half2float(w[i]);
    mn = fminf(mn, v);
    mx = fmaxf(mx, v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const half s = __float2half_rn(zero ? __fdiv_rn(__fsub_rn(mx, mn), 15.0f) : __fdiv_rn(fmaxf(-mn, mx), 7.0f));
  const float sf = __half2float(s);
  float z = 8.f;
  if (zero) {
    z = sf > 0.f ? rintf(__fdiv_rn(-mn, sf)) : 0.f;
    z = fminf(fmaxf(z, 0.f), 15.f);
    if (lane == 0) zero[gi] = __float2half_rn(z);
  }
  if (lane == 0) scale[gi] = s;
  uint8_t* qb = q + ((n * K + k0) >> 1);
  for (int j = lane; j < (len >> 1); j += 32) {
    uint32_t byte = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float t = sf > 0.f ? __fadd_rn(rintf(__fdiv_rn(__half2float(w[2 * j + i]), sf)), z) : z;
      byte |= static_cast<uint32_t>(fminf(fmaxf(t, 0.f), 15.f)) << (4 * i);
    }
    qb[j] = static_cast<uint8_t>(byte);
  }
}

__global__ void unpack_w4_group_kernel(int K, int shift, int groups, long long total, const uint8_t* __restrict__ q,
                                       const half* __restrict__ scale, const half* __restrict__ zero, half* __restrict__ W) {
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const long long n = i / K;
  const long long g = n * groups + (static_cast<int>(i - n * K) >> shift);
  const int qq = (i & 1) ? (q[i >> 1] >> 4) : (q[i >> 1] & 15);
  W[i] = __float2half_rn(__fmul_rn(__fsub_rn(static_cast<float>(qq), zero ? __half2float(zero[g]) : 8.f), __half2float(scale[g])));
}

int check_shape(const char* what, int N, int K, int group) {
  RK_REQUIRE(N > 0 && K > 0, kBadArg, "%s: dimensions must be positive", what);
  RK_REQUIRE(group == 32 || group == 64 || group == 128, kShape, "%s: groups of 32, 64 or 128 (got %d)", what, group);
  RK_REQUIRE(K % 32 == 0, kShape, "%s: K must be a multiple of 32 (got %d)", what, K);
  return kOk;
}

}  // namespace

int w4_group_linear(cudaStream_t stream, const W4GroupArgs& a) {
  const int s = check_shape("linear_w4a16_group", a.N, a.K, a.group);
  if (s != kOk) return s;
  RK_REQUIRE(a.M > 0 && a.x && a.q && a.scale && a.y, kBadArg, "linear_w4a16_group: bad argument");
  RK_REQUIRE(a.epi == kEpiNone || a.epi == kEpiRelu2 || a.epi == kEpiF32, kBadArg, "linear_w4a16_group: unknown epilogue %d", a.epi);
  RK_REQUIRE(((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.q)) & 15u) == 0, kBadArg,
             "linear_w4a16_group: x and q must be 16-byte aligned");
  for (int m0 = 0; m0 < a.M; m0 += 65535) {  // (the grid's second dimension)
    W4GroupArgs b = a;
    b.M = min(a.M - m0, 65535);
    b.x = a.x + static_cast<size_t>(m0) * a.K;
    b.y = static_cast<char*>(a.y) + static_cast<size_t>(m0) * a.N * (a.epi == kEpiF32 ? 4 : 2);
    w4_group_simple_kernel<<<dim3((a.N + 7) / 8, b.M), 256, 0, stream>>>(b);
    RK_LAUNCH_CHECK("linear_w4a16_group launch");
  }
  return kOk;
}

int quant_pack_w4_group(cudaStream_t stream, int N, int K, int group, const half* W, uint8_t* q, half* scale, half* zero) {
  const int s = check_shape("quant_pack_w4_group", N, K, group);
  if (s != kOk) return s;
  RK_REQUIRE(W && q && scale, kBadArg, "quant_pack_w4_group: null pointer");
  const int groups = (K + group - 1) / group;
  const long long total = static_cast<long long>(N) * groups;
  pack_w4_group_kernel<<<static_cast<unsigned>((total + 3) / 4), 128, 0, stream>>>(K, group, groups, total, W, q, scale, zero);
  RK_LAUNCH_CHECK("quant_pack_w4_group launch");
  return kOk;
}

int quant_unpack_w4_group(cudaStream_t stream, int N, int K, int group, const uint8_t* q, const half* scale, const half* zero, half* W) {
  const int s = check_shape("quant_unpack_w4_group", N, K, group);
  if (s != kOk) return s;
  RK_REQUIRE(W && q && scale, kBadArg, "quant_unpack_w4_group: null pointer");
  const long long total = static_cast<long long>(N) * K;
  const int shift = group == 32 ? 5 : group == 64 ? 6 : 7;
  unpack_w4_group_kernel<<<static_cast<unsigned>((total + 255) / 256), 256, 0, stream>>>(K, shift, (K + group - 1) / group, total, q, scale, zero, W);
  RK_LAUNCH_CHECK("quant_unpack_w4_group launch");
  return kOk;
}

}  // namespace rk
