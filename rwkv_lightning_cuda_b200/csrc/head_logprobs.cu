// The head product with its softmax statistics: for every row of x [rows, K] the log probability of a given token under
// softmax(x W^T), the entropy and the log of the sum of exponentials, W [V, K] being the head matrix in any of the
// models' weight formats.  The logits (rows * V fp32) are never written: a tile of them is reduced to (m, s, t) per row
// where it is computed, and a second kernel merges a row's tiles (logprob.cuh).  fp16 operands, fp32 sums; int8 weights
// are exact integers with the channel's scale on the sum, 4-bit weights half((q - zero) * scale).
//
// Bound by the weights' bytes up to some 256 rows, by the tensor cores above.  One CTA per SM walks the units (128 rows x
// 256 tokens), the row blocks of a token tile one after the other, so that neighbouring CTAs share a tile of weights and
// it comes from HBM once.  The rows take the MMA's M side and the tokens its N side: a lane of tensor memory is then a row
// of x, and an epilogue thread reduces its row's 256 logits without talking to any other.  Two accumulators, so that
// a unit's epilogue runs under the next one's products.
//
// Warp roles: 0 loads (TMA, 128-byte swizzle), 1 issues tcgen05.mma, 2..5 reduce.  Quantised weights: warp 0 brings
// packed tiles into a ring of their own, warp 6 the rows of x, and 16 more warps expand a packed tile into the swizzled
// fp16 tile that the MMA reads (two threads to a weight row).  Every wait is bounded: one that runs out sets the device's
// failure word, every role leaves its loop, and the CTA frees its tensor memory and returns.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "logprob.cuh"
#include "tensormap.h"

namespace rk {
namespace {

constexpr int kRows = 128;   // rows of x per unit = MMA M
constexpr int kToks = 256;   // tokens per unit = MMA N
constexpr int kBK = 64;      // halves per K block = one 128-byte swizzle row
constexpr uint32_t kXBytes = kRows * 128, kWBytes = kToks * 128, kStageBytes = kXBytes + kWBytes;
constexpr int kExpandWarps = 16;
constexpr uint32_t kTmemCols = 512;

// Stages of the tile ring and of the ring of packed tiles, bytes of a packed row and tile.
template <int kFmt> struct Ring;
template <> struct Ring<0> { static constexpr int tiles = 4, raws = 0, raw_row = 0, raw = 0; };
template <> struct Ring<1> { static constexpr int tiles = 3, raws = 4, raw_row = kBK, raw = kToks * raw_row; };
template <> struct Ring<2> { static constexpr int tiles = 3, raws = 8, raw_row = kBK / 2, raw = kToks * raw_row; };
template <int kFmt> constexpr size_t smem_bytes() { return 1024 + Ring<kFmt>::tiles * kStageBytes + Ring<kFmt>::raws * Ring<kFmt>::raw; }
template <int kFmt> constexpr int head_threads() { return kFmt == 0 ? 192 : 256 + kExpandWarps * 32; }

struct HeadMaps {
  CUtensorMap x, w;
};

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Shared-memory matrix descriptor: K-major tile, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Eight 4-bit codes to eight halves half((q - zero) * scale): a nibble under the exponent of 1024 is 1024 + q (the high ones
// arrive as 1024 + 16 q), so one subtraction or fused multiply-add leaves q - zero exactly and the product rounds once.
struct Group4 {
  __half2 scale, sub;  // (s, s) and (-(1024 + z), -(64 + z))
};
__device__ __forceinline__ Group4 group4(half s, float z) {
  return {__half2half2(s), __halves2half2(__float2half_rn(-1024.f - z), __float2half_rn(-64.f - z))};
}
__device__ __forceinline__ uint4 expand4(uint32_t w, const Group4& g) {
  const __half2 mul = __floats2half2_rn(1.0f, 0.0625f);
  uint32_t h[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t both = __byte_perm(w, 0u, 0x4040u + 0x0101u * b);  // the byte in both halves
    uint32_t pair = (both & 0x00f0000fu) | 0x64006400u;
    const __half2 v = __hmul2(__hfma2(*reinterpret_cast<__half2*>(&pair), mul, g.sub), g.scale);
    h[b] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}
// Four int8 codes to four halves, exactly: code + 128 under the exponent of 1024, less 1152.
__device__ __forceinline__ uint2 expand8(uint32_t w) {
  const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
  const uint32_t t = w ^ 0x80808080u;
  uint32_t lo = __byte_perm(t, 0x64646464u, 0x4140), hi = __byte_perm(t, 0x64646464u, 0x4342);
  const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&lo), bias), b = __hsub2(*reinterpret_cast<__half2*>(&hi), bias);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <int kFmt>
__global__ void __launch_bounds__(head_threads<kFmt>(), 1)
    head_tc_kernel(const __grid_constant__ HeadMaps maps, const HeadLogprobsArgs a, const int row_blocks, const int units, int* timeout) {
  constexpr int kTiles = Ring<kFmt>::tiles, kRaws = Ring<kFmt>::raws > 0 ? Ring<kFmt>::raws : 1;
  extern __shared__ unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kTiles], ready[kTiles], empty[kTiles], raw_full[kRaws], raw_empty[kRaws], acc_full[2], acc_empty[2];
  __shared__ float scales[kToks];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = (smem_u32(smem) + 1023u) & ~1023u, raw_ring = ring + kTiles * kStageBytes;
  const int kblocks = (a.K + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&ready[i]), kExpandWarps);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < kRaws; ++i) {
      mbar_init(smem_u32(&raw_full[i]), 1);
      mbar_init(smem_u32(&raw_empty[i]), kExpandWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&acc_full[i]), 1);
      mbar_init(smem_u32(&acc_empty[i]), 4);
    }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_trigger();

  auto wait = [&](uint64_t& bar, int parity) { return !failed && mbar_wait(smem_u32(&bar), parity); };
  bool ok = true;
  if (warp == 0 || (kFmt != 0 && warp == 6)) {
    // ---- loads: the fp16 tiles of both operands, or the packed weights (warp 0) and the rows (warp 6) on rings of their own
    if (lane == 0) {
      const bool packed = kFmt != 0 && warp == 0;
      const int stages = packed ? kRaws : kTiles;
      int it = 0;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const int r0 = (u % row_blocks) * kRows, n0 = (u / row_blocks) * kToks;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % stages;
          if (it >= stages && !(ok = wait(packed ? raw_empty[s] : empty[s], (it / stages - 1) & 1))) break;
          const uint32_t bar = smem_u32(packed ? &raw_full[s] : &full[s]), dst = ring + s * kStageBytes;
          if (packed) {
            mbar_expect_tx(bar, Ring<kFmt>::raw);
            tma_2d(raw_ring + s * Ring<kFmt>::raw, &maps.w, bar, kb * Ring<kFmt>::raw_row, n0);
          } else {
            mbar_expect_tx(bar, kFmt == 0 ? kStageBytes : kXBytes);
            tma_2d(dst, &maps.x, bar, kb * kBK, r0);
            if (kFmt == 0) tma_2d(dst + kXBytes, &maps.w, bar, kb * kBK, n0);
          }
        }
      }
      if (!ok)  // leave no copy in flight behind
        for (int i = it > stages ? it - stages : 0; i < it; ++i) mbar_wait(smem_u32(packed ? &raw_full[i % stages] : &full[i % stages]), (i / stages) & 1);
    }
  } else if (warp == 1) {
    // ---- products: K blocks of 64 as four instructions into the unit's accumulator
    if (lane == 0) {
      constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(kToks >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
      int it = 0, n = 0;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++n) {
        if (n >= 2 && !(ok = wait(acc_empty[n & 1], ((n >> 1) - 1) & 1))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + (n & 1) * kToks;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % kTiles;
          ok = wait(full[s], (it / kTiles) & 1) && (kFmt == 0 || wait(ready[s], (it / kTiles) & 1));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dx = tile_desc(ring + s * kStageBytes), dw = tile_desc(ring + s * kStageBytes + kXBytes);
#pragma unroll
          for (int k4 = 0; k4 < kBK / 16; ++k4) mma(acc, dx + 2 * k4, dw + 2 * k4, idesc, (kb | k4) != 0);
          commit(smem_u32(&empty[s]));
        }
        if (ok) commit(smem_u32(&acc_full[n & 1]));
      }
    }
  } else if (warp < 6) {
    // ---- reduction: a thread owns a row of x, its TMEM lane, and takes the unit's tokens 32 at a time
    const int quad = warp & 3, t = threadIdx.x - 64;
    int n = 0;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++n) {
      const int r = (u % row_blocks) * kRows + quad * 32 + lane, n0 = (u / row_blocks) * kToks, toks = min(kToks, a.V - n0);
      const int64_t id = a.tokens && r < a.rows ? a.tokens[r] : -1;
      if (kFmt == 1) {
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the last unit's scales have been read
        for (int i = t; i < kToks; i += 128) scales[i] = i < toks ? __half2float(a.scale[n0 + i]) : 0.f;
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      ok = __all_sync(0xffffffffu, wait(acc_full[n & 1], (n >> 1) & 1));
      if (kFmt == 1) {  // all four warps stay or leave together: they meet at the barriers above
        uint32_t all;
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\tbar.red.and.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(all) : "r"(static_cast<uint32_t>(ok)) : "memory");
        ok = all != 0;
      }
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      SoftStats st;
      for (int c = 0; c < toks; c += 32) {
        float z[32];
        tmem_ld32(tmem + (n & 1) * kToks + c + (static_cast<uint32_t>(quad * 32) << 16), z);
        const int here = min(32, toks - c);
        if (kFmt == 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) z[i] *= scales[c + i];
        }
        if (here < 32) {
#pragma unroll
          for (int i = 0; i < 32; ++i) z[i] = i < here ? z[i] : -INFINITY;
        }
        if (id >= n0 + c && id < n0 + c + here) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (id == n0 + c + i) a.given[r] = z[i];
        }
        float m = st.m;
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max_nan(m, z[i]);
        raise(st, m);
#pragma unroll
        for (int i = 0; i < 32; ++i) add(st, z[i]);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(smem_u32(&acc_empty[n & 1]));
      if (r < a.rows) a.part[static_cast<size_t>(u / row_blocks) * a.rows + r] = make_float4(st.m, st.s, st.t, 0.f);
    }
  } else if (kFmt != 0 && warp >= 8) {
    // ---- expansion: two threads to a weight row, 32 weights each.  Row r of the tile is 128 bytes at r * 128, its 16-byte
    // chunk c at chunk position c ^ (r & 7).
    const int e = threadIdx.x - 256, r = e >> 1, part = e & 1;
    unsigned char* const base = smem + (ring - smem_u32(smem));
    const int shift = a.group == 32 ? 5 : a.group == 64 ? 6 : 7, groups = (a.K + a.group - 1) >> shift;
    int it = 0;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const int row = (u / row_blocks) * kToks + r;
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const int s = it % kTiles, rs = it % kRaws;
        Group4 g = group4(__float2half_rn(0.f), 0.f);
        if (kFmt == 2 && row < a.V) {  // requested before the wait for the tile
          const size_t gi = static_cast<size_t>(row) * groups + min((kb * kBK + part * 32) >> shift, groups - 1);
          g = group4(a.scale[gi], a.zero ? __half2float(a.zero[gi]) : 8.f);
        }
        ok = __all_sync(0xffffffffu, wait(raw_full[rs], (it / kRaws) & 1) && (it < kTiles || wait(empty[s], (it / kTiles - 1) & 1)));
        if (!ok) break;
        const unsigned char* src = base + kTiles * kStageBytes + rs * Ring<kFmt>::raw + r * Ring<kFmt>::raw_row + part * (Ring<kFmt>::raw_row / 2);
        uint4* dst = reinterpret_cast<uint4*>(base + s * kStageBytes + kXBytes + r * 128);
        if (kFmt == 1) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint4 q = reinterpret_cast<const uint4*>(src)[c];
            const uint2 h0 = expand8(q.x), h1 = expand8(q.y), h2 = expand8(q.z), h3 = expand8(q.w);
            dst[(part * 4 + 2 * c) ^ (r & 7)] = make_uint4(h0.x, h0.y, h1.x, h1.y);
            dst[(part * 4 + 2 * c + 1) ^ (r & 7)] = make_uint4(h2.x, h2.y, h3.x, h3.y);
          }
        } else {
          const uint4 q = *reinterpret_cast<const uint4*>(src);
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[(part * 4 + i) ^ (r & 7)] = expand4(w[i], g);
        }
        // written through the generic proxy, read by the tensor core through the async one
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          arrive(smem_u32(&ready[s]));
          arrive(smem_u32(&raw_empty[rs]));
        }
      }
    }
  }
  if (!ok) failed = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && failed && timeout) atomicOr(timeout, kTimeoutGemm);
  __syncwarp();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// One warp per row merges the row's tiles.
__global__ void __launch_bounds__(256) head_merge_kernel(HeadLogprobsArgs a, int tiles) {
  pdl_wait();
  pdl_trigger();
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

// A 2-D tensor [rows, row_bytes / size of an element] in boxes of box_cols x box_rows, zeros outside.
int head_map(CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base, int rows, size_t cols, int box_cols, int box_rows, bool swizzle) {
  const TensorMapEncodeFn fn = tensor_map_encode_fn();
  RK_REQUIRE(fn, kCuda, "head_logprobs: cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[2] = {cols, static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {cols * elem_bytes};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RK_REQUIRE(r == CUDA_SUCCESS, kCuda, "head_logprobs: cuTensorMapEncodeTiled failed with %d (rows=%d, columns=%zu)", static_cast<int>(r), rows, cols);
  return kOk;
}

template <int kFmt>
int launch_head(cudaStream_t stream, const HeadLogprobsArgs& a, int sms) {
  HeadMaps maps;
  int s = head_map(&maps.x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, a.x, a.rows, a.K, kBK, kRows, true);
  if (s != kOk) return s;
  if (kFmt == 0) s = head_map(&maps.w, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, a.w, a.V, a.K, kBK, kToks, true);
  else s = head_map(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.w, a.V, kFmt == 1 ? a.K : a.K / 2, Ring<kFmt>::raw_row, kToks, false);
  if (s != kOk) return s;
  const int row_blocks = (a.rows + kRows - 1) / kRows, tiles = (a.V + kToks - 1) / kToks;
  RK_REQUIRE(static_cast<long long>(row_blocks) * tiles < (1ll << 31), kShape, "head_logprobs: too many rows");
  const int units = row_blocks * tiles;
  RK_CUDA(cudaFuncSetAttribute(head_tc_kernel<kFmt>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bytes<kFmt>())));
  RK_CUDA(launch_pdl(head_tc_kernel<kFmt>, dim3(std::min(units, sms)), dim3(head_threads<kFmt>()), smem_bytes<kFmt>(), stream, maps, a, row_blocks, units,
                     timeout_word_or_null()));
  RK_LAUNCH_CHECK("head_logprobs launch");
  RK_CUDA(launch_pdl(head_merge_kernel, dim3((a.rows + 7) / 8), dim3(256), 0, stream, a, tiles));
  RK_LAUNCH_CHECK("head_logprobs merge launch");
  return kOk;
}

}  // namespace

size_t head_logprobs_workspace(int rows, int V) {
  const size_t tiles = (static_cast<size_t>(V) + kToks - 1) / kToks;
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
  a.part = static_cast<float4*>(workspace);
  a.given = reinterpret_cast<float*>(a.part + (static_cast<size_t>(a.V) + kToks - 1) / kToks * a.rows);
  int sms = 0;
  const int status = device_sms(&sms);
  if (status != kOk) return status;
  if (a.fmt == 1) return launch_head<1>(stream, a, sms);
  if (a.fmt == 2) return launch_head<2>(stream, a, sms);
  return launch_head<0>(stream, a, sms);
}

}  // namespace rk
