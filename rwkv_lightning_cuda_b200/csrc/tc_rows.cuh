// x W^T for rows of x on the tensor cores, with whatever is done with the products left to the caller: the skeleton of the head
// product that keeps no logits (head_logprobs.cu) and of the 4-bit products of many rows (w4_group.cu).
//
// One CTA per SM walks units of 128 rows x up to 256 tokens (output channels) x a range of K.  The rows take the MMA's M
// side and the tokens its N side: a lane of tensor memory is then a row of x, and an epilogue thread sees its row's results one
// after the other without talking to any other thread.  Row blocks of a token tile follow one another, so that neighbouring CTAs
// share a tile of weights and it comes from HBM once.  Two accumulators: a unit's epilogue runs under the next one's products.
//
// Warp roles: 0 loads (TMA, 128-byte swizzle), 1 issues tcgen05.mma, 2..5 run the epilogue.  Quantised weights: warp 0 brings
// packed tiles into a ring of their own, warp 6 the rows of x, and 16 more warps expand a packed tile into the swizzled
// fp16 tile that the MMA reads (a thread to a weight row, the two halves of the warps taking turns).  Every wait is bounded:
// one that runs out sets the device's failure word, every role leaves its loop, and the CTA frees its tensor memory and returns.
#pragma once

#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tensormap.h"

namespace rk {
namespace tc {

constexpr int kRows = 128;   // rows of x per unit = MMA M
constexpr int kToks = 256;   // tokens per unit = MMA N, at most (Shape::toks)
constexpr int kBK = 64;      // halves per K block = one 128-byte swizzle row
constexpr int kExpandWarps = 16;
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxTiles = 8, kMaxRaws = 8;
constexpr size_t kSmemBytes = 225 * 1024;  // of 227 KB, beside the static part

template <int kFmt> constexpr int tc_threads() { return kFmt == 0 ? 192 : 256 + kExpandWarps * 32; }
template <int kFmt> __host__ __device__ constexpr int raw_row() { return kFmt == 0 ? 0 : kFmt == 1 ? kBK : kBK / 2; }  // bytes of a packed row of a K block

// The weights: fp16, int8 with a scale per row (applied to the sums), or 4 bits with scales and zeros per group (half((q - zero) * scale)).
struct Weights {
  int V, K;
  int group;                    // 4 bits: 32, 64 or 128
  const half *scale, *zero;     // zero nullptr: 8
};
struct Shape {
  int toks, tiles;          // tokens per unit (at most kToks), token tiles
  int row_blocks;           // blocks of 128 rows
  int splits, kb_per_split; // ranges of K and their K blocks (the last one may have fewer)
  int units;
  int x_rows;  // rows of x that a block loads: all there are, in eights, up to 128 (the rest of the tile is not read out)
  // shared memory, set by launch_rows: the rings of tiles (x, then weights) and of packed tiles
  int ring_tiles, ring_raws;
  uint32_t x_bytes, tile_bytes, raw_bytes;
};
struct Unit {
  int r0, n0, split, kb0, kblocks;
};
__device__ __forceinline__ Unit unit_of(const Shape& h, int u, int kblocks) {
  Unit r;
  r.r0 = u % h.row_blocks * kRows;
  u /= h.row_blocks;
  r.split = u % h.splits;
  r.n0 = u / h.splits * h.toks;
  r.kb0 = r.split * h.kb_per_split;
  r.kblocks = min(h.kb_per_split, kblocks - r.kb0);
  return r;
}

struct Maps {
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
// Bounded wait: out of line after the first try, and over as soon as another role has given up.
static __device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, const volatile int* failed) {
  for (uint32_t i = 0; i < kSpinLimit && !*failed; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
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
__device__ __forceinline__ Group4 group4(uint32_t s2, uint32_t z2) {  // the group's scale and zero, twice each
  return {*reinterpret_cast<const __half2*>(&s2), __hsub2(__floats2half2_rn(-1024.f, -64.f), *reinterpret_cast<const __half2*>(&z2))};
}
// Half i of eight, twice.
__device__ __forceinline__ uint32_t pick(const uint4& v, int i) {
  const uint32_t lo = i & 2 ? v.y : v.x, hi = i & 2 ? v.w : v.z;
  return __byte_perm(i & 4 ? hi : lo, 0u, i & 1 ? 0x3232 : 0x1010);
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

// Epi: a copy per epilogue thread and unit; begin(row, n0, tokens, split), then chunk(c, z, here) for every 32 tokens n0 + c .. (here of
// them valid), then end(); rows() is the number of rows, beyond which a thread is not asked.
template <int kFmt, class Epi>
__global__ void __launch_bounds__(tc_threads<kFmt>(), 1)
    tc_rows_kernel(const __grid_constant__ Maps maps, const Weights a, const Shape h, const Epi epilogue, int* timeout) {
  extern __shared__ unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kMaxTiles], ready[kMaxTiles], empty[kMaxTiles], raw_full[kMaxRaws], raw_empty[kMaxRaws], acc_full[2], acc_empty[2];
  __shared__ float scales[kToks];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = (smem_u32(smem) + 1023u) & ~1023u, raw_ring = ring + h.ring_tiles * h.tile_bytes;
  const int kblocks = (a.K + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int i = 0; i < h.ring_tiles; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&ready[i]), kExpandWarps / 2);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < h.ring_raws; ++i) {
      mbar_init(smem_u32(&raw_full[i]), 1);
      mbar_init(smem_u32(&raw_empty[i]), kExpandWarps / 2);
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

  auto wait = [&](uint64_t& bar, int parity) { return mbar_try_wait(smem_u32(&bar), parity) || wait_on(smem_u32(&bar), parity, &failed); };
  bool ok = true;
  if (warp == 0 || (kFmt != 0 && warp == 6)) {
    // ---- loads: the fp16 tiles of both operands, or the packed weights (warp 0) and the rows (warp 6) on rings of their own
    if (lane == 0) {
      const bool packed = kFmt != 0 && warp == 0;
      const int stages = packed ? h.ring_raws : h.ring_tiles;
      int it = 0, s = 0, phase = 0;
      for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
        const Unit un = unit_of(h, u, kblocks);
        for (int kb = un.kb0; kb < un.kb0 + un.kblocks; ++kb, ++it) {
          if (it >= stages && !(ok = wait(packed ? raw_empty[s] : empty[s], phase ^ 1))) break;
          const uint32_t bar = smem_u32(packed ? &raw_full[s] : &full[s]), dst = ring + s * h.tile_bytes;
          if (packed) {
            mbar_expect_tx(bar, h.toks * raw_row<kFmt>());
            tma_2d(raw_ring + s * h.raw_bytes, &maps.w, bar, kb * raw_row<kFmt>(), un.n0);
          } else {
            mbar_expect_tx(bar, 128 * (h.x_rows + (kFmt == 0 ? h.toks : 0)));
            tma_2d(dst, &maps.x, bar, kb * kBK, un.r0);
            if (kFmt == 0) tma_2d(dst + h.x_bytes, &maps.w, bar, kb * kBK, un.n0);
          }
          if (++s == stages) { s = 0; phase ^= 1; }
        }
      }
      if (!ok)  // leave no copy in flight behind
        for (int i = it > stages ? it - stages : 0; i < it; ++i) mbar_wait(smem_u32(packed ? &raw_full[i % stages] : &full[i % stages]), (i / stages) & 1);
    }
  } else if (warp == 1) {
    // ---- products: K blocks of 64 as four instructions into the unit's accumulator
    if (lane == 0) {
      const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(h.toks >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
      int n = 0, s = 0, phase = 0;
      for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x, ++n) {
        if (n >= 2 && !(ok = wait(acc_empty[n & 1], ((n >> 1) - 1) & 1))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + (n & 1) * kToks;
        const int here = unit_of(h, u, kblocks).kblocks;
        for (int kb = 0; kb < here; ++kb) {
          ok = wait(full[s], phase) && (kFmt == 0 || wait(ready[s], phase));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dx = tile_desc(ring + s * h.tile_bytes), dw = tile_desc(ring + s * h.tile_bytes + h.x_bytes);
#pragma unroll
          for (int k4 = 0; k4 < kBK / 16; ++k4) mma(acc, dx + 2 * k4, dw + 2 * k4, idesc, (kb | k4) != 0);
          commit(smem_u32(&empty[s]));
          if (++s == h.ring_tiles) { s = 0; phase ^= 1; }
        }
        if (ok) commit(smem_u32(&acc_full[n & 1]));
      }
    }
  } else if (warp < 6) {
    // ---- reduction: a thread owns a row of x, its TMEM lane, and takes the unit's tokens 32 at a time
    const int quad = warp & 3, t = threadIdx.x - 64;
    int n = 0;
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x, ++n) {
      const Unit un = unit_of(h, u, kblocks);
      const int r = un.r0 + quad * 32 + lane, toks = min(h.toks, a.V - un.n0);
      if (kFmt == 1) {
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the last unit's scales have been read
        for (int i = t; i < kToks; i += 128) scales[i] = i < toks ? __half2float(a.scale[un.n0 + i]) : 0.f;
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
      Epi epi = epilogue;
      const bool some = r - lane < epilogue.rows();  // (nothing to do for a warp beyond the last row)
      if (r < epilogue.rows()) epi.begin(r, un.n0, toks, un.split);
      for (int c = 0; c < toks && some; c += 32) {
        float z[32];
        tmem_ld32(tmem + (n & 1) * kToks + c + (static_cast<uint32_t>(quad * 32) << 16), z);
        if (kFmt == 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) z[i] *= scales[c + i];
        }
        if (r < epilogue.rows()) epi.chunk(c, z, min(32, toks - c));
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(smem_u32(&acc_empty[n & 1]));
      if (r < epilogue.rows()) epi.end();
    }
  } else if (kFmt != 0 && warp >= 8) {
    // ---- expansion: a thread owns a row of the tile, 64 weights a K block; half of the warps take the even K blocks, half the odd
    // ones.  Row r of the tile is 128 bytes at r * 128, its 16-byte chunk c at chunk position c ^ (r & 7); a packed row of 64 (32)
    // bytes has its chunk c at c ^ (r / 2 & 3) (c ^ (r / 4 & 1)): the swizzles of 128-, 64- and 32-byte rows, so that no two
    // lanes of a quarter warp meet in a bank.  (No barrier's phase is
    // missed by taking every other K block: the packed ring is even; and in the other ring of T >= 2 tiles block i waits until block
    // i - T is used, when block i - 2 has shown that i - 2 - T is, so the fill of this tile before that one, i - 2 T, is too.)
    const int r = threadIdx.x & 255, turn = (threadIdx.x >> 8) - 1;
    const uint32_t raw = raw_ring + r * raw_row<kFmt>(), raw_swz = kFmt == 1 ? ((r >> 1) & 3) << 4 : ((r >> 2) & 1) << 4;
    const int shift = a.group == 32 ? 5 : a.group == 64 ? 6 : 7, groups = (a.K + a.group - 1) >> shift;
    uint32_t at[8];  // where the chunks of this row go, in the first stage
#pragma unroll
    for (int c = 0; c < 8; ++c) at[c] = ring + h.x_bytes + r * 128 + ((16 * c) ^ ((r & 7) << 4));
    // Scales and zeros: eight groups at a time as one 16-byte load each, the next eight under way; where a row of them is no
    // multiple of 16 bytes, group by group.
    const bool eights = groups % 8 == 0 && ((reinterpret_cast<uintptr_t>(a.scale) | reinterpret_cast<uintptr_t>(a.zero)) & 15u) == 0;
    const uint16_t *sp = nullptr, *zp = nullptr;
    constexpr uint32_t kEight = 0x48004800u;
    uint4 sc = make_uint4(0u, 0u, 0u, 0u), ze = make_uint4(kEight, kEight, kEight, kEight), sc_next = sc, ze_next = ze;
    auto load8 = [&](int block) {
      if (block * 8 >= groups) return;
      sc_next = reinterpret_cast<const uint4*>(sp)[block];
      if (zp) ze_next = reinterpret_cast<const uint4*>(zp)[block];
    };
    auto load_runs = [&](int kb) {  // a K block's two runs of 32 weights into the first two halves
      const int g0 = min((kb * kBK) >> shift, groups - 1), g1 = min((kb * kBK + 32) >> shift, groups - 1);
      sc_next.x = sp[g0] | (static_cast<uint32_t>(sp[g1]) << 16);
      if (zp) ze_next.x = zp[g0] | (static_cast<uint32_t>(zp[g1]) << 16);
    };
    int it = 0, rs = turn, raw_phase = 0, s = turn, tile_phase = 0;
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      const Unit un = unit_of(h, u, kblocks);
      const int row = min(un.n0 + r, a.V - 1), kb_end = un.kb0 + un.kblocks;
      int kb = un.kb0 + ((it & 1) == turn ? 0 : 1);
      int block = -1;
      if (kFmt == 2 && kb < kb_end) {
        sp = reinterpret_cast<const uint16_t*>(a.scale) + static_cast<size_t>(row) * groups;
        if (a.zero) zp = reinterpret_cast<const uint16_t*>(a.zero) + static_cast<size_t>(row) * groups;
        if (eights) load8((kb * kBK) >> (shift + 3));
        else load_runs(kb);
      }
      for (; kb < kb_end; kb += 2) {
        const bool first_round = it + kb - un.kb0 < h.ring_tiles;
        if (kFmt == 2 && (!eights || (kb * kBK) >> (shift + 3) != block)) {
          sc = sc_next;
          ze = ze_next;
          block = (kb * kBK) >> (shift + 3);
          if (eights) load8(block + 1);
        }
        ok = __all_sync(0xffffffffu, wait(raw_full[rs], raw_phase) && (first_round || wait(empty[s], tile_phase ^ 1)));
        if (!ok) break;
        if (r < h.toks) {
          const uint32_t src = raw + rs * h.raw_bytes, stage = s * h.tile_bytes;
          if (kFmt == 1) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint4 q = lds16(src + ((16 * c) ^ raw_swz));
              const uint2 h0 = expand8(q.x), h1 = expand8(q.y), h2 = expand8(q.z), h3 = expand8(q.w);
              sts16(at[2 * c] + stage, make_uint4(h0.x, h0.y, h1.x, h1.y));
              sts16(at[2 * c + 1] + stage, make_uint4(h2.x, h2.y, h3.x, h3.y));
            }
          } else {
            const uint4 q0 = lds16(src + raw_swz), q1 = lds16(src + (16 ^ raw_swz));
            const uint32_t w[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int i = eights ? ((kb * kBK + 32 * c) >> shift) & 7 : c;
              const Group4 g = group4(pick(sc, i), pick(ze, i));
#pragma unroll
              for (int j = 0; j < 4; ++j) sts16(at[4 * c + j] + stage, expand4(w[4 * c + j], g));
            }
          }
        }
        if (kFmt == 2 && !eights && kb + 2 < kb_end) load_runs(kb + 2);  // under way until this thread's next turn
        // written through the generic proxy, read by the tensor core through the async one
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          arrive(smem_u32(&ready[s]));
          arrive(smem_u32(&raw_empty[rs]));
        }
        rs += 2;
        if (rs >= h.ring_raws) { rs -= h.ring_raws; raw_phase ^= 1; }
        s += 2;
        if (s >= h.ring_tiles) { s -= h.ring_tiles; tile_phase ^= 1; }
      }
      it += un.kblocks;
    }
  }
  if (!ok) failed = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && failed && timeout) atomicOr(timeout, kTimeoutGemm);
  __syncwarp();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// A 2-D tensor of rows of `cols` elements in boxes of box_cols x box_rows, zeros outside.
inline int encode_map(const char* what, CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base, int rows, size_t cols, int box_cols,
                      int box_rows, CUtensorMapSwizzle swizzle) {
  const TensorMapEncodeFn fn = tensor_map_encode_fn();
  RK_REQUIRE(fn, kCuda, "%s: cuTensorMapEncodeTiled is not available from this driver", what);
  const cuuint64_t dims[2] = {cols, static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {cols * elem_bytes};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RK_REQUIRE(r == CUDA_SUCCESS, kCuda, "%s: cuTensorMapEncodeTiled failed with %d (rows=%d, columns=%zu)", what, static_cast<int>(r), rows, cols);
  return kOk;
}

template <int kFmt, class Epi>
int launch_rows(cudaStream_t stream, const char* what, const half* x, int rows, const void* w, const Weights& a, Shape h, const Epi& epi, int sms) {
  Maps maps;
  int s = encode_map(what, &maps.x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x, rows, a.K, kBK, h.x_rows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s != kOk) return s;
  if (kFmt == 0) s = encode_map(what, &maps.w, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, w, a.V, a.K, kBK, h.toks, CU_TENSOR_MAP_SWIZZLE_128B);
  else s = encode_map(what, &maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, a.V, kFmt == 1 ? a.K : a.K / 2, raw_row<kFmt>(), h.toks,
                      kFmt == 1 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
  if (s != kOk) return s;
  // The rings: packed tiles want enough in flight for the HBM (64 KB or so), fp16 tiles one more than the expansion and the MMA hold
  // at a time: four where the packed ring keeps four, otherwise three.
  h.x_bytes = (h.x_rows * 128 + 1023) & ~1023;
  h.tile_bytes = std::max<uint32_t>(h.x_bytes + h.toks * 128, kRows * 128);  // (the MMA reads 128 rows of x, whatever is there)
  h.raw_bytes = (h.toks * raw_row<kFmt>() + 1023) & ~1023;
  const int budget = static_cast<int>(kSmemBytes) - 1024;
  if (kFmt == 0) {
    h.ring_tiles = std::min(kMaxTiles, budget / static_cast<int>(h.tile_bytes));
    h.ring_raws = 0;
  } else {
    h.ring_tiles = budget - 4 * static_cast<int>(h.tile_bytes) >= 4 * static_cast<int>(h.raw_bytes) ? 4 : 3;
    h.ring_raws = std::min(kMaxRaws, (budget - h.ring_tiles * static_cast<int>(h.tile_bytes)) / static_cast<int>(h.raw_bytes)) & ~1;
  }
  const size_t smem = 1024 + h.ring_tiles * static_cast<size_t>(h.tile_bytes) + h.ring_raws * static_cast<size_t>(h.raw_bytes);
  const auto kernel = tc_rows_kernel<kFmt, Epi>;
  RK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes)));
  RK_CUDA(launch_pdl(kernel, dim3(std::min(h.units, sms)), dim3(tc_threads<kFmt>()), smem, stream, maps, a, h, epi, timeout_word_or_null()));
  RK_LAUNCH_CHECK(what);
  return kOk;
}

}  // namespace tc
}  // namespace rk
