// 4-bit weights with group scales: y = epi(x W^T) with W[n,k] = (q[n,k] - zero[n,g]) * scale[n,g], g = k / group, for
// groups of 32, 64 or 128 input channels, the last of which may be short, and without zeros (then 8) or with them.
// Packing as the other 4-bit format: byte j of a row holds q[2j] (low nibble) and q[2j + 1] (high nibble).
//
// Up to eight rows of x (one launch each): bound by the weights' bytes, and next by instruction issue, so the kernel spends as
// little as it can on a weight.
//   - A nibble under a mask IS a half: 0x000q is the subnormal q 2^-24 and 0x00q0 is 16 q 2^-24, which the tensor cores
//     multiply exactly.  Turning a 32-bit word into four operand registers costs one shift and four ANDs, no conversion;
//     low and high nibbles go to sums of their own (lo, hi), joined as lo + hi / 16.
//   - Scales and zeros multiply the sums of a group, in fp32:  y = sum_g s_g (sum_k q x - z_g sum_k x), with the sums of x
//     made once per CTA.  A weight is never rounded to half, unlike in the format of groups of 128 that the models use.
//   - mma.sync m16n8k16 has eight columns.  With fewer rows of x the columns hold different 32-weight chunks (a
//     lane whose column is another chunk's reads zeros), so that with one row eight chunks end up in eight columns and the
//     scales are applied once for all of them.
// kRounded: the same walk for callers whose weights are half((q - zero) * scale) (the head product of head_logprobs.cu): a word
// becomes eight such halves (one subtraction or fused multiply-add and one product per two), the sums need no scales, and
// the columns are up to eight rows of x.
// One CTA of 16 warps per SM takes a contiguous range of output channels in tiles of up to 32.  The warps form 1, 2 or 4
// teams with a tile each; the tile's K extent is cut into boxes of 128 bytes per row, dealt out to the team's warps and
// fetched by one 2-D tensor copy each into the warp's ring.  The warps' partial sums of a tile are added in warp order:
// results do not depend on timing.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "tc_packed.cuh"

namespace rk {
namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kTileRows = 32;
constexpr int kBoxWeights = 256;  // 128 bytes along a row: eight chunks of 32 weights
// Rows up to which the weights are streamed and never rounded.  Nine to sixteen rows in two such launches took 70 to 82 us at
// 65536 x 4096, 24 at 16384 x 4096, 18 to 20 at 10240 x 2560 and 30 at 2560 x 10240; the kernel for many rows takes 58, 18, 14 and 12,
// and 85, 27, 17 and 15 with exact weights.
constexpr int kMaxRows = 8;
constexpr size_t kSmemLimit = 226 * 1024;

struct MatvecMaps {
  CUtensorMap q, scale, zero;
};

struct MatvecPlan {
  int teams = 0;                // of 16 / teams warps
  int h = 0, tiles = 0;         // rows of a tile and box, tiles per team
  int boxes = 0;                // along a weight row
  int slots = 0, slot_bytes = 0;  // a slot: the box, and behind it 16 bytes of scales and of zeros per row
  bool copied = false;            // whether tensor copies can bring those
  int x_pitch = 0;              // bytes from one staged row of x to the next: 64 modulo 128, two rows share no bank
  uint32_t part_off = 0, sums_off = 0, x_off = 0, zero_off = 0;  // from the aligned start of shared memory
  size_t smem = 0;
  int grid = 0;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first) {
  if (first)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&w)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// The eight weights of a word as pairs (0, 4), (1, 5), (2, 6), (3, 7): a nibble under the exponent of 1024 is 1024 + q, a high one
// 1024 + 16 q; less 1024 + zero (or / 16 less 64 + zero) that is q - zero, exactly where zero is whole, and the product rounds once.  one: 0x64006400 in a
// register of the caller's (as a literal beside the mask it would take an instruction of its own).
template <uint32_t kMask> __device__ __forceinline__ __half2 under_1024(uint32_t u, uint32_t one) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(u), "n"(kMask), "r"(one));  // (u & mask) | one
  return u2h(v);
}
__device__ __forceinline__ void round4(uint32_t u, uint32_t one, __half2 s, __half2 zlo, __half2 zhi, uint32_t (&o)[4]) {
  const uint32_t v = u >> 8;
  const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
  o[0] = h2u(__hmul2(__hsub2(under_1024<0x000f000fu>(u, one), zlo), s));
  o[1] = h2u(__hmul2(__hfma2(under_1024<0x00f000f0u>(u, one), sixteenth, zhi), s));
  o[2] = h2u(__hmul2(__hsub2(under_1024<0x000f000fu>(v, one), zlo), s));
  o[3] = h2u(__hmul2(__hfma2(under_1024<0x00f000f0u>(v, one), sixteenth, zhi), s));
}
// 0 where both of two zeros are whole numbers up to 1024, which 1024 + zero and 64 + zero hold exactly.
__device__ __forceinline__ uint32_t not_whole(uint32_t z2) {
  const uint32_t size = z2 & 0x7fff7fffu;
  const __half2 big = __floats2half2_rn(1024.f, 1024.f);
  return h2u(__hsub2(__hadd2(u2h(size), big), big)) ^ size;
}
// round4 for any zeros: the product in fp32, rounded from there.
__device__ __forceinline__ void round4_any(uint32_t u, float s, float z, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = h2u(__floats2half2_rn(__fmul_rn(__fsub_rn(static_cast<float>(u >> (4 * i) & 15), z), s),
                                 __fmul_rn(__fsub_rn(static_cast<float>(u >> (4 * i + 16) & 15), z), s)));
}
__device__ __forceinline__ float half_of(uint32_t pair, int i) {
  const float2 f = h2f2(pair);
  return i ? f.y : f.x;
}
// What becomes of an fp32 sum; the store rounds to half where y is half.
__device__ __forceinline__ float w4_epilogue(float v, int epi) {
  if (epi == kEpiRawF32) return v;
  const float h = __half2float(__float2half_rn(v));
  if (epi != kEpiRelu2) return h;
  const float u = fmaxf(h, 0.f);
  return u * u;
}
__device__ __forceinline__ void store_epi(const W4GroupArgs& a, size_t o, float v) {
  const float e = w4_epilogue(v, a.epi);
  if (a.epi == kEpiF32 || a.epi == kEpiRawF32) static_cast<float*>(a.y)[o] = e;
  else static_cast<half*>(a.y)[o] = __float2half_rn(e);
}

// kM: columns per chunk, the rows of x rounded up to 1, 2, 4 or 8; kShift: log2 of the group.  A box is worked off in passes of
// kPass chunks, after each of which the sums are scaled; chunk c of a pass goes to the columns of slot c mod kSlots.
// kBlk: blocks of 16 rows in a tile.  kCopied: scales and zeros come with their box, by tensor copies of the eight groups
// (16 bytes) of each row that hold the box's; otherwise (rows of groups that are not multiples of 16 bytes) through registers.
template <int kM, int kShift, int kBlk, bool kCopied, bool kRounded>
__global__ void __launch_bounds__(kThreads, 1) w4_matvec_kernel(const __grid_constant__ MatvecMaps maps, const W4GroupArgs a, const MatvecPlan p, int* timeout) {
  constexpr int kSlots = 8 / kM, kGroupChunks = 1 << (kShift - 5);
  constexpr int kPass = kSlots > kGroupChunks ? kSlots : kGroupChunks, kPasses = 8 / kPass;
  static_assert(!kRounded || kM == 8, "");
  constexpr float kUnit = 1.0f / 16777216.0f;  // what a code of 1 stands for in the products
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t bars[kWarps][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t dyn = smem_u32(smem_dyn), base = (dyn + 1023u) & ~1023u;
  unsigned char* const mem = smem_dyn + (base - dyn);
  const uint32_t ring = base + warp * p.slots * p.slot_bytes;
  float* const part = reinterpret_cast<float*>(mem + p.part_off);
  float* const sums = reinterpret_cast<float*>(mem + p.sums_off);
  const int team_warps = kWarps / p.teams, team = warp / team_warps, team_warp = warp - team * team_warps;
  // this team's tiles: team, team + teams, ... of the CTA's
  const int cta_row0 = blockIdx.x * p.teams * p.tiles * p.h, all_tiles = min(p.teams * p.tiles, (a.N - cta_row0 + p.h - 1) / p.h);
  const int row0 = cta_row0 + team * p.h, row_step = p.teams * p.h, tiles = all_tiles > team ? (all_tiles - team - 1) / p.teams + 1 : 0;
  const int groups = (a.K + (1 << kShift) - 1) >> kShift;

  if (lane == 0) {
    for (int i = 0; i < p.slots; ++i) mbar_init(smem_u32(&bars[warp][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.q) : "memory");
  }
  if (threadIdx.x < 32) *reinterpret_cast<uint4*>(mem + p.zero_off + threadIdx.x * 16) = make_uint4(0u, 0u, 0u, 0u);  // what idle columns read, at the offsets of eight chunks
  if (kRounded && kCopied && lane >= p.h) {  // what is read as the zeros of rows that the copies do not bring: 0, a whole number
    for (int i = 0; i < p.slots; ++i) *reinterpret_cast<uint4*>(mem + (ring - base) + (i + 1) * p.slot_bytes - 512 + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();

  // this warp's boxes: every team_warps-th of the team's flattened (tile, box) sequence
  auto advance = [&](int& tile, int& kb) {
    kb += team_warps;
    while (kb >= p.boxes && tile < tiles) { kb -= p.boxes; ++tile; }
  };
  int q_tile = 0, q_kb = team_warp - team_warps, q_slot = 0;
  advance(q_tile, q_kb);
  // used: 0, computed from what the slot's last contents went into, so that they have been read when the copy is issued.
  auto issue = [&](uint32_t used) {
    if (lane == 0) {
      const uint32_t bar = smem_u32(&bars[warp][q_slot]);
      const uint32_t dst = ring + q_slot * p.slot_bytes + used;
      const int n = row0 + q_tile * row_step;
      mbar_expect_tx(bar, p.h * (128 + (kCopied ? (a.zero ? 32 : 16) : 0)));
      tc::tma_2d(dst, &maps.q, bar, q_kb << 7, n);
      if (kCopied) {
        const int first = (q_kb << (8 - kShift)) & ~7;
        tc::tma_2d(dst + p.slot_bytes - 1024, &maps.scale, bar, first, n);
        if (a.zero) tc::tma_2d(dst + p.slot_bytes - 512, &maps.zero, bar, first, n);
      }
    }
    if (++q_slot == p.slots) q_slot = 0;
    advance(q_tile, q_kb);
  };
  for (int i = 0; i < p.slots && q_tile < tiles; ++i) issue(0u);

  // A lane's share of a box's scales and zeros, for the rows g, g + 8, g + 16, g + 24: groups of 32: the pair 2t, 2t + 1 of the
  // box's eight; of 64: group t of four; of 128: group t / 2 of two.
  uint32_t sc[2 * kBlk], ze[2 * kBlk], row_at[2 * kBlk];  // row_at: the row's first group (the host checks that 32 bits hold it)
  int row_tile = -1;
  const bool paired = (groups & 1) == 0 && ((reinterpret_cast<uintptr_t>(a.scale) | reinterpret_cast<uintptr_t>(a.zero)) & 3) == 0;
  const uint16_t *const scale = reinterpret_cast<const uint16_t*>(a.scale), *const zero = reinterpret_cast<const uint16_t*>(a.zero);
  auto fetch = [&](int tile, int kb) {
    if (tile != row_tile) {
#pragma unroll
      for (int i = 0; i < 2 * kBlk; ++i) row_at[i] = static_cast<uint32_t>(min(row0 + tile * row_step + g + 8 * i, a.N - 1)) * groups;
      row_tile = tile;
    }
    const int at = kShift == 5 ? kb * 8 + 2 * t : kShift == 6 ? kb * 4 + t : kb * 2 + (t >> 1);
    const uint32_t o0 = min(at, groups - (kShift == 5 && paired ? 2 : 1)), o1 = min(at + 1, groups - 1);
#pragma unroll
    for (int i = 0; i < 2 * kBlk; ++i) {
      ze[i] = 0x48004800u;  // 8, 8
      const uint16_t *s = scale + (row_at[i] + o0), *z = zero + (row_at[i] + o0);
      if (kShift == 5 && paired) {
        sc[i] = *reinterpret_cast<const uint32_t*>(s);
        if (zero) ze[i] = *reinterpret_cast<const uint32_t*>(z);
      } else {
        sc[i] = *s;
        if (zero) ze[i] = *z;
        if (kShift == 5) {
          sc[i] |= static_cast<uint32_t>(s[o1 - o0]) << 16;
          if (zero) ze[i] |= static_cast<uint32_t>(z[o1 - o0]) << 16;
        }
      }
    }
  };
  int c_tile = 0, c_kb = team_warp - team_warps;
  advance(c_tile, c_kb);
  if (!kCopied && c_tile < tiles) fetch(c_tile, c_kb);

  // x as halves in the order of the fragments: a block of eight as x0 x4 x2 x6 | x1 x5 x3 x7 (the operands of the low and of the high
  // nibbles of a word); zeros behind K.  The sums of the chunks of 32 go to shared memory beside it.
  const int blocks = p.boxes * 32, chunks = p.boxes * 8;
  float* const chunk_sums = part;  // [M][chunks], until the first tile's partial sums
  auto stage = [&](int m, int j, uint4 q) {
    *reinterpret_cast<uint4*>(mem + p.x_off + m * p.x_pitch + j * 16) =
        make_uint4(__byte_perm(q.x, q.z, 0x5410), __byte_perm(q.y, q.w, 0x5410), __byte_perm(q.x, q.z, 0x7632), __byte_perm(q.y, q.w, 0x7632));
    const float2 f0 = h2f2(q.x), f1 = h2f2(q.y), f2 = h2f2(q.z), f3 = h2f2(q.w);
    float sum = ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);  // (blocks is a multiple of 32: whole warps take part)
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if ((j & 3) == 0) chunk_sums[m * chunks + (j >> 2)] = sum;
  };
  auto walk = [&](int& m, int& j) {  // to the block kThreads further on
    j += kThreads;
    while (j >= blocks) { j -= blocks; ++m; }
  };
  constexpr int kDeep = 8;  // loads under way at a time
  int m_ld = 0, j_ld = static_cast<int>(threadIdx.x) - kThreads, m_st = 0, j_st = static_cast<int>(threadIdx.x) - kThreads;
  walk(m_ld, j_ld);
  walk(m_st, j_st);
  while (m_st < a.M) {
    uint4 q[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      q[d] = make_uint4(0u, 0u, 0u, 0u);
      if (m_ld < a.M) {
        if (j_ld * 8 < a.K) q[d] = *reinterpret_cast<const uint4*>(a.x + static_cast<size_t>(m_ld) * a.K + j_ld * 8);
        walk(m_ld, j_ld);
      }
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
      if (m_st < a.M) {
        stage(m_st, j_st, q[d]);
        walk(m_st, j_st);
      }
  }
  __syncthreads();
  // -2^-24 times the sum of x that belongs to each column of each pass: [box][pass][8]
  for (int i = threadIdx.x; i < p.boxes * kPasses * 8; i += kThreads) {
    const int col = i & 7, c0 = (i >> 3) * kPass + col / kM, m = min(col % kM, a.M - 1);
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < kPass; c += kSlots) sum += chunk_sums[m * chunks + c0 + c];
    sums[i] = -kUnit * sum;
  }
  __syncthreads();

  const uint32_t w_lane = (((lane >> 3) & 1) * 8 + (lane & 7)) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);  // see ldmatrix below
  const int slot_of_lane = g / kM;
  const uint32_t x_row = base + p.x_off + min(g % kM, a.M - 1) * p.x_pitch + (t << 4), zero_now = base + p.zero_off;
  float acc[kBlk][4];
#pragma unroll
  for (int b = 0; b < kBlk; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[b][i] = 0.f;
  const uint32_t none = base >> 30, one = 0x64006400u + none;  // (a shared-memory address is below 2^30, which the compiler does not know)
  int cur = 0, slot = 0, phase = 0;
  bool dead = false;  // a wait ran out: no more work, but the barriers are kept
  for (;;) {
    // Tile boundaries: every warp of the team leaves its sums, and one barrier later its threads add up the tile.
    for (const int upto = min(c_tile, tiles); cur < upto; ++cur) {
      float* const sums_of = part + ((cur & 1) * kWarps + team * team_warps) * kTileRows * kM;
      float* const mine = sums_of + team_warp * kTileRows * kM;
#pragma unroll
      for (int b = 0; b < kBlk; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = acc[b][i];  // row 16 b + g + 8 (i / 2), column 2 t + i % 2
          acc[b][i] = 0.f;
          if (kM == 1) {
            if (i & 1) continue;
            v += acc[b][i + 1];
            acc[b][i + 1] = 0.f;
          }
          if (kM <= 2) v += __shfl_xor_sync(0xffffffffu, v, 1);
          if (kM <= 4) v += __shfl_xor_sync(0xffffffffu, v, 2);
          const int m = kM == 1 ? 0 : (2 * t + (i & 1)) % kM;
          if (2 * t < kM) mine[(16 * b + g + 8 * (i >> 1)) * kM + m] = v;
        }
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(team_warps * 32) : "memory");
      for (int i = team_warp * 32 + lane; i < kTileRows * kM; i += team_warps * 32) {
        const int r = i % kTileRows, m = i / kTileRows, n = row0 + cur * row_step + r;
        if (r >= p.h || m >= a.M || n >= a.N) continue;
        float v = 0.f;
#pragma unroll 4
        for (int w = 0; w < team_warps; ++w) v += sums_of[w * kTileRows * kM + r * kM + m];
        store_epi(a, static_cast<size_t>(m) * a.N + n, kRounded ? v : v * 16777216.0f);
      }
    }
    if (c_tile >= tiles) break;

    const int kb = c_kb;
    uint32_t s_now[2 * kBlk], z_now[2 * kBlk];
    advance(c_tile, c_kb);
    if (!kCopied) {
#pragma unroll
      for (int i = 0; i < 2 * kBlk; ++i) { s_now[i] = sc[i]; z_now[i] = ze[i]; }
      if (c_tile < tiles) fetch(c_tile, c_kb);
    }
    const uint32_t bar = smem_u32(&bars[warp][slot]);
    if (!dead && !mbar_try_wait(bar, phase) && !mbar_wait(bar, phase)) {
      dead = true;
      if (lane == 0 && timeout) atomicOr(timeout, kTimeoutGemv);
    }
    if (!dead) {
      const uint32_t wbase = ring + slot * p.slot_bytes;
      if (kCopied) {
        const int at = (kb << (8 - kShift)) & 7;  // the box's first group among the eight
        const unsigned char* params = mem + (wbase - base) + p.slot_bytes - 1024 + g * 16 + 2 * (at + (kShift == 5 ? 2 * t : kShift == 6 ? t : t >> 1));
#pragma unroll
        for (int i = 0; i < 2 * kBlk; ++i) {
          s_now[i] = kShift == 5 ? *reinterpret_cast<const uint32_t*>(params + 128 * i) : *reinterpret_cast<const uint16_t*>(params + 128 * i);
          z_now[i] = 0x48004800u;
          if (a.zero) z_now[i] = kShift == 5 ? *reinterpret_cast<const uint32_t*>(params + 512 + 128 * i) : *reinterpret_cast<const uint16_t*>(params + 512 + 128 * i);
        }
      }
      const uint32_t x_now = x_row + (kb << 9);
      float lo[kBlk][4], hi[kBlk][4];
      __half2 scale2[2 * kBlk], zero_lo[2 * kBlk], zero_hi[2 * kBlk];  // kRounded
      auto work = [&](auto any) {
        // kRounded: whatever the zeros are (zero_lo then holds them as they are); in a loop, so that it leaves the other form its registers
        constexpr bool kAny = decltype(any)::value;
        constexpr int kUnroll = kAny ? 1 : 4;
#pragma unroll kUnroll
        for (int c2 = 0; c2 < 4; ++c2) {
          // Two chunks of 16 rows: the matrices are (rows 0-7, rows 8-15) x (chunk 2 c2, chunk 2 c2 + 1), 16 bytes a row, and a lane gets
          // the word t of row g.  The 128-byte swizzle puts chunk c of row r at c ^ (r mod 8).
          uint32_t w[kBlk][4];
#pragma unroll
          for (int b = 0; b < kBlk; ++b) ldmatrix4(w[b], wbase + b * 2048 + (w_lane ^ (c2 << 5)));
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const int c = 2 * c2 + cc;
            uint4 xv;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(xv.x), "=r"(xv.y), "=r"(xv.z), "=r"(xv.w)
                         : "r"((kSlots == 1 || slot_of_lane == c % kSlots ? x_now : zero_now) + (c << 6)));
            if (kRounded) {
              if (c % kGroupChunks == 0) {  // a new group: its parameters for the rows g and g + 8 of each block
                const int from = kShift == 7 ? (c >> 2) << 1 : c >> 1;
#pragma unroll
                for (int i = 0; i < 2 * kBlk; ++i) {
                  const uint32_t sp = __shfl_sync(0xffffffffu, s_now[i], (lane & ~3) | from), zp = __shfl_sync(0xffffffffu, z_now[i], (lane & ~3) | from);
                  const uint32_t sel = kShift == 5 && (c & 1) ? 0x3232 : 0x1010;
                  scale2[i] = u2h(__byte_perm(sp, 0u, sel));
                  const __half2 z2 = u2h(__byte_perm(zp, 0u, sel));
                  zero_lo[i] = kAny ? z2 : __hadd2(z2, __floats2half2_rn(1024.f, 1024.f));
                  zero_hi[i] = __hfma2(z2, __floats2half2_rn(-1.f, -1.f), __floats2half2_rn(-64.f, -64.f));
                }
              }
              if ((kb << 8) + 32 * c >= a.K) {  // behind K: code 0, which may stand for an infinite weight
#pragma unroll
                for (int i = 0; i < 2 * kBlk; ++i) scale2[i] = __floats2half2_rn(0.f, 0.f);
              }
#pragma unroll
              for (int b = 0; b < kBlk; ++b) {
                uint32_t ra[4], rb[4];
                if (!kAny) {
                  round4(w[b][2 * cc], one, scale2[2 * b], zero_lo[2 * b], zero_hi[2 * b], ra);
                  round4(w[b][2 * cc + 1], one, scale2[2 * b + 1], zero_lo[2 * b + 1], zero_hi[2 * b + 1], rb);
                } else {
                  round4_any(w[b][2 * cc], __low2float(scale2[2 * b]), __low2float(zero_lo[2 * b]), ra);
                  round4_any(w[b][2 * cc + 1], __low2float(scale2[2 * b + 1]), __low2float(zero_lo[2 * b + 1]), rb);
                }
                mma16816(lo[b], ra[0], rb[0], ra[2], rb[2], xv.x, xv.y, c == 0);
                mma16816(hi[b], ra[1], rb[1], ra[3], rb[3], xv.z, xv.w, c == 0);
                if (c == 7) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) acc[b][i] += lo[b][i] + hi[b][i];
                }
              }
              continue;
            }
            const bool first = c % kPass == 0;
#pragma unroll
            for (int b = 0; b < kBlk; ++b) {
              const uint32_t wa = w[b][2 * cc], wb = w[b][2 * cc + 1], va = wa >> 8, vb = wb >> 8;
              mma16816(lo[b], wa & 0x000f000fu, wb & 0x000f000fu, va & 0x000f000fu, vb & 0x000f000fu, xv.x, xv.y, first);
              mma16816(hi[b], wa & 0x00f000f0u, wb & 0x00f000f0u, va & 0x00f000f0u, vb & 0x00f000f0u, xv.z, xv.w, first);
            }
            if ((c + 1) % kPass != 0) continue;
            // the end of a pass: scales and zeros of the groups that this lane's two columns hold
            const int pass = c / kPass;
            const float2 xs = *reinterpret_cast<const float2*>(sums + (kb * kPasses + pass) * 8 + 2 * t);
            // the chunk of the column 2t, and where its group's parameters are: (lane of the quad, half of the pair)
            const int chunk = kM == 1 ? 2 * t : pass * kPass + (kM == 8 ? 0 : 2 * t / kM);
            const int from = kShift == 5 ? chunk >> 1 : kShift == 6 ? chunk >> 1 : (chunk >> 2) << 1;
#pragma unroll
            for (int b = 0; b < kBlk; ++b) {
              float s0[2], s1[2], z0[2], z1[2];  // rows g and g + 8: of the lane's first and second column
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t sp = s_now[2 * b + i], zp = z_now[2 * b + i];
                if (kM > 1) {
                  sp = __shfl_sync(0xffffffffu, sp, (lane & ~3) | from);
                  zp = __shfl_sync(0xffffffffu, zp, (lane & ~3) | from);
                }
                if (kM == 1 && kShift == 5) {
                  s0[i] = half_of(sp, 0); s1[i] = half_of(sp, 1);
                  z0[i] = half_of(zp, 0); z1[i] = half_of(zp, 1);
                } else {
                  const int odd = kShift == 5 ? chunk & 1 : 0;
                  s0[i] = s1[i] = half_of(sp, odd);
                  z0[i] = z1[i] = half_of(zp, odd);
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float u = fmaf(hi[b][i], 0.0625f, lo[b][i]);
                acc[b][i] = fmaf(i & 1 ? s1[i >> 1] : s0[i >> 1], fmaf(i & 1 ? z1[i >> 1] : z0[i >> 1], i & 1 ? xs.y : xs.x, u), acc[b][i]);
              }
            }
          }
        }
      };
      bool whole = true;  // the zeros of the box's groups are whole numbers
      if (kRounded && a.zero) {
        uint32_t odd = 0;
#pragma unroll
        for (int i = 0; i < 2 * kBlk; i += 2) {
          if (kShift == 5) odd |= not_whole(z_now[i]) | not_whole(z_now[i + 1]);
          else odd |= not_whole(__byte_perm(z_now[i], z_now[i + 1], 0x5410));
        }
        whole = __all_sync(0xffffffffu, odd == 0);
      }
      if (!kRounded || whole) work(std::false_type());
      else work(std::true_type());
    }
    // Every lane has read the slot: it may be overwritten.  The barrier alone orders the loads' issue, not their results, and the
    // products that take those might be placed behind the copy; its address waits for the sums that they and the scales went into (a
    // product takes all lanes' operands, so lane 0's sums stand for the warp's).
    __syncwarp();
    if (!dead && q_tile < tiles) {
      uint32_t used = 0;
#pragma unroll
      for (int b = 0; b < kBlk; ++b) used |= __float_as_uint(acc[b][0]) | __float_as_uint(acc[b][2]);
      issue(used & none);
    }
    if (++slot == p.slots) { slot = 0; phase ^= 1; }
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

namespace {

int columns(int M) { return M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : 8; }

// One tile height for all CTAs, so that a box is exactly what its team works on: N / SMs rows per CTA in equal tiles of at most
// 32.  Larger teams share a tile's K extent among more warps, smaller ones pay the end of a tile (sums through shared memory, a
// barrier) less often per box: as many teams as keep the number of 16-row blocks within 15 % of the least.
bool plan_matvec(const W4GroupArgs& a, int sms, MatvecPlan* out, bool rounded = false) {
  const int kM = rounded ? 8 : columns(a.M), group_chunks = a.group / 32, pass = std::max(8 / kM, group_chunks), passes = 8 / pass;
  const int target = (a.N + sms - 1) / sms, groups = (a.K + a.group - 1) / a.group;
  const bool copied = groups % 8 == 0 && ((reinterpret_cast<uintptr_t>(a.scale) | reinterpret_cast<uintptr_t>(a.zero)) & 15u) == 0;
  for (const int most : {kTileRows, 16}) {  // tiles of 16 where those of 32 leave no room for two boxes per warp
    MatvecPlan p;
    auto tile = [&](int teams) {
      p.teams = teams;
      p.tiles = (target + most * teams - 1) / (most * teams);
      p.h = (target + p.tiles * teams - 1) / (p.tiles * teams);
      return p.tiles * teams * ((p.h + 15) / 16);
    };
    const int least = std::min(tile(1), std::min(tile(2), tile(4)));
    if (tile(4) * 100 > least * 115 && tile(2) * 100 > least * 115) tile(1);
    p.grid = (a.N + p.teams * p.tiles * p.h - 1) / (p.teams * p.tiles * p.h);
    p.boxes = (a.K + kBoxWeights - 1) / kBoxWeights;
    p.copied = copied;
    p.slot_bytes = ((p.h * 128 + 1023) & ~1023) + (copied ? 1024 : 0);
    p.x_pitch = p.boxes * kBoxWeights * 2 + 64;
    const size_t part = std::max<size_t>(2u * kWarps * kTileRows * kM * sizeof(float), static_cast<size_t>(a.M) * p.boxes * 8 * sizeof(float));
    const size_t sums = static_cast<size_t>(p.boxes) * passes * 8 * sizeof(float), x = static_cast<size_t>(a.M) * p.x_pitch;
    const size_t fixed = 1024 + 512 + ((part + 127) & ~static_cast<size_t>(127)) + ((sums + 127) & ~static_cast<size_t>(127)) + x;
    const size_t per_slot = static_cast<size_t>(kWarps) * p.slot_bytes;
    if (fixed + 2 * per_slot > kSmemLimit) continue;
    p.slots = static_cast<int>(std::min<size_t>(4, (kSmemLimit - fixed) / per_slot));
    p.part_off = static_cast<uint32_t>(p.slots * per_slot);
    p.sums_off = p.part_off + static_cast<uint32_t>((part + 127) & ~static_cast<size_t>(127));
    p.zero_off = p.sums_off + static_cast<uint32_t>((sums + 127) & ~static_cast<size_t>(127));
    p.x_off = p.zero_off + 512;
    p.smem = fixed + p.slots * per_slot;
    *out = p;
    return true;
  }
  return false;
}

template <int kM, int kShift, int kBlk, bool kCopied, bool kRounded>
int launch_matvec(cudaStream_t stream, const MatvecMaps& maps, const W4GroupArgs& a, const MatvecPlan& p) {
  const auto kernel = w4_matvec_kernel<kM, kShift, kBlk, kCopied, kRounded>;
  RK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemLimit)));
  RK_CUDA(launch_pdl(kernel, dim3(p.grid), dim3(kThreads), p.smem, stream, maps, a, p, timeout_word_or_null()));
  RK_LAUNCH_CHECK("linear_w4a16_group launch");
  return kOk;
}
template <int kM, int kShift, bool kRounded>
int launch_matvec(cudaStream_t stream, const MatvecMaps& maps, const W4GroupArgs& a, const MatvecPlan& p) {
  if (p.copied) return p.h > 16 ? launch_matvec<kM, kShift, 2, true, kRounded>(stream, maps, a, p) : launch_matvec<kM, kShift, 1, true, kRounded>(stream, maps, a, p);
  return p.h > 16 ? launch_matvec<kM, kShift, 2, false, kRounded>(stream, maps, a, p) : launch_matvec<kM, kShift, 1, false, kRounded>(stream, maps, a, p);
}
template <int kM, bool kRounded = false>
int launch_matvec(cudaStream_t stream, const MatvecMaps& maps, const W4GroupArgs& a, const MatvecPlan& p) {
  if (a.group == 32) return launch_matvec<kM, 5, kRounded>(stream, maps, a, p);
  if (a.group == 64) return launch_matvec<kM, 6, kRounded>(stream, maps, a, p);
  return launch_matvec<kM, 7, kRounded>(stream, maps, a, p);
}

int matvec(cudaStream_t stream, const W4GroupArgs& a, const MatvecPlan& p, bool rounded = false) {
  MatvecMaps maps;
  const char* const what = "linear_w4a16_group";
  int s = tc::encode_map(what, &maps.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.q, a.N, a.K / 2, 128, p.h, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s != kOk) return s;
  maps.scale = maps.zero = maps.q;
  if (p.copied) {
    const size_t groups = (a.K + a.group - 1) / a.group;
    s = tc::encode_map(what, &maps.scale, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, a.scale, a.N, groups, 8, p.h, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (s == kOk && a.zero) s = tc::encode_map(what, &maps.zero, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, a.zero, a.N, groups, 8, p.h, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (s != kOk) return s;
  }
  if (rounded) return launch_matvec<8, true>(stream, maps, a, p);
  switch (columns(a.M)) {
    case 1: return launch_matvec<1>(stream, maps, a, p);
    case 2: return launch_matvec<2>(stream, maps, a, p);
    case 4: return launch_matvec<4>(stream, maps, a, p);
    default: return launch_matvec<8>(stream, maps, a, p);
  }
}

}  // namespace

bool w4_rounded_fits(const W4GroupArgs& a, int sms) {
  MatvecPlan p;
  const long long groups = (a.K + a.group - 1) / a.group;
  return a.M <= kMaxRows && a.N * groups < (1ll << 31) && plan_matvec(a, sms, &p, true);  // (a row's first group is kept in 32 bits)
}

int w4_rounded_linear(cudaStream_t stream, const W4GroupArgs& a, int sms) {
  MatvecPlan p;
  RK_REQUIRE(a.M > 0 && a.M <= kMaxRows && plan_matvec(a, sms, &p, true), kShape, "4-bit product: unsupported shape");
  return matvec(stream, a, p, true);
}

// ---- more rows: the tensor-core skeleton of tc_packed.cuh, weights rounded to half, or as two halves each where the caller wants none
// rounded: two instructions more per two weights, twice the stores and products, and stages of 64 (96 rows of 10240 x 2560 20.1 us, 14.0 rounded;
// 24 of 65536 x 4096 88 and 59; 256 of 16384 x 4096 49 and 30; nine of 10240 x 2560 17.0 and 13.8).
namespace {

__device__ __forceinline__ void sts4(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

// A token's (channel's) results for the unit's rows to y, or to the unit's plane of partial sums; a warp's 32 channels are neighbours.
struct ProductEpilogue {
  static constexpr bool kExact = false;  // (the result is rounded to half, beside which the sum's error is small)
  static int scratch(int) { return 4 * 2048; }
  void* y;
  float* partial;  // [splits][rows][N], or nullptr
  int n_rows, N, epi;
  int n;
  size_t at;  // of the first row's result
  float* plane;
  uint32_t tile;  // this warp's part of the scratch
  __device__ __forceinline__ void begin(int channel, int r0, int, int split, unsigned char* scratch) {
    n = channel;
    at = static_cast<size_t>(r0) * N + n;
    plane = partial ? partial + static_cast<size_t>(split) * n_rows * N : nullptr;
    tile = smem_u32(scratch) + (threadIdx.x >> 5 & 3) * 2048;
  }
  // A lane has a channel of 32 rows; a warp's stores of one row each, 64 or 128 bytes, took 90 to 110 clocks apiece (11,000 of a
  // unit of 96 rows), so the rows change places in shared memory and leave 16 bytes a lane.
  __device__ __forceinline__ void chunk(int c, float (&z)[32], int here) {
    const int lane = threadIdx.x & 31;
    const size_t o = at + static_cast<size_t>(c) * N;
    if (plane || epi == kEpiF32) {
      float* const to = plane ? plane : static_cast<float*>(y);
      if (N % 4 == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) sts4(tile + 128 * i + 4 * lane, __float_as_uint(plane ? z[16 * h + i] : w4_epilogue(z[16 * h + i], epi)));
          __syncwarp();
          const int col = n - lane + 4 * (lane & 7);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = 4 * j + (lane >> 3);
            if (16 * h + i < here && col < N) *reinterpret_cast<uint4*>(to + o - n + col + static_cast<size_t>(16 * h + i) * N) = tc::lds16(tile + 512 * j + 16 * lane);
          }
        }
      } else if (n < N) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < here) to[o + static_cast<size_t>(i) * N] = plane ? z[i] : w4_epilogue(z[i], epi);
      }
    } else if (N % 8 == 0) {  // two rows of a channel share a word: 8 words are 8 channels of both
      if (epi == kEpiRelu2) {
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = w4_epilogue(z[i], kEpiRelu2);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) sts4(tile + 128 * i + 4 * lane, h2u(__floats2half2_rn(z[2 * i], z[2 * i + 1])));
      __syncwarp();
      const int col = n - lane + 8 * (lane & 3);
      half* const to = static_cast<half*>(y) + o - n + col;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = 2 * (8 * j + (lane >> 2));
        const uint4 a = tc::lds16(tile + 1024 * j + 32 * lane), b = tc::lds16(tile + 1024 * j + 32 * lane + 16);
        const uint4 even = {__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410), __byte_perm(b.x, b.y, 0x5410), __byte_perm(b.z, b.w, 0x5410)};
        const uint4 odd = {__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632), __byte_perm(b.x, b.y, 0x7632), __byte_perm(b.z, b.w, 0x7632)};
        if (i < here && col < N) *reinterpret_cast<uint4*>(to + static_cast<size_t>(i) * N) = even;
        if (i + 1 < here && col < N) *reinterpret_cast<uint4*>(to + static_cast<size_t>(i + 1) * N) = odd;
      }
    } else if (n < N) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < here) static_cast<half*>(y)[o + static_cast<size_t>(i) * N] = __float2half_rn(w4_epilogue(z[i], epi));
    }
  }
  __device__ __forceinline__ void end() {}
};

// The same where a long K may be added up in ranges.
struct RangedEpilogue : ProductEpilogue {
  static constexpr bool kExact = true;
};

// Adds the planes in order (the result does not depend on timing) and applies the epilogue: four channels per thread.
__global__ void __launch_bounds__(256) w4_reduce_kernel(const ProductEpilogue p, int splits) {
  pdl_wait();
  pdl_trigger();
  const size_t total = static_cast<size_t>(p.n_rows) * p.N, i = (static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= total) return;
  float4 v = *reinterpret_cast<const float4*>(p.partial + i);
  for (int s = 1; s < splits; ++s) {
    const float4 w = *reinterpret_cast<const float4*>(p.partial + s * total + i);
    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
  }
  const float e[4] = {w4_epilogue(v.x, p.epi), w4_epilogue(v.y, p.epi), w4_epilogue(v.z, p.epi), w4_epilogue(v.w, p.epi)};
  if (p.epi == kEpiF32)
    *reinterpret_cast<float4*>(static_cast<float*>(p.y) + i) = make_float4(e[0], e[1], e[2], e[3]);
  else
    *reinterpret_cast<uint2*>(static_cast<half*>(p.y) + i) = make_uint2(h2u(__floats2half2_rn(e[0], e[1])), h2u(__floats2half2_rn(e[2], e[3])));
}

// K ranges with the least time by this account, in clocks of an SM: 64 of K take what is done per weight and stage 380, or the tensor
// cores 2.35 a row; a unit's results take 25 a row, hidden under the next unit's products where there are two accumulators; the
// second kernel 3000, 200 a range and its traffic.  (64 rows of 1024 x 1024: 7.5 us whole, 6.5 in eight ranges, 7.9 in sixteen; 96
// rows of 10240 x 2560: 15.7 whole, 19.0 in two, 16.2 in three; 96 rows of 2560 x 10240: 43.7 whole, 15.7 in seven, 19.6 in nine,
// which is a second wave: with stages of 64, those of 128 take a tenth less of all of them.)  Exact weights, two halves each, have
// stages of 64, which take 600 to 760 clocks, and twice the products.  Their long sums go in ranges, because the tensor cores cut off of
// what they add: 4.8e-6 of a result's size for 256 additions, which the result's rounding to half covers up to kLongExact, but not
// in a K of any length.
constexpr int kLongExact = 16384, kExactRange = 8192;
tc::PackedShape many_rows_shape(int M, int K, int N, bool exact, size_t scratch_floats, int sms) {
  tc::PackedShape best = {};
  double least = 0;
  tc::PackedShape rows = {};
  const bool ranges = exact && K > kLongExact;
  tc::set_row_blocks(&rows, M, ranges ? 128 : tc::kMaxBlockRows);
  const int stage = tc::kBK * (exact ? 1 : tc::subs(rows.block_rows)), kblocks = (K + stage - 1) / stage;
  const size_t plane = static_cast<size_t>(M) * N;
  for (int want = 1; want <= 16 && want <= kblocks; ++want) {
    tc::PackedShape h = rows;
    h.tiles = (N + tc::kTileToks - 1) / tc::kTileToks;
    h.kb_per_split = (kblocks + want - 1) / want;
    h.splits = (kblocks + h.kb_per_split - 1) / h.kb_per_split;
    h.seg = ranges ? std::min(h.kb_per_split, kExactRange / stage) : h.kb_per_split;
    if (h.splits > 1 && (N % 4 != 0 || h.splits * plane > scratch_floats)) continue;
    const long long units = static_cast<long long>(h.tiles) * h.row_blocks * h.splits;
    const double waves = static_cast<double>((units + sms - 1) / sms), results = 25.0 * h.block_rows;
    double cost = waves * (h.kb_per_split * std::max(stage * (exact ? 8.0 : 6.0), stage * h.block_rows / (exact ? 13.5 : 27.0))) + (h.block_rows <= 128 ? 500 * waves + results : results * waves);
    if (h.splits > 1) cost += 3000 + 200 * h.splits + 4.0 * (h.splits + 1) * plane / (48.0 * sms);
    h.units = static_cast<int>(std::min<long long>(units, 0x7fffffff));
    if (best.units == 0 || cost < least) { least = cost; best = h; }
  }
  return best;
}

int many_rows(cudaStream_t stream, const W4GroupArgs& a, float* scratch, size_t scratch_bytes, int sms) {
  const tc::PackedShape h = many_rows_shape(a.M, a.K, a.N, a.exact, scratch ? scratch_bytes / sizeof(float) : 0, sms);
  RK_REQUIRE(h.units < 0x7fffffff, kShape, "linear_w4a16_group: too many rows");
  tc::Packed w;
  w.V = a.N; w.K = a.K; w.group = a.group; w.scale = a.scale; w.zero = a.zero;
  RangedEpilogue epi;
  epi.y = a.y; epi.partial = h.splits > 1 ? scratch : nullptr; epi.n_rows = a.M; epi.N = a.N; epi.epi = a.epi;
  const ProductEpilogue& plain = epi;
  const int s = a.exact ? tc::launch_packed<3>(stream, "linear_w4a16_group", a.x, a.q, w, h, epi, sms)
                        : tc::launch_packed<2>(stream, "linear_w4a16_group", a.x, a.q, w, h, plain, sms);
  if (s != kOk || h.splits == 1) return s;
  const size_t quads = static_cast<size_t>(a.M) * a.N / 4;
  RK_CUDA(launch_pdl(w4_reduce_kernel, dim3(static_cast<unsigned>((quads + 255) / 256)), dim3(256), 0, stream, plain, h.splits));
  RK_LAUNCH_CHECK("linear_w4a16_group reduction launch");
  return kOk;
}

}  // namespace

size_t w4_group_workspace(int M, int K, int N) {
  if (M <= kMaxRows || N % 4 != 0) return 0;
  int sms = 148;
  if (device_sms(&sms) != kOk) sms = 148;
  const size_t any = ~static_cast<size_t>(0) / 8;
  const int splits = std::max(many_rows_shape(M, K, N, false, any, sms).splits, many_rows_shape(M, K, N, true, any, sms).splits);
  return splits > 1 ? static_cast<size_t>(splits) * M * N * sizeof(float) : 0;
}

int w4_group_linear(cudaStream_t stream, const W4GroupArgs& a, void* workspace, size_t workspace_bytes) {
  const int s = check_shape("linear_w4a16_group", a.N, a.K, a.group);
  if (s != kOk) return s;
  RK_REQUIRE(a.M > 0 && a.x && a.q && a.scale && a.y, kBadArg, "linear_w4a16_group: bad argument");
  RK_REQUIRE(a.epi == kEpiNone || a.epi == kEpiRelu2 || a.epi == kEpiF32, kBadArg, "linear_w4a16_group: unknown epilogue %d", a.epi);
  RK_REQUIRE(((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.y) |
               reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0, kBadArg, "linear_w4a16_group: x, q, y and the workspace must be 16-byte aligned");
  RK_REQUIRE(static_cast<long long>(a.N) * ((a.K + a.group - 1) / a.group) < (1ll << 31), kShape, "linear_w4a16_group: too many groups");
  int sms = 0, status = device_sms(&sms);
  if (status != kOk) return status;
  W4GroupArgs one = a;
  MatvecPlan p;
  one.M = 1;
  const bool streamed = a.M <= kMaxRows && plan_matvec(one, sms, &p);
  if (!streamed) {
    W4GroupArgs b = a;
    b.exact = a.exact || a.M <= kMaxRows;  // (a K of which not one row fits into shared memory, some 58,000: no weight is rounded either)
    return many_rows(stream, b, static_cast<float*>(workspace), workspace_bytes, sms);
  }
  for (int m0 = 0; m0 < a.M;) {
    W4GroupArgs b = a;
    b.M = std::min(a.M - m0, kMaxRows);
    while (!plan_matvec(b, sms, &p)) b.M = (b.M + 1) / 2;  // (one row fits)
    b.x = a.x + static_cast<size_t>(m0) * a.K;
    b.y = static_cast<char*>(a.y) + static_cast<size_t>(m0) * a.N * (a.epi == kEpiF32 ? 4 : 2);
    if ((status = matvec(stream, b, p)) != kOk) return status;
    m0 += b.M;
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
