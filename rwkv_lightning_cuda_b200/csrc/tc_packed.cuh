// x W^T for rows of x and quantised weights on the tensor cores, with whatever is done with the products left to the caller: the skeleton
// of the 4-bit products of many rows (w4_group.cu) and of the quantised head product that keeps no logits (head_logprobs.cu).
//
// The weights take the MMA's M side, 128 tokens (output channels) per unit, as an operand in tensor memory: a thread expands a
// token's packed weights in registers and stores them to its lane, so that the fp16 weights never pass through shared
// memory.  (Expanded into shared memory, as the operand of the N side, a K block of 224 tokens took some 1000 clocks, of which
// its stores, the MMA's reads of both operands and the copies filled shared memory for 900.)  The N side are up to 256 rows of x.
// Units: 128 tokens x a block of rows x a range of K, the row blocks of a token tile one after the other.  A lane of tensor
// memory is a token, a column a row of x.  Up to 128 rows in a block there are two accumulators, and a unit's epilogue runs
// under the next one's products; with more there is one.
//
// Bound up to 128 rows by what the roles do per stage and weight: of 128 of K, some 800 clocks, in which the expansion of 4-bit weights
// has 300 to 350 issue slots of each scheduler; above by the tensor cores.  (24 rows of 65536 x 4096 in 59 us, with stages of 64
// in 65; 128 rows of 16384 x 4096 in 22; 256 in 30 us, 1.15 PFLOP/s.  Where a weight is
// two halves: 88, 32 and 49.)
//
// Warp roles: 0 loads packed tiles, 1 issues tcgen05.mma, 2..5 run the epilogue, 6 loads rows of x, 8..23 expand, four warps to a
// stage in turn.  Every wait is bounded: one that runs out sets the device's failure word, every role leaves its loop, and the
// CTA frees its tensor memory and returns.
#pragma once

#include "tc_common.cuh"

namespace rk {
namespace tc {

constexpr int kTileToks = 128;    // tokens per unit = MMA M
constexpr int kMaxBlockRows = 256;
constexpr int kTurns = 4;         // groups of four warps that expand stages in turn
constexpr int kMaxRing = 8;
constexpr int kPackedThreads = 256 + kTurns * 128;
constexpr int kOperandAt = 256;    // columns of tensor memory behind the accumulators: 256 for stages of expanded weights

// kSub: K blocks of 64 to a stage.  Two with up to 128 rows, where what every role does once per stage bounds; with more rows there is
// no room for four such stages.
__host__ __device__ constexpr int subs(int block_rows) { return block_rows <= 128 ? 2 : 1; }
// kFmt: 1 int8; 2 and 3 4-bit, the weights as halves, or (3) as two halves whose sum they are exactly, each multiplied with x.
// Two halves take twice the columns of a stage, so that stages are of 64 then.
template <int kFmt, int kSub> __host__ __device__ constexpr int stage_cols() { return kSub * kBK / 2 * (kFmt == 3 ? 2 : 1); }
template <int kFmt, int kSub> __host__ __device__ constexpr int raw_row() { return kSub * (kFmt == 1 ? kBK : kBK / 2); }  // bytes of a packed row of a stage

// int8 with a scale per token (applied to the sums), or 4 bits with scales and zeros per group: half((q - zero) * scale), or that and the
// half that is missing to (q - zero) * scale.
struct Packed {
  int V, K;
  int group;                 // 4 bits: 32, 64 or 128
  const half *scale, *zero;  // zero nullptr: 8
};
struct PackedShape {
  int tiles;                 // of 128 tokens
  int rows, row_blocks, block_rows;  // rows of x; block_rows: a multiple of 16, at most kMaxBlockRows
  int splits, kb_per_split;  // ranges of K and their stages of 64 subs(block_rows) (the last one may have fewer)
  int units;
  int seg;                   // stages that are added up in one accumulator: all of a unit's, or kRangeK's where K is long (block_rows at most 128 then)
  int ring, raws;            // stages of x and weights, and of packed tiles (set by launch_packed)
};
struct PackedMaps {
  CUtensorMap x, w;
};
struct PackedUnit {
  int r0, n0, split, kb0, kblocks;
};
__device__ __forceinline__ PackedUnit unit_of(const PackedShape& h, int u, int kblocks) {
  PackedUnit r;
  r.r0 = u % h.row_blocks * h.block_rows;
  u /= h.row_blocks;
  r.split = u % h.splits;
  r.n0 = u / h.splits * kTileToks;
  r.kb0 = r.split * h.kb_per_split;
  r.kblocks = min(h.kb_per_split, kblocks - r.kb0);
  return r;
}

// Eight 4-bit codes to eight halves half((q - zero) * scale): a nibble in the middle of a byte under the exponent of 1024 is 1024 + 16 q, so
// that a sixteenth of it less 64 + zero, in one fused multiply-add, is q - zero, and a second one multiplies and rounds.  64 + zero is
// itself rounded, to sixteenths for zeros up to 64; what that leaves over, times the scale, is the second one's addend: nothing for whole
// zeros, and otherwise at most a 32nd of the scale, whose own rounding puts a weight off by 2^-17 of the scale.  (q - zero so rounded
// is a half exactly for zeros from -32 on.)
struct Group4 {
  __half2 scale, sub, rest;  // twice each: s, -(64 + z) rounded, -(what z has beyond that) s
};
__device__ __forceinline__ __half2 zero_sub(__half2 z) { return __hsub2(__floats2half2_rn(-64.f, -64.f), z); }
__device__ __forceinline__ __half2 zero_rest(__half2 z, __half2 sub, __half2 scale) {
  return __hmul2(__hsub2(__hsub2(__floats2half2_rn(-64.f, -64.f), sub), z), scale);
}
__device__ __forceinline__ Group4 group4(uint32_t s2, uint32_t z2) {  // the group's scale and zero, twice each
  const __half2 s = *reinterpret_cast<const __half2*>(&s2), z = *reinterpret_cast<const __half2*>(&z2), sub = zero_sub(z);
  return {s, sub, zero_rest(z, sub, s)};
}
// Half i of eight, twice.
__device__ __forceinline__ uint32_t pick(const uint4& v, int i) {
  const uint32_t lo = i & 2 ? v.y : v.x, hi = i & 2 ? v.w : v.z;
  return __byte_perm(i & 4 ? hi : lo, 0u, i & 1 ? 0x3232 : 0x1010);
}
// The constants are the caller's registers: as literals, mask and bias of the AND-OR would not fit into one instruction.
struct Expand4 {
  uint32_t nibbles, bias;  // 0x00f000f0, 0x64006400
  __half2 mul;             // 1/16 twice
  // Byte b's codes as 1024 + 16 q; up: the word shifted up by a nibble.
  __device__ __forceinline__ __half2 pair(uint32_t up, uint32_t w, int b) const {
    const uint32_t both = __byte_perm(up, w, 0x4400u + 0x1111u * b);
    uint32_t p;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p) : "r"(both), "r"(nibbles), "r"(bias));
    return *reinterpret_cast<const __half2*>(&p);
  }
};
__device__ __forceinline__ uint4 expand4(uint32_t w, const Group4& g, const Expand4& e) {
  uint32_t h[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const __half2 v = __hfma2(__hfma2(e.pair(w << 4, w, b), e.mul, g.sub), g.scale, g.rest);
    h[b] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}
// The same and what the rounding took off.  With a whole zero (q - zero) * scale is a multiple of the scale's last place, and so is what it is
// off its rounding: a half, which the fused multiply-add gives exactly.  With others the low half is off by up to 2^-17 of the scale more.
__device__ __forceinline__ void expand4(uint32_t w, const Group4& g, const Expand4& e, uint4* high, uint4* low) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const __half2 d = __hfma2(e.pair(w << 4, w, b), e.mul, g.sub), v = __hmul2(d, g.scale), o = __hadd2(__hfma2(d, g.scale, __hneg2(v)), g.rest);
    h[b] = *reinterpret_cast<const uint32_t*>(&v);
    l[b] = *reinterpret_cast<const uint32_t*>(&o);
  }
  *high = make_uint4(h[0], h[1], h[2], h[3]);
  *low = make_uint4(l[0], l[1], l[2], l[3]);
}
// Four int8 codes to four halves, exactly: code + 128 under the exponent of 1024, less 1152.
__device__ __forceinline__ uint2 expand8(uint32_t w) {
  const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
  const uint32_t t = w ^ 0x80808080u;
  uint32_t lo = __byte_perm(t, 0x64646464u, 0x4140), hi = __byte_perm(t, 0x64646464u, 0x4342);
  const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&lo), bias), b = __hsub2(*reinterpret_cast<__half2*>(&hi), bias);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Epi: a copy per epilogue thread and unit, all 128 of which are asked; begin(token, r0, rows, split, scratch) while the products are under
// way, then chunk(c, z, here) for every 32 rows r0 + c .. (here of them valid), where z[i] is the result of row r0 + c + i, then end();
// scratch: Epi::scratch(block_rows) bytes of shared memory; Epi::kExact: a long K may be added up in ranges.  The threads may meet at barrier 1.
template <int kFmt, int kSub, bool kRanges, class Epi>
__global__ void __launch_bounds__(kPackedThreads, 1)
    tc_packed_kernel(const __grid_constant__ PackedMaps maps, const Packed a, const PackedShape h, const Epi epilogue, int* timeout) {
  extern __shared__ unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kMaxRing], empty[kMaxRing], raw_full[kMaxRing], raw_empty[kMaxRing], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  constexpr int kStage = kSub * kBK;  // weights of a token per stage
  constexpr bool kTwo = kFmt == 3;    // two halves to a weight
  constexpr int kCols = stage_cols<kFmt, kSub>();
  static_assert(kTurns * kCols <= static_cast<int>(kTmemCols) - kOperandAt, "four stages of expanded weights at least");
  constexpr uint32_t kRawRow = raw_row<kFmt, kSub>(), kRawBytes = kTileToks * kRawRow;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t x_sub = h.block_rows * 128, x_bytes = kSub * x_sub, ring = (smem_u32(smem) + 1023u) & ~1023u, raw_ring = ring + h.ring * x_bytes;
  const int kblocks = (a.K + kStage - 1) / kStage;
  const int accs = h.block_rows <= (kRanges ? 64 : 128) ? 2 : 1, seg = kRanges ? h.seg : kblocks;
  constexpr int acc_cols = kRanges ? 64 : 128;
  constexpr uint32_t kSumAt = 128;  // of the ranges of a long K, behind the accumulators

  if (threadIdx.x == 0) {
    for (int i = 0; i < h.ring; ++i) {
      mbar_init(smem_u32(&full[i]), 1 + 4);  // the rows of x, and the four warps' parts of the weights
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < h.raws; ++i) {
      mbar_init(smem_u32(&raw_full[i]), 1);
      mbar_init(smem_u32(&raw_empty[i]), 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&acc_full[i]), 1);
      mbar_init(smem_u32(&acc_empty[i]), 4);
    }
    mbar_init(smem_u32(&drained), 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.w) : "memory");
  if (warp == 6 && lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.x) : "memory");
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = uniform(tmem_slot);
  pdl_wait();
  pdl_trigger();

  auto wait = [&](uint64_t& bar, int parity) { return mbar_try_wait(smem_u32(&bar), parity) || wait_on(smem_u32(&bar), parity, &failed); };
  bool ok = true;
  int it = 0;  // stages so far, of the roles that count them
  // Copies: as below the whole warp goes through the loop, one lane issues, and the next stage is asked for ahead.  (One lane alone took
  // 480 to 560 clocks a K block, more than anything else.)
  auto fetch = [&](uint64_t* filled, uint64_t* used, int stages, uint32_t bytes, auto&& copy) {
    const bool issuer = elect_one();
    int s = 0, phase = 1;
    bool free = true;  // the first round's stages are
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      const PackedUnit un = unit_of(h, u, kblocks);
      for (int kb = un.kb0; kb < un.kb0 + un.kblocks; ++kb) {
        if (!__all_sync(0xffffffffu, free) && !(ok = __all_sync(0xffffffffu, wait(used[s], phase)))) break;
        if (issuer) {
          const uint32_t bar = smem_u32(&filled[s]);
          mbar_expect_tx(bar, bytes);
          copy(s, bar, kb, un);
        }
        ++it;
        if (++s == stages) { s = 0; phase ^= 1; }
        free = it < stages || mbar_test(smem_u32(&used[s]), phase);
        __syncwarp();
      }
    }
  };
  if (warp == 0) {
    fetch(raw_full, raw_empty, h.raws, kRawBytes,
          [&](int s, uint32_t bar, int kb, const PackedUnit& un) { tma_2d(raw_ring + s * kRawBytes, &maps.w, bar, kb * kRawRow, un.n0); });
  } else if (warp == 6) {
    fetch(full, empty, h.ring, x_bytes, [&](int s, uint32_t bar, int kb, const PackedUnit& un) {
#pragma unroll
      for (int i = 0; i < kSub; ++i) tma_2d(ring + s * x_bytes + i * x_sub, &maps.x, bar, kb * kStage + i * kBK, un.r0);
    });
  } else if (warp == 1) {
    // ---- products: four instructions for each 64 of K into the unit's accumulator.  The whole warp goes through the loop, so that the
    // operands are computed in uniform registers, and one lane issues (700 clocks a K block when one lane did all of it, between
    // the instructions of 16 other warps); the next stage's barrier is asked, without waiting, before this one's products are issued.
    const uint32_t idesc = instruction_desc(h.block_rows);
    const bool issuer = elect_one();
    int n = 0, s = 0, phase = 0;
    bool ready = false;
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      const int here = unit_of(h, u, kblocks).kblocks;
      for (int first = 0; first < here && ok; first += seg, ++n) {
        const int acc = accs == 2 ? n & 1 : 0, use = accs == 2 ? n >> 1 : n, upto = min(here, first + seg);
        if (use >= 1 && !(ok = __all_sync(0xffffffffu, wait(acc_empty[acc], (use - 1) & 1)))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = first; kb < upto; ++kb) {
          if (!ready && !(ok = __all_sync(0xffffffffu, wait(full[s], phase)))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dx = tile_desc(ring + s * x_bytes);
          const uint32_t dw = tmem + kOperandAt + s * kCols, done = smem_u32(&empty[s]);
          if (++s == h.ring) { s = 0; phase ^= 1; }
          const bool next = mbar_test(smem_u32(&full[s]), phase);
          if (issuer) {
#pragma unroll
            for (int k = 0; k < kStage / 16; ++k) {
              const uint64_t dxk = dx + (k / 4) * (x_sub >> 4) + 2 * (k % 4);
              mma_from_tmem(tmem + acc * acc_cols, dw + 8 * k, dxk, idesc, kb != first || k != 0);
              if (kTwo) mma_from_tmem(tmem + acc * acc_cols, dw + kCols / 2 + 8 * k, dxk, idesc, 1);
            }
            commit(done);
          }
          ready = __all_sync(0xffffffffu, next);
        }
        if (ok && issuer) commit(smem_u32(&acc_full[acc]));
        __syncwarp();
      }
    }
  } else if (warp >= 2 && warp < 6) {
    // ---- epilogue: a thread owns a token, its TMEM lane, and takes the unit's rows 32 at a time
    const int quad = warp & 3;
    unsigned char* const scratch = smem + (raw_ring - smem_u32(smem)) + h.raws * kRawBytes;
    int n = 0;
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      const PackedUnit un = unit_of(h, u, kblocks);
      const int token = un.n0 + quad * 32 + lane, rows = min(h.block_rows, h.rows - un.r0);
      const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
      const float scale = kFmt == 1 && token < a.V ? __half2float(a.scale[token]) : 1.f;
      Epi epi = epilogue;
      epi.begin(token, un.r0, rows, un.split, scratch);
      for (int first = 0; first < un.kblocks; first += seg, ++n) {
        const int acc = accs == 2 ? n & 1 : 0, use = accs == 2 ? n >> 1 : n;
        const bool last = !kRanges || first + seg >= un.kblocks;
        // (asleep: these four warps' polling of a wait this long cost the expansion a quarter of its time)
        for (uint32_t i = 0; i < kSpinLimit && !(ok = mbar_test(smem_u32(&acc_full[acc]), use & 1)) && !failed; ++i) __nanosleep(100);
        {  // all four warps stay or leave together: an epilogue may have them meet at a barrier
          uint32_t all;
          asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\tbar.red.and.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(all) : "r"(static_cast<uint32_t>(ok)) : "memory");
          ok = all != 0;
        }
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int c = 0; c < rows; c += 32) {
          float z[32];
          tmem_ld32(tmem + lanes + acc * acc_cols + c, z);
          if (kRanges && first > 0) {
            float before[32];
            tmem_ld32(tmem + lanes + kSumAt + c, before);
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] += before[i];
          }
          if (!last) {
            tmem_st32(tmem + lanes + kSumAt + c, z);
            continue;
          }
          if (kFmt == 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] *= scale;
          }
          epi.chunk(c, z, min(32, rows - c));
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&acc_empty[acc]));
      }
      if (ok) epi.end();
    }
  } else if (warp >= 8) {
    // ---- expansion: a thread owns a token of the tile, all its weights of a stage; four warps take every fourth stage.  A packed row of
    // 128 (64, 32) bytes has its 16-byte chunk c at c ^ (r & 7) (c ^ (r / 2 & 3), c ^ (r / 4 & 1)), the swizzles of such rows, so that
    // no two lanes of a quarter warp meet in a bank.  (No barrier's phase is missed by taking every fourth stage: the packed ring is a
    // multiple of four; and in the other ring of T >= 4 places block i waits until block i - T is used, when block i - 4 has shown that
    // i - 4 - T is, so the fill of this place before that one, i - 2 T, is too.)
    const int r = threadIdx.x & 127, turn = (warp - 8) >> 2;
    const uint32_t raw = raw_ring + r * kRawRow, raw_swz = (kRawRow == 32 ? (r >> 2) & 1 : kRawRow == 64 ? (r >> 1) & 3 : r & 7) << 4;
    const uint32_t operand = tmem + kOperandAt + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's 32 lanes
    const int shift = a.group == 32 ? 5 : a.group == 64 ? 6 : 7, groups = (a.K + a.group - 1) >> shift;
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
    auto load_runs = [&](int kb) {  // a stage's runs of 32 weights into the first halves
      auto run = [&](const uint16_t* of, int i) {
        return of[min((kb * kStage + 64 * i) >> shift, groups - 1)] | (static_cast<uint32_t>(of[min((kb * kStage + 64 * i + 32) >> shift, groups - 1)]) << 16);
      };
      sc_next.x = run(sp, 0);
      if (kSub == 2) sc_next.y = run(sp, 1);
      if (zp) {
        ze_next.x = run(zp, 0);
        if (kSub == 2) ze_next.y = run(zp, 1);
      }
    };
    auto eight_of = [&](int kb) { return (kb * kStage) >> (shift + 3); };
    const uint32_t none = ring >> 30;  // 0, which the compiler does not know, so that the constants stay in registers
    const uint32_t mul = 0x2c002c00u + none;
    const Expand4 e4 = {0x00f000f0u + none, 0x64006400u + none, *reinterpret_cast<const __half2*>(&mul)};
    // A stage is handed over when this warp has the next one's weights in registers: the stores end under those loads.  (A packed tile
    // waits for nothing later than the stage four before it, and a place for the one T before, so no wait closes a circle.)
    int stored = -1;
    auto hand_over = [&](int stage) {
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(smem_u32(&full[stage]));
    };
    int rs = turn, raw_phase = 0, s = turn, phase = 0;
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      const PackedUnit un = unit_of(h, u, kblocks);
      const int row = min(un.n0 + r, a.V - 1), kb_end = un.kb0 + un.kblocks;
      int kb = un.kb0 + ((turn - it) & (kTurns - 1));
      int block = -1, ahead = -1;
      if (kFmt != 1 && kb < kb_end) {
        sp = reinterpret_cast<const uint16_t*>(a.scale) + static_cast<size_t>(row) * groups;
        if (a.zero) zp = reinterpret_cast<const uint16_t*>(a.zero) + static_cast<size_t>(row) * groups;
        if (eights) load8(ahead = eight_of(kb));
        else load_runs(kb);
      }
      for (; kb < kb_end; kb += kTurns) {
        const bool first_round = it + kb - un.kb0 < h.ring;
        if (kFmt != 1 && (!eights || ahead != block)) {
          sc = sc_next;
          ze = ze_next;
          block = ahead;
        }
        if (kFmt != 1 && eights && eight_of(kb + kTurns) != block) load8(ahead = eight_of(kb + kTurns));
        ok = __all_sync(0xffffffffu, wait(raw_full[rs], raw_phase));
        if (!ok) break;
        const uint32_t src = raw + rs * kRawBytes;
        Group4 g;
#pragma unroll
        for (int sub = 0; sub < kSub; ++sub) {
          constexpr int kLoads = kFmt == 1 ? 4 : 2;
          uint4 q[kLoads];
#pragma unroll
          for (int c = 0; c < kLoads; ++c) q[c] = lds16(src + ((16 * (kLoads * sub + c)) ^ raw_swz));
          if (sub == 0) {
            if (stored >= 0) hand_over(stored);
            ok = __all_sync(0xffffffffu, first_round || wait(empty[s], phase ^ 1));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // 32 weights at a time: more would take too many registers
            uint32_t o[16], rest[16];  // (rest: kTwo)
            if (kFmt == 1) {
              const uint32_t w[8] = {q[2 * c].x, q[2 * c].y, q[2 * c].z, q[2 * c].w, q[2 * c + 1].x, q[2 * c + 1].y, q[2 * c + 1].z, q[2 * c + 1].w};
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint2 p = expand8(w[i]);
                o[2 * i] = p.x;
                o[2 * i + 1] = p.y;
              }
            } else {
              const int run = 2 * sub + c, k = kb * kStage + 32 * run;
              if (run == 0 || shift == 5 || (shift == 6 && c == 0)) {
                const int i = eights ? (k >> shift) & 7 : run;
                g = group4(pick(sc, i), pick(ze, i));
              }
              if (run > 0 && k >= a.K) g.scale = g.rest = __floats2half2_rn(0.f, 0.f);  // behind K: code 0, which may stand for an infinite weight
              const uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint4 p, r = make_uint4(0u, 0u, 0u, 0u);
                if (kTwo) expand4(w[j], g, e4, &p, &r);
                else p = expand4(w[j], g, e4);
                o[4 * j] = p.x;
                o[4 * j + 1] = p.y;
                o[4 * j + 2] = p.z;
                o[4 * j + 3] = p.w;
                rest[4 * j] = r.x;
                rest[4 * j + 1] = r.y;
                rest[4 * j + 2] = r.z;
                rest[4 * j + 3] = r.w;
              }
            }
            tmem_st16(operand + s * kCols + 32 * sub + 16 * c, o);
            if (kTwo) tmem_st16(operand + s * kCols + kCols / 2 + 32 * sub + 16 * c, rest);
          }
        }
        if (!ok) break;
        // The packed tile is given back only now that its words have gone into the stores above: an arrival right behind the loads did
        // not wait for them, and the next tile came in under them.
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&raw_empty[rs]));
        if (kFmt != 1 && !eights && kb + kTurns < kb_end) load_runs(kb + kTurns);  // under way until this thread's next turn
        stored = s;
        rs += kTurns;
        if (rs >= h.raws) { rs -= h.raws; raw_phase ^= 1; }
        s += kTurns;
        if (s >= h.ring) { s -= h.ring; phase ^= 1; }
      }
      it += un.kblocks;
    }
    if (stored >= 0 && ok) hand_over(stored);
  }
  if (!ok) failed = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && failed && timeout) atomicOr(timeout, kTimeoutGemm);
  // One gave up: the copies in flight and the products issued end before the CTA does.
  if (failed && (warp == 0 || warp == 6) && lane == 0) {
    for (int i = max(it - (warp ? h.ring : h.raws), 0); i < it; ++i) settle(smem_u32(warp ? &full[i % h.ring] : &raw_full[i % h.raws]), (i / (warp ? h.ring : h.raws)) & 1);
  }
  if (failed && warp == 1 && elect_one()) {
    commit(smem_u32(&drained));
    settle(smem_u32(&drained), 0);
  }
  __syncwarp();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// Blocks of rows as equal as sixteens allow, at most `most` each.
inline void set_row_blocks(PackedShape* h, int rows, int most = kMaxBlockRows) {
  h->rows = rows;
  h->row_blocks = (rows + most - 1) / most;
  h->block_rows = ((rows + h->row_blocks - 1) / h->row_blocks + 15) & ~15;
}

template <int kFmt, int kSub, bool kRanges, class Epi>
int launch_stages(cudaStream_t stream, const char* what, const half* x, const void* w, const Packed& a, PackedShape h, const Epi& epi, int sms) {
  constexpr int kRawRow = raw_row<kFmt, kSub>(), kRawBytes = kTileToks * kRawRow, kMost = std::min<int>(kMaxRing, (kTmemCols - kOperandAt) / stage_cols<kFmt, kSub>());
  PackedMaps maps;
  int s = encode_map(what, &maps.x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x, h.rows, a.K, kBK, h.block_rows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s == kOk)
    s = encode_map(what, &maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, a.V, kFmt == 1 ? a.K : a.K / 2, kRawRow, kTileToks,
                   kRawRow == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : kRawRow == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
  if (s != kOk) return s;
  const int x_bytes = kSub * h.block_rows * 128, scratch = Epi::scratch(h.block_rows), budget = static_cast<int>(kSmemBytes) - 1024 - scratch;
  for (h.raws = kMaxRing;; h.raws = kTurns) {  // the rows of x go first: four stages of them at least
    h.ring = std::min(kMost, (budget - h.raws * kRawBytes) / x_bytes);
    if (h.ring >= kTurns || h.raws == kTurns) break;
  }
  const size_t smem = 1024 + scratch + static_cast<size_t>(h.ring) * x_bytes + static_cast<size_t>(h.raws) * kRawBytes;
  RK_REQUIRE(h.ring >= kTurns, kShape, "%s: no room for four stages", what);
  const auto kernel = tc_packed_kernel<kFmt, kSub, kRanges, Epi>;
  RK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes)));
  RK_CUDA(launch_pdl(kernel, dim3(std::min(h.units, sms)), dim3(kPackedThreads), smem, stream, maps, a, h, epi, timeout_word_or_null()));
  RK_LAUNCH_CHECK(what);
  return kOk;
}
template <int kFmt, class Epi>
int launch_packed(cudaStream_t stream, const char* what, const half* x, const void* w, const Packed& a, const PackedShape& h, const Epi& epi, int sms) {
  if constexpr (Epi::kExact)
    if (h.seg < h.kb_per_split) return launch_stages<kFmt, kFmt == 3 ? 1 : 2, true>(stream, what, x, w, a, h, epi, sms);
  if constexpr (kFmt == 3) return launch_stages<kFmt, 1, false>(stream, what, x, w, a, h, epi, sms);
  else return subs(h.block_rows) == 2 ? launch_stages<kFmt, 2, false>(stream, what, x, w, a, h, epi, sms) : launch_stages<kFmt, 1, false>(stream, what, x, w, a, h, epi, sms);
}

}  // namespace tc
}  // namespace rk
