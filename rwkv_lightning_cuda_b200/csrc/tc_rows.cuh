// x W^T for rows of x and fp16 weights on the tensor cores, with whatever is done with the products left to the caller: the skeleton of
// the head product that keeps no logits (head_logprobs.cu).  tc_packed.cuh is the same for quantised weights.
//
// One CTA per SM walks units of 128 rows x up to 256 tokens (output channels).  The rows take the MMA's M side and the
// tokens its N side: a lane of tensor memory is then a row of x, and an epilogue thread sees its row's results one after the
// other without talking to any other thread.  Row blocks of a token tile follow one another, so that neighbouring CTAs share a
// tile of weights and it comes from HBM once.  Two accumulators: a unit's epilogue runs under the next one's products.
//
// Warp roles: 0 loads (TMA, 128-byte swizzle), 1 issues tcgen05.mma, 2..5 run the epilogue.  Every wait is bounded: one that runs
// out sets the device's failure word, every role leaves its loop, and the CTA frees its tensor memory and returns.
#pragma once

#include "tc_common.cuh"

namespace rk {
namespace tc {

constexpr int kRows = 128;  // rows of x per unit = MMA M
constexpr int kToks = 256;  // tokens per unit = MMA N, at most (Shape::toks)
constexpr int kRangeToks = 160;  // two accumulators and the sum of the ranges fit into tensor memory
constexpr int kMaxTiles = 8;
constexpr int kRowsThreads = 192;

struct Shape {
  int toks, tiles;  // tokens per unit, token tiles
  int row_blocks;   // blocks of 128 rows
  int units;
  int x_rows;       // rows of x that a block loads: all there are, in eights, up to 128 (the rest of the tile is not read out)
  int seg;          // K blocks that are added up in one accumulator: all, or kRangeK's where K is long (toks at most kRangeToks then)
  int ring;         // stages; a stage is a tile of x, then one of weights (set by launch_rows, like the next two)
  uint32_t x_bytes, tile_bytes;
};
struct Maps {
  CUtensorMap x, w;
};

// Epi: a copy per epilogue thread and unit; begin(row, n0, tokens), then chunk(c, z, here) for every 32 tokens n0 + c .. (here of them
// valid), then end(); rows() is the number of rows, beyond which a thread is not asked.
template <class Epi>
__global__ void __launch_bounds__(kRowsThreads, 1)
    tc_rows_kernel(const __grid_constant__ Maps maps, const int K, const int V, const Shape h, const Epi epilogue, int* timeout) {
  extern __shared__ unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kMaxTiles], empty[kMaxTiles], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t ring = (smem_u32(smem) + 1023u) & ~1023u;
  const int kblocks = (K + kBK - 1) / kBK;
  const uint32_t acc_cols = h.seg < kblocks ? kRangeToks : kToks, sum_at = 2 * kRangeToks;

  if (threadIdx.x == 0) {
    for (int i = 0; i < h.ring; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&acc_full[i]), 1);
      mbar_init(smem_u32(&acc_empty[i]), 4);
    }
    mbar_init(smem_u32(&drained), 1);
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
  const uint32_t tmem = uniform(tmem_slot);
  pdl_wait();
  pdl_trigger();

  auto wait = [&](uint64_t& bar, int parity) { return mbar_try_wait(smem_u32(&bar), parity) || wait_on(smem_u32(&bar), parity, &failed); };
  bool ok = true;
  int it = 0;  // K blocks so far, of the roles that count them
  if (warp == 0) {
    // ---- copies: as below the whole warp goes through the loop, one lane issues, and the next stage is asked for ahead
    const bool issuer = elect_one();
    int s = 0, phase = 1;
    bool free = true;  // the first round's stages are
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      const int r0 = u % h.row_blocks * kRows, n0 = u / h.row_blocks * h.toks;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!__all_sync(0xffffffffu, free) && !(ok = __all_sync(0xffffffffu, wait(empty[s], phase)))) break;
        if (issuer) {
          const uint32_t bar = smem_u32(&full[s]), dst = ring + s * h.tile_bytes;
          mbar_expect_tx(bar, 128 * (h.x_rows + h.toks));
          tma_2d(dst, &maps.x, bar, kb * kBK, r0);
          tma_2d(dst + h.x_bytes, &maps.w, bar, kb * kBK, n0);
        }
        ++it;
        if (++s == h.ring) { s = 0; phase ^= 1; }
        free = it < h.ring || mbar_test(smem_u32(&empty[s]), phase);
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ---- products: K blocks of 64 as four instructions into the unit's accumulator.  The whole warp goes through the loop, so that the
    // operands are computed in uniform registers, and one lane issues; the next stage's barrier is asked, without
    // waiting, before this one's products are issued.
    const uint32_t idesc = instruction_desc(h.toks);
    const bool issuer = elect_one();
    int n = 0, s = 0, phase = 0;
    bool ready = false;
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      for (int first = 0; first < kblocks && ok; first += h.seg, ++n) {
        if (n >= 2 && !(ok = __all_sync(0xffffffffu, wait(acc_empty[n & 1], ((n >> 1) - 1) & 1)))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + (n & 1) * acc_cols;
        for (int kb = first, upto = min(kblocks, first + h.seg); kb < upto; ++kb) {
          if (!ready && !(ok = __all_sync(0xffffffffu, wait(full[s], phase)))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t dx = tile_desc(ring + s * h.tile_bytes), dw = tile_desc(ring + s * h.tile_bytes + h.x_bytes);
          const uint32_t done = smem_u32(&empty[s]);
          if (++s == h.ring) { s = 0; phase ^= 1; }
          const bool next = mbar_test(smem_u32(&full[s]), phase);
          if (issuer) {
#pragma unroll
            for (int k4 = 0; k4 < kBK / 16; ++k4) mma(acc, dx + 2 * k4, dw + 2 * k4, idesc, kb != first || k4 != 0);
            commit(done);
          }
          ready = __all_sync(0xffffffffu, next);
        }
        if (ok && issuer) commit(smem_u32(&acc_full[n & 1]));
        __syncwarp();
      }
    }
  } else {
    // ---- epilogue: a thread owns a row of x, its TMEM lane, and takes the unit's tokens 32 at a time
    const int quad = warp & 3;
    int n = 0;
    for (int u = blockIdx.x; u < h.units && ok; u += gridDim.x) {
      const int r = u % h.row_blocks * kRows + quad * 32 + lane, n0 = u / h.row_blocks * h.toks, toks = min(h.toks, V - n0);
      const bool some = r - lane < epilogue.rows();  // (nothing to do for a warp beyond the last row)
      const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
      Epi epi = epilogue;
      for (int first = 0; first < kblocks; first += h.seg, ++n) {
        const bool last = first + h.seg >= kblocks;
        ok = __all_sync(0xffffffffu, wait(acc_full[n & 1], (n >> 1) & 1));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (last && r < epilogue.rows()) epi.begin(r, n0, toks);
        for (int c = 0; c < toks && some; c += 32) {
          float z[32];
          tmem_ld32(tmem + lanes + (n & 1) * acc_cols + c, z);
          if (first > 0) {
            float before[32];
            tmem_ld32(tmem + lanes + sum_at + c, before);
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] += before[i];
          }
          if (!last) tmem_st32(tmem + lanes + sum_at + c, z);
          else if (r < epilogue.rows()) epi.chunk(c, z, min(32, toks - c));
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&acc_empty[n & 1]));
      }
      if (ok && r < epilogue.rows()) epi.end();
    }
  }
  if (!ok) failed = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && failed && timeout) atomicOr(timeout, kTimeoutGemm);
  // One gave up: the copies in flight and the products issued end before the CTA does.
  if (failed && warp == 0 && lane == 0) {
    for (int i = max(it - h.ring, 0); i < it; ++i) settle(smem_u32(&full[i % h.ring]), (i / h.ring) & 1);
  }
  if (failed && warp == 1 && elect_one()) {
    commit(smem_u32(&drained));
    settle(smem_u32(&drained), 0);
  }
  __syncwarp();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <class Epi>
int launch_rows(cudaStream_t stream, const char* what, const half* x, int rows, const half* w, int K, int V, Shape h, const Epi& epi, int sms) {
  Maps maps;
  int s = encode_map(what, &maps.x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, x, rows, K, kBK, h.x_rows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s == kOk) s = encode_map(what, &maps.w, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, w, V, K, kBK, h.toks, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s != kOk) return s;
  h.x_bytes = (h.x_rows * 128 + 1023) & ~1023;
  h.tile_bytes = std::max<uint32_t>(h.x_bytes + h.toks * 128, kRows * 128);  // (the MMA reads 128 rows of x, whatever is there)
  h.ring = std::min<int>(kMaxTiles, (kSmemBytes - 1024) / h.tile_bytes);
  const auto kernel = tc_rows_kernel<Epi>;
  RK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes)));
  RK_CUDA(launch_pdl(kernel, dim3(std::min(h.units, sms)), dim3(kRowsThreads), 1024 + h.ring * static_cast<size_t>(h.tile_bytes), stream, maps, K, V, h,
                     epi, timeout_word_or_null()));
  RK_LAUNCH_CHECK(what);
  return kOk;
}

}  // namespace tc
}  // namespace rk
