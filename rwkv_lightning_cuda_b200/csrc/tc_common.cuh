// What the kernels on tcgen05.mma share: copies, barriers, descriptors, tensor memory, and the tensor maps.
#pragma once

#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tensormap.h"

namespace rk {
namespace tc {

constexpr int kBK = 64;  // halves per K block = one 128-byte swizzle row
constexpr uint32_t kTmemCols = 512;
constexpr size_t kSmemBytes = 225 * 1024;  // of 227 KB, beside the static part

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// A value that is the same in all lanes, in a form that the compiler knows to be.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Whether the phase is over, without waiting: a try_wait may hold its thread for microseconds where nothing more will come.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Bounded wait: out of line after the first try, and over as soon as another role has given up.
static __device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, const volatile int* failed) {
  for (uint32_t i = 0; i < kSpinLimit && !*failed; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}
// 32 columns of this warp's lanes, there when the call returns.
__device__ __forceinline__ void tmem_st32(uint32_t addr, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
        "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]),
        "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// The tensor cores cut off what they add to a running sum, so its error grows faster than the sum: logits of 4096 products came out
// 4.8e-6 of their size off (root mean square) and of 8192 9.5e-6, against 1.2e-6 at any K when ranges of 1024 are added up by themselves,
// each rounded to nearest into a sum beside the accumulators.  So the head does above kWholeK; at 65536 x 4096 that costs nothing at 128 fp16 rows,
// 4 % at 16 quantised ones, 8 % at 2048 fp16 ones (narrower tiles) and 16 % at 2048 quantised ones (128 rows to a block, not 256).
constexpr int kWholeK = 2048, kRangeK = 1024;
// The wait of a kernel that has given up for its own copies and products in flight: a fraction of a second at most.
static __device__ __noinline__ void settle(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 16); ++i)
    if (mbar_try_wait(bar, parity)) return;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
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
__device__ __forceinline__ uint32_t instruction_desc(int n) {  // fp16 operands, both K-major, fp32 sums: M = 128, N = n
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
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

}  // namespace tc
}  // namespace rk
