// The head product with its softmax statistics: for every row of x [rows, K] the log probability of a given token under
// softmax(x W^T), the entropy and the log of the sum of exponentials, W [V, K] being the head matrix in any of the
// models' weight formats.  The logits (rows * V fp32) are never written: a tile of them is reduced to (m, s, t) per row
// where it is computed, and a second kernel merges a row's tiles (logprob.cuh).  fp16 operands, fp32 sums; int8 weights
// are exact integers with the channel's scale on the sum, 4-bit weights half((q - zero) * scale).
//
// Bound by the weights' bytes up to some 256 rows of fp16 weights, by the tensor cores above, and by the expansion of quantised ones in
// between (128 x 65536 x 4096 fp16: 94 us, 5.7 TB/s; 2048 rows: 800 to 940 us as the power cap lets it).  The products are tc_rows.cuh's (fp16 weights) and
// tc_packed.cuh's (quantised ones); here are their epilogues, which reduce a tile of logits to (m, s, t) per row, the merging of the
// tiles, and the route for a few rows.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "logprob.cuh"
#include "tc_packed.cuh"
#include "tc_rows.cuh"

namespace rk {
namespace {

constexpr int kMinToks = 128;  // the narrowest token tile
static_assert(kMinToks <= tc::kTileToks, "");

// A row's tokens of a unit: m, s and t over them, and the given token's logit where it is among them.  A thread has one row.
struct StatsEpilogue {
  float4* part;   // [tiles][rows]
  float* given;   // [rows]
  const int64_t* tokens;
  int n_rows, toks;
  int r, n0;
  int64_t id;
  SoftStats st;
  __device__ __forceinline__ int rows() const { return n_rows; }
  __device__ __forceinline__ void begin(int row, int first, int) {
    r = row;
    n0 = first;
    id = tokens ? tokens[row] : -1;
    st = SoftStats();
  }
  __device__ __forceinline__ void chunk(int c, float (&z)[32], int here) {
    if (here < 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) z[i] = i < here ? z[i] : -INFINITY;
    }
    if (id >= n0 + c && id < n0 + c + here) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (id == n0 + c + i) given[r] = z[i];
    }
    float m = st.m;
#pragma unroll
    for (int i = 0; i < 32; ++i) m = max_nan(m, z[i]);
    raise(st, m);
#pragma unroll
    for (int i = 0; i < 32; ++i) add(st, z[i]);
  }
  __device__ __forceinline__ void end() { part[static_cast<size_t>(n0 / toks) * n_rows + r] = make_float4(st.m, st.s, st.t, 0.f); }
};

// The same where a thread has one token and all rows: 32 tokens x 32 rows at a time go through shared memory, after which a lane has
// one row's 32 tokens; the four warps' parts of a row are merged at the end of the unit.
struct PackedStatsEpilogue {
  static constexpr int kPitch = 36, kWarpFloats = 32 * kPitch;
  static constexpr bool kExact = true;
  static int scratch(int block_rows) { return 4 * kWarpFloats * 4 + 4 * block_rows * 16; }
  float4* part;   // [tiles][rows]
  float* given;   // [rows]
  const int64_t* tokens;
  int n_rows, V;
  int token, r0, rows, lane, quad;
  int64_t id;       // asked of the next chunk's row, on its way since the chunk before
  float* box;       // this warp's [row][token]: written by columns, read by 16 bytes, neither with a conflict
  float4* parts;    // [warp][row of the block]
  __device__ __forceinline__ int64_t asked(int c) const { return tokens && c + lane < rows ? tokens[r0 + c + lane] : -1; }
  __device__ __forceinline__ void begin(int tok, int first, int rows_here, int, unsigned char* scratch) {
    token = tok;
    r0 = first;
    rows = rows_here;
    lane = threadIdx.x & 31;
    quad = (threadIdx.x >> 5) & 3;
    box = reinterpret_cast<float*>(scratch) + quad * kWarpFloats;
    parts = reinterpret_cast<float4*>(scratch + 4 * kWarpFloats * 4);
    id = asked(0);
  }
  __device__ __forceinline__ void chunk(int c, float (&z)[32], int here) {
    const int64_t at = id - (token - lane);  // relative to the warp's first token
    const bool mine = id >= 0 && at >= 0 && at < 32 && id < V;
    id = asked(c + 32);
#pragma unroll
    for (int i = 0; i < 32; ++i) box[i * kPitch + lane] = token < V ? z[i] : -INFINITY;
    __syncwarp();
    if (lane < here) {
      const float4* row = reinterpret_cast<const float4*>(box + lane * kPitch);
      float v[32];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 q = row[i];
        v[4 * i] = q.x;
        v[4 * i + 1] = q.y;
        v[4 * i + 2] = q.z;
        v[4 * i + 3] = q.w;
      }
      if (mine) given[r0 + c + lane] = box[lane * kPitch + at];
      SoftStats st[4];  // chains of their own
#pragma unroll
      for (int i = 0; i < 32; ++i) st[i & 3].m = max_nan(st[i & 3].m, v[i]);
      const float m = max_nan(max_nan(st[0].m, st[1].m), max_nan(st[2].m, st[3].m));
#pragma unroll
      for (int i = 0; i < 4; ++i) st[i].m = m;
#pragma unroll
      for (int i = 0; i < 32; ++i) add(st[i & 3], v[i]);
      parts[quad * rows + c + lane] =
          make_float4(m, (st[0].s + st[1].s) + (st[2].s + st[3].s), (st[0].t + st[1].t) + (st[2].t + st[3].t), 0.f);
    }
    __syncwarp();
  }
  __device__ __forceinline__ void end() {
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int tile = (token - lane) / tc::kTileToks;
    for (int r = threadIdx.x & 127; r < rows; r += 128) {
      SoftStats all;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 p = parts[w * rows + r];
        SoftStats b;
        b.m = p.x; b.s = p.y; b.t = p.z;
        all = merge(all, b);
      }
      part[static_cast<size_t>(tile) * n_rows + r0 + r] = make_float4(all.m, all.s, all.t, 0.f);
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the parts have been read
  }
};

// One CTA per row merges the row's tiles: a load or two per thread, all under way at once.
constexpr int kMergeThreads = 256;
__global__ void __launch_bounds__(kMergeThreads) head_merge_kernel(HeadLogprobsArgs a, int tiles) {
  __shared__ SoftStats warps[kMergeThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.x, t = threadIdx.x;
  SoftStats st;
  for (int i = t; i < tiles; i += kMergeThreads) {
    const float4 p = a.part[static_cast<size_t>(i) * a.rows + r];
    SoftStats b;
    b.m = p.x; b.s = p.y; b.t = p.z;
    st = merge(st, b);
  }
  st = warp_merge(st);
  if ((t & 31) == 0) warps[t >> 5] = st;
  __syncthreads();
  if (t != 0) return;
#pragma unroll
  for (int w = 1; w < kMergeThreads / 32; ++w) st = merge(st, warps[w]);
  const RowResult res = finish(st);
  if (a.entropy) a.entropy[r] = res.entropy;
  if (a.lse) a.lse[r] = res.lse;
  if (a.tokens) a.logprobs[r] = given_logprob(res, a.tokens[r], a.V, [&](int64_t) { return a.given[r]; });
}

// The token tile that lets the units come out in the fewest full rounds over the SMs (65536 tokens in tiles of 256 are 1.7 rounds
// of 148, in tiles of 224 two full ones); a unit is counted as its tokens and 32 more for its beginning and end.
tc::Shape head_shape(int rows, int V, int K, int sms) {
  tc::Shape best = {};
  long long least = -1;
  const bool whole = K <= tc::kWholeK;
  for (int toks = whole ? tc::kToks : tc::kRangeToks; toks >= kMinToks; toks -= 16) {
    tc::Shape h;
    h.toks = toks;
    h.tiles = (V + toks - 1) / toks;
    h.row_blocks = (rows + tc::kRows - 1) / tc::kRows;
    h.seg = (whole ? tc::kWholeK : tc::kRangeK) / tc::kBK;
    h.x_rows = std::min(tc::kRows, (rows + 7) & ~7);
    const long long units = static_cast<long long>(h.tiles) * h.row_blocks, cost = (units + sms - 1) / sms * (toks + 32);
    h.units = static_cast<int>(std::min<long long>(units, 0x7fffffff));
    if (least < 0 || cost < least) { least = cost; best = h; }
  }
  return best;
}

int merge_tiles(cudaStream_t stream, const HeadLogprobsArgs& a, int tiles) {
  RK_CUDA(launch_pdl(head_merge_kernel, dim3(a.rows), dim3(kMergeThreads), 0, stream, a, tiles));
  RK_LAUNCH_CHECK("head_logprobs merge launch");
  return kOk;
}

int head_f16(cudaStream_t stream, HeadLogprobsArgs a, int sms) {
  const tc::Shape h = head_shape(a.rows, a.V, a.K, sms);
  RK_REQUIRE(h.units < 0x7fffffff, kShape, "head_logprobs: too many rows");
  a.given = reinterpret_cast<float*>(a.part + static_cast<size_t>(h.tiles) * a.rows);
  StatsEpilogue epi;
  epi.part = a.part; epi.given = a.given; epi.tokens = a.tokens; epi.n_rows = a.rows; epi.toks = h.toks;
  const int s = tc::launch_rows(stream, "head_logprobs", a.x, a.rows, static_cast<const half*>(a.w), a.K, a.V, h, epi, sms);
  return s != kOk ? s : merge_tiles(stream, a, h.tiles);
}

template <int kFmt>
int head_packed(cudaStream_t stream, HeadLogprobsArgs a, int sms) {
  tc::PackedShape h = {};
  const bool whole = a.K <= tc::kWholeK;
  tc::set_row_blocks(&h, a.rows, whole ? tc::kMaxBlockRows : 128);
  h.tiles = (a.V + tc::kTileToks - 1) / tc::kTileToks;
  h.splits = 1;
  const int stage = tc::kBK * tc::subs(h.block_rows);
  h.kb_per_split = (a.K + stage - 1) / stage;
  h.seg = whole ? h.kb_per_split : tc::kRangeK / stage;
  const long long units = static_cast<long long>(h.tiles) * h.row_blocks;
  RK_REQUIRE(units < 0x7fffffff, kShape, "head_logprobs: too many rows");
  h.units = static_cast<int>(units);
  a.given = reinterpret_cast<float*>(a.part + static_cast<size_t>(h.tiles) * a.rows);
  tc::Packed w;
  w.V = a.V; w.K = a.K; w.group = a.group; w.scale = a.scale; w.zero = a.zero;
  PackedStatsEpilogue epi;
  epi.part = a.part; epi.given = a.given; epi.tokens = a.tokens; epi.n_rows = a.rows; epi.V = a.V;
  const int s = tc::launch_packed<kFmt>(stream, "head_logprobs", a.x, a.w, w, h, epi, sms);
  return s != kOk ? s : merge_tiles(stream, a, h.tiles);
}

}  // namespace

// Few rows: where the weight-streaming kernels read the weights at a better rate than the kernels above with their 128-row or
// 128-token tiles, the logits of so few rows are small.  Measured at 65536 tokens (K = 4096 unless said otherwise), this route
// against the other: 4-bit 55 us against 64 at eight rows (31 against 35 at two and K = 2048, 24 against 25 at eight and K = 1024, but
// 17 against 13 at eight rows of 32003 x 768); fp16 84 to 86 against 90 at one row, but 111 against 94 at four, and below 128 MB of
// weights the second pass takes what is saved.   int8 has no such route: 58 against 51 at four rows, 42 against 35 at two and
// K = 2560.
constexpr int kFewRowsF16 = 1, kFewRowsW4 = 8;
constexpr double kFewRowsBytes = 128e6;

size_t head_logprobs_workspace(int rows, int V) {
  const size_t tiles = (static_cast<size_t>(V) + kMinToks - 1) / kMinToks;
  const size_t need = static_cast<size_t>(rows) * (tiles * sizeof(float4) + sizeof(float));
  return rows <= kFewRowsW4 ? std::max(need, static_cast<size_t>(rows) * V * sizeof(float)) : need;
}

namespace {

// (K: what the products stage of x in shared memory.)
bool few_rows(const HeadLogprobsArgs& a, int sms) {
  if (a.fmt == 2) {
    W4GroupArgs w;
    w.M = a.rows; w.K = a.K; w.N = a.V; w.group = a.group; w.scale = a.scale; w.zero = a.zero;
    return a.rows <= kFewRowsW4 && w4_rounded_fits(w, sms);
  }
  return a.fmt == 0 && a.rows <= kFewRowsF16 && a.K <= 16384 && 2.0 * a.V * a.K >= kFewRowsBytes;
}
// Logits into the workspace, then their statistics.
int logits_then_stats(cudaStream_t stream, const HeadLogprobsArgs& a, float* logits, int sms) {
  int s;
  if (a.fmt == 2) {
    W4GroupArgs w;
    w.M = a.rows; w.K = a.K; w.N = a.V; w.group = a.group; w.x = a.x; w.q = static_cast<const uint8_t*>(a.w); w.scale = a.scale; w.zero = a.zero;
    w.epi = kEpiRawF32; w.y = logits;
    s = w4_rounded_linear(stream, w, sms);
  } else {
    LinearArgs l;
    l.M = a.rows; l.K = a.K; l.N = a.V; l.x = a.x; l.w = a.w; l.fmt = a.fmt; l.epi = kEpiRawF32; l.y = logits;
    l.after = !a.resident;  // (a caller may have made the weights just before)
    s = linear(stream, l);
  }
  if (s != kOk) return s;
  TokenLogprobsArgs t;
  t.rows = a.rows; t.V = a.V; t.logits = logits; t.ld = a.V; t.tokens = a.tokens; t.n_tokens = a.tokens ? 1 : 0;
  t.logprobs = a.logprobs; t.entropy = a.entropy; t.lse = a.lse;
  return token_logprobs(stream, t);
}

}  // namespace

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
  int sms = 0;
  const int status = device_sms(&sms);
  if (status != kOk) return status;
  if (few_rows(a, sms)) return logits_then_stats(stream, a, static_cast<float*>(workspace), sms);
  if (a.fmt == 1) return head_packed<1>(stream, a, sms);
  if (a.fmt == 2) return head_packed<2>(stream, a, sms);
  return head_f16(stream, a, sms);
}

}  // namespace rk
