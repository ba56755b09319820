// Log probabilities of given tokens over logits [rows, V], with the entropy, the log of the sum of exponentials and the
// likeliest alternatives of every row (definitions and corner cases: logprob.cuh).
//
// Bound by reading the logits once; a single row by latency.  A row goes to one CTA, or to the CTAs of a cluster when
// there are too few rows to fill the GPU: each takes a contiguous part, and the first one merges the others' statistics
// and alternatives out of their shared memory, so there is no scratch, no second launch and no atomic whose order could show.
// A thread keeps 16 logits in registers and the next 16 under way, and its own running maximum (one rescaling per 16).
//
// Alternatives without a second pass: after the first 16 logits per thread the k-th largest of the maxima of disjoint groups
// of four threads is a lower bound of the k-th largest logit; whatever reaches it goes to a list in shared memory.  The
// bound is raised after 2, 4 and 8 steps, so some 5 k of the logits are ever listed, and the list is put in order by
// counting, for every entry, the larger ones.  A row that fills the list (thousands of equal logits, rows sorted upwards)
// takes k passes over its part instead.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "logprob.cuh"

namespace cg = cooperative_groups;

namespace rk {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kCtasPerSm = 4;
constexpr int kGroups = kThreads / 4;  // groups of four lanes whose maxima bound the k-th largest logit
constexpr int kList = 1536;            // candidates a part can list
constexpr int kMaxParts = 8;           // portable cluster size

using Key = unsigned long long;

// Orders (value, id) pairs as whole numbers: larger value first, then the lower id.  -0 counts as +0.  Never 0 for a number.
__device__ __forceinline__ Key rank_key(float v, int id) {
  const uint32_t u = __float_as_uint(v + 0.f);
  const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<Key>(o) << 32) | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ int key_id(Key k) { return static_cast<int>(~static_cast<uint32_t>(k)); }
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

// 16 bytes that are read once.  (Not the read-only path: the kernel may have been launched before its predecessor wrote them.)
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// A row as 16-byte vectors: it may start `lead` elements into the first one and end inside the last one; what is outside
// reads as -inf, a token that counts for nothing.
template <typename T>
struct RowView {
  static constexpr int kVec = 16 / sizeof(T);
  const T* z;  // the row's first logit
  int V, lead, vecs;
  __device__ __forceinline__ RowView(const T* row, int n) : z(row), V(n) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kVec);
    vecs = static_cast<int>((static_cast<long long>(n) + lead + kVec - 1) / kVec);
  }
  __device__ __forceinline__ int column(int vec) const { return vec * kVec - lead; }
  __device__ __forceinline__ uint4 load(int vec) const {
    const int c = column(vec);
    if (c >= 0 && c <= V - kVec) return load16(z + c);
    union { uint4 q; T e[kVec]; } u;
#pragma unroll
    for (int i = 0; i < kVec; ++i) u.e[i] = c + i >= 0 && c + i < V ? z[c + i] : static_cast<T>(-INFINITY);
    return u.q;
  }
};
template <typename T>
__device__ __forceinline__ uint4 nothing() {  // a vector of -inf
  const uint32_t w = sizeof(T) == 4 ? 0xff800000u : 0xfc00fc00u;
  return make_uint4(w, w, w, w);
}
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
  v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = h2f2(w[i]);
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(half v) { return __half2float(v); }

struct Shared {
  SoftStats stats[kWarps];
  float groups[kGroups];
  float bound[2];                        // of this refresh and the one before (threads may still read that)
  int count;
  Key best[kWarps];
  Key top[kMaxTopLogprobs];              // this part's alternatives, best first, 0: none
  Key list[kList];
  Key merged[kMaxParts * kMaxTopLogprobs];
  RowResult result;
};

// The k largest of n distinct keys (0: no key), in order.
__device__ __forceinline__ void order(const Key* keys, int n, int k, Key* out) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const Key mine = keys[i];
    int larger = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) larger += keys[j] > mine ? 1 : 0;
    if (mine != 0 && larger < k) out[larger] = mine;
  }
}

template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) token_logprobs_kernel(const TokenLogprobsArgs a, const int parts) {
  constexpr int kVec = RowView<T>::kVec, kVecs = 16 / kVec;  // 16 logits per thread and step
  __shared__ Shared s;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, threads = blockDim.x;
  const int r = blockIdx.x / parts, part = blockIdx.x - r * parts;
  pdl_wait();
  pdl_trigger();
  const RowView<T> row(static_cast<const T*>(a.logits) + static_cast<long long>(r) * a.ld, a.V);
  const int per = (row.vecs + parts - 1) / parts;
  const int begin = min(part * per, row.vecs), end = min(begin + per, row.vecs);
  const int step = threads * kVecs, steps = (end - begin + step - 1) / step;
  auto fetch = [&](int i, uint4 (&q)[kVecs]) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int vec = begin + i * step + j * threads + t;
      q[j] = vec < end ? row.load(vec) : nothing<T>();
    }
  };
  uint4 next[kVecs];
  fetch(0, next);
  int64_t id = -1;  // the first tokens' logits are requested with the row's own
  float given = 0.f;
  if (part == 0 && t < a.n_tokens) {
    id = a.tokens[static_cast<size_t>(r) * a.n_tokens + t];
    if (id >= 0 && id < a.V) given = to_float(row.z[id]);
  }
  if (kTop) {
    if (t == 0) s.count = 0;
    if (t < a.top_k) s.top[t] = 0;
  }

  SoftStats st;
  float bound = -INFINITY;
  int refresh = 0;
  for (int i = 0; i < steps; ++i) {
    uint4 q[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) q[j] = next[j];
    if (i + 1 < steps) fetch(i + 1, next);
    float v[kVecs][kVec];
    float m = st.m, here = -INFINITY;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      unpack(q[j], v[j]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) here = max_nan(here, v[j][e]);
    }
    m = max_nan(m, here);
    if (m != st.m) raise(st, m);
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int e = 0; e < kVec; ++e) add(st, v[j][e]);
    if (kTop) {
      if ((i & (i + 1)) == 0 && i < 8) {  // steps 0, 1, 3, 7: the bound
        float g = fmaxf(st.m, __shfl_xor_sync(0xffffffffu, st.m, 1));
        g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
        if ((lane & 3) == 0) s.groups[t >> 2] = g;
        refresh ^= 1;
        if (t == 0) s.bound[refresh] = -INFINITY;
        __syncthreads();
        const int n = threads >> 2;
        if (t < n) {
          const float mine = s.groups[t];
          int before = 0;
          for (int j = 0; j < n; ++j) before += s.groups[j] > mine || (s.groups[j] == mine && j < t) ? 1 : 0;
          if (before == a.top_k - 1) s.bound[refresh] = mine > -FLT_MAX ? mine : -INFINITY;  // (-FLT_MAX: a group with nothing but masked tokens)
        }
        __syncthreads();
        bound = s.bound[refresh];
      }
      if (here >= bound && here > -INFINITY) {
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (v[j][e] >= bound && v[j][e] > -INFINITY) {
              const int slot = atomicAdd(&s.count, 1);
              if (slot < kList) s.list[slot] = rank_key(v[j][e], row.column(begin + i * step + j * threads + t) + e);
            }
      }
    }
  }
  st = warp_merge(st);
  if (lane == 0) s.stats[warp] = st;
  __syncthreads();
  if (kTop) {
    const int count = s.count;
    if (count <= kList) {
      order(s.list, count, a.top_k, s.top);
    } else {  // (the same in all threads) one pass per alternative: the largest key below the one before
      Key last = ~0ull;
      for (int k = 0; k < a.top_k && last != 0; ++k) {
        Key best = 0;
        for (int vec = begin + t; vec < end; vec += threads) {
          float v[kVec];
          unpack(row.load(vec), v);
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const Key key = v[e] > -INFINITY ? rank_key(v[e], row.column(vec) + e) : 0;
            if (key < last && key > best) best = key;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const Key other = __shfl_xor_sync(0xffffffffu, best, o);
          best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) s.best[warp] = best;
        __syncthreads();
        for (int w = 0; w < threads >> 5; ++w) best = s.best[w] > best ? s.best[w] : best;
        last = best;
        if (t == 0) s.top[k] = best;
      }
    }
  }
  const int warps = threads >> 5;
  const Key* top = s.top;
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (part == 0) {
      if (warp == 0) {
        SoftStats all;
        for (int i = lane; i < parts * warps; i += 32) all = merge(all, cluster.map_shared_rank(s.stats, i / warps)[i % warps]);
        all = warp_merge(all);
        if (lane == 0) s.result = finish(all);
      }
      if (kTop) {
        const int n = parts * a.top_k;
        for (int i = t; i < n; i += threads) s.list[i] = cluster.map_shared_rank(s.top, i / a.top_k)[i % a.top_k];
        if (t < a.top_k) s.merged[t] = 0;
        __syncthreads();
        order(s.list, n, a.top_k, s.merged);
        top = s.merged;
      }
    }
    cluster.sync();  // the others' shared memory has been read
    if (part != 0) return;
  } else if (warp == 0) {
    SoftStats all;
    if (lane < warps) all = s.stats[lane];
    all = warp_merge(all);
    if (lane == 0) s.result = finish(all);
  }
  __syncthreads();
  const RowResult res = s.result;
  if (t == 0) {
    if (a.entropy) a.entropy[r] = res.entropy;
    if (a.lse) a.lse[r] = res.lse;
  }
  for (int i = t; i < a.n_tokens; i += threads) {
    const size_t o = static_cast<size_t>(r) * a.n_tokens + i;
    a.logprobs[o] = i == t ? given_logprob(res, id, a.V, [&](int64_t) { return given; })
                           : given_logprob(res, a.tokens[o], a.V, [&](int64_t j) { return to_float(row.z[j]); });
  }
  if (kTop && t < a.top_k) {
    const size_t o = static_cast<size_t>(r) * a.top_k + t;
    const Key key = res.poisoned ? 0 : top[t];
    a.top_ids[o] = key ? key_id(key) : -1;
    a.top_logprobs[o] = key ? res.logprob(key_value(key)) : res.poisoned ? res.lse : -INFINITY;
  }
}

template <typename T>
int launch(cudaStream_t stream, const TokenLogprobsArgs& a, int sms) {
  // One CTA per row while that fills the GPU; with fewer rows, the largest cluster that leaves a thread its 16 logits and
  // all parts resident at once.
  const long long slots = static_cast<long long>(sms) * kCtasPerSm;
  int parts = 1;
  while (parts < kMaxParts && 2 * parts * static_cast<long long>(a.rows) <= slots && a.V >= 2 * parts * kThreads * 16) parts *= 2;
  const int per = (a.V + parts - 1) / parts;
  const int threads = std::min(kThreads, (per + 16 * 32 - 1) / (16 * 32) * 32);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * parts);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  RK_CUDA(cudaLaunchKernelEx(&cfg, a.top_k > 0 ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>, a, parts));
  RK_LAUNCH_CHECK("token_logprobs launch");
  return kOk;
}

}  // namespace

int token_logprobs(cudaStream_t stream, const TokenLogprobsArgs& a) {
  RK_REQUIRE(a.rows > 0 && a.V > 0 && a.logits, kBadArg, "token_logprobs: bad argument");
  RK_REQUIRE(a.V < (1 << 30), kShape, "token_logprobs: vocabulary of %d or more", 1 << 30);
  RK_REQUIRE(a.ld >= a.V, kShape, "token_logprobs: row stride %lld below the vocabulary size %d", a.ld, a.V);
  RK_REQUIRE(reinterpret_cast<uintptr_t>(a.logits) % (a.is_half ? 2 : 4) == 0, kBadArg, "token_logprobs: misaligned logits");
  RK_REQUIRE(a.n_tokens >= 0 && (a.n_tokens == 0 || (a.tokens && a.logprobs)), kBadArg, "token_logprobs: tokens without their output");
  RK_REQUIRE(a.top_k >= 0 && a.top_k <= kMaxTopLogprobs, kBadArg, "token_logprobs: top_k %d outside [0, %d]", a.top_k, kMaxTopLogprobs);
  RK_REQUIRE(a.top_k == 0 || (a.top_ids && a.top_logprobs), kBadArg, "token_logprobs: alternatives without their outputs");
  int sms = 0;
  const int status = device_sms(&sms);
  if (status != kOk) return status;
  return a.is_half ? launch<half>(stream, a, sms) : launch<float>(stream, a, sms);
}

}  // namespace rk
