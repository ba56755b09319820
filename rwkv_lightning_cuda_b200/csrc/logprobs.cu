// Log probabilities of given tokens over logits [rows, V], with the entropy, the log of the sum of exponentials and the
// likeliest alternatives of every row (definitions and corner cases: logprob.cuh).
//
// Bound by reading the logits once; a single row by latency.  A row goes to one CTA, or to the CTAs of a cluster when
// there are too few rows to fill the GPU: each takes a contiguous part and leaves its statistics and alternatives in the
// first one's shared memory, so there is no scratch, no second launch and no atomic whose order could show.
// A thread keeps 16 logits in registers and the next 16 under way, and its own running maximum (one rescaling per 16).  What a
// logit costs counts: half a maximum (a third with fp32), an exp2, and the multiply-adds and additions of its sums two logits at a
// time.  4096 rows of 65536: fp32 164 us, what the HBM takes (6.5 TB/s); fp16 105 us (5.1 TB/s), the exp2 units busy for 72 of them
// and the issue slots for 73.  (Two steps of fp16 under way instead of one: 114 us.)
//
// Alternatives without a pass over the rest: the k-th largest of the maxima of 64 disjoint groups of threads is a lower
// bound of the k-th largest logit, and only about k logits reach it.  Every thread has left the maxima of 16 stretches
// of its logits in shared memory, so the few stretches that reach the bound are known; they are loaded again (out of the
// L2, one vector per thread, all at once), what reaches the bound is listed, and the list is put in order by counting,
// for every entry, the larger ones.  A row with too many such stretches or logits (thousands of equal ones) takes k
// passes over its part instead.
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
constexpr int kGroups = 64;            // groups of neighbouring threads whose maxima bound the k-th largest logit
constexpr int kList = 512;             // candidates a part can list
constexpr int kStretches = 16;
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
__device__ __forceinline__ void unpack(const uint4& q, float* v, float) {
  v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void unpack(const uint4& q, float* v, half) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = h2f2(w[i]);
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(half v) { return __half2float(v); }

// Three operands, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The largest of a step's logits, NaN if there is one.
template <int kVecs>
__device__ __forceinline__ float largest_of(const uint4 (&q)[kVecs], float) {
  float a = __uint_as_float(q[0].x);
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const float x = __uint_as_float(q[j].x), y = __uint_as_float(q[j].y), z = __uint_as_float(q[j].z), w = __uint_as_float(q[j].w);
    a = max3_nan(max3_nan(a, x, y), z, w);
  }
  return a;
}
template <int kVecs>
__device__ __forceinline__ float largest_of(const uint4 (&q)[kVecs], half) {
  __half2 a = *reinterpret_cast<const __half2*>(&q[0].x);
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const uint32_t w[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) a = __hmax2_nan(a, *reinterpret_cast<const __half2*>(&w[i]));
  }
  const float2 x = __half22float2(a);
  return max_nan(x.x, x.y);
}

// Two fp32 at a time: an instruction each, with the roundings of the single ones.
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ float2 both() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r(0.f, 0.f);
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r(0.f, 0.f);
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// A step's 16 logits at the maximum that is in place.  2^((z - m) log2 e) as 2^(y - r) with y = z log2 e - M, M = fl(m log2 e)
// and r = m log2 e - M, each one rounding of an exact product: r is the same for all and comes off the sums.  r is up to half a
// step of M: 8 for |m| up to 1e8, but 128 and more, where 2^y and 2^-r overflow, from some 1.5e9 on.  A larger maximum, be it only that
// of a thread whose first logits are all masked with a large finite number, goes logit by logit.  So does a step with a product that
// overflows, of a logit below -2.3e38 or a masked token: a y of -inf, whose 0 * y makes t NaN.  (Looking for the smallest logit instead took half an instruction
// per logit of the ten or so that bound this kernel; the sums two at a time save one and a half.)
__device__ __forceinline__ void add_step(SoftStats& st, const float* v) {
  const float M = st.m * kLog2e, r = fmaf(st.m, kLog2e, -M);
  const F2 scale(kLog2e, kLog2e), less(-M, -M);
  F2 s2(0.f, 0.f), t2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const F2 y = fma2(F2(v[i], v[i + 1]), scale, less);
    const float2 p = y.both();
    const F2 e(exp2f(p.x), exp2f(p.y));
    s2 = add2(s2, e);
    t2 = fma2(e, y, t2);
  }
  const float2 s = s2.both(), t = t2.both();
  const float sum = s.x + s.y, weighted = t.x + t.y;
  if (fabsf(st.m) <= 1e8f && weighted == weighted) {
    const float f = exp2f(-r);
    st.s = fmaf(f, sum, st.s);
    st.t = fmaf(f * 0.6931471805599453f, fmaf(-r, sum, weighted), st.t);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) add(st, v[i]);
  }
}

constexpr int kHits = 256;

struct Stats {  // SoftStats without its initial values
  float m, s, t;
};
struct Shared {
  Stats stats[kWarps];
  Stats parts[kMaxParts];  // of the first part: all parts' statistics and alternatives
  alignas(16) Key part_top[kMaxParts * kMaxTopLogprobs + 2];
  alignas(16) float groups[kGroups];
  float bound;
  int count, hits;
  Key best[kWarps];
  Key top[kMaxTopLogprobs];  // this part's alternatives, best first, 0: none
  Key merged[kMaxTopLogprobs];
  alignas(16) Key list[kList + 2];
  unsigned short hit[kHits];  // stretches that reach the bound: stretch * kThreads + thread
  float stretch[1];           // [kStretches][threads]: the largest logit of each stretch of a thread's steps
};
__host__ __device__ constexpr size_t shared_bytes(int threads) { return sizeof(Shared) + sizeof(float) * kStretches * threads; }

// The k largest of n distinct keys (0: no key), in order; keys[n] and keys[n + 1] are overwritten.
__device__ __forceinline__ void order(Key* keys, int n, int k, Key* out) {
  if (threadIdx.x < 2) keys[n + threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const Key mine = keys[i];
    int larger = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + j);
      larger += (two.x > mine ? 1 : 0) + (two.y > mine ? 1 : 0);
    }
    if (mine != 0 && larger < k) out[larger] = mine;
  }
}

template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) token_logprobs_kernel(const TokenLogprobsArgs a, const int parts) {
  constexpr int kVec = RowView<T>::kVec, kVecs = 16 / kVec;  // 16 logits per thread and step
  extern __shared__ __align__(16) unsigned char shared_mem[];
  Shared& s = *reinterpret_cast<Shared*>(shared_mem);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, threads = blockDim.x;
  const int r = blockIdx.x / parts, part = blockIdx.x - r * parts;
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA has begun: waited for before it is written to
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
    if (t == 0) s.count = s.hits = 0;
    if (t < a.top_k) s.top[t] = 0;
  }

  SoftStats st;
  const int stretch = (steps + kStretches - 1) / kStretches;  // in steps
  float highest = -INFINITY;
  uint4 q[kVecs];
  for (int i = 0, in = 0, at = 0; i < steps; ++i) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) q[j] = next[j];
    if (i + 1 < steps) fetch(i + 1, next);
    const float hi = largest_of(q, T(0));
    const float m = max_nan(st.m, hi);
    if (m != st.m) raise(st, m);
    float v[16];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) unpack(q[j], v + j * kVec, T(0));
    add_step(st, v);
    if (kTop) {
      highest = in == 0 ? hi : fmaxf(highest, hi);
      if (++in == stretch || i + 1 == steps) {
        s.stretch[at++ * threads + t] = highest;
        in = 0;
      }
    }
  }
  const float mine = st.m;  // this thread's largest logit, -FLT_MAX if it has none that counts
  st = warp_merge(st);
  if (lane == 0) s.stats[warp] = Stats{st.m, st.s, st.t};
  __syncthreads();
  if (kTop) {
    // the bound: -inf when there are fewer groups with a logit than alternatives
    const int share = threads > kGroups ? threads / kGroups : 1;  // threads to a group: 1, 2 or 4
    float g = mine;
    if (share > 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 1));
    if (share > 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
    if ((t & (share - 1)) == 0) s.groups[t / share] = g;
    if (threads < kGroups) s.groups[t + threads] = -FLT_MAX;  // what one warp lacks
    __syncthreads();
    for (int j = t >> 2; j < kGroups; j += threads >> 2) {  // four threads count a quarter each of what is before group j
      const float largest = s.groups[j];
      int before = 0;
#pragma unroll
      for (int e = 0; e < kGroups / 4; ++e) {
        const int o = 4 * e + (lane & 3);
        const float other = s.groups[o];
        before += other > largest || (other == largest && o < j) ? 1 : 0;
      }
      before += __shfl_xor_sync(0xffffffffu, before, 1);
      before += __shfl_xor_sync(0xffffffffu, before, 2);
      if ((lane & 3) == 0 && before == a.top_k - 1) s.bound = largest > -FLT_MAX ? largest : -INFINITY;
    }
    __syncthreads();
    const float bound = s.bound;
    auto list = [&](const float (&v)[kVec], int vec) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (v[e] >= bound && v[e] > -INFINITY) {
          const int slot = atomicAdd(&s.count, 1);
          if (slot < kList) s.list[slot] = rank_key(v[e], row.column(vec) + e);
        }
    };
    if (steps == 1) {  // short rows: the logits are still here
      if (mine >= bound) {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          float v[kVec];
          unpack(q[j], v, T(0));
          list(v, begin + j * threads + t);
        }
      }
    } else if (mine >= bound) {
      for (int w = 0; w * stretch < steps; ++w) {
        const float high = s.stretch[w * threads + t];
        if (high < bound || !(high > -INFINITY)) continue;
        const int slot = atomicAdd(&s.hits, 1);
        if (slot < kHits) s.hit[slot] = static_cast<unsigned short>(w * kThreads + t);
      }
    }
    __syncthreads();
    const int hits = s.hits, vectors = stretch * kVecs;
    for (int i = t; i < min(hits, kHits) * vectors; i += threads) {
      const int hit = s.hit[i / vectors], of = i % vectors;
      const int vec = begin + (hit / kThreads * stretch + of / kVecs) * step + of % kVecs * threads + hit % kThreads;
      if (vec >= end) continue;
      float v[kVec];
      unpack(row.load(vec), v, T(0));
      list(v, vec);
    }
    __syncthreads();
    const int count = s.count;
    if (hits <= kHits && count <= kList) {
      order(s.list, count, a.top_k, s.top);
    } else {  // (the same in all threads) one pass per alternative: the largest key below the one before
      Key last = ~0ull;
      for (int k = 0; k < a.top_k && last != 0; ++k) {
        Key best = 0;
        for (int vec = begin + t; vec < end; vec += threads) {
          float v[kVec];
          unpack(row.load(vec), v, T(0));
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
  // Every warp merges this part's statistics; with several parts they and the alternatives go to the first one.
  auto merged = [&](const Stats* of, int n) {
    SoftStats b;
    if (lane < n) { b.m = of[lane].m; b.s = of[lane].s; b.t = of[lane].t; }
    return warp_merge(b);
  };
  SoftStats all = merged(s.stats, threads >> 5);
  const Key* top = s.top;
  if (parts > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    Shared* first = cluster.map_shared_rank(&s, 0);
    if (t == 0) first->parts[part] = Stats{all.m, all.s, all.t};
    if (kTop) {
      __syncthreads();
      if (t < a.top_k) first->part_top[part * a.top_k + t] = s.top[t];
    }
    cluster.sync();
    if (part != 0) return;
    all = merged(s.parts, parts);
    if (kTop) {
      if (t < a.top_k) s.merged[t] = 0;
      order(s.part_top, parts * a.top_k, a.top_k, s.merged);
      top = s.merged;
    }
  }
  if (kTop) __syncthreads();
  const RowResult res = finish(all);
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
  // Several CTAs to a row while that leaves them a thread 16 logits and about two to an SM (clusters are not placed as densely
  // as single CTAs, and each row ends in a microsecond or two of merging).  Measured with 65536 fp32 logits and five alternatives,
  // 1 / 2 / 4 / 8 parts: 148 rows 19.0 / 15.0 / 19.5 / 22.7 us, 64 rows 17.9 / 12.5 / 9.9 / 11.0, 32 rows 17.5 / 12.0 / 8.8 / 7.8;
  // 256 rows and 20 alternatives 21.9 / 20.5 / 26.2 / 38.5.
  int parts = 1;
  while (parts < kMaxParts && 2LL * parts * a.rows <= (parts == 1 ? 4 : 11 * 0.25) * sms && a.V >= 2 * parts * kThreads * 16) parts *= 2;
  // Blocks of 256 threads, or about as many as have 16 to 32 logits each; smaller ones where there are rows for every SM several
  // times over, because every warp of a row's block takes part in the merging (3850 rows of 2475: 29.5 us with 256 threads or what
  // they come to, 23.6 with 64; 4096 x 65536 fp16: 116 us with 256, 110 with 128).
  const int per = (a.V + parts - 1) / parts;
  int threads = 32;
  while (threads < kThreads && threads * 24 < per) threads *= 2;
  if (static_cast<long long>(a.rows) * parts >= 4LL * sms) threads = std::min(threads, a.V <= 4096 ? 64 : 128);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * parts);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared_bytes(threads);
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
