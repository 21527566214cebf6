// Log probabilities of given tokens with rank, entropy and the top
// alternatives (ov_token_logprobs).  With m = max x and d = x - m,
//   Z = sum e^d,  logprob = d_target - log Z,  entropy = log Z - (sum e^d d) / Z,
// in one pass over the logits: a running maximum and two sums, rescaled when
// the maximum grows (float32, whatever the logits' type).  Bound by reading
// the logits once.
//
// Alternatives order by (logit descending, index ascending), one 64-bit key
// each.  Instead of sorting, a threshold that at least top_k values reach is
// taken from the maxima that the threads hold anyway; the few values that
// pass it are ranked against one another.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "internal.hpp"
#include "kv_cache.hpp"
#include "launch.hpp"
#include "ov_kernels.h"
#include "ptx.cuh"

namespace ovb {
namespace {

constexpr int kMaxTopK = 32;
constexpr float kLog2E = 1.4426950408889634f;

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  int64_t rows;
  int codebooks;
  int vocab;
  const int32_t* targets;
  int top_k;
  float* logprob;
  float* entropy;       // or null
  int32_t* rank;        // or null
  int32_t* top_ids;
  float* top_logprobs;
  uint32_t* err;
};

__device__ __forceinline__ float ToFloat(float x) { return x; }
__device__ __forceinline__ float ToFloat(__half x) { return __half2float(x); }

// Maximum that keeps a NaN.
__device__ __forceinline__ float MaxNan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float Exp2Approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order of alternatives: greater logit first, then lower index.  No key is 0.
__device__ __forceinline__ uint64_t AlternativeKey(float x, int index) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // one key for +0 and -0
  const uint32_t ordered = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<uint64_t>(ordered) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ float KeyValue(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ int KeyIndex(uint64_t key) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

__device__ __forceinline__ uint64_t WarpMaxKey(uint64_t key) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xFFFFFFFFu, key, o);
    key = other > key ? other : key;
  }
  return key;
}

// The k-th greatest of the warp's 32 values (bitonic sort, descending).
__device__ __forceinline__ float WarpKth(float v, int k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const float other = __shfl_xor_sync(0xFFFFFFFFu, v, step);
      const bool descending = (lane & size) == 0;
      const bool lower = (lane & step) == 0;
      v = lower == descending ? fmaxf(v, other) : fminf(v, other);
    }
  }
  return __shfl_sync(0xFFFFFFFFu, v, k - 1);
}

// What a row without a distribution gives.
__device__ __forceinline__ void StoreNothing(const LogprobArgs& a, int64_t out, int lane) {
  const float nan = __uint_as_float(0x7FC00000u);
  if (lane == 0) {
    a.logprob[out] = nan;
    if (a.entropy != nullptr) a.entropy[out] = nan;
    if (a.rank != nullptr) a.rank[out] = -1;
  }
  if (lane < a.top_k) {
    a.top_ids[out * a.top_k + lane] = -1;
    a.top_logprobs[out * a.top_k + lane] = nan;
  }
}

// The item's target, or -1.
__device__ __forceinline__ int Target(const LogprobArgs& a, int64_t out, bool report) {
  const int t = a.targets[out];
  if (t < a.vocab) return t < 0 ? -1 : t;
  if (report) atomicOr(a.err, kErrBadArgument);
  return -1;
}

// ------------------------------------------- short rows: one warp per item

constexpr int kWarps = 8;
constexpr int kWarpKeys = 64;

// The whole group sits in registers, value j in lane j % 32.
template <typename T, int kPer>
__global__ void __launch_bounds__(kWarps * 32) logprobs_warp_kernel(const LogprobArgs a) {
  __shared__ uint64_t s_keys[kWarps][kWarpKeys];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= a.rows * a.codebooks) return;
  const int64_t row = item / a.codebooks;
  const int codebook = static_cast<int>(item % a.codebooks);
  const int64_t out = codebook * a.rows + row;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + static_cast<int64_t>(codebook) * a.vocab;
  float x[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = lane + 32 * i;
    x[i] = j < a.vocab ? ToFloat(src[j]) : -INFINITY;
  }
  const int target = Target(a, out, lane == 0);
  const float xt = target >= 0 ? ToFloat(src[target]) : 0.0f;
  float top = x[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) top = MaxNan(top, x[i]);
  float m = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = MaxNan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (!(fabsf(m) < INFINITY)) {
    StoreNothing(a, out, lane);
    return;
  }
  float z = 0.0f, w = 0.0f;
  int ahead = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float d = fmaxf(x[i] - m, -1e30f);  // finite, so that 0 * d is 0 for a closed token
    const float e = Exp2Approx(d * kLog2E);
    z += e;
    w = fmaf(e, d, w);
  }
  if (a.rank != nullptr) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = lane + 32 * i;
      ahead += (x[i] > xt || (x[i] == xt && j < target)) ? 1 : 0;
    }
    ahead = __reduce_add_sync(0xFFFFFFFFu, ahead);
  }
  z = warp_sum(z);
  w = warp_sum(w);
  const float log_z = logf(z);
  if (lane == 0) {
    a.logprob[out] = target >= 0 ? (xt - m) - log_z : 0.0f;
    if (a.entropy != nullptr) a.entropy[out] = log_z - w / z;
    if (a.rank != nullptr) a.rank[out] = target >= 0 ? ahead : -1;
  }
  const int k = a.top_k;
  if (k == 0) return;
  int32_t* ids = a.top_ids + out * k;
  float* logprobs = a.top_logprobs + out * k;
  // k lanes hold a value of at least the k-th greatest lane maximum.
  const float threshold = WarpKth(top, k);
  uint64_t* keys = s_keys[threadIdx.x >> 5];
  int n = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool pass = x[i] >= threshold && lane + 32 * i < a.vocab;
    const uint32_t mask = __ballot_sync(0xFFFFFFFFu, pass);
    if (mask == 0) continue;
    const int at = n + __popc(mask & ((1u << lane) - 1u));
    if (pass && at < kWarpKeys) keys[at] = AlternativeKey(x[i], lane + 32 * i);
    n += __popc(mask);
  }
  __syncwarp();
  if (n <= kWarpKeys) {
    const uint64_t k0 = lane < n ? keys[lane] : 0, k1 = lane + 32 < n ? keys[lane + 32] : 0;
    int r0 = 0, r1 = 0;
    for (int j = 0; j < n; ++j) {
      const uint64_t other = keys[j];
      r0 += other > k0 ? 1 : 0;
      r1 += other > k1 ? 1 : 0;
    }
    if (k0 != 0 && r0 < k) {
      ids[r0] = KeyIndex(k0);
      logprobs[r0] = (KeyValue(k0) - m) - log_z;
    }
    if (k1 != 0 && r1 < k) {
      ids[r1] = KeyIndex(k1);
      logprobs[r1] = (KeyValue(k1) - m) - log_z;
    }
    return;
  }
  // Many equal or closed values: one alternative after the other.
  uint64_t last = ~uint64_t{0};
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = lane + 32 * i;
      const uint64_t key = j < a.vocab ? AlternativeKey(x[i], j) : 0;
      if (key < last && key > best) best = key;
    }
    last = WarpMaxKey(best);
    if (lane == 0) {
      ids[r] = KeyIndex(last);
      logprobs[r] = (KeyValue(last) - m) - log_z;
    }
  }
}

// ------------------------------ long rows: one CTA, or a cluster, per item

constexpr int kThreads = 512;
constexpr int kKeys = 1024;      // room for passing values between prunings
constexpr int kPruneAt = 512;

// Running maximum, Z and sum e^d d of what was read.
struct RowStats {
  float m, z, w;
  // To a maximum m2 >= m.
  __device__ __forceinline__ void Rebase(float m2) {
    if (m == -INFINITY) {
      m = m2;
      return;
    }
    const float d = m - m2, f = Exp2Approx(d * kLog2E);
    w = f * fmaf(d, z, w);
    z *= f;
    m = m2;
  }
  __device__ __forceinline__ void Merge(RowStats o) {
    const float top = MaxNan(m, o.m);
    if (!(fabsf(top) < INFINITY)) {  // nothing yet, or no distribution
      m = top;
      return;
    }
    Rebase(top);
    o.Rebase(top);
    z += o.z;
    w += o.w;
  }
};

__device__ __forceinline__ uint32_t LoadCluster32(uint32_t address) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t LoadCluster64(uint32_t address) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(address) : "memory");
  return v;
}

// 16 bytes of logits as floats.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void Unpack(const uint4& q, float* x) {
    x[0] = __uint_as_float(q.x);
    x[1] = __uint_as_float(q.y);
    x[2] = __uint_as_float(q.z);
    x[3] = __uint_as_float(q.w);
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void Unpack(const uint4& q, float* x) {
    const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

struct LongShared {
  uint64_t keys[kKeys];
  uint64_t sorted[8 * kMaxTopK];
  uint64_t warp_key[kThreads / 32];
  float kth[kThreads / 32];
  RowStats stats[kThreads / 32];
  int ahead[kThreads / 32];
  RowStats total;
  int total_ahead;
  int count;
  int found;
  float threshold;
};

// Leaves the top_k greatest of the `count` keys in order in keys[0 ..) and
// sets count and threshold.  Every thread calls it, after a barrier.
__device__ __forceinline__ void Prune(LongShared& s, int k) {
  const int n = s.count;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = s.keys[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += s.keys[j] > key ? 1 : 0;
    if (r < k) s.sorted[r] = key;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < min(n, k)) s.keys[threadIdx.x] = s.sorted[threadIdx.x];
  if (threadIdx.x == 0) {
    s.count = min(n, k);
    s.threshold = n >= k ? KeyValue(s.sorted[k - 1]) : -INFINITY;
  }
  __syncthreads();
}

template <typename T, int kU>
__global__ void __launch_bounds__(kThreads, 2)
    logprobs_long_kernel(const LogprobArgs a, int cluster) {
  constexpr int kE = Vec<T>::kN;
  constexpr int kN = kU * kE;
  __shared__ LongShared s;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(cluster));
  const int64_t item = blockIdx.x / static_cast<unsigned>(cluster);
  const int64_t row = item / a.codebooks;
  const int codebook = static_cast<int>(item % a.codebooks);
  const int64_t out = codebook * a.rows + row;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + static_cast<int64_t>(codebook) * a.vocab;
  const int k = a.top_k;
  const int target = Target(a, out, tid == 0 && part == 0);
  const float xt = target >= 0 ? ToFloat(src[target]) : INFINITY;
  if (tid == 0) {
    s.count = 0;
    s.threshold = -INFINITY;
  }
  // Vectors of 16 aligned bytes; vector v holds values [kE v - skip, ...).
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(src - skip);
  const int vectors = (skip + a.vocab + kE - 1) / kE;
  const int per = (vectors + cluster - 1) / cluster;
  const int begin = part * per, end = min(vectors, begin + per);

  auto load = [&](int v, float* x) {
    const int j = v * kE - skip;
    if (v < end && j >= 0 && j + kE <= a.vocab) {
      Vec<T>::Unpack(base[v], x);
    } else {
#pragma unroll
      for (int e = 0; e < kE; ++e)
        x[e] = v < end && j + e >= 0 && j + e < a.vocab ? ToFloat(src[j + e]) : -INFINITY;
    }
  };

  RowStats st = {-INFINITY, 0.0f, 0.0f};
  int ahead = 0;
  bool first = true;
  for (int v0 = begin; v0 < end; v0 += kThreads * kU) {
    float x[kN];
#pragma unroll
    for (int u = 0; u < kU; ++u) load(v0 + u * kThreads + tid, x + u * kE);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < kN; ++i) top = MaxNan(top, x[i]);
    const float grown = MaxNan(st.m, top);
    if (grown != st.m) {
      if (fabsf(grown) < INFINITY) st.Rebase(grown);
      else st.m = grown;  // NaN or +inf: no distribution
    }
    if (fabsf(st.m) < INFINITY) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float d = fmaxf(x[i] - st.m, -1e30f);
        const float e = Exp2Approx(d * kLog2E);
        st.z += e;
        st.w = fmaf(e, d, st.w);
      }
    }
    if (a.rank != nullptr) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int v = v0 + u * kThreads + tid;
        const int j = v * kE - skip;
#pragma unroll
        for (int e = 0; e < kE; ++e) ahead += x[u * kE + e] > xt ? 1 : 0;
        if (v < end && j < target) {  // equal values ahead of the target
#pragma unroll
          for (int e = 0; e < kE; ++e)
            ahead += x[u * kE + e] == xt && j + e < target && j + e >= 0 ? 1 : 0;
        }
      }
    }
    if (k == 0) continue;
    // The first values take their threshold from the threads' maxima: k
    // lanes of a warp hold a value of at least its k-th greatest maximum.
    float threshold;
    if (first) {
      const float kth = WarpKth(top, k);
      if (lane == 0) s.kth[warp] = kth;
      __syncthreads();
      threshold = -INFINITY;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) threshold = fmaxf(threshold, s.kth[i]);
    } else {
      threshold = s.threshold;
    }
    // Later values lose to an equal earlier one, so they have to be greater.
    bool crowded = first;
    if (top > threshold || (first && top == threshold)) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int j = (v0 + u * kThreads + tid) * kE - skip;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const float v = x[u * kE + e];
          if (v > threshold || (first && v == threshold && v > -INFINITY)) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kKeys) s.keys[at] = AlternativeKey(v, j + e);
            crowded |= at >= kPruneAt;
          }
        }
      }
    }
    if (__syncthreads_or(crowded)) {
      if (s.count > kKeys) {
        // No room (many equal values, or rising ones): the k greatest of
        // these and of the keys from before, one after the other.
        const int chunk = v0 * kE - skip;  // first index of these values
        uint64_t last = ~uint64_t{0};
        for (int r = 0; r < k; ++r) {
          uint64_t best = 0;
          for (int i = tid; i < kKeys; i += kThreads) {
            const uint64_t key = s.keys[i];
            if (KeyIndex(key) < chunk && key < last && key > best) best = key;
          }
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const int j = (v0 + (i / kE) * kThreads + tid) * kE - skip + i % kE;
            const uint64_t key = x[i] > -INFINITY ? AlternativeKey(x[i], j) : 0;
            if (key < last && key > best) best = key;
          }
          best = WarpMaxKey(best);
          if (lane == 0) s.warp_key[warp] = best;
          __syncthreads();
          last = 0;
#pragma unroll
          for (int i = 0; i < kThreads / 32; ++i) last = max(last, s.warp_key[i]);
          if (tid == 0) s.sorted[r] = last;  // never 0: more than kKeys values passed
          __syncthreads();
        }
        if (tid < k) s.keys[tid] = s.sorted[tid];
        if (tid == 0) {
          s.count = k;
          s.threshold = KeyValue(s.sorted[k - 1]);
        }
        __syncthreads();
      } else {
        Prune(s, k);
      }
    }
    first = false;
  }

  // The CTA's sums, in a fixed order.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RowStats other;
    other.m = __shfl_xor_sync(0xFFFFFFFFu, st.m, o);
    other.z = __shfl_xor_sync(0xFFFFFFFFu, st.z, o);
    other.w = __shfl_xor_sync(0xFFFFFFFFu, st.w, o);
    st.Merge(other);
  }
  ahead = __reduce_add_sync(0xFFFFFFFFu, ahead);
  if (lane == 0) {
    s.stats[warp] = st;
    s.ahead[warp] = ahead;
  }
  __syncthreads();
  if (k > 0) Prune(s, k);
  if (tid == 0) {
    RowStats total = s.stats[0];
    int sum = s.ahead[0];
    for (int i = 1; i < kThreads / 32; ++i) {
      total.Merge(s.stats[i]);
      sum += s.ahead[i];
    }
    s.total = total;
    s.total_ahead = sum;
  }
  if (cluster > 1) {
    __syncthreads();
    cluster_sync();
    if (part == 0) {
      // The other parts' alternatives behind this one's; their sums in part
      // order.  Parts hold ascending indices, and the keys order ties.
      if (k > 0) {
        for (int i = tid; i < (cluster - 1) * kMaxTopK; i += kThreads) {
          const int peer = 1 + i / kMaxTopK, at = i % kMaxTopK;
          const int n = static_cast<int>(LoadCluster32(mapa_shared(smem_u32(&s.count), peer)));
          uint64_t key = 0;
          if (at < n) key = LoadCluster64(mapa_shared(smem_u32(&s.keys[at]), peer));
          s.sorted[i] = key;
        }
        __syncthreads();
        for (int i = tid; i < (cluster - 1) * kMaxTopK; i += kThreads)
          if (s.sorted[i] != 0) s.keys[atomicAdd(&s.count, 1)] = s.sorted[i];
        __syncthreads();
        Prune(s, k);
      }
      if (tid == 0) {
        RowStats total = s.total;
        int sum = s.total_ahead;
        for (int peer = 1; peer < cluster; ++peer) {
          const uint32_t at = mapa_shared(smem_u32(&s.total), peer);
          RowStats o;
          o.m = __uint_as_float(LoadCluster32(at));
          o.z = __uint_as_float(LoadCluster32(at + 4));
          o.w = __uint_as_float(LoadCluster32(at + 8));
          total.Merge(o);
          sum += static_cast<int>(LoadCluster32(mapa_shared(smem_u32(&s.total_ahead), peer)));
        }
        s.total = total;
        s.total_ahead = sum;
      }
    }
    __syncthreads();
    cluster_sync();  // the peers' shared memory was read
    if (part != 0) return;
  }
  __syncthreads();
  const RowStats total = s.total;
  if (!(fabsf(total.m) < INFINITY)) {
    StoreNothing(a, out, tid);
    return;
  }
  const float log_z = logf(total.z);
  if (tid == 0) {
    a.logprob[out] = target >= 0 ? (xt - total.m) - log_z : 0.0f;
    if (a.entropy != nullptr) a.entropy[out] = log_z - total.w / total.z;
    if (a.rank != nullptr) a.rank[out] = target >= 0 ? s.total_ahead : -1;
  }
  const int n = min(s.count, k);
  if (tid < n) {
    a.top_ids[out * k + tid] = KeyIndex(s.keys[tid]);
    a.top_logprobs[out * k + tid] = (KeyValue(s.keys[tid]) - total.m) - log_z;
  }
  // Fewer than top_k open tokens: closed ones by index.
  if (warp == 0 && n < k) {
    int filled = n;
    for (int j0 = 0; j0 < a.vocab && filled < k; j0 += 32) {
      const int j = j0 + lane;
      const bool closed = j < a.vocab && ToFloat(src[j]) == -INFINITY;
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, closed);
      const int at = filled + __popc(mask & ((1u << lane) - 1u));
      if (closed && at < k) {
        a.top_ids[out * k + at] = j;
        a.top_logprobs[out * k + at] = -INFINITY;
      }
      filled += __popc(mask);
    }
  }
}

template <typename T>
void LaunchLogprobs(const LogprobArgs& a, cudaStream_t stream) {
  const int64_t items = a.rows * a.codebooks;
  const char* what = "log probability kernel launch";
  if (a.vocab <= 66 * 32) {
    const dim3 grid(static_cast<unsigned>((items + kWarps - 1) / kWarps));
    Launch(a.vocab <= 33 * 32 ? logprobs_warp_kernel<T, 33> : logprobs_warp_kernel<T, 66>, grid,
           dim3(kWarps * 32), 0, stream, what, a);
    return;
  }
  // Few rows: up to eight CTAs of a cluster share one, as long as each has
  // vectors for all of its threads.
  unsigned cluster = 1;
  while (cluster < 8 && items * cluster * 2 <= 2 * SmCount() &&
         a.vocab >= static_cast<int>(cluster) * 2 * kThreads * Vec<T>::kN)
    cluster *= 2;
  LaunchEx(logprobs_long_kernel<T, 16 / Vec<T>::kN>, dim3(static_cast<unsigned>(items) * cluster),
           dim3(kThreads), 0, stream, what, cluster, a, static_cast<int>(cluster));
}

}  // namespace
}  // namespace ovb

using namespace ovb;

extern "C" int ov_token_logprobs(const void* logits, int logits_type, size_t ld, size_t rows,
                                 size_t codebooks, size_t vocab, const int32_t* targets,
                                 size_t top_k, float* logprob, float* entropy, int32_t* rank,
                                 int32_t* top_ids, float* top_logprobs, ov_stream_t stream) {
  return Guard("ov_token_logprobs: ", [&] {
    OV_REQUIRE(logits_type == OV_LOGITS_F32 || logits_type == OV_LOGITS_F16, "logits type");
    OV_REQUIRE(codebooks > 0 && codebooks <= 65535, "codebooks must be 1 to 65535");
    OV_REQUIRE(vocab > 0 && vocab <= (size_t{1} << 20), "vocab must be 1 to 2^20");
    OV_REQUIRE(ld >= codebooks * vocab, "logits stride");
    OV_REQUIRE(top_k <= kMaxTopK && top_k <= vocab, "top_k must be at most 32 and at most vocab");
    OV_REQUIRE(rows < (size_t{1} << 27) / codebooks, "rows * codebooks must stay below 2^27");
    if (rows == 0) return;
    RequireAligned(logits, logits_type == OV_LOGITS_F16 ? 2 : 4, "logits");
    RequireAligned(targets, 4, "targets");
    RequireAligned(logprob, 4, "logprob");
    if (entropy != nullptr) RequireAligned(entropy, 4, "entropy");
    if (rank != nullptr) RequireAligned(rank, 4, "rank");
    if (top_k > 0) RequireAligned(top_ids, 4, "top_ids");
    if (top_k > 0) RequireAligned(top_logprobs, 4, "top_logprobs");
    RequireOnDevice(logits, "logits");
    RequireOnDevice(targets, "targets");
    RequireOnDevice(logprob, "logprob");
    if (entropy != nullptr) RequireOnDevice(entropy, "entropy");
    if (rank != nullptr) RequireOnDevice(rank, "rank");
    if (top_k > 0) RequireOnDevice(top_ids, "top_ids");
    if (top_k > 0) RequireOnDevice(top_logprobs, "top_logprobs");
    LogprobArgs a;
    a.logits = logits;
    a.ld = static_cast<int64_t>(ld);
    a.rows = static_cast<int64_t>(rows);
    a.codebooks = static_cast<int>(codebooks);
    a.vocab = static_cast<int>(vocab);
    a.targets = targets;
    a.top_k = static_cast<int>(top_k);
    a.logprob = logprob;
    a.entropy = entropy;
    a.rank = rank;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.err = DeviceErrorWord();
    if (logits_type == OV_LOGITS_F16) LaunchLogprobs<__half>(a, AsStream(stream));
    else LaunchLogprobs<float>(a, AsStream(stream));
  });
}
