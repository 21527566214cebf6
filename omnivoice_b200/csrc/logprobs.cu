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
//
// Measured on one B200: the audio head's 500 rows of 8 x 1,025 float32 values
// (16.6 MB) 8.0 us; 512 half rows of 151,936 values (156 MB) with 20
// alternatives 52 us, 3.0 TB/s: not the reading but about 14 instructions for
// a value bound it (6 for the sums and the rank, the rest for alternatives and
// what a chunk costs; with the sums' operations one by one instead of in pairs,
// 56 us); one float32 row of that length 12.6 us, its clusters' barriers and
// joins included.
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
constexpr float kLn2 = 0.6931471805599453f;

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

// The same for a small k, one maximum after the other.
__device__ __forceinline__ float WarpKthOfFew(float v, int k) {
  const uint32_t u = __float_as_uint(v);
  uint32_t key = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  uint32_t top = __reduce_max_sync(0xFFFFFFFFu, key);
  for (int i = 1; i < k; ++i) {
    const uint32_t holders = __ballot_sync(0xFFFFFFFFu, key == top);
    if ((threadIdx.x & 31) == __ffs(holders) - 1) key = 0;
    top = __reduce_max_sync(0xFFFFFFFFu, key);
  }
  return __uint_as_float((top & 0x80000000u) ? (top & 0x7FFFFFFFu) : ~top);
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

// n / d, in 32 bits where they hold it.
__device__ __forceinline__ int64_t Quotient(int64_t n, int d) {
  if (n >> 31 == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

// The item's target, or -1.
__device__ __forceinline__ int Target(const LogprobArgs& a, int64_t out, bool report) {
  const int t = a.targets[out];
  if (t < a.vocab) return t < 0 ? -1 : t;
  if (report) atomicOr(a.err, kErrBadArgument);
  return -1;
}

// ------------------------------------------------- exponents by logits type

constexpr int kVectors = 4;      // 16-byte vectors of a thread and chunk (Row::Top takes four)

// 16 bytes of logits, and how their exponent t = (x - m) log2(e) is formed.
// For float32 the difference comes first: a mask of the type's lowest value
// times log2(e) would overflow.  For halves it cannot, and one fused
// multiply-add against Scaled(m) does.
template <typename T>
struct Row;

template <>
struct Row<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ uint4 Closed() {  // all -inf
    return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
  }
  static __device__ __forceinline__ float Scaled(float m) { return m; }
  static __device__ __forceinline__ float Exponent(float x, float scaled) {
    return (x - scaled) * kLog2E;
  }
  // Those of values i and i + 1; finite, so that a closed token's 0 * t is 0.
  static __device__ __forceinline__ float2 Exponents(const uint4& q, int i, float scaled) {
    return Finite(mul2(add2(make_float2(At(q, i), At(q, i + 1)), make_float2(-scaled, -scaled)),
                       make_float2(kLog2E, kLog2E)));
  }
  static __device__ __forceinline__ float2 Finite(float2 t) {
    return make_float2(fmaxf(t.x, -16384.0f), fmaxf(t.y, -16384.0f));
  }
  // log p of a value, with log_z = log Z.
  static __device__ __forceinline__ float LogProb(float x, float m, float log_z) {
    return (x - m) - log_z;
  }
  static __device__ __forceinline__ float At(const uint4& q, int i) {
    return __uint_as_float(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w);
  }
  // Exponent of the step from one maximum to another.
  static __device__ __forceinline__ float Step(float from, float to) {
    return (from - to) * kLog2E;
  }
  static __device__ __forceinline__ float Top(const uint4& q) {
    return MaxNan(MaxNan(At(q, 0), At(q, 1)), MaxNan(At(q, 2), At(q, 3)));
  }
  static __device__ __forceinline__ float Top(const uint4 (&q)[kVectors]) {
    return MaxNan(MaxNan(Top(q[0]), Top(q[1])), MaxNan(Top(q[2]), Top(q[3])));
  }
  // Values above x (kEqual: or equal to it).
  template <bool kEqual>
  static __device__ __forceinline__ int Above(const uint4 (&q)[kVectors], float x) {
    int n = 0;
#pragma unroll
    for (int u = 0; u < kVectors; ++u)
#pragma unroll
      for (int i = 0; i < kN; ++i) n += kEqual ? At(q[u], i) >= x : At(q[u], i) > x;
    return n;
  }
  // Bit i: value i is above x.
  static __device__ __forceinline__ uint32_t MaskAbove(const uint4& q, float x) {
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) mask |= At(q, i) > x ? 1u << i : 0u;
    return mask;
  }
  // Value i, i not known when compiling.
  static __device__ __forceinline__ float Pick(const uint4& q, int i) {
    return __uint_as_float(i < 2 ? (i == 0 ? q.x : q.y) : (i == 2 ? q.z : q.w));
  }
  // The greatest value below x.
  static __device__ __forceinline__ float Below(float x) {
    return __uint_as_float(x > 0.0f ? __float_as_uint(x) - 1
                                    : x == 0.0f ? 0x80000001u : __float_as_uint(x) + 1);
  }
};

template <>
struct Row<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ uint4 Closed() {
    return make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
  }
  // Rounded by itself: a contracted product would make Step(m, m) its residue.
  static __device__ __forceinline__ float Scaled(float m) { return __fmul_rn(m, kLog2E); }
  static __device__ __forceinline__ float Exponent(float x, float scaled) {
    return fmaf(x, kLog2E, -scaled);
  }
  static __device__ __forceinline__ float2 Exponents(const uint4& q, int i, float scaled) {
    const uint32_t w = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return Row<float>::Finite(
        fma2(__half22float2(Pair(w)), make_float2(kLog2E, kLog2E), make_float2(-scaled, -scaled)));
  }
  static __device__ __forceinline__ float LogProb(float x, float m, float log_z) {
    return fmaf(Exponent(x, Scaled(m)), kLn2, -log_z);
  }
  static __device__ __forceinline__ float At(const uint4& q, int i) {
    const uint32_t w = i < 2 ? q.x : i < 4 ? q.y : i < 6 ? q.z : q.w;
    return __half2float(__ushort_as_half(static_cast<uint16_t>(i & 1 ? w >> 16 : w)));
  }
  static __device__ __forceinline__ float Step(float from, float to) {
    return Scaled(from) - Scaled(to);
  }
  static __device__ __forceinline__ __half2 Pair(uint32_t w) {
    return *reinterpret_cast<const __half2*>(&w);
  }
  static __device__ __forceinline__ __half2 Top2(const uint4& q) {
    return __hmax2_nan(__hmax2_nan(Pair(q.x), Pair(q.y)), __hmax2_nan(Pair(q.z), Pair(q.w)));
  }
  static __device__ __forceinline__ float Top(const uint4& q) {
    const __half2 top = Top2(q);
    return MaxNan(__low2float(top), __high2float(top));
  }
  static __device__ __forceinline__ float Top(const uint4 (&q)[kVectors]) {
    const __half2 top = __hmax2_nan(__hmax2_nan(Top2(q[0]), Top2(q[1])),
                                    __hmax2_nan(Top2(q[2]), Top2(q[3])));
    return MaxNan(__low2float(top), __high2float(top));
  }
  template <bool kEqual>
  static __device__ __forceinline__ int Above(const uint4 (&q)[kVectors], float x) {
    const __half2 h = __float2half2_rn(x);  // a half to begin with
    auto test = [&](uint32_t w) { return kEqual ? __hge2(Pair(w), h) : __hgt2(Pair(w), h); };
    __half2 n = __half2half2(__ushort_as_half(0));
#pragma unroll
    for (int u = 0; u < kVectors; ++u)
      n = __hadd2(n, __hadd2(__hadd2(test(q[u].x), test(q[u].y)), __hadd2(test(q[u].z), test(q[u].w))));
    return static_cast<int>(__low2float(n) + __high2float(n));
  }
  static __device__ __forceinline__ uint32_t MaskAbove(const uint4& q, float x) {
    const __half2 h = __float2half2_rn(x);
    const uint32_t m = (__hgt2_mask(Pair(q.x), h) & 0x00020001u) | (__hgt2_mask(Pair(q.y), h) & 0x00080004u) |
                       (__hgt2_mask(Pair(q.z), h) & 0x00200010u) | (__hgt2_mask(Pair(q.w), h) & 0x00800040u);
    return (m | (m >> 16)) & 0xFFu;
  }
  static __device__ __forceinline__ float Pick(const uint4& q, int i) {
    const uint32_t w = i < 4 ? (i < 2 ? q.x : q.y) : (i < 6 ? q.z : q.w);
    return __half2float(__ushort_as_half(static_cast<uint16_t>(w >> (i & 1) * 16)));
  }
  static __device__ __forceinline__ float Below(float x) {
    const uint16_t h = __half_as_ushort(__float2half_rn(x));
    return __half2float(__ushort_as_half(static_cast<uint16_t>(
        x > 0.0f ? h - 1 : x == 0.0f ? 0x8001 : h + 1)));
  }
};

// ------------------------------------------- short rows: one warp per item

constexpr int kWarps = 8;
constexpr int kWarpKeys = 64;

// The whole group sits in registers, value j in lane j % 32: a load, a
// maximum, an exponential, two comparisons and a handful of sums for a value.
// What bounds it is the instructions (35 for a value of 8 x 1,025 with five
// alternatives, what a row costs once among them; 12 bytes of a thread spill),
// with the loads' latency hidden by the SM's 32 warps.
template <typename T, int kPer>
__global__ void __launch_bounds__(kWarps * 32, kPer <= 33 ? 4 : 2)
    logprobs_warp_kernel(const LogprobArgs a) {
  using R = Row<T>;
  constexpr int kMasks = (kPer + 31) / 32;
  __shared__ uint64_t s_keys[kWarps][kWarpKeys];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= a.rows * a.codebooks) return;
  const int64_t row = Quotient(item, a.codebooks);
  const int codebook = static_cast<int>(item - row * a.codebooks);
  const int64_t out = codebook * a.rows + row;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + static_cast<int64_t>(codebook) * a.vocab;
  float x[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = lane + 32 * i;
    x[i] = j < a.vocab ? ToFloat(src[j]) : -INFINITY;
  }
  const int target = Target(a, out, lane == 0);
  const float xt = target >= 0 ? ToFloat(src[target]) : INFINITY;
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
  const float scaled = R::Scaled(m);
  float z = 0.0f, w = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    // Finite, so that 0 * t is 0 for a closed token.
    const float t = fmaxf(R::Exponent(x[i], scaled), -16384.0f);
    const float e = Exp2Approx(t);
    z += e;
    w = fmaf(e, t, w);
  }
  z = warp_sum(z);
  w = warp_sum(w);
  const float log_z = logf(z);
  int ahead = 0;
  if (a.rank != nullptr && target >= 0) {
    bool equal = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      ahead += x[i] > xt ? 1 : 0;
      equal |= x[i] == xt;
    }
    // More lanes than the target's hold its value, or that one may hold it
    // twice: those with a lower index are ahead as well.
    if (__popc(__ballot_sync(0xFFFFFFFFu, equal)) > 1 || xt == -INFINITY) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) ahead += x[i] == xt && lane + 32 * i < target ? 1 : 0;
    } else if (equal) {
      for (int j = lane; j < target; j += 32) ahead += ToFloat(src[j]) == xt ? 1 : 0;
    }
    ahead = __reduce_add_sync(0xFFFFFFFFu, ahead);
  }
  if (lane == 0) {
    a.logprob[out] = target >= 0 ? R::LogProb(xt, m, log_z) : 0.0f;
    if (a.entropy != nullptr) a.entropy[out] = fmaf(w / z, -kLn2, log_z);
    if (a.rank != nullptr) a.rank[out] = target >= 0 ? ahead : -1;
  }
  const int k = a.top_k;
  if (k == 0) return;
  int32_t* ids = a.top_ids + out * k;
  float* logprobs = a.top_logprobs + out * k;
  // k lanes hold a value of at least the k-th greatest lane maximum.  Taking
  // maxima one after the other is shorter than a sort up to about eight.
  const float threshold = k <= 8 ? WarpKthOfFew(top, k) : WarpKth(top, k);
  uint32_t masks[kMasks] = {};  // bit i % 32 of masks[i / 32]: x[i] passes
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (x[i] >= threshold) masks[i / 32] |= 1u << (i % 32);
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kMasks; ++i) {
    // Values behind the group pass only where -inf does.
    const int valid = (a.vocab - lane + 31) / 32 - 32 * i;
    masks[i] &= valid >= 32 ? ~0u : valid <= 0 ? 0u : (1u << valid) - 1u;
    mine += __popc(masks[i]);
  }
  int at = mine;  // inclusive, then exclusive count of the lanes before
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int before = __shfl_up_sync(0xFFFFFFFFu, at, o);
    if (lane >= o) at += before;
  }
  const int n = __shfl_sync(0xFFFFFFFFu, at, 31);
  at -= mine;
  if (n <= kWarpKeys) {
    uint64_t* keys = s_keys[threadIdx.x >> 5];
#pragma unroll
    for (int i = 0; i < kMasks; ++i) {
      uint32_t mask = masks[i];
      while (mask != 0) {
        const int j = lane + 32 * (32 * i + __ffs(mask) - 1);
        mask &= mask - 1;
        keys[at++] = AlternativeKey(ToFloat(src[j]), j);
      }
    }
    __syncwarp();
    const uint64_t k0 = lane < n ? keys[lane] : 0, k1 = lane + 32 < n ? keys[lane + 32] : 0;
    int r0 = 0, r1 = 0;
    for (int j = 0; j < n; ++j) r0 += keys[j] > k0 ? 1 : 0;
    if (n > 32)
      for (int j = 0; j < n; ++j) r1 += keys[j] > k1 ? 1 : 0;
    if (k0 != 0 && r0 < k) {
      ids[r0] = KeyIndex(k0);
      logprobs[r0] = R::LogProb(KeyValue(k0), m, log_z);
    }
    if (k1 != 0 && r1 < k) {
      ids[r1] = KeyIndex(k1);
      logprobs[r1] = R::LogProb(KeyValue(k1), m, log_z);
    }
    return;
  }
  // Many equal or closed values: one alternative after the other.
  uint64_t last = ~uint64_t{0};
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    for (int j = lane; j < a.vocab; j += 32) {
      const uint64_t key = AlternativeKey(ToFloat(src[j]), j);
      if (key < last && key > best) best = key;
    }
    last = WarpMaxKey(best);
    if (lane == 0) {
      ids[r] = KeyIndex(last);
      logprobs[r] = R::LogProb(KeyValue(last), m, log_z);
    }
  }
}

// ------------------------------ long rows: one CTA, or a cluster, per item

constexpr int kKeys = 1024;      // room for passing values between prunings

// Running maximum, Z = sum 2^t and W = sum 2^t t of what was read, with
// t = Row<T>::Exponent(x, m).
struct RowStats {
  float m, z, w;
};

// To a maximum m >= s.m.
template <typename T>
__device__ __forceinline__ void Rebase(RowStats& s, float m) {
  if (s.m != -INFINITY) {
    const float d = fmaxf(Row<T>::Step(s.m, m), -16384.0f);
    const float f = Exp2Approx(d);
    s.w = f * fmaf(d, s.z, s.w);
    s.z *= f;
  }
  s.m = m;
}
// The whole warp's sums, in all lanes; in a fixed order.
template <typename T>
__device__ __forceinline__ void MergeWarp(RowStats& s) {
  float top = s.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = MaxNan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (!(fabsf(top) < INFINITY)) {  // nothing yet, or no distribution
    s.m = top;
    return;
  }
  Rebase<T>(s, top);
  s.z = warp_sum(s.z);
  s.w = warp_sum(s.w);
}

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

template <int kThreads>
struct LongShared {
  uint64_t keys[kKeys];
  uint64_t sorted[8 * kMaxTopK];
  uint64_t warp_key[kThreads / 32];
  float fourth[kThreads / 32];
  RowStats stats[kThreads / 32];
  int ahead[kThreads / 32];
  RowStats total;
  int total_ahead;
  int count;
  float threshold;
};

// Leaves the top_k greatest of the keys in order in keys[0 ..) and sets count
// and threshold; `slots` slots hold `present` keys, the others 0.  Every
// thread calls it, after a barrier.
template <int kThreads>
__device__ __forceinline__ void Prune(LongShared<kThreads>& s, int k, int slots, int present) {
  // Four lanes count the keys ahead of one.
  const int lanes = threadIdx.x & 3;
  for (int i0 = 0; i0 < slots; i0 += kThreads / 4) {
    const int i = i0 + (threadIdx.x >> 2);
    const uint64_t key = i < slots ? s.keys[i] : 0;
    int r = 0;
#pragma unroll 4
    for (int j = lanes; j < slots; j += 4) r += s.keys[j] > key ? 1 : 0;
    r += __shfl_xor_sync(0xFFFFFFFFu, r, 1);
    r += __shfl_xor_sync(0xFFFFFFFFu, r, 2);
    if (key != 0 && lanes == 0 && r < k) s.sorted[r] = key;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < min(present, k)) s.keys[threadIdx.x] = s.sorted[threadIdx.x];
  if (threadIdx.x == 32) {
    s.count = min(present, k);
    s.threshold = present >= k ? KeyValue(s.sorted[k - 1]) : -INFINITY;
  }
  __syncthreads();
}

// Threads: 256 (four CTAs an SM hide one another's barriers), or 512 for the
// few rows that clusters share, whose time is that of one chunk after another.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    logprobs_long_kernel(const LogprobArgs a, int cluster) {
  using R = Row<T>;
  constexpr int kE = R::kN;
  __shared__ LongShared<kThreads> s;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(cluster));
  const int64_t item = blockIdx.x / static_cast<unsigned>(cluster);
  const int64_t row = Quotient(item, a.codebooks);
  const int codebook = static_cast<int>(item - row * a.codebooks);
  const int64_t out = codebook * a.rows + row;
  const T* src = static_cast<const T*>(a.logits) + row * a.ld + static_cast<int64_t>(codebook) * a.vocab;
  const int k = a.top_k;
  // Up to the first 16-byte boundary and behind the last whole vector: the
  // row's ends, read value by value, the first end before and the last one
  // behind the vectors (alternatives arrive by ascending index).
  const int head = min(a.vocab, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(src) & 15u)) % 16u /
                                                 sizeof(T)));
  const uint4* base = reinterpret_cast<const uint4*>(src + head);
  const int vectors = (a.vocab - head) / kE;
  const int per = (vectors + cluster - 1) / cluster;
  const int begin = part * per, end = min(vectors, begin + per);
  constexpr int kStep = kThreads * kVectors;  // vectors of a chunk
  auto load = [&](int v0, uint4 (&q)[kVectors]) {
    const uint4* p = base + v0 + tid;
    if (v0 + kStep <= end) {
#pragma unroll
      for (int u = 0; u < kVectors; ++u) q[u] = __ldg(p + u * kThreads);
    } else {
#pragma unroll
      for (int u = 0; u < kVectors; ++u)
        q[u] = v0 + u * kThreads + tid < end ? __ldg(p + u * kThreads) : R::Closed();
    }
  };
  uint4 next[kVectors];
  load(begin, next);
  const int target = Target(a, out, tid == 0 && part == 0);
  const float xt = target >= 0 ? ToFloat(src[target]) : 0.0f;
  const bool ranks = a.rank != nullptr && target >= 0;
  if (tid == 0) {
    s.count = 0;
    s.threshold = -INFINITY;
  }
  __syncthreads();

  RowStats st = {-INFINITY, 0.0f, 0.0f};
  int ahead = 0;
  auto grow = [&](float top) {  // NaN or +inf stays: no distribution
    const float grown = MaxNan(st.m, top);
    if (grown == st.m) return;
    if (fabsf(grown) < INFINITY) Rebase<T>(st, grown);
    else st.m = grown;
  };
  auto push = [&](float x, int j) {
    const int at = atomicAdd(&s.count, 1);
    if (at < kKeys) s.keys[at] = AlternativeKey(x, j);
  };
  // One value of the row's ends, for threads below 8.
  auto scalar = [&](int j, float threshold) {
    const float x = ToFloat(src[j]);
    grow(x);
    if (fabsf(st.m) < INFINITY) {
      const float t = fmaxf(R::Exponent(x, R::Scaled(st.m)), -16384.0f);
      const float p = Exp2Approx(t);
      st.z += p;
      st.w = fmaf(p, t, st.w);
    }
    ahead += ranks && (x > xt || (x == xt && j < target)) ? 1 : 0;
    if (k > 0 && x > threshold) push(x, j);
  };
  // Leaves the k best so far in order in s.keys, and their threshold.  Values
  // [low, high) came since the last time.
  auto settle = [&](int low, int high) {
    __syncthreads();
    if (s.count > kKeys) {
      // No room (many equal values, or rising ones): the best of these and of
      // the keys from before, one after the other.
      uint64_t last = ~uint64_t{0};
      for (int r = 0; r < k; ++r) {
        uint64_t best = 0;
        for (int i = tid; i < kKeys; i += kThreads) {
          const uint64_t key = s.keys[i];
          if (KeyIndex(key) < low && key < last && key > best) best = key;
        }
        for (int j = low + tid; j < high; j += kThreads) {
          const float x = ToFloat(src[j]);
          const uint64_t key = x > -INFINITY ? AlternativeKey(x, j) : 0;
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
      Prune(s, k, s.count, s.count);
    }
  };
  if (part == 0) {
    if (tid < head) scalar(tid, -INFINITY);
    __syncthreads();  // the row's first keys are stored, whatever follows
  }
  int settled = head + begin * kE;  // values below are in order in s.keys
  int chunk = 0;
  for (int v0 = begin; v0 < end; v0 += kStep, ++chunk) {
    uint4 q[kVectors];
#pragma unroll
    for (int u = 0; u < kVectors; ++u) q[u] = next[u];
    if (v0 + kStep < end) load(v0 + kStep, next);
    const float top = R::Top(q);
    grow(top);
    if (fabsf(st.m) < INFINITY) {
      const float scaled = R::Scaled(st.m);
#pragma unroll
      for (int u = 0; u < kVectors; ++u) {
        float2 z = {0.0f, 0.0f}, w = {0.0f, 0.0f};  // of one vector: longer sums lose less
#pragma unroll
        for (int e = 0; e < kE; e += 2) {
          const float2 t = R::Exponents(q[u], e, scaled);
          const float2 p = make_float2(Exp2Approx(t.x), Exp2Approx(t.y));
          z = add2(z, p);
          w = fma2(p, t, w);
        }
        st.z += z.x + z.y;
        st.w += w.x + w.y;
      }
    }
    if (ranks) {
      // Ahead of the target an equal value counts, behind it none; closed
      // values behind the part's end must not count as equal ones.
      const int low = head + v0 * kE, high = low + kStep * kE;
      if (low > target) {
        ahead += R::template Above<false>(q, xt);
      } else if (high <= target && high <= head + end * kE) {
        ahead += R::template Above<true>(q, xt);
      } else {
#pragma unroll 1
        for (int u = 0; u < kVectors; ++u) {
          const int v = v0 + u * kThreads + tid, j = head + v * kE;
          if (v >= end) break;
          const uint4 vector = __ldg(base + v);
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float x = R::At(vector, e);
            ahead += x > xt || (x == xt && j + e < target) ? 1 : 0;
          }
        }
      }
    }
    if (k == 0) continue;
    // The first values take their threshold from the threads' maxima: in each
    // of ceil(k / 4) warps four lanes hold a value of at least the warp's
    // fourth greatest maximum.
    // Later values lose to an equal earlier one, so they have to be greater.
    float threshold;
    if (chunk == 0) {
      const float fourth = WarpKthOfFew(top, 4);
      if (lane == 0) s.fourth[warp] = fourth;
      __syncthreads();
      threshold = WarpKthOfFew(lane < kThreads / 32 ? s.fourth[lane] : -INFINITY, (k + 3) / 4);
      if (threshold > -INFINITY) threshold = R::Below(threshold);
    } else {
      threshold = s.threshold;
    }
    if (top > threshold) {
      uint32_t masks[kVectors];
      int n = 0;
#pragma unroll
      for (int u = 0; u < kVectors; ++u) {
        masks[u] = R::MaskAbove(q[u], threshold);
        n += __popc(masks[u]);
      }
      int at = atomicAdd(&s.count, n);
#pragma unroll
      for (int u = 0; u < kVectors; ++u) {
        uint32_t mask = masks[u];
        const int j = head + (v0 + u * kThreads + tid) * kE;
        while (mask != 0) {
          const int e = __ffs(mask) - 1;
          mask &= mask - 1;
          if (at < kKeys) s.keys[at] = AlternativeKey(R::Pick(q[u], e), j + e);
          ++at;
        }
      }
    }
    // After chunks 1, 2, 4, 8, ...: about top_k values pass in between.  Over
    // 512 half rows of 151,936 values this took 61 us, settling after every
    // chunk 70 us and after chunks 1, 4, 16, ... 79 us.
    if ((chunk & (chunk + 1)) == 0 && v0 + kStep < end) {
      const int high = head + min(end, v0 + kStep) * kE;
      settle(settled, high);
      settled = high;
    }
  }
  const bool row_end = part == cluster - 1;
  if (row_end && head + vectors * kE + tid < a.vocab) scalar(head + vectors * kE + tid, s.threshold);
  if (k > 0) settle(settled, row_end ? a.vocab : head + end * kE);

  // The CTA's sums.
  MergeWarp<T>(st);
  ahead = __reduce_add_sync(0xFFFFFFFFu, ahead);
  if (lane == 0) {
    s.stats[warp] = st;
    s.ahead[warp] = ahead;
  }
  __syncthreads();
  if (warp == 0) {
    RowStats total = {-INFINITY, 0.0f, 0.0f};
    int sum = 0;
    if (lane < kThreads / 32) {
      total = s.stats[lane];
      sum = s.ahead[lane];
    }
    MergeWarp<T>(total);
    sum = __reduce_add_sync(0xFFFFFFFFu, sum);
    if (lane == 0) {
      s.total = total;
      s.total_ahead = sum;
    }
  }
  if (cluster > 1) {
    __syncthreads();
    cluster_sync();
    if (part == 0) {
      if (warp == 0) {  // lane p: part p's sums
        RowStats total = {-INFINITY, 0.0f, 0.0f};
        int sum = 0;
        if (lane < cluster) {
          const uint32_t at = mapa_shared(smem_u32(&s.total), lane);
          total.m = __uint_as_float(LoadCluster32(at));
          total.z = __uint_as_float(LoadCluster32(at + 4));
          total.w = __uint_as_float(LoadCluster32(at + 8));
          sum = static_cast<int>(LoadCluster32(mapa_shared(smem_u32(&s.total_ahead), lane)));
        }
        MergeWarp<T>(total);
        sum = __reduce_add_sync(0xFFFFFFFFu, sum);
        __syncwarp();
        if (lane == 0) {
          s.total = total;
          s.total_ahead = sum;
        }
      }
      // The other parts' alternatives behind this one's.  Parts hold ascending
      // indices, and the keys order ties.
      if (k > 0) {
        const int own = s.count, others = (cluster - 1) * k;
        int found = 0;
        for (int i0 = 0; i0 < others; i0 += kThreads) {  // the same turns for all threads
          const int i = i0 + tid, peer = 1 + i / k, at = i % k;
          uint64_t key = 0;
          if (i < others) {
            const int n = static_cast<int>(LoadCluster32(mapa_shared(smem_u32(&s.count), peer)));
            key = LoadCluster64(mapa_shared(smem_u32(&s.keys[at]), peer));
            if (at >= n) key = 0;
            s.keys[own + i] = key;
          }
          found += __syncthreads_count(key != 0);
        }
        Prune(s, k, own + others, own + found);
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
    a.logprob[out] = target >= 0 ? R::LogProb(xt, total.m, log_z) : 0.0f;
    if (a.entropy != nullptr)
      a.entropy[out] = fmaf(total.w / total.z, -kLn2, log_z);
    if (a.rank != nullptr) a.rank[out] = target >= 0 ? s.total_ahead : -1;
  }
  const int n = min(s.count, k);
  if (tid < n) {
    a.top_ids[out * k + tid] = KeyIndex(s.keys[tid]);
    a.top_logprobs[out * k + tid] = R::LogProb(KeyValue(s.keys[tid]), total.m, log_z);
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
  // Few rows: up to eight CTAs of a cluster share one, while each has vectors
  // for all of its threads and they fit the SMs twice over, or, with four
  // chunks for each and more, four times (an SM holds four).  One row of
  // 151,936 floats, with CTAs of 256 threads: 17.5 us with eight of them, 19.6
  // with sixteen (eight of 512 threads: 12.6); 100 such rows:
  // 22.3 us with four, 26.1 us with two; 64 rows of 32,000: 10.5 us with four,
  // 13.7 us with eight.
  constexpr int kVector = Row<T>::kN;
  int cluster = 1;
  while (cluster < 8 && a.vocab >= cluster * 2 * 256 * kVector) {
    const bool long_parts = a.vocab >= cluster * 2 * 4 * 256 * kVectors * kVector;
    if (items * cluster * 2 > (long_parts ? 4 : 2) * SmCount()) break;
    cluster *= 2;
  }
  // Large CTAs where all fit at once and have chunks enough.
  const bool large = items * cluster <= SmCount() && a.vocab >= cluster * 2 * 256 * kVectors * kVector;
  LaunchEx(large ? logprobs_long_kernel<T, 512> : logprobs_long_kernel<T, 256>,
           dim3(static_cast<unsigned>(items * cluster)), dim3(large ? 512 : 256), 0, stream, what,
           static_cast<unsigned>(cluster), a, cluster);
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
