// Grouped-query attention over the paged 8-bit key/value cache
// (ov_attention_kv_cache).
//
// With codes K', V' and scales a (keys) and b (values) of a token's page,
//   out = sum_j p_j b_j V'_j / sum_j p_j,   p_j = 2^(c_j q . K'_j),
//   c_j = scale * log2(e) * a_j.
// The value scale goes into the exponent: P_j = 2^(c_j q . K'_j + log2 b_j - m)
// is p_j b_j relative to the row's largest, so out = (sum P_j V'_j) /
// (sum P_j / b_j), and both products take the codes themselves, which are
// exact in half.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "attention_device.cuh"
#include "internal.hpp"
#include "kv_cache.hpp"
#include "launch.hpp"
#include "ov_kernels.h"
#include "ptx.cuh"

namespace ovb {
namespace {

// Division of 0 <= n < 2^31 by d through a multiplication (Granlund &
// Montgomery, "Division by invariant integers using multiplication", 1994).
struct FastDiv {
  int d;
  uint32_t mul, shift;
  explicit FastDiv(int divisor) : d(divisor), mul(0), shift(0) {
    while ((1ll << shift) < d) ++shift;
    mul = static_cast<uint32_t>((((1ull << shift) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), mul) + n) >> shift);
  }
};

struct CacheAttnArgs {
  CacheView cache;
  const __half* q;
  int64_t ld_q;
  __half* out;
  int64_t ld_out;
  const int32_t* cu_rows;
  const int32_t* lengths;
  int rows;
  int max_rows;
  int max_length;
  FastDiv group;  // heads / kv_heads
  int causal;
  float scale_log2;  // softmax scale * log2(e)
  uint32_t* err;
};

// Stands for a value scale below it, 0 above all, whose log2 the exponent
// could not take: such codes add nothing that a half could hold (128 * 2^-33
// is a quarter of the least one and rounds to 0, as what they stand for does),
// but their tokens count in the denominator.  The least scale that a page of
// halves is written with is 2^-24 / 127, four times as large.
constexpr float kLeastScale = 0x1.0p-33f;

// log2 and inverse of a value scale.  A NaN one (or a negative one, which
// none is) makes the exponent NaN where it is seen, and must not reach a sum
// where it is not.
__device__ __forceinline__ void ValueScale(float scale, float* shift, float* inverse) {
  const float b = scale >= 0.0f && scale < kLeastScale ? kLeastScale : scale;
  *shift = __log2f(b);
  *inverse = b == b ? __fdividef(1.0f, b) : 0.0f;
}

// Tokens of a sequence, bounded by what the call announced.
__device__ __forceinline__ int CheckLength(const CacheAttnArgs& a, int length) {
  if (length < 0 || length > a.max_length) {
    atomicOr(a.err, kErrBadArgument);
    return length < 0 ? 0 : a.max_length;
  }
  return length;
}

// ------------------------------------------- few rows: keys streamed by warps
//
// Up to 16 query rows share a kv head (tokens x heads of the group), so the
// products have M or N of 8 to 16 and the time is that of reading the codes.
// Tensor memory and its 128-row tiles would be mostly padding; here the keys
// take the 16-row side of mma.sync instead, S^T = K Q^T and O^T = V^T P^T,
// and the rows its 8-column side.
//
// Work is cut into units of 32 keys of one item (sequence, kv head), numbered
// along heads and sequences, and every warp of the grid takes the same count
// of consecutive units, whatever the lengths, through a ring of its own (TMA,
// 128B swizzle).  Producer warps fill the rings, a lane for each: issuing a
// TMA load takes a warp about a hundred cycles, and done by the computing
// warps themselves it took as long as half a unit's products.  An item inside
// one warp's range is stored by it; one that spans warps is joined in shared
// memory when the CTA's warps are done, one that spans CTAs by the last of
// them to arrive, always over the parts in order.  When all items fit, each
// starts at a CTA of its own, which spares most of them the join across CTAs.
//
// Fragments straight from the swizzled tiles: lane 4g + c, MMA row g is key
// kappa(g) of a slab of 16 (and 8 + kappa(g)).  kappa puts neighbouring g
// into different halves of a 128-byte line, so that K reads (16 bytes of key
// g, dims 64 j + 16 c) and V reads (16 bytes of key kappa(2c), dims 16 g) are
// both free of bank conflicts.  The order of dims in the first product, and
// of keys in the second, is the same for both operands and needs no move.
//
// Measured on one B200: 64 sequences of up to 4,096 tokens, 16 heads over 8
// (303 MB of codes): 58 us, 5.2 TB/s; in its middle the kernel reads at the
// rate of a plain copy, the rest is about 4 us before the first keys arrive
// (lengths, page table, TMA, each waiting for the one before) and 4 us of
// joins.  4 sequences of 65,537 tokens, 16 heads over 2 (134 MB): 36 us, of
// which 18 for 15 units a warp, 5 before the first keys and 7 of joins.  One
// token over 705: 10 us, all of it such waits.  Spills 36 bytes a thread (52
// with two blocks of 8 rows).

constexpr int kUnit = 32;               // keys
constexpr int kUnitTile = kUnit * kCacheHeadDim;  // bytes of K or V of a unit
constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = kStreamWarps * 32;  // of the warps that compute
// Units of a warp where items get CTAs of their own: more make a short item's
// warps work longer, fewer split it over CTAs and add their join.  3 is for
// batches of short histories: 16 sequences of up to 700 tokens took 12.6 us
// with 2, 10.5 with 3, 11.7 with 4, and a CTA's 768 tokens hold a prompt of
// 705.  One sequence, whose items leave most of the GPU idle, is as fast or
// faster with 2: 8 kv heads over 300 / 1,500 / 8,192 tokens 8.7 / 11.0 / 12.5
// us with 2, 8.6 / 12.2 / 13.3 with 3, 9.5 / 13.4 / 13.9 with 4.
constexpr int kMinUnits = 3;

// Ring slot beside the codes: scales and pages of the unit's two 16-key
// slabs, and the barrier of all that arrives in the slot.
struct alignas(16) SlotInfo {
  float scale[4];  // key, value of slab 0, of slab 1
  int page[2];     // -1: nothing to see
  uint64_t full;
};

struct StreamArgs {
  CacheAttnArgs a;
  uint32_t* counters;  // of the item that goes on behind each CTA; null: no item is split
  float* parts;        // [CTA][2][JoinFloats(join_rows)]: of the item begun before, of the last
  int join_rows;       // rows of a (sequence, kv head) at most
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9},"
      " {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Bytes 2i, 2i + 1 (kSel 0x4140, 0x4342) of four codes offset by 128, as
// halves: 0x6400 | u is 1024 + u, less 1152 the code, all exact.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t CodePair(uint32_t offset_codes) {
  const uint32_t biased = __byte_perm(offset_codes, 0x64646464u, kSel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&biased),
                            __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ void cp_async_4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
// 16 bytes, or zeros where `there` is false (`src` is not read then).
__device__ __forceinline__ void cp_async_16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}

// Arrives on `bar` when this thread's cp.asyncs so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// A load that stays where it is written, ahead of its use.
__device__ __forceinline__ int load_early(const int32_t* p) {
  int v;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// Factor of a key scale in the exponent.  Not 0, which would make NaN of a
// hidden score's -inf: a page of zeros has scale 0 and scores 0, which any
// finite factor keeps, and scores that a smaller one tells apart are equal.
__device__ __forceinline__ float KeyFactor(float scale, float scale_log2) {
  const float factor = scale * scale_log2;
  return factor >= 0.0f && factor < 0x1.0p-126f ? 0x1.0p-126f : factor;
}

// Adds a part's maximum and sum (ms) to a row's; returns the factors of the
// O so far and of the part's O.
__device__ __forceinline__ float2 JoinFactors(float* top, float* sum, float2 ms) {
  const float grown = fmaxf(*top, ms.x);
  const float base = grown == -INFINITY ? 0.0f : grown;
  const float f = ex2_approx(*top - base), h = ex2_approx(ms.x - base);
  *sum = fmaf(ms.y, h, *sum * f);
  *top = grown;
  return make_float2(f, h);
}

// One (sequence, kv head).  Its units have numbers begin, begin + 1, ...; the
// next item's begin `room` behind its own.
struct ItemAt {
  int seq, head;
  int first, count, length;  // packed rows, tokens
  int units, room;
  int64_t begin;

  // The rows and units of `seq`: one unit (with nothing to see) where rows
  // need their zeros, none without rows.
  __device__ __forceinline__ void Load(const CacheAttnArgs& a, int align) {
    const int from = a.cu_rows[seq], to = a.cu_rows[seq + 1], tokens = a.lengths[seq];
    const RowSpan span = CheckRows(from, to, a.rows, a.max_rows, a.err);
    first = span.first;
    count = span.count;
    length = CheckLength(a, tokens);
    units = count == 0 ? 0 : max(1, (length - 1) / kUnit + 1);
    room = (units + align - 1) / align * align;
  }
  __device__ __forceinline__ int64_t end() const { return begin + units; }
  // To the next one that has units; false behind the last.
  __device__ __forceinline__ bool Next(const CacheAttnArgs& a, int align) {
    begin += room;
    if (++head < a.cache.kv_heads) return true;
    head = 0;
    while (++seq < a.cache.num_seqs) {
      Load(a, align);
      if (units > 0) return true;
    }
    return false;
  }
};

struct alignas(16) StreamShared {
  ItemAt group[kStreamWarps + 1];  // items to join: one begun before the CTA, then by warp
  int rows[kStreamWarps + 1];      // their rows; 0: none
  ItemAt part[2];                  // items that this CTA shares with others
  int has[2], last[2];
};

template <int kNT>
constexpr int StreamStages() {
  return kNT == 1 ? 3 : 2;
}
// A part of an item with `rows` query rows: O, then maxima and sums.
__host__ __device__ constexpr size_t JoinFloats(int rows) {
  return (static_cast<size_t>(rows) * (kCacheHeadDim + 2) + 3) / 4 * 4;
}
template <int kNT>
constexpr size_t StreamSmem(int rows) {
  return 1024 + static_cast<size_t>(StreamStages<kNT>()) * kStreamWarps *
                    (2 * kUnitTile + sizeof(SlotInfo) + sizeof(uint64_t)) +
         sizeof(StreamShared) + kStreamWarps * JoinFloats(rows) * sizeof(float);
}

// n / d, in 32 bits where they hold it.
__device__ __forceinline__ int64_t Divide(int64_t n, int64_t d) {
  if (((n | d) >> 31) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

// Sum of a value over the warp; `before`: over the lanes before this one.
__device__ __forceinline__ int64_t WarpSum(int64_t mine, int64_t* before) {
  int64_t inclusive = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xFFFFFFFFu, inclusive, o);
    if ((threadIdx.x & 31) >= o) inclusive += v;
  }
  *before = inclusive - mine;
  return __shfl_sync(0xFFFFFFFFu, inclusive, 31);
}

// How the units are numbered and shared out; every warp works it out for
// itself, lane i from sequences [i * per, (i + 1) * per).
struct Division {
  ItemAt item;       // the lane's only sequence, where per is 1
  int per;
  int align;         // room of an item is a multiple of this
  int64_t width;     // numbers of a warp
  int64_t begin, end;  // of the lane's sequences

  __device__ __forceinline__ explicit Division(const CacheAttnArgs& a) {
    const int lane = threadIdx.x & 31, seqs = a.cache.num_seqs;
    per = (seqs + 31) / 32;
    const int first = min(seqs, lane * per), last = min(seqs, first + per);
    int64_t mine = 0, before;
    item.units = 0;
    for (item.seq = first; item.seq < last; ++item.seq) {
      item.Load(a, 1);
      mine += item.units;
    }
    const int64_t units = WarpSum(mine, &before) * a.cache.kv_heads;
    width = Divide(units + gridDim.x * kStreamWarps - 1, gridDim.x * kStreamWarps);
    align = 1;
    // Items with a begin of their own at a CTA, if they all fit.
    if (seqs * a.cache.kv_heads <= static_cast<int>(gridDim.x)) {
      const int wide = static_cast<int>(max(width, static_cast<int64_t>(kMinUnits))) * kStreamWarps;
      int64_t ctas = 0, ctas_before;
      if (per == 1) {
        ctas = (item.units + wide - 1) / wide;
      } else {
        for (item.seq = first; item.seq < last; ++item.seq) {
          item.Load(a, wide);
          ctas += item.room / wide;
        }
      }
      const int64_t all = WarpSum(ctas, &ctas_before) * a.cache.kv_heads;
      if (all <= gridDim.x) {
        align = wide;
        width = wide / kStreamWarps;
        mine = ctas * align;
        before = ctas_before * align;
      }
    }
    if (per == 1) {
      item.seq = first;
      item.room = static_cast<int>(mine);
    }
    begin = before * a.cache.kv_heads;
    end = begin + mine * a.cache.kv_heads;
  }

  // The item at number p (the same in all lanes); seq -1 behind the last.
  __device__ __forceinline__ ItemAt Find(const CacheAttnArgs& a, int64_t p) const {
    ItemAt at;
    at.seq = -1;
    const uint32_t here = __ballot_sync(0xFFFFFFFFu, begin <= p && p < end);
    if (here == 0) return at;
    const int lane = __ffs(here) - 1;
    at.begin = __shfl_sync(0xFFFFFFFFu, begin, lane);
    if (per == 1) {
      at.seq = __shfl_sync(0xFFFFFFFFu, item.seq, lane);
      at.first = __shfl_sync(0xFFFFFFFFu, item.first, lane);
      at.count = __shfl_sync(0xFFFFFFFFu, item.count, lane);
      at.length = __shfl_sync(0xFFFFFFFFu, item.length, lane);
      at.units = __shfl_sync(0xFFFFFFFFu, item.units, lane);
      at.room = __shfl_sync(0xFFFFFFFFu, item.room, lane);
    } else {
      for (at.seq = lane * per;; ++at.seq) {
        at.Load(a, align);
        const int64_t heads = static_cast<int64_t>(at.room) * a.cache.kv_heads;
        if (p < at.begin + heads) break;
        at.begin += heads;
      }
    }
    at.head = static_cast<int>(Divide(p - at.begin, at.room));
    at.begin += static_cast<int64_t>(at.head) * at.room;
    return at;
  }
};

template <int kNT>
__global__ void __launch_bounds__(kStreamThreads + 128, 1)
    cache_attention_stream_kernel(const __grid_constant__ CUtensorMap map_k,
                                  const __grid_constant__ CUtensorMap map_v,
                                  const StreamArgs args) {
  constexpr int kStages = StreamStages<kNT>();
  const CacheAttnArgs& a = args.a;
  const CacheView& cache = a.cache;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
  const int g = lane >> 2, c = lane & 3;
  // The rings of this warp, or (producers) of the one that this lane serves.
  const bool producer = warp >= kStreamWarps;
  const int mine_warp = producer ? (warp - kStreamWarps) * 2 + (lane & 1) : warp;
  uint8_t* ring = smem + mine_warp * (kStages * 2 * kUnitTile);
  SlotInfo* info = reinterpret_cast<SlotInfo*>(smem + kStreamWarps * kStages * 2 * kUnitTile) +
                   mine_warp * kStages;
  uint64_t* empty = reinterpret_cast<uint64_t*>(
                        smem + kStreamWarps * kStages * (2 * kUnitTile + sizeof(SlotInfo))) +
                    mine_warp * kStages;
  StreamShared& shared = *reinterpret_cast<StreamShared*>(
      smem + kStreamWarps * kStages * (2 * kUnitTile + sizeof(SlotInfo) + sizeof(uint64_t)));
  float* join = reinterpret_cast<float*>(&shared + 1);  // [warp][JoinFloats(join_rows)]
  const size_t join_floats = JoinFloats(args.join_rows);
  const int stats = args.join_rows * kCacheHeadDim;  // of a part: maxima and sums
  pdl_trigger();
  if (producer && lane < 2) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&info[i].full, 2);  // for the codes and for the scales
      mbar_init(&empty[i], 1);
    }
    fence_mbar_init();
    if (warp == kStreamWarps) {
      tma_prefetch_map(lane == 0 ? &map_k : &map_v);
      shared.has[lane] = 0;
    }
  }
  pdl_wait();

  // This warp's numbers [p0, p1), of the CTA's from `base` on, and the item
  // at p0 (producers: those of the lane's warp).
  ItemAt item;
  int align = 1;
  int64_t width, base, p0, p1;
  if (args.counters == nullptr) {  // the CTA has an item to itself
    item.seq = static_cast<int>(blockIdx.x) / cache.kv_heads;
    item.head = static_cast<int>(blockIdx.x) % cache.kv_heads;
    item.begin = 0;
    item.Load(a, 1);
    if (item.units == 0) return;  // uniform over the CTA
    width = (item.units + kStreamWarps - 1) / kStreamWarps;
    base = 0;
    // The CTA's numbers end with its item: the next one is another CTA's.
    p0 = mine_warp * width;
    p1 = min(p0 + width, static_cast<int64_t>(item.units));
    if (p0 >= item.units) item.seq = -1;
  } else {
    const Division division(a);
    align = division.align;
    width = division.width;
    base = width * kStreamWarps * blockIdx.x;
    p0 = base + mine_warp * width;
    p1 = p0 + width;
    item = division.Find(a, __shfl_sync(0xFFFFFFFFu, p0, 0));
    if (producer) {
      const ItemAt second = division.Find(a, __shfl_sync(0xFFFFFFFFu, p0, 1));
      if (lane & 1) item = second;
    }
  }
  __syncthreads();  // the barriers are initialised

  // Registers: 384 threads start with 168 each.  The warpgroups that compute
  // take 224 and leave the producer's 56.
  if (producer) {
    registers_shrink<56>();
    // Lanes 0 and 1 fill a warp's ring each: the codes of a unit (one box, or two of 16
    // keys), its scales and pages, the page numbers looked up one unit ahead.
    const int box = min(kUnit, 1 << cache.page_shift);  // rows of a TMA box
    int64_t at = lane < 2 && item.seq >= 0 ? p0 : p1;
    int page[2] = {-1, -1}, tokens = 0, sent = 0;
    auto look_up = [&] {
      while (at < p1 && at >= item.end()) at = item.Next(a, align) ? item.begin : p1;
      if (at >= p1) return;
      const int token = static_cast<int>(at - item.begin) * kUnit;
      tokens = item.length - token;
      const int32_t* table = cache.table + static_cast<int64_t>(item.seq) * cache.max_pages;
      if (tokens > 0) page[0] = load_early(table + (token >> cache.page_shift));
      if (tokens > 16 && box < kUnit) page[1] = load_early(table + ((token + 16) >> cache.page_shift));
    };
    look_up();
    uint64_t idle_since = 0;
    while (__any_sync(0xFFFFFFFFu, at < p1)) {
      const int stage = sent % kStages;
      // Free, and what was copied there before has landed: a warp that gave up
      // waiting for it frees the slot without.
      const uint32_t used = static_cast<uint32_t>(sent / kStages - 1) & 1u;
      const bool ready = at < p1 && (sent < kStages || (mbar_test_wait(&empty[stage], used) &&
                                                        mbar_test_wait(&info[stage].full, used)));
      if (ready) {
        int now[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // the pages of the unit's slabs
          now[h] = tokens > h * 16 ? page[box < kUnit ? h : 0] : -1;
          if (tokens > h * 16 && (now[h] < 0 || now[h] >= cache.pages)) {
            atomicOr(a.err, kErrBadArgument);
            now[h] = -1;
          }
          info[stage].page[h] = now[h];
          if (now[h] >= 0) {
            const int64_t scale = static_cast<int64_t>(now[h]) * cache.kv_heads + item.head;
            cp_async_4(&info[stage].scale[2 * h], cache.key_scales + scale);
            cp_async_4(&info[stage].scale[2 * h + 1], cache.value_scales + scale);
          } else {
            info[stage].scale[2 * h] = info[stage].scale[2 * h + 1] = 1.0f;
          }
        }
        const int loads = (now[0] >= 0) + (box < kUnit && now[1] >= 0);
        mbar_arrive_expect_tx(&info[stage].full, static_cast<uint32_t>(2 * loads * box * kCacheHeadDim));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (now[h] < 0 || (h == 1 && box == kUnit)) continue;
          const int token = static_cast<int>(at - item.begin) * kUnit + h * 16;
          const int row = ((now[h] * cache.kv_heads + item.head) << cache.page_shift) +
                          (token & ((1 << cache.page_shift) - 1));
          uint8_t* dst = ring + stage * 2 * kUnitTile + h * 16 * kCacheHeadDim;
          tma_load_2d(dst, &map_k, &info[stage].full, 0, row);
          tma_load_2d(dst + kUnitTile, &map_v, &info[stage].full, 0, row);
        }
        cp_async_arrive(&info[stage].full);
        ++sent;
        ++at;
        look_up();
      }
      // Bounded: warps that give up waiting still free their slots, so this
      // one ends too.
      if (__any_sync(0xFFFFFFFFu, ready)) {
        idle_since = 0;
      } else if (idle_since == 0) {
        idle_since = global_timer_ns();
      } else if (global_timer_ns() - idle_since > 2 * kWaitLimitNs) {
        if (lane == 0) atomicOr(a.err, kErrWaitTimeout);
        break;
      }
    }
    cp_async_wait_all();
    // No copy outlives the CTA.
    for (int u = max(0, sent - kStages); u < sent; ++u)
      (void)mbar_wait(&info[u % kStages].full, static_cast<uint32_t>(u / kStages) & 1u, a.err);
    return;
  }
  registers_grow<224>();

  // kappa(g) and kappa(2c), see above.
  const int key_g = ((g & 1) << 2) | (g & 2) | (g >> 2);
  const int key_c = ((c & 1) << 1) | (c >> 1);
  // Lanes of c >= 2 read the later key of a pair first.
  const bool later = c >= 2;
  const uint32_t pair_lo = later ? 0x1504u : 0x5140u, pair_hi = later ? 0x3726u : 0x7362u;
  int k_at[2], v_at[2];  // byte offsets in a slab of this lane's first reads
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    k_at[j] = key_g * kCacheHeadDim + (((4 * j + c) ^ key_g) << 4);
    const int key = key_c + (later != (j == 1) ? 4 : 0);
    v_at[j] = key * kCacheHeadDim + ((g ^ key) << 4);
  }
  // Where row r of an item is stored.
  auto out_row = [&](const ItemAt& it, int r) {
    const int token = a.group(r);
    return a.out + static_cast<int64_t>(it.first + token) * a.ld_out +
           (it.head * a.group.d + r - token * a.group.d) * kCacheHeadDim;
  };

  const ItemAt started = item;
  int64_t at = p0;
  int done = 0;  // units of this warp so far
  bool ok = true;  // once a wait ran out, no other is begun
  bool tail = false;  // `item` goes on behind p1 and began here
  while (item.seq >= 0 && at < p1) {
    const int64_t end = min(p1, item.end());
    if (at < end) {
      const int rows = item.count * a.group.d;  // row r: token r / group, head r % group
      const bool begun = at == item.begin;
      float m[kNT][2], l[kNT][2], o[8][kNT][4];
      int seen[kNT][2];  // tokens that column 2c + e sees
      uint32_t q[2][4][kNT][2];
      const int least = a.causal ? item.length - item.count + 1 : item.length;
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
        const int r = t * 8 + g;
        const bool live = r < rows;
        const __half* src = a.q;
        if (live) {
          const int token = a.group(r);
          src += static_cast<int64_t>(item.first + token) * a.ld_q +
                 (item.head * a.group.d + r - token * a.group.d) * kCacheHeadDim + 16 * c;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint4 x = make_uint4(0, 0, 0, 0), y = x;
          if (live) {
            x = *reinterpret_cast<const uint4*>(src + 64 * j);
            y = *reinterpret_cast<const uint4*>(src + 64 * j + 8);
          }
          q[j][0][t][0] = x.x, q[j][0][t][1] = x.y;
          q[j][1][t][0] = x.z, q[j][1][t][1] = x.w;
          q[j][2][t][0] = y.x, q[j][2][t][1] = y.y;
          q[j][3][t][0] = y.z, q[j][3][t][1] = y.w;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          m[t][e] = -INFINITY;
          l[t][e] = 0.0f;
          const int column = t * 8 + 2 * c + e;
          seen[t][e] = a.causal && column < rows ? least + a.group(column) : item.length;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][t][e] = 0.0f;
      }
      for (; at < end; ++at) {
        const int stage = done % kStages;
        ok = ok && mbar_wait(&info[stage].full, static_cast<uint32_t>(done / kStages) & 1u, a.err);
        __syncwarp();
        const uint8_t* keys = ring + stage * 2 * kUnitTile;
        const uint8_t* values = keys + kUnitTile;
        const int token0 = static_cast<int>(at - item.begin) * kUnit;
        float s[2][kNT][4], shift[2], inverse[2];
        const float4 scales = *reinterpret_cast<const float4*>(info[stage].scale);
        const int2 pages = *reinterpret_cast<const int2*>(info[stage].page);
        const float factor[2] = {KeyFactor(scales.x, a.scale_log2), KeyFactor(scales.z, a.scale_log2)};
        ValueScale(scales.y, &shift[0], &inverse[0]);
        ValueScale(scales.w, &shift[1], &inverse[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < kNT; ++t) s[h][t][0] = s[h][t][1] = s[h][t][2] = s[h][t][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t x[2][2][4];  // slab, keys of rows g and g + 8
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(keys + (h * 16 + i * 8) * kCacheHeadDim + k_at[j]);
              x[h][i][0] = v.x ^ 0x80808080u;
              x[h][i][1] = v.y ^ 0x80808080u;
              x[h][i][2] = v.z ^ 0x80808080u;
              x[h][i][3] = v.w ^ 0x80808080u;
            }
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t f[4] = {CodePair<0x4140>(x[h][0][r]), CodePair<0x4140>(x[h][1][r]),
                                     CodePair<0x4342>(x[h][0][r]), CodePair<0x4342>(x[h][1][r])};
#pragma unroll
              for (int t = 0; t < kNT; ++t) mma_16816(s[h][t], f, q[j][r][t][0], q[j][r][t][1]);
            }
        }
        // Exponents, then the maximum, raised only when one passes it by 2^8.
        const bool partial = token0 + kUnit > least || pages.x < 0 || pages.y < 0;
        bool grow = false;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < kNT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& v = s[h][t][e];
              v = fmaf(v, factor[h], shift[h]);
              if (partial) {
                const int key = token0 + h * 16 + key_g + (e >> 1) * 8;
                if (key >= seen[t][e & 1] || (h == 0 ? pages.x : pages.y) < 0) v = -INFINITY;
              }
              grow |= v > m[t][e & 1] + 8.0f;
            }
        if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
          for (int t = 0; t < kNT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = fmaxf(fmaxf(s[0][t][e], s[0][t][e + 2]), fmaxf(s[1][t][e], s[1][t][e + 2]));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
              if (top > m[t][e]) {
                const float old = ex2_approx(m[t][e] - top);
                m[t][e] = top;
                l[t][e] *= old;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  o[i][t][e] *= old;
                  o[i][t][e + 2] *= old;
                }
              }
            }
        }
        uint32_t pb[2][kNT][2];
#pragma unroll
        for (int t = 0; t < kNT; ++t) {
          const float m0 = m[t][0] == -INFINITY ? 0.0f : m[t][0];
          const float m1 = m[t][1] == -INFINITY ? 0.0f : m[t][1];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float e0 = ex2_approx(s[h][t][0] - m0), e1 = ex2_approx(s[h][t][1] - m1);
            const float e2 = ex2_approx(s[h][t][2] - m0), e3 = ex2_approx(s[h][t][3] - m1);
            l[t][0] = fmaf(e0 + e2, inverse[h], l[t][0]);
            l[t][1] = fmaf(e1 + e3, inverse[h], l[t][1]);
            pb[h][t][0] = transpose_8x8(pack_half2(e0, e1));
            pb[h][t][1] = transpose_8x8(pack_half2(e2, e3));
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* p = values + h * 16 * kCacheHeadDim;
          const uint4 x0 = *reinterpret_cast<const uint4*>(p + v_at[0]);
          const uint4 x1 = *reinterpret_cast<const uint4*>(p + v_at[1]);
          const uint4 x2 = *reinterpret_cast<const uint4*>(p + v_at[0] + 8 * kCacheHeadDim);
          const uint4 x3 = *reinterpret_cast<const uint4*>(p + v_at[1] + 8 * kCacheHeadDim);
          const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
          const uint32_t w2[4] = {x2.x, x2.y, x2.z, x2.w}, w3[4] = {x3.x, x3.y, x3.z, x3.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t u0 = w0[r] ^ 0x80808080u, u1 = w1[r] ^ 0x80808080u;
            const uint32_t u2 = w2[r] ^ 0x80808080u, u3 = w3[r] ^ 0x80808080u;
#pragma unroll
            for (int b = 0; b < 2; ++b) {  // dims 16 g + 4 r + 2 b, and one more
              const uint32_t sel = b == 0 ? pair_lo : pair_hi;
              const uint32_t near = __byte_perm(u0, u1, sel), far = __byte_perm(u2, u3, sel);
              const uint32_t f[4] = {CodePair<0x4140>(near), CodePair<0x4342>(near),
                                     CodePair<0x4140>(far), CodePair<0x4342>(far)};
#pragma unroll
              for (int t = 0; t < kNT; ++t) mma_16816(o[2 * r + b][t], f, pb[h][t][0], pb[h][t][1]);
            }
          }
        }
        ++done;
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }

      // Out, or a part: of an item begun before p0 in `join`, of one that goes
      // on behind p1 in this warp's ring, which is idle by then.
      const bool whole = begun && end == item.end();
      tail = begun && !whole;
      float* part = tail ? reinterpret_cast<float*>(ring) : join + warp * join_floats;
#pragma unroll
      for (int t = 0; t < kNT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[t][e];
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
          const int r = t * 8 + 2 * c + e;
          if (r >= rows) continue;
          if (whole) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            uint4* dst = reinterpret_cast<uint4*>(out_row(item, r) + 16 * g);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              dst[i] = make_uint4(pack_half2(o[4 * i][t][e] * inv, o[4 * i][t][e + 2] * inv),
                                  pack_half2(o[4 * i + 1][t][e] * inv, o[4 * i + 1][t][e + 2] * inv),
                                  pack_half2(o[4 * i + 2][t][e] * inv, o[4 * i + 2][t][e + 2] * inv),
                                  pack_half2(o[4 * i + 3][t][e] * inv, o[4 * i + 3][t][e + 2] * inv));
          } else {
            float4* dst = reinterpret_cast<float4*>(part + r * kCacheHeadDim + 16 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              dst[i] = make_float4(o[2 * i][t][e], o[2 * i][t][e + 2], o[2 * i + 1][t][e],
                                   o[2 * i + 1][t][e + 2]);
            if (g == 0)
              *reinterpret_cast<float2*>(part + stats + 2 * r) = make_float2(m[t][e], sum);
          }
        }
    }
    at = min(p1, item.begin + item.room);
    if (at >= p1 || !item.Next(a, align)) break;
  }
  if (lane == 0) {
    shared.group[warp + 1] = item;
    shared.rows[warp + 1] = tail ? item.count * a.group.d : 0;
    if (warp == 0) {
      const bool begun_before = started.seq >= 0 && started.begin < base && base < started.end();
      shared.group[0] = started;
      shared.rows[0] = begun_before ? started.count * a.group.d : 0;
    }
  }
  named_barrier(1, kStreamThreads);

  // Joins: rows of the items that span warps, dealt out over the warps.
  const int64_t cta_end = base + width * kStreamWarps;
  auto store_vector = [&](const ItemAt& it, int r, int d, float4 v, float sum) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<uint2*>(out_row(it, r) + d) =
        make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
  };
  int task = warp;  // this warp's next row among all groups' rows
#pragma unroll 1
  for (int i = 0, before = 0; i <= kStreamWarps; ++i) {
    const int rows = shared.rows[i];
    if (task >= before + rows) {
      before += rows;
      continue;
    }
    // Group 0 is the item begun before the CTA, group w + 1 the one begun by
    // warp w: that part lies in the warp's ring, the others' in `join`.
    const ItemAt it = shared.group[i];
    const bool begun = i > 0;
    const int from = begun ? i - 1 : 0;
    // Bit w: warp w has a part.
    const uint32_t members = __ballot_sync(
        0xFFFFFFFFu, lane >= from && lane < kStreamWarps && base + lane * width < it.end());
    auto part_of = [&](int w) {
      return begun && w == from ? reinterpret_cast<const float*>(smem + w * (kStages * 2 * kUnitTile))
                                : join + w * join_floats;
    };
    const bool whole = begun && it.end() <= cta_end;
    float* dst = whole ? nullptr : args.parts + (static_cast<int64_t>(blockIdx.x) * 2 + begun) * join_floats;
    for (; task < before + rows; task += kStreamWarps) {
      const int r = task - before, d = lane * 4;
      // Lane w looks after the statistics of warp w's part.
      float2 ms = make_float2(-INFINITY, 0.0f);
      if (members >> lane & 1u)
        ms = *reinterpret_cast<const float2*>(part_of(lane) + stats + 2 * r);
      const float top = warp_max(ms.x);
      const float f = ex2_approx(ms.x - (top == -INFINITY ? 0.0f : top));
      const float sum = warp_sum(ms.y * f);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kStreamWarps; ++w) {
        const float fw = __shfl_sync(0xFFFFFFFFu, f, w);
        if ((members >> w & 1u) == 0) continue;
        const float4 y = *reinterpret_cast<const float4*>(part_of(w) + r * kCacheHeadDim + d);
        v.x = fmaf(y.x, fw, v.x);
        v.y = fmaf(y.y, fw, v.y);
        v.z = fmaf(y.z, fw, v.z);
        v.w = fmaf(y.w, fw, v.w);
      }
      if (whole) {
        store_vector(it, r, d, v, sum);
      } else {
        *reinterpret_cast<float4*>(dst + r * kCacheHeadDim + d) = v;
        if (lane == 0) *reinterpret_cast<float2*>(dst + stats + 2 * r) = make_float2(top, sum);
      }
    }
    before += rows;
    if (!whole && lane == 0) {
      shared.part[begun] = it;
      shared.has[begun] = 1;
    }
  }
  named_barrier(1, kStreamThreads);

  // The last CTA of an item to arrive joins its parts, in CTA order.
  if (shared.has[0] + shared.has[1] == 0) return;
  const int64_t cta_width = width * kStreamWarps;
  if (tid < 2 && shared.has[tid] != 0) {
    const ItemAt it = shared.part[tid];
    const int64_t first = Divide(it.begin, cta_width);  // at most one item goes on behind a CTA
    const int64_t parts = Divide(it.end() - 1, cta_width) - first;
    uint32_t* counter = args.counters + first;
    const bool last = atom_add_acq_rel(counter, 1u) == static_cast<uint32_t>(parts);
    if (last) *counter = 0;
    shared.last[tid] = last;
  }
  named_barrier(1, kStreamThreads);
  for (int slot = 0; slot < 2; ++slot) {
    if (shared.has[slot] == 0 || shared.last[slot] == 0) continue;
    const ItemAt it = shared.part[slot];
    const int first = static_cast<int>(Divide(it.begin, cta_width));
    const int last = static_cast<int>(Divide(it.end() - 1, cta_width));
    for (int i = tid; i < it.count * a.group.d * (kCacheHeadDim / 4); i += kStreamThreads) {
      const int r = i / (kCacheHeadDim / 4), d = i % (kCacheHeadDim / 4) * 4;
      // The first CTA began the item: its part is its second, the others' their first.
      auto part_of = [&](int x) {
        return args.parts + (static_cast<int64_t>(x) * 2 + (x == first ? 1 : 0)) * join_floats;
      };
      float top = -INFINITY, sum = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int x0 = first; x0 <= last; x0 += 8) {  // eight parts' loads in flight
        float2 ms[8];
        float4 y[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          ms[x] = make_float2(-INFINITY, 0.0f);
          y[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (x0 + x > last) continue;
          ms[x] = __ldcg(reinterpret_cast<const float2*>(part_of(x0 + x) + stats + 2 * r));
          y[x] = __ldcg(reinterpret_cast<const float4*>(part_of(x0 + x) + r * kCacheHeadDim + d));
        }
        float grown = top;
#pragma unroll
        for (int x = 0; x < 8; ++x) grown = fmaxf(grown, ms[x].x);
        const float zero = grown == -INFINITY ? 0.0f : grown;
        const float old = ex2_approx(top - zero);
        top = grown;
        v.x *= old, v.y *= old, v.z *= old, v.w *= old, sum *= old;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float f = ex2_approx(ms[x].x - zero);
          v.x = fmaf(y[x].x, f, v.x);
          v.y = fmaf(y[x].y, f, v.y);
          v.z = fmaf(y[x].z, f, v.z);
          v.w = fmaf(y[x].w, f, v.w);
          sum = fmaf(ms[x].y, f, sum);
        }
      }
      store_vector(it, r, d, v, sum);
    }
  }
}

// ---------------------------------------- many rows: tiles on tcgen05
//
// The rows of a kv head (row r: token r / group, head r % group) in tiles of
// 128, with attention_device.cuh's schedule: S = Q K^T into tensor memory,
// the softmax's P written over it as half, O += P V.  What differs is how K
// and V arrive: a warp loads their codes by TMA (32 KB for 128 keys instead
// of 64), a converter warpgroup writes them as half into the swizzled tiles
// that the MMAs read, once for two row tiles.  Two forms of a CTA:
//   pairs   more than 128 rows: two tiles, one per softmax warpgroup, that
//           share every K and V tile;
//   single  up to 128 rows: both warpgroups take the same tile, one the even
//           and one the odd key tiles, and join at the end.
// A softmax step takes 64 keys of a tile and S has two buffers for each
// warpgroup, so that the S of the next 64 keys is there when it starts: with
// one S of 128 keys the softmax and the products of a row tile took turns
// (215 us for the case below, 205 with the two buffers).  The products are
// issued by the elected thread of a converged warp: from a divergent branch
// each instruction cost about 100 cycles, of 64 that the tensor core needs
// (324 us with these 48 products a key tile, 240 with 32 of 128 keys).
//
// Bound by the softmax warps' latencies: 64 keys of both warpgroups take 2,200
// cycles (waits 300, scores read and their maxima 500, exponentials and the
// probabilities' way back 1,300; the MMAs take 1,280 beside that, K's and V's
// conversion 1,600 a tile), and by what comes before and after a CTA's key
// tiles, 7,400 and 3,100 cycles.  Measured on one B200: 16 causal sequences of
// up to 2,175 rows, 16 heads over 8: 198 us, 630 TFLOP/s of what is seen; 375
// rows over 705 tokens: 15.7 us, where a CTA sees 2 key tiles.
//
// Registers: 512 threads start with 128 each; the softmax warpgroups take 152,
// the other two keep 104.

constexpr int kSlabs = kKeys / 16;  // 16-key groups of a key tile: one page each at least
constexpr int kUnitKeys = 64;       // keys of one softmax step: half a key tile
constexpr int kUnitSlabs = kUnitKeys / 16;
constexpr int kScaleSlots = 8;
constexpr int kMinKeyTiles = 2;  // of a split; 2 to 4 measured alike (375 rows over 705 tokens
                                 // 18.0 to 17.2 us), 8 took 24.2 us for 19.6 over 2,048 tokens
constexpr uint32_t kCodeTile = kKeys * kCacheHeadDim;  // 16 KB
constexpr int kTileThreads = 512;
constexpr int kConvertWarp = 8, kLoadWarp = 12, kMmaWarp = 13;

// A slab's factor, shift and inverse value scale (ValueScale); bad: 1 where
// its page does not exist.
struct alignas(16) SlabScale {
  float factor, shift, inverse;
  int bad;
};

struct TileShared {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2][2], p_full[2][2];     // [group][buffer]
  uint64_t codes_full[2], codes_empty[2];  // of keys, of values
  uint64_t scale_full[kScaleSlots];
  uint32_t tmem;
  int last;
  alignas(16) SlabScale scales[kScaleSlots][kSlabs];
};

constexpr size_t kTileSmem = 1024 + 6 * kTile + 2 * kCodeTile + sizeof(TileShared);
// One part of a split item: O[32 vectors of 4 columns][row], then (maximum,
// sum) of its rows.
__host__ __device__ constexpr size_t TilePartFloats(int tile_rows) {
  return static_cast<size_t>(tile_rows) * (kCacheHeadDim + 2);
}
static_assert(kTileSmem <= 232448, "shared memory of a CTA");

struct TileArgs {
  CacheAttnArgs a;
  uint32_t* counters;  // one for each (row tile of this grid, sequence, kv head)
  float* parts;        // [counter][split]
  int tile_rows;       // rows of a CTA: 128 or 256
  int tiles;           // CTAs along the rows
  int splits;          // CTAs along the keys, at most
};

__device__ __forceinline__ float Max16(const uint32_t* r) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = fmaxf(__uint_as_float(r[j]), __uint_as_float(r[j + 8]));
#pragma unroll
  for (int w = 4; w > 0; w >>= 1)
#pragma unroll
    for (int j = 0; j < w; ++j) v[j] = fmaxf(v[j], v[j + w]);
  return v[0];
}

// 16 codes to 16 halves, in two 16-byte pieces.
__device__ __forceinline__ void Convert16(const uint4& q, uint8_t* low, uint8_t* high) {
  const uint32_t x = q.x ^ 0x80808080u, y = q.y ^ 0x80808080u;
  const uint32_t z = q.z ^ 0x80808080u, w = q.w ^ 0x80808080u;
  *reinterpret_cast<uint4*>(low) =
      make_uint4(CodePair<0x4140>(x), CodePair<0x4342>(x), CodePair<0x4140>(y), CodePair<0x4342>(y));
  *reinterpret_cast<uint4*>(high) =
      make_uint4(CodePair<0x4140>(z), CodePair<0x4342>(z), CodePair<0x4140>(w), CodePair<0x4342>(w));
}

// Codes of 128 keys to a swizzled half tile ([2 boxes][128][64]), by 128
// threads: 16 codes of each 64-dim half of every 32nd row.  Even and odd rows
// take their halves in opposite order, so that 8 neighbouring lanes read and
// write all banks.
__device__ __forceinline__ void ConvertTile(const uint8_t* codes, uint8_t* tile, int tid) {
  const int part = tid & 3, row = tid >> 2, box = row & 1;
  const uint8_t* src = codes + row * kCacheHeadDim + part * 16;
  uint8_t* low = tile + row * 128 + (((2 * part) ^ (row & 7)) << 4);
  uint8_t* high = tile + row * 128 + (((2 * part + 1) ^ (row & 7)) << 4);
  const uint32_t first = box * kHalfTile, second = kHalfTile - first;
  const uint8_t* src_first = src + box * 64;
  const uint8_t* src_second = src + 64 - box * 64;
  uint4 q[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    q[2 * i] = *reinterpret_cast<const uint4*>(src_first + i * 32 * kCacheHeadDim);
    q[2 * i + 1] = *reinterpret_cast<const uint4*>(src_second + i * 32 * kCacheHeadDim);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    Convert16(q[2 * i], low + first + i * 32 * 128, high + first + i * 32 * 128);
    Convert16(q[2 * i + 1], low + second + i * 32 * 128, high + second + i * 32 * 128);
  }
}

// One arrival for a warp, behind what all its lanes did.
__device__ __forceinline__ void WarpArrive(uint64_t* bar) {
  __syncwarp();
  if (elect_one()) mbar_arrive(bar);
}

// The products of one CTA, issued by one thread of a converged warp.  A step
// along the head dimension or the keys only adds to a descriptor's address field.
struct TileIssue {
  uint32_t tmem;
  uint64_t q, k, v;  // descriptors of row tile 0 and of stage 0

  __device__ __forceinline__ TileIssue(uint32_t tmem_, const uint8_t* q_s, const uint8_t* k_s,
                                       const uint8_t* v_s)
      : tmem(tmem_),
        q(smem_desc_sw128(smem_u32(q_s), 16, 1024)),
        k(smem_desc_sw128(smem_u32(k_s), 16, 1024)),
        v(smem_desc_sw128(smem_u32(v_s), kHalfTile, 1024)) {}
  // S of group g, buffer `half` = Q of row tile `tile` x that half of K of `stage`.
  __device__ __forceinline__ void Scores(int g, int tile, int stage, int half) const {
    constexpr uint32_t idesc = idesc_f16_f32(kQ, kUnitKeys, 0);
    const uint64_t qd = q + static_cast<uint32_t>(tile) * (kTile >> 4);
    const uint64_t kd = k + static_cast<uint32_t>(stage) * (kTile >> 4) +
                        static_cast<uint32_t>(half) * (kUnitKeys * 128 >> 4);
    const uint32_t d = tmem + static_cast<uint32_t>(g * 256 + half * kUnitKeys);
    if (!elect_one()) return;
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk) {
      const uint32_t off = ((kk >> 2) * kHalfTile + (kk & 3) * 32) >> 4;
      umma_f16_ss(d, qd + off, kd + off, idesc, kk > 0 ? 1u : 0u);
    }
  }
  // O of group g (+)= P of buffer `half` x that half of V of `stage`.
  __device__ __forceinline__ void Values(int g, int stage, int half, bool add) const {
    constexpr uint32_t idesc = idesc_f16_f32(kQ, kD, 1);
    const uint64_t vd = v + static_cast<uint32_t>(stage) * (kTile >> 4) +
                        static_cast<uint32_t>(half) * (kUnitKeys * 128 >> 4);
    const uint32_t o = tmem + static_cast<uint32_t>(g * 256 + 128);
    const uint32_t p = tmem + static_cast<uint32_t>(g * 256 + half * kUnitKeys);
    if (!elect_one()) return;
#pragma unroll
    for (int kk = 0; kk < kUnitKeys / 16; ++kk)
      umma_f16_ts(o, p + static_cast<uint32_t>(kk * 8), vd + ((kk * 16 * 128) >> 4), idesc,
                  add || kk > 0 ? 1u : 0u);
  }
};

__device__ __forceinline__ void Commit(uint64_t* bar) {
  if (elect_one()) umma_commit(bar);
}

// A wait of the whole warp, converged behind it, with one outcome for all.
__device__ __forceinline__ bool WarpWait(uint64_t* bar, uint32_t parity, uint32_t* err) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, err));
}

// Phases of the barriers: s_full[g][b] completes once for the first S of the
// buffer, then once for each of its P V (and the S after it, where there is
// one); p_full[g][b] once for each P.  So S of unit u is there after phase
// u / 2, and P V of unit u is done after phase u / 2 + 1.

// Two row tiles share every key tile.  units0, units1: 64-key units of which the
// groups' rows see something; one of the groups reaches the last key tile.
__device__ __forceinline__ void IssuePairs(const TileIssue& mma, TileShared& s, int nt, int units0,
                                           int units1, uint32_t* err) {
  if (!WarpWait(&s.q_full, 0, err) || !WarpWait(&s.k_full[0], 0, err)) return;
  tc_fence_after_sync();
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int half = i >> 1, g = i & 1;
    if (half >= (g == 0 ? units0 : units1)) continue;
    mma.Scores(g, g, 0, half);
    Commit(&s.s_full[g][half]);
  }
  Commit(&s.k_empty[0]);
#pragma unroll 1
  for (int t = 0; t < nt; ++t) {
    const int stage = t & 1, next = stage ^ 1;
    bool k_ready = false;
    if (!WarpWait(&s.v_full[stage], static_cast<uint32_t>(t >> 1) & 1u, err)) return;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const int half = i >> 1, g = i & 1, u = 2 * t + half, units = g == 0 ? units0 : units1;
      if (u >= units) continue;
      if (!WarpWait(&s.p_full[g][half], static_cast<uint32_t>(t) & 1u, err)) return;
      tc_fence_after_sync();
      mma.Values(g, stage, half, u > 0);
      if (u + 2 < units) {
        if (!k_ready && !WarpWait(&s.k_full[next], static_cast<uint32_t>((t + 1) >> 1) & 1u, err)) return;
        k_ready = true;
        tc_fence_after_sync();
        mma.Scores(g, g, next, half);
      }
      Commit(&s.s_full[g][half]);
    }
    Commit(&s.v_empty[stage]);
    if (t + 1 < nt) Commit(&s.k_empty[next]);
  }
}

// One row tile: key tile t belongs to group t & 1, in stage t & 1.  (Products in
// the order in which their operands arrive, polled, were alike here and 5 % slower
// for pairs; a second issuing warp was 3 % slower.)
__device__ __forceinline__ void IssueSingle(const TileIssue& mma, TileShared& s, int nt, int units0,
                                            int units1, uint32_t* err) {
  if (!WarpWait(&s.q_full, 0, err)) return;
  for (int t = -2; t < nt; t += 2) {  // tiles t and t + 1; before the first, only their S
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      // A tile's two units before the other group's: keys of tile t + 3 are
      // converted behind the values of t + 2, which wait for those of tile t.
      const int half = i & 1, g = i >> 1;
      const int u = t + half, units = g == 0 ? units0 : units1;
      const uint32_t phase = static_cast<uint32_t>(t >> 1) & 1u;
      if (t >= 0 && u < units) {
        if (!WarpWait(&s.p_full[g][half], phase, err)) return;
        if (half == 0 && !WarpWait(&s.v_full[g], phase, err)) return;
        tc_fence_after_sync();
        mma.Values(g, g, half, u > 0);
        if (half == 1 || u + 1 == units) Commit(&s.v_empty[g]);
      }
      if (u + 2 < units) {
        if (half == 0 && !WarpWait(&s.k_full[g], phase ^ 1u, err)) return;
        tc_fence_after_sync();
        mma.Scores(g, 0, g, half);
        if (half == 1 || u + 3 == units) Commit(&s.k_empty[g]);
      }
      if (u + 2 < units || (t >= 0 && u < units)) Commit(&s.s_full[g][half]);
    }
  }
}

// Joins `parts` parts of a CTA's `here` rows, by 256 threads. Each L2 latency
// costs about 1 us here, so a thread has two pieces (16 columns of a row) of two
// parts in flight: 375 rows over 705 tokens took 18.2 us with one piece and four
// parts, 16.3 with two and two, 18.3 with four and one.
template <typename OutRow>
__device__ __forceinline__ void JoinTile(const TileArgs& args, const float* first, int parts, int here,
                                         const OutRow& out_row) {
  constexpr int kItems = 2;
  const int stats_at = args.tile_rows * kCacheHeadDim;
  for (int i0 = threadIdx.x; i0 < 8 * here; i0 += 256 * kItems) {
    float top[kItems], sum[kItems], o[kItems][16];
    int row[kItems], d16[kItems];
#pragma unroll
    for (int n = 0; n < kItems; ++n) {
      const int i = min(i0 + n * 256, 8 * here - 1);  // behind the last: its sums again
      d16[n] = i / here;
      row[n] = i - d16[n] * here;
      top[n] = -INFINITY;
      sum[n] = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) o[n][j] = 0.0f;
    }
#pragma unroll 2
    for (int x = 0; x < parts; ++x) {
      const float* p = first + x * TilePartFloats(args.tile_rows);
      float2 ms[kItems];
      float4 y[kItems][4];
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        ms[n] = __ldcg(reinterpret_cast<const float2*>(p + stats_at + 2 * row[n]));
#pragma unroll
        for (int j = 0; j < 4; ++j)
          y[n][j] = __ldcg(reinterpret_cast<const float4*>(p) + (d16[n] * 4 + j) * args.tile_rows + row[n]);
      }
#pragma unroll
      for (int n = 0; n < kItems; ++n) {
        const float2 f = JoinFactors(&top[n], &sum[n], ms[n]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[n][4 * j] = fmaf(y[n][j].x, f.y, o[n][4 * j] * f.x);
          o[n][4 * j + 1] = fmaf(y[n][j].y, f.y, o[n][4 * j + 1] * f.x);
          o[n][4 * j + 2] = fmaf(y[n][j].z, f.y, o[n][4 * j + 2] * f.x);
          o[n][4 * j + 3] = fmaf(y[n][j].w, f.y, o[n][4 * j + 3] * f.x);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < kItems; ++n) {
      if (i0 + n * 256 >= 8 * here) continue;
      const float inv = sum[n] == 0.0f ? 0.0f : 1.0f / sum[n];
      uint4* dst = reinterpret_cast<uint4*>(out_row(row[n]) + d16[n] * 16);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        dst[j] = make_uint4(pack_half2(o[n][8 * j] * inv, o[n][8 * j + 1] * inv),
                            pack_half2(o[n][8 * j + 2] * inv, o[n][8 * j + 3] * inv),
                            pack_half2(o[n][8 * j + 4] * inv, o[n][8 * j + 5] * inv),
                            pack_half2(o[n][8 * j + 6] * inv, o[n][8 * j + 7] * inv));
    }
  }
}

__global__ void __launch_bounds__(kTileThreads, 1)
    cache_attention_tile_kernel(const __grid_constant__ CUtensorMap map_k,
                                const __grid_constant__ CUtensorMap map_v, const TileArgs args) {
  const CacheAttnArgs& a = args.a;
  const CacheView& cache = a.cache;
  pdl_trigger();
  pdl_wait();
  // Heads first: CTAs that run together read whole rows of q and whole pages.
  // The last row tiles of causal sequences see most: they start first, those
  // of all sequences before the next.
  int at_grid = static_cast<int>(blockIdx.x);
  const int kv_head = at_grid % cache.kv_heads;
  at_grid /= cache.kv_heads;
  const int split = at_grid % args.splits;
  at_grid /= args.splits;
  const int seq = at_grid % cache.num_seqs;
  const int tile = args.tiles - 1 - at_grid / cache.num_seqs;
  const int announced = a.lengths[seq];
  const RowSpan span = SequenceRows(a.cu_rows, seq, a.rows, a.max_rows, a.err);
  const int rows = span.count * a.group.d;  // at most 2^31 (host check)
  const int row0 = tile * args.tile_rows;
  if (row0 >= rows) return;  // uniform over the CTA, before any barrier
  const int length = CheckLength(a, announced);
  const bool pair = rows - row0 > kQ && args.tile_rows > kQ;
  const int here = min(rows - row0, args.tile_rows);
  const int before = length - span.count;  // tokens that row token 0 has before it
  // Tokens that some row up to (and with) row0 + n sees.
  auto reach_of = [&](int n) { return a.causal ? max(0, before + a.group(row0 + n) + 1) : length; };
  const int reach = reach_of(here - 1);
  const int all_tiles = (reach + kKeys - 1) / kKeys;
  const int per = max(1, (all_tiles + args.splits - 1) / args.splits);
  const int parts = max(1, (all_tiles + per - 1) / per);
  if (split >= parts) return;
  const int t0 = split * per;
  const int nt = min(all_tiles, t0 + per) - t0;
  // 64-key units of the groups: of a pair's first tile up to what its rows see,
  // else the even and the odd key tiles'.
  auto units_of = [&](int r) { return max(0, min(2 * nt, (r - t0 * kKeys + kUnitKeys - 1) / kUnitKeys)); };
  const int all_units = units_of(reach);
  const int units0 = pair ? units_of(reach_of(kQ - 1)) : (nt + 1) / 2 * 2 - ((nt & 1) != 0 ? all_units & 1 : 0);
  const int units1 = pair ? all_units : nt / 2 * 2 - ((nt & 1) == 0 ? all_units & 1 : 0);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* q_s = smem;               // [2 row tiles] x 32 KB
  uint8_t* k_s = q_s + 2 * kTile;    // [2 stages] x 32 KB
  uint8_t* v_s = k_s + 2 * kTile;    // [2 stages] x 32 KB
  uint8_t* code_s = v_s + 2 * kTile; // keys, values: 16 KB each
  TileShared& s = *reinterpret_cast<TileShared*>(code_s + 2 * kCodeTile);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
  // Query rows into the swizzled tiles, 16 lanes a row, by the softmax warps:
  // on their way while the CTA sets itself up.
  const int piece = tid & 15;
  if (tid < kConvertWarp * 32) {
    for (int r = tid >> 4; r < (pair ? 2 * kQ : kQ); r += 16) {
      const int row = row0 + min(r, here - 1), token = a.group(row);
      cp_async_16(q_s + (r >> 7) * kTile + (piece >> 3) * kHalfTile + (r & 127) * 128 +
                      (((piece & 7) ^ (r & 7)) << 4),
                  a.q + static_cast<int64_t>(span.first + token) * a.ld_q +
                      (kv_head * a.group.d + row - token * a.group.d) * kCacheHeadDim + piece * 8,
                  r < here);
    }
  }
  if (tid == 0) {
    mbar_init(&s.q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.k_full[i], 4);
      mbar_init(&s.v_full[i], 4);
      mbar_init(&s.codes_full[i], kSlabs);
      mbar_init(&s.codes_empty[i], 4);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.v_empty[i], 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s.s_full[i][b], 1);
        mbar_init(&s.p_full[i][b], 4);
      }
    }
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&s.scale_full[i], kSlabs);
    fence_mbar_init();
    tma_prefetch_map(&map_k);
    tma_prefetch_map(&map_v);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&s.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, s.tmem, 0);
  const int64_t item = (static_cast<int64_t>(tile) * cache.num_seqs + seq) * cache.kv_heads + kv_head;
  float* part = parts > 1 ? args.parts + (item * args.splits + split) * TilePartFloats(args.tile_rows) : nullptr;
  const int stats_at = args.tile_rows * kCacheHeadDim;

  if (warp >= kConvertWarp) registers_shrink<104>();
  if (warp == kLoadWarp) {
    // Lane i < 8 looks after slab i of a key tile; the first slab of a box
    // loads it.  Codes wait for the converters, one key tile ahead of them.
    const int box = min(kKeys, 1 << cache.page_shift);
    auto look_up = [&](int t) {
      const int token = (t0 + t) * kKeys + lane * 16;
      return lane < kSlabs && t < nt && token < length
                 ? cache.table[static_cast<int64_t>(seq) * cache.max_pages + (token >> cache.page_shift)]
                 : -1;
    };
    int next = look_up(0);
    for (int t = 0; t < nt; ++t) {
      const int token = (t0 + t) * kKeys + lane * 16;
      int page = next;
      next = look_up(t + 1);
      const bool wanted = token < length;
      if (lane < kSlabs && wanted && (page < 0 || page >= cache.pages)) {
        atomicOr(a.err, kErrBadArgument);
        page = -1;
      }
      const int row = ((page * cache.kv_heads + kv_head) << cache.page_shift) +
                      (token & ((1 << cache.page_shift) - 1));
      bool ok = true;
      for (int w = 0; w < 2 && ok; ++w) {
        // The whole warp together: a lane that came late could find a barrier
        // two phases on, by the others' arrivals.  Landed, too: converters that
        // gave up waiting for codes free them all the same.
        const uint32_t used = static_cast<uint32_t>(t - 1) & 1u;
        if (t > 0)
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(&s.codes_empty[w], used, a.err) &&
                                           mbar_wait(&s.codes_full[w], used, a.err));
        if (lane < kSlabs && ok) {
          if (page >= 0 && lane * 16 % box == 0) {
            mbar_arrive_expect_tx(&s.codes_full[w], box * kCacheHeadDim);
            tma_load_2d(code_s + w * kCodeTile + lane * 16 * kCacheHeadDim, w == 0 ? &map_k : &map_v,
                        &s.codes_full[w], 0, row);
          } else {
            mbar_arrive(&s.codes_full[w]);
          }
        }
      }
      if (lane < kSlabs) {
        SlabScale v = {1.0f, 0.0f, 1.0f, wanted ? 1 : 0};
        if (page >= 0) {
          const int64_t at = static_cast<int64_t>(page) * cache.kv_heads + kv_head;
          v.factor = KeyFactor(cache.key_scales[at], a.scale_log2);
          ValueScale(cache.value_scales[at], &v.shift, &v.inverse);
          v.bad = 0;
        }
        s.scales[t % kScaleSlots][lane] = v;
        mbar_arrive(&s.scale_full[t % kScaleSlots]);
      }
      __syncwarp();
      if (!__all_sync(0xFFFFFFFFu, ok)) break;
    }
    // No copy outlives the CTA (behind a wait that ran out, all had its time).
    if (nt > 0)
      for (int w = 0; w < 2; ++w)
        (void)mbar_wait(&s.codes_full[w], static_cast<uint32_t>(nt - 1) & 1u, a.err);
  } else if (warp >= kConvertWarp && warp < kLoadWarp) {
    const int ctid = tid - kConvertWarp * 32;
    bool ok = true;  // once a wait ran out, no other is begun
    for (int t = 0; t < nt; ++t) {
      const int stage = t & 1;
      const uint32_t reuse = static_cast<uint32_t>((t >> 1) - 1) & 1u;
      ok = ok && mbar_wait(&s.codes_full[0], static_cast<uint32_t>(t) & 1u, a.err);
      if (t >= 2) ok = ok && mbar_wait(&s.k_empty[stage], reuse, a.err);
      ConvertTile(code_s, k_s + stage * kTile, ctid);
      fence_proxy_async_smem();
      WarpArrive(&s.k_full[stage]);
      WarpArrive(&s.codes_empty[0]);
      ok = ok && mbar_wait(&s.codes_full[1], static_cast<uint32_t>(t) & 1u, a.err);
      if (t >= 2) ok = ok && mbar_wait(&s.v_empty[stage], reuse, a.err);
      ConvertTile(code_s + kCodeTile, v_s + stage * kTile, ctid);
      fence_proxy_async_smem();
      WarpArrive(&s.v_full[stage]);
      WarpArrive(&s.codes_empty[1]);
    }
  } else if (warp == kMmaWarp) {
    if (nt > 0) {
      const TileIssue mma(tmem, q_s, k_s, v_s);
      if (pair) IssuePairs(mma, s, nt, units0, units1, a.err);
      else IssueSingle(mma, s, nt, units0, units1, a.err);
    }
    __syncwarp();
    named_barrier(2, 256 + 32);  // O was read
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  } else if (warp < kConvertWarp) {
    registers_grow<152>();
    cp_async_wait_all();
    fence_proxy_async_smem();
    WarpArrive(&s.q_full);

    const int g = warp >> 2;
    const int r = tid & 127;               // tensor-memory lane, row of the tile
    const int mine = row0 + (pair ? g * kQ : 0) + r;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + static_cast<uint32_t>(g * 256) + lanes;
    const uint32_t o_addr = s_addr + 128;
    const int seen = a.causal ? min(length, before + a.group(mine) + 1) : length;
    // The fewest tokens that a row of this tile sees.
    const int least = a.causal ? before + a.group(mine - r) + 1 : length;
    const int units = g == 0 ? units0 : units1;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int u = 0; u < units; ++u) {
      const int half = u & 1, t = pair ? u >> 1 : (u & ~1) + g;
      const uint32_t p_addr = s_addr + static_cast<uint32_t>(half * kUnitKeys);
      ok = ok && mbar_wait(&s.scale_full[t % kScaleSlots],
                           static_cast<uint32_t>(t / kScaleSlots) & 1u, a.err);
      const SlabScale* slab = s.scales[t % kScaleSlots] + half * kUnitSlabs;
      ok = ok && mbar_wait(&s.s_full[g][half], static_cast<uint32_t>(u >> 1) & 1u, a.err);
      __syncwarp();
      tc_fence_after_sync();
      const int token0 = (t0 + t) * kKeys + half * kUnitKeys;
      int bad = 0;
#pragma unroll
      for (int i = 0; i < kUnitSlabs; ++i) bad |= slab[i].bad;
      const bool partial = token0 + kUnitKeys > least || bad != 0;
      uint32_t x[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld_32x32b_x32(p_addr + c * 32, x[c]);
      tmem_ld_wait();
      if (partial) {
        const int valid = seen - token0;
#pragma unroll
        for (int i = 0; i < kUnitSlabs; ++i) {
          const int slab_valid = slab[i].bad != 0 ? 0 : valid - i * 16;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (j >= slab_valid) x[i >> 1][(i & 1) * 16 + j] = 0xFF800000u;
        }
      }
      // A slab that the row sees nothing of must not bring a NaN scale.
      auto scale_of = [&](int i) {
        SlabScale k = slab[i];
        if (partial && (k.bad != 0 || seen - token0 <= i * 16)) k.factor = 1.0f, k.shift = 0.0f;
        return k;
      };
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kUnitSlabs; ++i) {
        const SlabScale k = scale_of(i);
        top = fmaxf(top, fmaf(Max16(&x[i >> 1][(i & 1) * 16]), k.factor, k.shift));
      }
      bool rescale = false;
      float alpha = 1.0f;
      if (u == 0) {
        m = top;
      } else {
        const bool grow = top > m + kRescaleThreshold;
        rescale = __any_sync(0xFFFFFFFFu, grow);
        if (grow) {
          alpha = ex2_approx(m - top);
          m = top;
        }
      }
      const float base = m == -INFINITY ? 0.0f : m;
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t packed[16];
        float e[32];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const SlabScale k = scale_of(c * 2 + i);
          const float shift = k.shift - base;
#pragma unroll
          for (int j = 0; j < 16; ++j) e[i * 16 + j] = fmaf(__uint_as_float(x[c][i * 16 + j]), k.factor, shift);
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) e[j] = ex2_approx(e[j]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float p0 = 0.0f, p1 = 0.0f;
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            p0 += e[i * 16 + j];
            p1 += e[i * 16 + j + 1];
            packed[i * 8 + j / 2] = pack_half2(e[i * 16 + j], e[i * 16 + j + 1]);
          }
          sum = fmaf(p0 + p1, scale_of(c * 2 + i).inverse, sum);
        }
        tmem_st_32x32b_x16(p_addr + c * 16, packed);
      }
      if (rescale) {  // O so far: behind the P V of the unit before
        l *= alpha;
        ok = ok && mbar_wait(&s.s_full[g][half ^ 1], static_cast<uint32_t>(((u - 1) >> 1) + 1) & 1u, a.err);
        __syncwarp();
        tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t x[32];
          tmem_ld_32x32b_x32(o_addr + c * 32, x);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * alpha);
          tmem_st_32x32b_x16(o_addr + c * 32, *reinterpret_cast<const uint32_t(*)[16]>(&x[0]));
          tmem_st_32x32b_x16(o_addr + c * 32 + 16, *reinterpret_cast<const uint32_t(*)[16]>(&x[16]));
        }
      }
      l += sum;
      tmem_st_wait();
      tc_fence_before_sync();
      WarpArrive(&s.p_full[g][half]);
    }

    // O of this warpgroup's tile.  In the single form the warpgroups have the
    // even and the odd key tiles' parts of one tile: each takes half of the
    // columns, the other's half comes through shared memory (every MMA is
    // done by then, so the rings are idle).  Columns here: [col0, col0 + 32 n).
    // A warpgroup without units has no MMA to wait for, but its query tile still
    // takes both warpgroups' copies: its zeros go there behind all of them.
    if (units > 0)
      ok = ok && mbar_wait(&s.s_full[g][(units - 1) & 1], static_cast<uint32_t>(((units - 1) >> 1) + 1) & 1u, a.err);
    else
      ok = ok && mbar_wait(&s.q_full, 0, a.err);
    if (!pair) named_barrier(1, 256);
    __syncwarp();
    tc_fence_after_sync();
    const bool mine_any = units > 0, other_any = !pair && (g == 0 ? units1 : units0) > 0;
    const int chunks = pair ? 4 : 2, col0 = pair ? 0 : g * 64;
    float4* exchange = reinterpret_cast<float4*>(k_s);  // [group][16 vectors][128 rows]
    float2* stats = reinterpret_cast<float2*>(v_s);     // [group][128 rows]
    float scale_mine = 1.0f, scale_other = 0.0f;
    if (!pair) {
      if (mine_any) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t x[32];
          tmem_ld_32x32b_x32(o_addr + (64 - col0) + c * 32, x);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(exchange + (g * 16 + c * 8 + j) * kQ + r) =
                make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        }
      }
      stats[g * kQ + r] = make_float2(m, l);
      named_barrier(1, 256);
      const float2 o = stats[(g ^ 1) * kQ + r];
      const float top = fmaxf(m, o.x);
      const float base = top == -INFINITY ? 0.0f : top;
      scale_mine = ex2_approx(m - base);
      scale_other = ex2_approx(o.x - base);
      // In group order, so that both halves of a row divide by the same sum.
      l = g == 0 ? fmaf(o.y, scale_other, l * scale_mine) : fmaf(l, scale_mine, o.y * scale_other);
      m = top;
    }
    const int at = mine - row0;  // row of this CTA
    if (part == nullptr) {
      scale_mine = l == 0.0f ? 0.0f : scale_mine / l;
      scale_other = l == 0.0f ? 0.0f : scale_other / l;
    }
    // Halves go through the query tile, idle too, so that rows leave whole.
    uint8_t* stage = q_s + (pair ? g * kTile : 0);
    for (int c = 0; c < chunks; ++c) {
      const int col = col0 + c * 32;
      uint32_t x[32];
      float o[32];
      if (mine_any) {
        tmem_ld_32x32b_x32(o_addr + col, x);
        tmem_ld_wait();
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) o[j] = mine_any ? __uint_as_float(x[j]) * scale_mine : 0.0f;
      if (other_any) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 y = exchange[((g ^ 1) * 16 + c * 8 + j) * kQ + r];
          o[4 * j] = fmaf(y.x, scale_other, o[4 * j]);
          o[4 * j + 1] = fmaf(y.y, scale_other, o[4 * j + 1]);
          o[4 * j + 2] = fmaf(y.z, scale_other, o[4 * j + 2]);
          o[4 * j + 3] = fmaf(y.w, scale_other, o[4 * j + 3]);
        }
      }
      if (part != nullptr) {  // vector v of all rows, then vector v + 1
        if (at < here) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            reinterpret_cast<float4*>(part)[(col / 4 + j) * args.tile_rows + at] =
                make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
      } else {
        uint8_t* dst = stage + (col >> 6) * kHalfTile + r * 128;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int piece = ((col & 63) >> 3) + j;
          *reinterpret_cast<uint4*>(dst + ((piece ^ (r & 7)) << 4)) =
              make_uint4(pack_half2(o[8 * j], o[8 * j + 1]), pack_half2(o[8 * j + 2], o[8 * j + 3]),
                         pack_half2(o[8 * j + 4], o[8 * j + 5]), pack_half2(o[8 * j + 6], o[8 * j + 7]));
        }
      }
    }
    tc_fence_before_sync();
    named_barrier(2, 256 + 32);
    auto out_row = [&](int r_) {
      const int row = row0 + r_, token = a.group(row);
      return a.out + static_cast<int64_t>(span.first + token) * a.ld_out +
             (kv_head * a.group.d + row - token * a.group.d) * kCacheHeadDim;
    };
    if (part == nullptr) {
      const int count = min(here, pair ? 2 * kQ : kQ);
#pragma unroll 4
      for (int i = tid >> 4; i < count; i += 16)
        *reinterpret_cast<uint4*>(out_row(i) + piece * 8) = *reinterpret_cast<const uint4*>(
            q_s + (i >> 7) * kTile + (piece >> 3) * kHalfTile + (i & 127) * 128 + (((piece & 7) ^ (i & 7)) << 4));
      return;
    }
    if (at < here && (pair || g == 0))
      *reinterpret_cast<float2*>(part + stats_at + 2 * at) = make_float2(m, l);
    // The last part to arrive joins all of them, in split order.
    named_barrier(1, 256);
    uint32_t* counter = args.counters + item;
    if (tid == 0) {
      s.last = atom_add_acq_rel(counter, 1u) == static_cast<uint32_t>(parts - 1);
      if (s.last) *counter = 0;
    }
    named_barrier(1, 256);
    if (!s.last) return;
    const float* base_part = args.parts + item * args.splits * TilePartFloats(args.tile_rows);
    JoinTile(args, base_part, parts, here, out_row);
  }
}

// A workspace begins with counters, as many for every shape, so that calls of
// different shapes can share it: none finds another's parts in their place.
constexpr size_t kCounterBytes = 4096;

// CTAs of a call that splits items (each may need a counter).
size_t SplitCtas() {
  return std::min<size_t>(static_cast<size_t>(SmCount()), kCounterBytes / sizeof(uint32_t));
}

// How a call runs: the streaming kernel's rows for a (sequence, kv head), its
// CTAs and the scratch that splitting takes.
struct StreamPlan {
  int rows;       // 0: too many for it
  unsigned ctas;
  size_t part_bytes;
};

StreamPlan PlanStream(const ov_kv_cache* cache, size_t max_rows, size_t max_length, size_t heads) {
  StreamPlan plan{};
  const size_t rows = max_rows * (heads / cache->kv_heads);
  if (rows > 16) return plan;
  plan.rows = static_cast<int>(rows);
  const size_t items = cache->num_seqs * cache->kv_heads;
  const size_t units = std::max<size_t>(1, (max_length + kUnit - 1) / kUnit);
  const size_t least = kMinUnits * kStreamWarps;
  plan.ctas = static_cast<unsigned>(
      std::min(SplitCtas(), items * ((units + least - 1) / least)));
  plan.part_bytes = 2 * plan.ctas * JoinFloats(plan.rows) * sizeof(float);
  return plan;
}

// The tile kernel's CTAs and scratch.
struct TilePlan {
  int tile_rows, tiles, splits;
  size_t part_bytes;
};

TilePlan PlanTiles(const ov_kv_cache* cache, size_t max_rows, size_t max_length, size_t heads) {
  TilePlan plan{};
  const size_t rows = max_rows * (heads / cache->kv_heads);
  const size_t pairs = cache->num_seqs * cache->kv_heads;  // of sequence and kv head
  const size_t sms = SplitCtas();
  // Single tiles while they all fit the GPU at once, else tile pairs.
  plan.tile_rows = (rows + kQ - 1) / kQ * pairs <= sms ? kQ : 2 * kQ;
  plan.tiles = static_cast<int>((rows + plan.tile_rows - 1) / plan.tile_rows);
  const size_t items = plan.tiles * pairs;
  const size_t key_tiles = (max_length + kKeys - 1) / kKeys;
  plan.splits = static_cast<int>(
      std::max<size_t>(1, std::min(sms / items, key_tiles / kMinKeyTiles)));
  if (plan.splits > 1)
    plan.part_bytes = items * plan.splits * TilePartFloats(plan.tile_rows) * sizeof(float);
  return plan;
}

template <int kNT>
void LaunchStream(const StreamArgs& args, unsigned ctas, const CUtensorMap& map_k,
                  const CUtensorMap& map_v, cudaStream_t stream) {
  SetMaxDynamicSmem(reinterpret_cast<const void*>(cache_attention_stream_kernel<kNT>),
                    static_cast<int>(StreamSmem<kNT>(8 * kNT)));
  Launch(cache_attention_stream_kernel<kNT>, dim3(ctas), dim3(kStreamThreads + 128),
         StreamSmem<kNT>(args.join_rows), stream, "cache attention kernel launch", map_k, map_v,
         args);
}

// A cache's codes as 128-byte rows, boxes of `box_rows` of them.
void EncodeCodesMap(CUtensorMap* map, const int8_t* codes, const ov_kv_cache* cache,
                    size_t box_rows, CUtensorMapSwizzle swizzle) {
  EncodeTensorMap2D(map, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, kCacheHeadDim,
                    cache->pages * cache->kv_heads * cache->page_tokens, kCacheHeadDim,
                    kCacheHeadDim, static_cast<uint32_t>(box_rows), swizzle);
}

// What both entry points refuse, so that no plan overflows.
void RequireSizes(const ov_kv_cache* cache, size_t rows, size_t max_rows, size_t max_length,
                  size_t heads) {
  OV_REQUIRE(heads > 0 && heads % cache->kv_heads == 0, "heads must be a multiple of kv_heads");
  OV_REQUIRE(heads <= 1024, "more than 1024 heads");
  OV_REQUIRE(rows < (size_t{1} << 31), "rows must stay below 2^31");
  OV_REQUIRE(max_length <= cache->max_pages * cache->page_tokens,
             "max_length exceeds the page table");
  // Room for lengths rounded up to a key tile, and a loader's lanes behind it.
  OV_REQUIRE(max_length <= (size_t{1} << 31) - 1024, "max_length must be at most 2^31 - 1024");
  OV_REQUIRE(std::min(max_rows, rows) <= ((size_t{1} << 31) - 512) / heads,
             "max_rows * heads must stay below 2^31");
}

}  // namespace
}  // namespace ovb

using namespace ovb;

extern "C" {

size_t ov_attention_kv_cache_workspace_bytes(const ov_kv_cache* cache, size_t rows,
                                             size_t max_rows, size_t max_length, size_t heads) {
  size_t bytes = 0;
  const int status = Guard("ov_attention_kv_cache_workspace_bytes: ", [&] {
    RequireShape(cache);
    RequireSizes(cache, rows, max_rows, max_length, heads);
    if (std::min(max_rows, rows) == 0 || cache->num_seqs == 0) return;
    const StreamPlan plan = PlanStream(cache, std::min(max_rows, rows), max_length, heads);
    const size_t parts = plan.rows > 0
                             ? plan.part_bytes
                             : PlanTiles(cache, std::min(max_rows, rows), max_length, heads).part_bytes;
    if (parts > 0) bytes = kCounterBytes + parts;
  });
  return status == OV_OK ? bytes : 0;
}

int ov_attention_kv_cache(const ov_kv_cache* cache, const uint16_t* q, size_t ld_q, size_t rows,
                          const int32_t* cu_rows, size_t max_rows, const int32_t* lengths,
                          size_t max_length, size_t heads, int causal, float scale, uint16_t* out,
                          size_t ld_out, void* workspace, size_t workspace_bytes,
                          ov_stream_t stream) {
  return Guard("ov_attention_kv_cache: ", [&] {
    const CacheView c = ViewCache(cache);
    RequireSizes(cache, rows, max_rows, max_length, heads);
    OV_REQUIRE(std::isfinite(scale) && scale > 0.0f, "scale must be positive and finite");
    OV_REQUIRE(ld_q % 8 == 0 && ld_q >= heads * kCacheHeadDim, "q stride");
    OV_REQUIRE(ld_out % 8 == 0 && ld_out >= heads * kCacheHeadDim, "out stride");
    if (rows == 0 || max_rows == 0 || c.num_seqs == 0) return;
    RequireAligned(q, 16, "q");
    RequireAligned(out, 16, "out");
    RequireAligned(cu_rows, 4, "cu_rows");
    RequireAligned(lengths, 4, "lengths");
    if (workspace != nullptr) RequireAligned(workspace, 16, "workspace");
    RequireOnDevice(cache);
    RequireOnDevice(q, "q");
    RequireOnDevice(out, "out");
    RequireOnDevice(cu_rows, "cu_rows");
    RequireOnDevice(lengths, "lengths");
    if (workspace != nullptr) RequireOnDevice(workspace, "workspace");
    CacheAttnArgs a{.group = FastDiv(static_cast<int>(heads / cache->kv_heads))};
    a.cache = c;
    a.q = reinterpret_cast<const __half*>(q);
    a.ld_q = static_cast<int64_t>(ld_q);
    a.out = reinterpret_cast<__half*>(out);
    a.ld_out = static_cast<int64_t>(ld_out);
    a.cu_rows = cu_rows;
    a.lengths = lengths;
    a.rows = static_cast<int>(rows);
    a.max_rows = static_cast<int>(std::min(max_rows, rows));
    a.max_length = static_cast<int>(max_length);
    a.causal = causal != 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.err = DeviceErrorWord();
    const StreamPlan plan = PlanStream(cache, a.max_rows, max_length, heads);
    if (plan.rows > 0) {
      const size_t box = std::min<size_t>(kUnit, cache->page_tokens);
      CUtensorMap map_k, map_v;
      EncodeCodesMap(&map_k, c.keys, cache, box, CU_TENSOR_MAP_SWIZZLE_128B);
      EncodeCodesMap(&map_v, c.values, cache, box, CU_TENSOR_MAP_SWIZZLE_128B);
      StreamArgs args{a, nullptr, nullptr, plan.rows};
      unsigned ctas = static_cast<unsigned>(c.num_seqs * c.kv_heads);
      if (workspace != nullptr && workspace_bytes >= kCounterBytes + plan.part_bytes) {
        args.counters = static_cast<uint32_t*>(workspace);
        args.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
        ctas = plan.ctas;
      }
      if (plan.rows <= 8) LaunchStream<1>(args, ctas, map_k, map_v, AsStream(stream));
      else LaunchStream<2>(args, ctas, map_k, map_v, AsStream(stream));
      return;
    }
    TilePlan tiles = PlanTiles(cache, a.max_rows, max_length, heads);
    TileArgs args{a, nullptr, nullptr, tiles.tile_rows, tiles.tiles, tiles.splits};
    if (tiles.splits > 1) {
      if (workspace != nullptr && workspace_bytes >= kCounterBytes + tiles.part_bytes) {
        args.counters = static_cast<uint32_t*>(workspace);
        args.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
      } else {
        args.splits = 1;
      }
    }
    const size_t grid = static_cast<size_t>(args.tiles) * args.splits * cache->kv_heads * cache->num_seqs;
    OV_REQUIRE(grid <= INT32_MAX, "max_rows times the sequences and heads is above what one launch takes");
    const size_t box = std::min<size_t>(kKeys, cache->page_tokens);
    CUtensorMap map_k, map_v;
    EncodeCodesMap(&map_k, c.keys, cache, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    EncodeCodesMap(&map_v, c.values, cache, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    SetMaxDynamicSmem(reinterpret_cast<const void*>(cache_attention_tile_kernel),
                      static_cast<int>(kTileSmem));
    Launch(cache_attention_tile_kernel,
           dim3(static_cast<unsigned>(grid)),
           dim3(kTileThreads), kTileSmem, AsStream(stream), "cache attention kernel launch", map_k,
           map_v, args);
  });
}

}  // extern "C"
