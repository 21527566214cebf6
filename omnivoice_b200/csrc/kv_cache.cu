// The paged 8-bit key/value cache: quantising packed rows into its pages
// (ov_kv_cache_write) and reading tokens back as half (ov_kv_cache_read).
//
//   scale = max(kept scale, amax * fl(1/127)),  code = rint(x * fl(1/scale)),
//   value = half(code * scale)
//
// with amax over the rows that a page and head take in this call.  The codes
// are rounded to 8 bits, which is the operator; everything before that is
// float32.  Both kernels move bytes and nothing else: a written element costs
// 2 bytes read and 1 written, a read one 1 and 2.  Measured on one B200, 8 kv
// heads: 131,000 tokens written and read back in 272 us (1.62 GB, 5.9 TB/s),
// the prompts of 64 utterances in 122 us (679 MB, 5.6 TB/s); 64 sequences read
// in 100 us (535 MB, 5.4 TB/s); one token written and its page read in 6.8 us.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "internal.hpp"
#include "kv_cache.hpp"
#include "launch.hpp"
#include "ov_kernels.h"
#include "ptx.cuh"

namespace ovb {
namespace {

constexpr int kThreads = 256;
constexpr float kStep = 1.0f / 127.0f;

// Two halves to two int8 codes (low bytes of the result): the rounded
// product plus 1.5 * 2^23 has the code in its low byte.
__device__ __forceinline__ uint32_t Codes2(uint32_t pair, float inverse) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&pair));
  const uint32_t a = __float_as_uint(__fadd_rn(__fmul_rn(x.x, inverse), 12582912.0f));
  const uint32_t b = __float_as_uint(__fadd_rn(__fmul_rn(x.y, inverse), 12582912.0f));
  return __byte_perm(a, b, 0x0040);
}

// The codes of four int8 values on a grid `ratio` times as coarse.
__device__ __forceinline__ uint32_t Rescale4(uint32_t codes, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = static_cast<int8_t>(codes >> (8 * i));
    const uint32_t q = __float_as_uint(
        __fadd_rn(__fmul_rn(static_cast<float>(c), ratio), 12582912.0f));
    out |= (q & 255u) << (8 * i);
  }
  return out;
}

// One CTA per (page of a sequence that this call touches, sequence, kv head
// and keys or values): a page's scale needs all of its rows, so they are held
// in registers (kPage / 16 vectors of 8 halves a thread) between the maximum
// and the rounding, and memory is read once.
template <int kPage>
__global__ void __launch_bounds__(kThreads, kPage <= 64 ? 8 : 4)
    cache_write_kernel(const CacheView c, const __half* __restrict__ k, int64_t ld_k,
                       const __half* __restrict__ v, int64_t ld_v, int rows,
                       const int32_t* __restrict__ cu_rows, const int32_t* __restrict__ starts,
                       int max_rows, uint32_t* err) {
  constexpr int kVec = kPage / 16;
  __shared__ uint32_t s_max[kThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.y;
  const int head = blockIdx.z >> 1;
  const bool value = blockIdx.z & 1;
  const RowSpan span = SequenceRows(cu_rows, seq, rows, max_rows, err);
  const int start = starts[seq];
  if (start < 0) {
    if (threadIdx.x == 0) atomicOr(err, kErrBadArgument);
    return;
  }
  // Tokens [lo, hi) of this page's slots come from the rows.
  const int64_t index = start / kPage + static_cast<int64_t>(blockIdx.x);
  const int64_t first_token = index * kPage;
  const int64_t end = static_cast<int64_t>(start) + span.count;
  if (span.count == 0 || first_token >= end) return;
  const int lo = blockIdx.x == 0 ? start % kPage : 0;
  const int hi = static_cast<int>(end - first_token < kPage ? end - first_token : kPage);
  const int page = CachePage(c, seq, index, err);
  if (page < 0) return;

  const int piece = threadIdx.x & 15;  // 8 of the 128 head dimensions
  const int row0 = threadIdx.x >> 4;
  const int64_t ld = value ? ld_v : ld_k;
  const __half* src = (value ? v : k) + (span.first + (first_token + row0 - start)) * ld +
                      head * kCacheHeadDim + piece * 8;
  const bool full = lo == 0 && hi == kPage;
  uint4 x[kVec];
  uint32_t top = 0;  // non-negative halves order as integers, NaN above infinity
  if (full) {
#pragma unroll
    for (int i = 0; i < kVec; ++i, src += 16 * ld)
      x[i] = *reinterpret_cast<const uint4*>(src);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i, src += 16 * ld) {
      const int slot = i * 16 + row0;
      x[i] = make_uint4(0, 0, 0, 0);
      if (slot >= lo && slot < hi) x[i] = *reinterpret_cast<const uint4*>(src);
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    top = __vmaxu2(top, x[i].x & 0x7FFF7FFFu);
    top = __vmaxu2(top, x[i].y & 0x7FFF7FFFu);
    top = __vmaxu2(top, x[i].z & 0x7FFF7FFFu);
    top = __vmaxu2(top, x[i].w & 0x7FFF7FFFu);
  }
  float* scales = value ? c.value_scales : c.key_scales;
  const int64_t scale_at = static_cast<int64_t>(page) * c.kv_heads + head;
  const float old = lo > 0 ? scales[scale_at] : 0.0f;
  top = __reduce_max_sync(0xFFFFFFFFu, max(top & 0xFFFFu, top >> 16));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
  __syncthreads();  // also: every thread has the old scale
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = max(top, s_max[w]);
  const float need = __fmul_rn(__half2float(__ushort_as_half(static_cast<uint16_t>(top))), kStep);
  float scale = fmaxf(need, old);
  if (top >= 0x7C00u || !(old < INFINITY)) scale = __uint_as_float(0x7FC00000u);
  const float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
  if (threadIdx.x == 0) scales[scale_at] = scale;

  int8_t* dst = (value ? c.values : c.keys) + CacheTile(c, page, head);
  int8_t* mine = dst + row0 * kCacheHeadDim + piece * 8;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int slot = i * 16 + row0;
    uint2 codes;
    codes.x = __byte_perm(Codes2(x[i].x, inverse), Codes2(x[i].y, inverse), 0x5410);
    codes.y = __byte_perm(Codes2(x[i].z, inverse), Codes2(x[i].w, inverse), 0x5410);
    if (full || (slot >= lo && slot < hi))
      *reinterpret_cast<uint2*>(mine + i * 16 * kCacheHeadDim) = codes;
  }
  // The kept slots [0, lo) onto the new grid.
  if (lo > 0 && scale > old) {
    const float ratio = __fdiv_rn(old, scale);
    for (int i = threadIdx.x; i < lo * (kCacheHeadDim / 16); i += kThreads) {
      uint4* p = reinterpret_cast<uint4*>(dst) + i;
      uint4 q = *p;
      q.x = Rescale4(q.x, ratio);
      q.y = Rescale4(q.y, ratio);
      q.z = Rescale4(q.z, ratio);
      q.w = Rescale4(q.w, ratio);
      *p = q;
    }
  }
}

// Tokens per CTA of the read
// (64 ragged sequences: 100 us with 16, 122 us with 8, 107 us with 32).
constexpr int kReadTokens = 16;

__device__ __forceinline__ uint32_t Halves2(uint32_t codes, int byte, float scale) {
  const int a = static_cast<int8_t>(codes >> (8 * byte));
  const int b = static_cast<int8_t>(codes >> (8 * byte + 8));
  return pack_half2(static_cast<float>(a) * scale, static_cast<float>(b) * scale);
}

// One CTA per kReadTokens tokens of a sequence, all heads, keys and values:
// 8 lanes read a token's 128 codes of a head, neighbouring tokens follow, so
// a warp reads 512 consecutive bytes and writes four 256-byte runs.
__global__ void __launch_bounds__(kThreads)
    cache_read_kernel(const CacheView c, const int32_t* __restrict__ cu_rows,
                      const int32_t* __restrict__ starts, int rows, int max_rows,
                      __half* __restrict__ k, int64_t ld_k, __half* __restrict__ v, int64_t ld_v,
                      uint32_t* err) {
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.y;
  const RowSpan span = SequenceRows(cu_rows, seq, rows, max_rows, err);
  const int start = starts[seq];
  const int row0 = static_cast<int>(blockIdx.x) * kReadTokens;
  if (row0 >= span.count) return;
  if (start < 0) {
    if (threadIdx.x == 0) atomicOr(err, kErrBadArgument);
    return;
  }
  const int piece = threadIdx.x & 7;
  const int token = (threadIdx.x >> 3) & (kReadTokens - 1);
  if (row0 + token >= span.count) return;
  const int64_t position = static_cast<int64_t>(start) + row0 + token;
  const int page = CachePage(c, seq, position >> c.page_shift, err);
  if (page < 0) return;
  const int slot = static_cast<int>(position & ((1 << c.page_shift) - 1));
  const int64_t row = span.first + row0 + token;
#pragma unroll 4
  for (int i = threadIdx.x >> 7; i < 2 * c.kv_heads; i += kThreads / 128) {
    const int head = i >> 1;
    const bool value = i & 1;
    const float scale = (value ? c.value_scales : c.key_scales)[static_cast<int64_t>(page) * c.kv_heads + head];
    const int8_t* src = (value ? c.values : c.keys) + CacheTile(c, page, head) +
                        slot * kCacheHeadDim + piece * 16;
    const uint4 q = *reinterpret_cast<const uint4*>(src);
    __half* dst = (value ? v + row * ld_v : k + row * ld_k) + head * kCacheHeadDim + piece * 16;
    uint4 a, b;
    a.x = Halves2(q.x, 0, scale);
    a.y = Halves2(q.x, 2, scale);
    a.z = Halves2(q.y, 0, scale);
    a.w = Halves2(q.y, 2, scale);
    b.x = Halves2(q.z, 0, scale);
    b.y = Halves2(q.z, 2, scale);
    b.z = Halves2(q.w, 0, scale);
    b.w = Halves2(q.w, 2, scale);
    *reinterpret_cast<uint4*>(dst) = a;
    *reinterpret_cast<uint4*>(dst + 8) = b;
  }
}

}  // namespace

void RequireAligned(const void* pointer, size_t align, const char* name) {
  if (pointer == nullptr) throw Error(OV_ERR_INVALID, std::string(name) + " must not be null");
  if (reinterpret_cast<uintptr_t>(pointer) % align != 0)
    throw Error(OV_ERR_INVALID, std::string(name) + " must be " + std::to_string(align) +
                                    "-byte aligned");
}

namespace {

// The driver's single-attribute query: a third of the runtime's cost, and
// each call asks it for about ten tensors.
using PointerAttributeFn = CUresult (*)(void*, CUpointer_attribute, CUdeviceptr);
PointerAttributeFn GetPointerAttribute() {
  static PointerAttributeFn fn = [] {
    void* symbol = nullptr;
    cudaDriverEntryPointQueryResult query{};
    const cudaError_t e =
        cudaGetDriverEntryPoint("cuPointerGetAttribute", &symbol, cudaEnableDefault, &query);
    if (e != cudaSuccess || query != cudaDriverEntryPointSuccess) return PointerAttributeFn{nullptr};
    return reinterpret_cast<PointerAttributeFn>(symbol);
  }();
  return fn;
}

}  // namespace

void RequireOnDevice(const void* pointer, const char* name) {
  int device = 0;
  Check(cudaGetDevice(&device), "cudaGetDevice");
  int owner = -1;
  const PointerAttributeFn query = GetPointerAttribute();
  if (query != nullptr &&
      query(&owner, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
            reinterpret_cast<CUdeviceptr>(pointer)) == CUDA_SUCCESS &&
      owner == device)
    return;
  cudaPointerAttributes attr{};  // another device's, unified or host memory
  Check(cudaPointerGetAttributes(&attr, pointer), "pointer attributes");
  if (attr.type == cudaMemoryTypeUnregistered ||
      (attr.type == cudaMemoryTypeDevice && attr.device != device))
    throw Error(OV_ERR_INVALID, std::string(name) + " is not memory of the current device");
}

void RequireOnDevice(const ov_kv_cache* cache) {
  RequireOnDevice(cache->keys, "keys");
  RequireOnDevice(cache->values, "values");
  RequireOnDevice(cache->key_scales, "key_scales");
  RequireOnDevice(cache->value_scales, "value_scales");
  RequireOnDevice(cache->page_table, "page_table");
}

void RequireShape(const ov_kv_cache* cache) {
  OV_REQUIRE(cache != nullptr, "cache must not be null");
  OV_REQUIRE(cache->head_dim == kCacheHeadDim, "head_dim must be 128");
  const size_t p = cache->page_tokens;
  OV_REQUIRE(p == 16 || p == 32 || p == 64 || p == 128, "page_tokens must be 16, 32, 64 or 128");
  OV_REQUIRE(cache->kv_heads > 0 && cache->kv_heads <= 1024, "kv_heads must be 1 to 1024");
  OV_REQUIRE(cache->num_seqs <= 65535, "more than 65535 sequences");
  OV_REQUIRE(cache->pages > 0 && cache->max_pages > 0, "the cache has no pages");
  OV_REQUIRE(cache->pages < (size_t{1} << 31) / (cache->kv_heads * p),
             "pages * kv_heads * page_tokens must stay below 2^31");
  OV_REQUIRE(cache->max_pages <= (size_t{1} << 31) / p - 1,
             "max_pages * page_tokens must stay below 2^31");
}

CacheView ViewCache(const ov_kv_cache* cache) {
  RequireShape(cache);
  const size_t p = cache->page_tokens;
  RequireAligned(cache->keys, 16, "keys");
  RequireAligned(cache->values, 16, "values");
  RequireAligned(cache->key_scales, 4, "key_scales");
  RequireAligned(cache->value_scales, 4, "value_scales");
  RequireAligned(cache->page_table, 4, "page_table");
  CacheView c;
  c.keys = cache->keys;
  c.values = cache->values;
  c.key_scales = cache->key_scales;
  c.value_scales = cache->value_scales;
  c.table = cache->page_table;
  c.pages = static_cast<int32_t>(cache->pages);
  c.page_shift = p == 16 ? 4 : p == 32 ? 5 : p == 64 ? 6 : 7;
  c.kv_heads = static_cast<int32_t>(cache->kv_heads);
  c.num_seqs = static_cast<int32_t>(cache->num_seqs);
  c.max_pages = static_cast<int32_t>(cache->max_pages);
  return c;
}

namespace {

// What the two entry points' rows have in common.
void CheckRows(const ov_kv_cache* cache, const uint16_t* k, size_t ld_k, const uint16_t* v,
               size_t ld_v, size_t rows, const int32_t* cu_rows, const int32_t* starts) {
  const size_t width = cache->kv_heads * kCacheHeadDim;
  OV_REQUIRE(rows < (size_t{1} << 31), "rows must stay below 2^31");
  OV_REQUIRE(ld_k % 8 == 0 && ld_k >= width, "k stride");
  OV_REQUIRE(ld_v % 8 == 0 && ld_v >= width, "v stride");
  RequireAligned(k, 16, "k");
  RequireAligned(v, 16, "v");
  RequireAligned(cu_rows, 4, "cu_rows");
  RequireAligned(starts, 4, "starts");
  RequireOnDevice(cache);
  RequireOnDevice(k, "k");
  RequireOnDevice(v, "v");
  RequireOnDevice(cu_rows, "cu_rows");
  RequireOnDevice(starts, "starts");
}

}  // namespace

}  // namespace ovb

using namespace ovb;

extern "C" {

int ov_kv_cache_write(const ov_kv_cache* cache, const uint16_t* k, size_t ld_k, const uint16_t* v,
                      size_t ld_v, size_t rows, const int32_t* cu_rows, const int32_t* starts,
                      size_t max_rows, ov_stream_t stream) {
  return Guard("ov_kv_cache_write: ", [&] {
    const CacheView c = ViewCache(cache);
    if (rows == 0 || max_rows == 0 || c.num_seqs == 0) return;
    CheckRows(cache, k, ld_k, v, ld_v, rows, cu_rows, starts);
    max_rows = std::min(max_rows, rows);
    // A start inside a page makes max_rows tokens touch one page more.
    const size_t page = cache->page_tokens;
    const dim3 grid(static_cast<unsigned>((max_rows + page - 2) / page + 1),
                    static_cast<unsigned>(c.num_seqs), static_cast<unsigned>(2 * c.kv_heads));
    auto kernel = page == 16   ? cache_write_kernel<16>
                  : page == 32 ? cache_write_kernel<32>
                  : page == 64 ? cache_write_kernel<64>
                               : cache_write_kernel<128>;
    Launch(kernel, grid, dim3(kThreads), 0, AsStream(stream), "cache write kernel launch", c,
           reinterpret_cast<const __half*>(k), static_cast<int64_t>(ld_k),
           reinterpret_cast<const __half*>(v), static_cast<int64_t>(ld_v), static_cast<int>(rows),
           cu_rows, starts, static_cast<int>(max_rows), DeviceErrorWord());
  });
}

int ov_kv_cache_read(const ov_kv_cache* cache, const int32_t* cu_rows, const int32_t* starts,
                     size_t rows, size_t max_rows, uint16_t* k, size_t ld_k, uint16_t* v,
                     size_t ld_v, ov_stream_t stream) {
  return Guard("ov_kv_cache_read: ", [&] {
    const CacheView c = ViewCache(cache);
    if (rows == 0 || max_rows == 0 || c.num_seqs == 0) return;
    CheckRows(cache, k, ld_k, v, ld_v, rows, cu_rows, starts);
    max_rows = std::min(max_rows, rows);
    const dim3 grid(static_cast<unsigned>((max_rows + kReadTokens - 1) / kReadTokens),
                    static_cast<unsigned>(c.num_seqs));
    Launch(cache_read_kernel, grid, dim3(kThreads), 0, AsStream(stream),
           "cache read kernel launch", c, cu_rows, starts, static_cast<int>(rows),
           static_cast<int>(max_rows), reinterpret_cast<__half*>(k), static_cast<int64_t>(ld_k),
           reinterpret_cast<__half*>(v), static_cast<int64_t>(ld_v), DeviceErrorWord());
  });
}

}  // extern "C"
