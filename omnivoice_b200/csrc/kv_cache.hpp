// The paged 8-bit key/value cache as its kernels see it (kv_cache.cu writes
// and reads it, attention_cache.cu attends over it), and the host checks its
// entry points share.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "internal.hpp"
#include "ov_kernels.h"

namespace ovb {

constexpr int kCacheHeadDim = 128;

struct CacheView {
  int8_t* keys;
  int8_t* values;
  float* key_scales;
  float* value_scales;
  const int32_t* table;
  int32_t pages;
  int32_t page_shift;  // log2(page_tokens)
  int32_t kv_heads;
  int32_t num_seqs;
  int32_t max_pages;
};

// Refuses sizes of a cache that the kernels do not take.
void RequireShape(const ov_kv_cache* cache);

// Checks a cache description (without its pointers' device) and returns the
// kernels' view of it.
CacheView ViewCache(const ov_kv_cache* cache);

// Refuses a tensor that is null or not `align`-byte aligned.
void RequireAligned(const void* pointer, size_t align, const char* name);

// Refuses memory that the current device does not own: another device's, or
// unregistered host memory, would fault in a kernel.
void RequireOnDevice(const void* pointer, const char* name);
void RequireOnDevice(const ov_kv_cache* cache);

#ifdef __CUDACC__

// Page of table entry `index` of a sequence, or -1 (reported) when the table
// or the cache has no such page.
__device__ __forceinline__ int CachePage(const CacheView& c, int seq, int64_t index,
                                         uint32_t* err) {
  if (index >= c.max_pages) {
    atomicOr(err, kErrBadArgument);
    return -1;
  }
  const int page = c.table[static_cast<int64_t>(seq) * c.max_pages + index];
  if (page < 0 || page >= c.pages) {
    atomicOr(err, kErrBadArgument);
    return -1;
  }
  return page;
}

// First element of slot 0 of (page, head); below 2^38 for the 2^31 rows that
// ViewCache allows, hence 64 bits.
__device__ __forceinline__ int64_t CacheTile(const CacheView& c, int page, int head) {
  return ((static_cast<int64_t>(page) * c.kv_heads + head) << c.page_shift) * kCacheHeadDim;
}

struct RowSpan {
  int first;
  int count;
};

// Packed rows [begin, end) of a sequence; none (reported) when its bounds are
// not valid.
__device__ __forceinline__ RowSpan CheckRows(int begin, int end, int rows, int max_rows,
                                             uint32_t* err) {
  if (begin < 0 || end < begin || end > rows || end - begin > max_rows) {
    atomicOr(err, kErrBadArgument);
    return {0, 0};
  }
  return {begin, end - begin};
}
__device__ __forceinline__ RowSpan SequenceRows(const int32_t* cu_rows, int seq, int rows,
                                                int max_rows, uint32_t* err) {
  return CheckRows(cu_rows[seq], cu_rows[seq + 1], rows, max_rows, err);
}

#endif  // __CUDACC__

}  // namespace ovb
