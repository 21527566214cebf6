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
  int heads;
  int group;  // heads / kv_heads
  int causal;
  float scale_log2;  // softmax scale * log2(e)
  uint32_t* err;
};

// Stands for a value scale of 0: its codes add nothing, its tokens still
// count in the denominator.  Below the least scale of a nonzero half page.
constexpr float kZeroScale = 0x1.0p-31f;

// Tokens of a sequence, bounded by what the call announced.
__device__ __forceinline__ int SequenceLength(const CacheAttnArgs& a, int seq) {
  const int length = a.lengths[seq];
  if (length < 0 || length > a.max_length) {
    atomicOr(a.err, kErrBadArgument);
    return length < 0 ? 0 : a.max_length;
  }
  return length;
}

// One warp per (row, head): lane l holds head dimensions 4l .. 4l + 3, one
// token after the other.
__global__ void __launch_bounds__(128) cache_attention_row_kernel(const CacheAttnArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.z;
  const int kv_head = head / a.group;
  const int seq = blockIdx.y;
  const RowSpan span = SequenceRows(a.cu_rows, seq, a.rows, a.max_rows, a.err);
  const int i = static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (i >= span.count) return;
  const int length = SequenceLength(a, seq);
  const int seen = a.causal ? max(0, length - span.count + i + 1) : length;
  const int64_t row = span.first + i;
  const uint2 qp = *reinterpret_cast<const uint2*>(a.q + row * a.ld_q + head * kCacheHeadDim + lane * 4);
  const float2 q0 = __half22float2(*reinterpret_cast<const __half2*>(&qp.x));
  const float2 q1 = __half22float2(*reinterpret_cast<const __half2*>(&qp.y));
  float m = -INFINITY, l = 0.0f, o[4] = {};
  const int page_tokens = 1 << a.cache.page_shift;
  for (int first = 0; first < seen; first += page_tokens) {
    const int page = CachePage(a.cache, seq, first >> a.cache.page_shift, a.err);
    if (page < 0) continue;
    const int64_t at = static_cast<int64_t>(page) * a.cache.kv_heads + kv_head;
    const float c = a.scale_log2 * a.cache.key_scales[at];
    float b = a.cache.value_scales[at];
    b = b == 0.0f ? kZeroScale : b;
    const float shift = log2f(b), inverse = 1.0f / b;
    const int64_t tile = CacheTile(a.cache, page, kv_head) + lane * 4;
    const int n = min(page_tokens, seen - first);
    for (int j = 0; j < n; ++j) {
      const char4 kc = *reinterpret_cast<const char4*>(a.cache.keys + tile + j * kCacheHeadDim);
      const char4 vc = *reinterpret_cast<const char4*>(a.cache.values + tile + j * kCacheHeadDim);
      const float t = fmaf(warp_sum(q0.x * kc.x + q0.y * kc.y + q1.x * kc.z + q1.y * kc.w), c, shift);
      const float top = fmaxf(m, t);
      const float old = exp2f(m - top), p = exp2f(t - top);
      m = top;
      l = l * old + p * inverse;
      o[0] = o[0] * old + p * vc.x;
      o[1] = o[1] * old + p * vc.y;
      o[2] = o[2] * old + p * vc.z;
      o[3] = o[3] * old + p * vc.w;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<uint2*>(a.out + row * a.ld_out + head * kCacheHeadDim + lane * 4) =
      make_uint2(pack_half2(o[0] * inv, o[1] * inv), pack_half2(o[2] * inv, o[3] * inv));
}

}  // namespace
}  // namespace ovb

using namespace ovb;

extern "C" {

size_t ov_attention_kv_cache_workspace_bytes(const ov_kv_cache* cache, size_t rows,
                                             size_t max_rows, size_t max_length, size_t heads) {
  (void)cache, (void)rows, (void)max_rows, (void)max_length, (void)heads;
  return 0;
}

int ov_attention_kv_cache(const ov_kv_cache* cache, const uint16_t* q, size_t ld_q, size_t rows,
                          const int32_t* cu_rows, size_t max_rows, const int32_t* lengths,
                          size_t max_length, size_t heads, int causal, float scale, uint16_t* out,
                          size_t ld_out, void* workspace, size_t workspace_bytes,
                          ov_stream_t stream) {
  return Guard("ov_attention_kv_cache: ", [&] {
    (void)workspace_bytes;
    const CacheView c = ViewCache(cache);
    OV_REQUIRE(heads > 0 && heads % cache->kv_heads == 0, "heads must be a multiple of kv_heads");
    OV_REQUIRE(heads <= 1024, "more than 1024 heads");
    OV_REQUIRE(std::isfinite(scale) && scale > 0.0f, "scale must be positive and finite");
    OV_REQUIRE(rows < (size_t{1} << 31), "rows must stay below 2^31");
    OV_REQUIRE(max_length <= cache->max_pages * cache->page_tokens,
               "max_length exceeds the page table");
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
    CacheAttnArgs a;
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
    a.heads = static_cast<int>(heads);
    a.group = static_cast<int>(heads / cache->kv_heads);
    a.causal = causal != 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.err = DeviceErrorWord();
    const dim3 grid(static_cast<unsigned>((a.max_rows + 3) / 4), static_cast<unsigned>(c.num_seqs),
                    static_cast<unsigned>(heads));
    Launch(cache_attention_row_kernel, grid, dim3(128), 0, AsStream(stream),
           "cache attention kernel launch", a);
  });
}

}  // extern "C"
