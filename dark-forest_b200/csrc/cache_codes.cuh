// cache_codes.cuh - the 8-bit codes of the paged cache (include/darkforest_kernels.h: DF_CACHE_*), shared by the kernels that write and read it.
#pragma once

#include <cuda_fp16.h>

#include "df_common.cuh"

namespace df {

constexpr uint32_t kCacheMaxHead = 128, kCacheMaxPage = 256;

// d_head and page_size that the cache kernels take: slices of a page and head are then whole 128-byte lines, rows whole 16-byte pieces.
inline bool cache_shape_supported(uint32_t d_head, uint32_t page_size) {
  return d_head % 16 == 0 && d_head <= kCacheMaxHead && page_size % 16 == 0 && page_size <= kCacheMaxPage;
}
inline bool cache_shape_valid(uint32_t n_kv_heads, uint32_t d_head, uint32_t page_size, uint32_t n_pages) {
  return n_kv_heads != 0 && d_head != 0 && page_size != 0 && (uint64_t)n_pages * page_size < (1ull << 31) && (uint64_t)n_pages * n_kv_heads < (1ull << 31);
}

// The value of one code. An 8-bit float has the fields s eeee fff (bias 7): its seven low bits moved up by seven are those of a half with bias 15, i.e.
// the value times 2^-8, subnormals included, so that no table and no special case is needed (and 0x7f reads as 480, not NaN:
// df_cache_append never writes it; the attention kernels' own conversion gives NaN).
template <int FORMAT>
__device__ __forceinline__ float cache_value(uint32_t code) {
  if (FORMAT == DF_CACHE_INT8) return (float)(int8_t)(uint8_t)code;
  const uint16_t h = (uint16_t)(((code & 0x80u) << 8) | ((code & 0x7fu) << 7));
  return __half2float(__ushort_as_half(h)) * 256.0f;
}

}  // namespace df
