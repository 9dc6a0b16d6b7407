// cache_attention.cu - attention of ragged queries over an 8-bit paged cache, for B200 (sm_100a).
//
// For query row (token j of request r, head h), with kv = h / (n_heads / n_kv_heads) and last = lens[r] - q_len + j:
//   s_t = scale * k_scale[page(t), kv] * (q . k_code_t),  t = 0 .. last        m = max s, l = sum exp(s_t - m)
//   out = sum exp(s_t - m) / l * v_scale[page(t), kv] * v_code_t               lse = m + log l
// One pass with a running maximum and sum per row.
#include <float.h>
#include <math.h>

#include "cache_codes.cuh"
#include "sm100_ptx.cuh"

namespace df {
namespace {

struct AttendParams {
  const void *q;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  const int32_t *table, *lens, *starts;
  void *out;
  float *lse;
  unsigned long long q_stride;
  uint32_t n_requests, n_tokens, heads, kv_heads, D, P, n_pages, width;
  float scale;
};

template <bool BF16>
__device__ __forceinline__ float load1(const void *base, size_t e) {
  if (BF16) return __uint_as_float((uint32_t)__ldg(static_cast<const uint16_t *>(base) + e) << 16);
  return __ldg(static_cast<const float *>(base) + e);
}

template <bool BF16, int FORMAT>
__global__ void __launch_bounds__(128) k_cache_attention(const AttendParams p) {
  ptx::pdl_wait();
  __shared__ float sm_m[4], sm_l[4], sm_o[4][128];
  const uint32_t token = blockIdx.x, h = blockIdx.y, kv = h / (p.heads / p.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t r = 0;
  for (; r < p.n_requests; ++r)
    if ((int)token >= __ldg(p.starts + r) && (int)token < __ldg(p.starts + r + 1)) break;
  if (r == p.n_requests) return;
  const long long len = min((long long)max(__ldg(p.lens + r), 0), (long long)p.width * p.P);
  const long long see = len - __ldg(p.starts + r + 1) + (long long)token + 1;  // keys that the row sees
  float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -FLT_MAX, l = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t d = lane + 32 * i;
    q[i] = d < p.D ? load1<BF16>(p.q, (size_t)token * p.q_stride + (size_t)h * p.D + d) * (p.scale * kLog2e) : 0.0f;
  }
  for (long long t = warp; t < see; t += 4) {
    const uint32_t page = (uint32_t)__ldg(p.table + (size_t)r * p.width + t / p.P);
    const bool in = page < p.n_pages;
    const size_t slice = (size_t)(in ? page : 0) * p.kv_heads + kv, at = (slice * p.P + t % p.P) * p.D;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = lane + 32 * i;
      if (d < p.D && in) dot = fmaf(q[i], cache_value<FORMAT>(__ldg(p.k + at + d)), dot);
    }
#pragma unroll
    for (int o2 = 16; o2 > 0; o2 >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o2);
    const float s = dot * (in ? __ldg(p.k_scale + slice) : 0.0f);
    const float top = fmaxf(m, s), alpha = exp2f(m - top), e = exp2f(s - top);
    const float w = e * (in ? __ldg(p.v_scale + slice) : 0.0f);
    m = top;
    l = fmaf(l, alpha, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = lane + 32 * i;
      if (d < p.D) o[i] = fmaf(w, in ? cache_value<FORMAT>(__ldg(p.v + at + d)) : 0.0f, o[i] * alpha);
    }
  }
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
  for (int i = 0; i < 4; ++i) sm_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  const uint32_t d = threadIdx.x;
  float M = -FLT_MAX, L = 0.0f, O = 0.0f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w]);
  for (int w = 0; w < 4; ++w) {
    const float f = exp2f(sm_m[w] - M);
    L = fmaf(sm_l[w], f, L);
    O = fmaf(sm_o[w][d], f, O);
  }
  if (d < p.D) {
    const float x = L == 0.0f ? 0.0f : O / L;
    const size_t e = ((size_t)token * p.heads + h) * p.D + d;
    if (BF16) {
      uint16_t b;
      asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(b) : "f"(x));
      static_cast<uint16_t *>(p.out)[e] = b;
    } else {
      static_cast<float *>(p.out)[e] = x;
    }
  }
  if (d == 0 && p.lse) p.lse[(size_t)token * p.heads + h] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

int finish(int st) {
  note_status(st);
  return st;
}

}  // namespace
}  // namespace df

using namespace df;

extern "C" int df_cache_attention(const void *q, const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale,
                                  const int32_t *block_table, const int32_t *lens, const int32_t *starts, void *out, float *lse, void *workspace,
                                  uint64_t workspace_bytes, uint32_t n_requests, uint32_t n_tokens, uint32_t n_heads, uint32_t n_kv_heads,
                                  uint32_t d_head, uint32_t page_size, uint32_t n_pages, uint32_t table_width, uint64_t q_row_stride, float scale,
                                  uint32_t q_bf16, uint32_t format, void *stream) {
  DF_RANGE("df_cache_attention");
  if (!cache_shape_valid(n_kv_heads, d_head, page_size, n_pages) || n_tokens >= (1u << 31) || n_requests >= (1u << 31)) return finish(DF_ERR_INVALID_ARG);
  if (format != DF_CACHE_INT8 && format != DF_CACHE_E4M3) return finish(DF_ERR_INVALID_ARG);
  if (n_heads == 0 || n_heads % n_kv_heads != 0 || n_heads > 65535u || !isfinite(scale)) return finish(DF_ERR_INVALID_ARG);
  if (n_tokens > 1 && q_row_stride < (uint64_t)n_heads * d_head) return finish(DF_ERR_INVALID_ARG);
  if (!cache_shape_supported(d_head, page_size)) return finish(DF_ERR_UNSUPPORTED);
  if (n_tokens == 0 || n_requests == 0) return DF_OK;
  if (!q || !lens || !starts || !out || (n_pages && (!k_cache || !v_cache || !k_scale || !v_scale)) || (table_width && !block_table))
    return finish(DF_ERR_INVALID_ARG);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return finish(DF_ERR_INVALID_ARG);
  if (workspace_bytes < DF_CACHE_WORKSPACE_BYTES) return finish(DF_ERR_WORKSPACE);
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15u) != 0) return finish(DF_ERR_UNSUPPORTED);
  const AttendParams p = {q, static_cast<const uint8_t *>(k_cache), static_cast<const uint8_t *>(v_cache), k_scale, v_scale, block_table, lens, starts, out, lse,
                          q_row_stride, n_requests, n_tokens, n_heads, n_kv_heads, d_head, page_size, n_pages, table_width, scale};
  auto kernel = q_bf16 ? (format == DF_CACHE_INT8 ? k_cache_attention<true, DF_CACHE_INT8> : k_cache_attention<true, DF_CACHE_E4M3>)
                       : (format == DF_CACHE_INT8 ? k_cache_attention<false, DF_CACHE_INT8> : k_cache_attention<false, DF_CACHE_E4M3>);
  const int st = check_cuda(launch_kernel(kernel, dim3(n_tokens, n_heads), dim3(128), 0, static_cast<cudaStream_t>(stream), p));
  note_launch();
  return finish(st);
}
