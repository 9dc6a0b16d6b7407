// token_logprobs.cu - log probabilities of given tokens with entropy and the best alternatives, and their gradient, for B200 (sm_100a).
//
// Per row of logits x, z = scale x, m = max z, S = sum exp(z - m):
//   lse = m + log S      logp = (z_t - m) - log S      entropy = log S - (sum exp(z - m) (z - m)) / S      top k of x, equal ones by index
//   dx = scale (g (onehot - p) - h p (log p + entropy)),  p = exp(z - lse),  g, h the gradients of logp and entropy
// The entropy is formed from differences to the maximum, so that nothing large cancels; a column with exp(z - m) = 0 adds nothing (its z - m
// may be -inf). All sums in fp32.
#include <float.h>
#include <math.h>

#include "df_common.cuh"
#include "sm100_ptx.cuh"

namespace df {
namespace {

constexpr int kThreads = 512;

template <bool BF16>
__device__ __forceinline__ float load1(const void *base, size_t e) {
  if (BF16) return __uint_as_float((uint32_t)__ldg(static_cast<const uint16_t *>(base) + e) << 16);
  return __ldg(static_cast<const float *>(base) + e);
}
__device__ __forceinline__ uint16_t to_bf16(float x) {
  uint16_t r;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(x));
  return r;
}

// A total order of floats as unsigned integers: -inf lowest, NaN highest, -0 equal to +0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (isnan(x)) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct LogprobParams {
  const void *logits;
  const int32_t *targets;
  float *logp, *entropy, *lse, *top_logp;
  int32_t *top_ids;
  unsigned long long stride;
  uint32_t rows, cols, top_k;
  float scale;
};

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, Op op, T *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  T r = red[0];
  for (int w = 1; w < kThreads / 32; ++w) r = op(r, red[w]);
  return r;
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads) k_token_logprobs(const LogprobParams p) {
  ptx::pdl_wait();
  __shared__ float red[kThreads / 32];
  __shared__ unsigned long long red_key[kThreads / 32];
  const uint32_t row = blockIdx.x, t = threadIdx.x;
  const size_t base = (size_t)row * p.stride;
  auto add = [](float a, float b) { return a + b; };
  float top = -INFINITY;
  bool bad = false;
  for (uint32_t i = t; i < p.cols; i += kThreads) {
    const float z = load1<BF16>(p.logits, base + i) * p.scale;
    bad |= isnan(z) || z == INFINITY;
    top = fmaxf(top, z);
  }
  bad = __syncthreads_or(bad);
  top = block_reduce(top, [](float a, float b) { return fmaxf(a, b); }, red);
  const float m = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, weighted = 0.0f;
  for (uint32_t i = t; i < p.cols; i += kThreads) {
    const float y = load1<BF16>(p.logits, base + i) * p.scale - m, e = expf(y);
    sum += e;
    weighted += e > 0.0f ? e * y : 0.0f;
  }
  sum = block_reduce(sum, add, red);
  weighted = block_reduce(weighted, add, red);
  const float log_sum = bad ? NAN : logf(sum);
  // z - m first: their difference is exact where it matters, while m + log S would round log S away beside a large m
  auto logp_of = [&](float x) { return bad ? NAN : top == -INFINITY ? -INFINITY : (x * p.scale - m) - log_sum; };
  if (t == 0) {
    const int32_t target = __ldg(p.targets + row);
    p.lse[row] = bad ? NAN : top == -INFINITY ? -INFINITY : m + log_sum;
    p.entropy[row] = bad ? NAN : top == -INFINITY ? 0.0f : log_sum - weighted / sum;
    p.logp[row] = target >= 0 && (uint32_t)target < p.cols ? logp_of(load1<BF16>(p.logits, base + target)) : 0.0f;
  }
  unsigned long long last = ~0ull;  // key of the alternative before: order of the value, then the lower index
  for (uint32_t k = 0; k < p.top_k; ++k) {
    unsigned long long best = 0;
    for (uint32_t i = t; i < p.cols; i += kThreads) {
      const unsigned long long key = ((unsigned long long)order_of(load1<BF16>(p.logits, base + i)) << 32) | (0xffffffffu - i);
      if ((k == 0 || key < last) && key > best) best = key;
    }
    last = best = block_reduce(best, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; }, red_key);
    if (t == 0) {
      const uint32_t id = 0xffffffffu - (uint32_t)best;
      p.top_ids[(size_t)row * p.top_k + k] = (int32_t)id;
      p.top_logp[(size_t)row * p.top_k + k] = logp_of(load1<BF16>(p.logits, base + id));
    }
  }
}

struct LogprobGradParams {
  const void *logits;
  const int32_t *targets;
  const float *lse, *entropy, *grad_logp, *grad_entropy;
  void *d_logits;
  unsigned long long stride, d_stride;
  uint32_t rows, cols;
  float scale;
};

template <bool BF16>
__global__ void __launch_bounds__(kThreads) k_token_logprobs_backward(const LogprobGradParams p) {
  ptx::pdl_wait();
  const uint32_t row = blockIdx.x, t = threadIdx.x;
  const int32_t target = __ldg(p.targets + row);
  const bool has = target >= 0 && (uint32_t)target < p.cols;
  const float lse = __ldg(p.lse + row), entropy = __ldg(p.entropy + row);
  const float g = has && p.grad_logp ? __ldg(p.grad_logp + row) : 0.0f, h = p.grad_entropy ? __ldg(p.grad_entropy + row) : 0.0f;
  for (uint32_t i = t; i < p.cols; i += kThreads) {
    const float y = load1<BF16>(p.logits, (size_t)row * p.stride + i) * p.scale - lse, prob = expf(y);
    const float d = p.scale * ((has && i == (uint32_t)target ? g : 0.0f) - (prob == 0.0f ? 0.0f : prob * (g + h * (y + entropy))));
    if (BF16) static_cast<uint16_t *>(p.d_logits)[(size_t)row * p.d_stride + i] = to_bf16(d);
    else static_cast<float *>(p.d_logits)[(size_t)row * p.d_stride + i] = d;
  }
}

int finish(int st) {
  note_status(st);
  return st;
}

}  // namespace
}  // namespace df

using namespace df;

extern "C" {

int df_token_logprobs(const void *logits, const int32_t *targets, float *logp, float *entropy, float *lse, int *top_ids, float *top_logp,
                      uint32_t rows, uint32_t cols, uint64_t row_stride, uint32_t top_k, float scale, uint32_t logits_bf16, void *stream) {
  DF_RANGE("df_token_logprobs");
  if (top_k > DF_LOGPROBS_MAX_TOP || top_k > cols || cols == 0 || cols >= (1u << 31) || rows >= (1u << 31)) return finish(DF_ERR_INVALID_ARG);
  if (!(scale > 0.0f) || !isfinite(scale) || (rows > 1 && row_stride < cols)) return finish(DF_ERR_INVALID_ARG);
  if (rows == 0) return DF_OK;
  if (!logits || !targets || !logp || !entropy || !lse || (top_k && (!top_ids || !top_logp))) return finish(DF_ERR_INVALID_ARG);
  const LogprobParams p = {logits, targets, logp, entropy, lse, top_logp, top_ids, row_stride, rows, cols, top_k, scale};
  const int st = check_cuda(launch_kernel(logits_bf16 ? k_token_logprobs<true> : k_token_logprobs<false>, dim3(rows), dim3(kThreads), 0,
                                          static_cast<cudaStream_t>(stream), p));
  note_launch();
  return finish(st);
}

int df_token_logprobs_backward(const void *logits, const int32_t *targets, const float *lse, const float *entropy, const float *grad_logp,
                               const float *grad_entropy, void *d_logits, uint32_t rows, uint32_t cols, uint64_t row_stride,
                               uint64_t d_row_stride, float scale, uint32_t logits_bf16, void *stream) {
  DF_RANGE("df_token_logprobs_backward");
  if (cols == 0 || cols >= (1u << 31) || rows >= (1u << 31) || !(scale > 0.0f) || !isfinite(scale)) return finish(DF_ERR_INVALID_ARG);
  if (rows > 1 && (row_stride < cols || d_row_stride < cols)) return finish(DF_ERR_INVALID_ARG);
  if (rows == 0) return DF_OK;
  if (!logits || !targets || !lse || !entropy || !d_logits) return finish(DF_ERR_INVALID_ARG);
  if (logits == d_logits && rows > 1 && row_stride != d_row_stride) return finish(DF_ERR_INVALID_ARG);
  const LogprobGradParams p = {logits, targets, lse, entropy, grad_logp, grad_entropy, d_logits, row_stride, d_row_stride, rows, cols, scale};
  const int st = check_cuda(launch_kernel(logits_bf16 ? k_token_logprobs_backward<true> : k_token_logprobs_backward<false>, dim3(rows),
                                          dim3(kThreads), 0, static_cast<cudaStream_t>(stream), p));
  note_launch();
  return finish(st);
}

}  // extern "C"
