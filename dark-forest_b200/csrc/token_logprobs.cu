// token_logprobs.cu - log probabilities of given tokens with entropy and the best alternatives, and their gradient, for B200 (sm_100a).
//
// Per row of logits x, z = scale x, m = max z, S = sum exp(z - m):
//   lse = m + log S      logp = (z_t - m) - log S      entropy = log S - (sum exp(z - m) (z - m)) / S      top k of x, equal ones by index
//   dx = scale (g (onehot - p) - h p (log p + entropy)),  p = exp(z - lse),  g, h the gradients of logp and entropy
// The entropy is formed from differences to the maximum, so that nothing large cancels; a column with exp(z - m) = 0 adds nothing (its z - m
// may be -inf). All sums in fp32.
//
// Both directions are bound by HBM: the forward reads every logit once, the gradient reads and writes it once. In the forward a row is cut
// into slices, one for each CTA of a cluster, and a slice lies in the shared memory of its CTA, at most kUsual 16-byte groups a thread (104 KB: two CTAs
// of an SM load and compute at different times; four of half the size spent as much on their ends as on their elements) unless the row is longer than eight such slices. The CTAs' parts (maximum, sums, best
// keys) meet in the shared memory of the cluster's first.
// Alternatives without sorting a row: the ceil(k / 16)-th largest of its lanes' maxima is found in each of sixteen warps; the smallest of
// these is a bound that at least k elements of the slice reach, and for logits in no particular order a few dozen do. Only the lanes whose maximum
// reaches it are looked through, by their whole warp, and what is found is put in a list and ranked by counting (key: the value's order, then the
// lower index). Where more than the list's length reach the bound (equal logits, masked rows) the k best are taken one after another.
// Rows beyond 8 CTAs of kMost groups (442368 fp32 columns, 884736 bf16) are walked in global memory by one CTA each.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <float.h>
#include <math.h>

#include <mutex>

#include "df_common.cuh"
#include "sm100_ptx.cuh"

namespace cg = cooperative_groups;

namespace df {
namespace {

using ptx::ex2_approx;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxSlices = 8, kList = 256, kTop = DF_LOGPROBS_MAX_TOP;
constexpr uint32_t kMost = 27, kUsual = 13;  // groups of a thread: one CTA of an SM, two of them
static_assert(kMaxSlices * kTop <= kThreads, "a thread for each of the CTAs' alternatives");

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

// A total order of floats as unsigned integers: -inf lowest, NaN highest, -0 equal to +0; and back.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (isnan(x)) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return order == 0xffffffffu ? NAN : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ float bound_of(uint32_t order) { return order < 0x00800000u ? -INFINITY : value_of(order); }  // (the last bit may be off)
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t i) { return ((unsigned long long)order_of(x) << 32) | (0xffffffffu - i); }

struct LogprobParams {
  const void *logits;
  const int32_t *targets;
  float *logp, *entropy, *lse, *top_logp;
  int32_t *top_ids;
  unsigned long long stride;
  uint32_t rows, cols, top_k, slices, groups;
  float scale;
};

// A row as a scalar head up to the next 16-byte boundary, 16-byte groups, and a scalar tail.
template <bool BF16>
struct RowSplit {
  static constexpr uint32_t kElements = BF16 ? 8 : 4;
  uint32_t head, groups;
  __device__ __forceinline__ RowSplit(const void *row, uint32_t cols) {
    const uint32_t past = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u) / (16 / kElements);
    head = min((kElements - past) % kElements, cols);
    groups = (cols - head) / kElements;
  }
  __device__ __forceinline__ uint32_t body_end() const { return head + groups * kElements; }
};
template <bool BF16>
__device__ __forceinline__ const void *row_at(const void *base, uint32_t row, unsigned long long stride) {
  return static_cast<const uint8_t *>(base) + (size_t)row * stride * (BF16 ? 2 : 4);
}
// element e of a 16-byte group
template <bool BF16>
__device__ __forceinline__ float element(const uint4 &v, int e) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if (BF16) return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
  return __uint_as_float(w[e]);
}

// Two elements' exp(z - m) and its product with z - m, in units of log 2: y = (x - max x) * (scale * log2 e). The difference first: it is exact where it
// matters, and neither a large maximum nor its product with the scale can round it away or overflow.
struct Sums2 {
  float2 sum = {0.0f, 0.0f}, weighted = {0.0f, 0.0f};
  __device__ __forceinline__ void add(float a, float b, float2 scale_log2, float2 minus_top) {
    float2 y = ptx::mul2(ptx::add2(make_float2(a, b), minus_top), scale_log2);
    const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
    y = make_float2(fmaxf(y.x, -2000.0f), fmaxf(y.y, -2000.0f));  // -inf: its e is 0, the product 0 too
    sum = ptx::add2(sum, e);
    weighted = ptx::fma2(e, y, weighted);
  }
  __device__ __forceinline__ void add(const Sums2 &o) {
    sum = ptx::add2(sum, o.sum);
    weighted = ptx::add2(weighted, o.weighted);
  }
};

// A finished row: its largest logit (-inf where nothing can come), and sums in units of log 2.
struct RowResult {
  float top, sum, weighted;
  bool bad;  // a NaN or +inf
  __device__ __forceinline__ float logp(float x, float scale) const {
    return bad ? NAN : top == -INFINITY ? -INFINITY : fmaf(x - top, scale, -log2f(sum) * kLn2);
  }
  template <bool BF16>
  __device__ __forceinline__ void write(const LogprobParams &p, uint32_t row, const void *grow) const {
    const int32_t target = __ldg(p.targets + row);
    p.lse[row] = bad ? NAN : top == -INFINITY ? -INFINITY : fmaf(top, p.scale, log2f(sum) * kLn2);
    p.entropy[row] = bad ? NAN : top == -INFINITY ? 0.0f : (log2f(sum) - weighted / sum) * kLn2;
    p.logp[row] = target >= 0 && (uint32_t)target < p.cols ? logp(load1<BF16>(grow, target), p.scale) : 0.0f;
  }
  __device__ __forceinline__ void write_top(const LogprobParams &p, uint32_t row, uint32_t k, unsigned long long key) const {
    p.top_ids[(size_t)row * p.top_k + k] = (int32_t)(0xffffffffu - (uint32_t)key);
    p.top_logp[(size_t)row * p.top_k + k] = logp(value_of((uint32_t)(key >> 32)), p.scale);
  }
};

// What a CTA knows of its slice, and in the cluster's first CTA what the others send.
struct SliceSmem {
  unsigned long long list[kList];
  unsigned long long best[kMaxSlices * kTop];  // (first CTA) every CTA's best, in order
  float4 part[kMaxSlices];                     // (first CTA) maximum, sum, weighted sum, bad
  float red[3][kWarps];
  unsigned long long red_key[kWarps];
  uint32_t bound[kWarps];
  uint32_t n_list;
};

// The k best of `n` keys in `list`, in order, to `out`: a thread's key comes where as many are larger. All keys differ.
__device__ __forceinline__ void rank_list(const unsigned long long *list, uint32_t n, uint32_t k, unsigned long long *out) {
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long key = list[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += list[j] > key ? 1u : 0u;
    if (rank < k) out[rank] = key;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 2) k_token_logprobs(const LogprobParams p) {
  ptx::pdl_wait();
  constexpr int E = RowSplit<BF16>::kElements;
  extern __shared__ __align__(16) uint4 body_smem[];  // [groups][kThreads]
  __shared__ SliceSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
  if (p.slices > 1) cluster.barrier_arrive();  // waited for before the first write to another CTA's shared memory
  if (t == 0) sm.n_list = 0;
  const void *grow = row_at<BF16>(p.logits, row, p.stride);
  const RowSplit<BF16> split(grow, p.cols);
  // this CTA: groups [g0, g1) of the row's body; the first also has its head, the last its tail
  const uint32_t per = p.groups * kThreads, g0 = min(split.groups, slice * per), g1 = min(split.groups, g0 + per);
  const uint4 *body = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(grow) + (size_t)split.head * (16 / E));
  uint32_t extra = p.cols;  // the scalar element of this thread, if any
  if (slice == 0 && t < split.head) extra = t;
  if (slice == p.slices - 1 && t >= 32 && t - 32 < p.cols - split.body_end()) extra = split.body_end() + (t - 32);
  const uint32_t groups = g1 > g0 + t ? (g1 - g0 - t + kThreads - 1) / kThreads : 0;  // of this thread
  const uint32_t dst = ptx::smem_u32(body_smem + t);
  for (uint32_t i = 0; i < groups; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * (kThreads * 16u)), "l"(body + g0 + i * kThreads + t) : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  const float x_extra = extra < p.cols ? load1<BF16>(grow, extra) : -INFINITY;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();

  // ---- maximum (NaN apart)
  float top = x_extra;
  auto bf2 = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); };
  const uint32_t low2 = 0xff80ff80u;  // -inf, twice
  __nv_bfloat162 top2 = bf2(low2);
#pragma unroll 4
  for (uint32_t i = 0; i < groups; ++i) {
    const uint4 v = body_smem[i * kThreads + t];
    if (BF16) {
      top2 = __hmax2(top2, __hmax2(__hmax2(bf2(v.x), bf2(v.y)), __hmax2(bf2(v.z), bf2(v.w))));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) top = fmaxf(top, element<BF16>(v, e));
    }
  }
  if (BF16) top = fmaxf(top, fmaxf(__low2float(top2), __high2float(top2)));
  const float mine = top;  // of this thread
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sm.red[0][warp] = top;
  const uint32_t full_warps = min((g1 - g0) / 32, (uint32_t)kWarps);  // every lane of them has a maximum
  if (p.top_k && warp < full_warps) {  // this warp's bound: its ceil(k / full_warps)-th largest lane maximum
    uint32_t left = order_of(mine) | 1u, bound = 0;  // (the last bit off: a lane that is out has 0)
    for (uint32_t n = 0; n < (p.top_k + full_warps - 1) / full_warps; ++n) {
      bound = __reduce_max_sync(0xffffffffu, left);
      const uint32_t holds = __ballot_sync(0xffffffffu, left == bound);
      if (lane == __ffs(holds) - 1) left = 0;
    }
    if (lane == 0) sm.bound[warp] = bound & ~1u;
  }
  __syncthreads();
  top = sm.red[0][lane % kWarps];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));

  // ---- sums
  const float2 scale2 = make_float2(p.scale * kLog2e, p.scale * kLog2e), minus_top = top == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-top, -top);
  Sums2 sums;
  sums.add(x_extra, -INFINITY, scale2, minus_top);
#pragma unroll 2
  for (uint32_t i = 0; i < groups; ++i) {  // a group by itself first: a thread's sum is then of some dozens of terms, not hundreds
    const uint4 v = body_smem[i * kThreads + t];
    Sums2 group;
#pragma unroll
    for (int e = 0; e < E; e += 2) group.add(element<BF16>(v, e), element<BF16>(v, e + 1), scale2, minus_top);
    sums.add(group);
  }
  float sum = sums.sum.x + sums.sum.y, weighted = sums.weighted.x + sums.weighted.y;
  const bool nan_here = isnan(sum);  // this thread has a NaN (or +inf, or there is one in the slice)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    weighted += __shfl_xor_sync(0xffffffffu, weighted, o);
  }
  if (lane == 0) { sm.red[1][warp] = sum; sm.red[2][warp] = weighted; }

  // ---- the slice's best
  if (p.top_k) {
    const float bound = full_warps ? bound_of(__reduce_min_sync(0xffffffffu, lane < full_warps ? sm.bound[lane] : 0xffffffffu)) : -INFINITY;  // else everything
    auto consider = [&](float x, uint32_t i) {
      if (!(x < bound)) {  // a NaN is nobody's maximum, but comes first
        const uint32_t at = atomicAdd(&sm.n_list, 1u);
        if (at < kList) sm.list[at] = key_of(x, i);
      }
    };
    if (extra < p.cols) consider(x_extra, extra);
    uint32_t look = __ballot_sync(0xffffffffu, groups > 0 && (mine >= bound || nan_here));
    while (look) {
      const uint32_t owner = __ffs(look) - 1, n = __shfl_sync(0xffffffffu, groups, owner);
      look &= look - 1;
      for (uint32_t i = lane; i < n; i += 32) {
        const uint32_t at = i * kThreads + warp * 32 + owner;
        const uint4 v = body_smem[at];
#pragma unroll
        for (int e = 0; e < E; ++e) consider(element<BF16>(v, e), split.head + (g0 + at) * E + e);
      }
    }
  }
  __syncthreads();
  sum = sm.red[1][lane % kWarps];
  weighted = sm.red[2][lane % kWarps];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    weighted += __shfl_xor_sync(0xffffffffu, weighted, o);
  }
  const bool bad = isnan(sum) || top == INFINITY;  // a NaN or +inf reaches the sum

  // ---- to the first CTA
  SliceSmem *first = &sm;
  if (p.slices > 1) {
    cluster.barrier_wait();
    first = cluster.map_shared_rank(&sm, 0);
  }
  if (t == 0) first->part[slice] = make_float4(top, sum, weighted, bad ? 1.0f : 0.0f);
  unsigned long long *best = first->best + slice * p.top_k;
  if (p.top_k) {
    const uint32_t n = sm.n_list;
    if (n <= kList) {
      for (uint32_t k = n + t; k < p.top_k; k += kThreads) best[k] = 0;  // a slice with fewer elements than k
      rank_list(sm.list, n, p.top_k, best);
    } else {  // one after another
      unsigned long long last = ~0ull;
      for (uint32_t k = 0; k < p.top_k; ++k) {
        unsigned long long most = 0;
        auto consider = [&](float x, uint32_t i) {
          const unsigned long long key = key_of(x, i);
          if (key < last && key > most) most = key;
        };
        if (extra < p.cols) consider(x_extra, extra);
        for (uint32_t i = 0; i < groups; ++i) {
          const uint4 v = body_smem[i * kThreads + t];
#pragma unroll
          for (int e = 0; e < E; ++e) consider(element<BF16>(v, e), split.head + (g0 + i * kThreads + t) * E + e);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        __syncthreads();
        if (lane == 0) sm.red_key[warp] = most;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) most = max(most, sm.red_key[w]);
        if (t == 0) best[k] = most;
        last = most;
      }
    }
  }
  if (p.slices > 1) {
    cluster.sync();
    if (slice != 0) return;
  } else {
    __syncthreads();
  }
  if (t >= max(32u, p.slices * p.top_k)) return;
  RowResult r = {-INFINITY, 0.0f, 0.0f, false};
  for (uint32_t s = 0; s < p.slices; ++s) {
    r.top = fmaxf(r.top, sm.part[s].x);
    r.bad |= sm.part[s].w != 0.0f;
  }
  for (uint32_t s = 0; s < p.slices; ++s) {
    const float4 q = sm.part[s];
    if (q.x == -INFINITY) continue;  // nothing of this slice can come
    const float down = (q.x - r.top) * (p.scale * kLog2e), f = ex2_approx(down);
    r.sum = fmaf(q.y, f, r.sum);
    r.weighted = fmaf(fmaf(q.y, fmaxf(down, -2000.0f), q.z), f, r.weighted);  // y to the slice's maximum becomes y + down
  }
  if (t == 0) r.write<BF16>(p, row, grow);
  if (p.top_k) {
    if (p.slices == 1) {
      if (t < p.top_k) r.write_top(p, row, t, sm.best[t]);
    } else {  // keys that are not there are 0 and differ from each other in nothing: they are never among the k best, which exist
      const uint32_t n = p.slices * p.top_k;
      const unsigned long long key = t < n ? sm.best[t] : 0ull;
      uint32_t rank = 0;
      if (key)
        for (uint32_t j = 0; j < n; ++j) rank += sm.best[j] > key ? 1u : 0u;
      if (key && rank < p.top_k) r.write_top(p, row, rank, key);
    }
  }
}

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, Op op, T *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  T r = red[0];
  for (int w = 1; w < kWarps; ++w) r = op(r, red[w]);
  return r;
}

// Rows of any length: passes over global memory (they come out of L2 after the first).
template <bool BF16>
__global__ void __launch_bounds__(kThreads) k_token_logprobs_any(const LogprobParams p) {
  ptx::pdl_wait();
  __shared__ float red[kWarps];
  __shared__ unsigned long long red_key[kWarps];
  const uint32_t row = blockIdx.x, t = threadIdx.x;
  const void *grow = row_at<BF16>(p.logits, row, p.stride);
  auto add = [](float a, float b) { return a + b; };
  RowResult r = {-INFINITY, 0.0f, 0.0f, false};
  float top = -INFINITY;
  for (uint32_t i = t; i < p.cols; i += kThreads) {
    const float x = load1<BF16>(grow, i);
    r.bad |= isnan(x) || x == INFINITY;
    top = fmaxf(top, x);
  }
  r.bad = __syncthreads_or(r.bad);
  top = block_reduce(top, [](float a, float b) { return fmaxf(a, b); }, red);
  r.top = top;
  const float2 scale2 = make_float2(p.scale * kLog2e, p.scale * kLog2e), minus_top = top == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-top, -top);
  for (uint32_t i0 = t; i0 < p.cols; i0 += 32 * kThreads) {  // 32 terms by themselves first: thousands in a row would lose the last bits
    Sums2 some;
    for (uint32_t i = i0; i < min(p.cols, i0 + 32 * kThreads); i += 2 * kThreads)
      some.add(load1<BF16>(grow, i), i + kThreads < p.cols ? load1<BF16>(grow, i + kThreads) : -INFINITY, scale2, minus_top);
    r.sum += some.sum.x + some.sum.y;
    r.weighted += some.weighted.x + some.weighted.y;
  }
  r.sum = block_reduce(r.sum, add, red);
  r.weighted = block_reduce(r.weighted, add, red);
  if (t == 0) r.write<BF16>(p, row, grow);
  unsigned long long last = ~0ull;
  for (uint32_t k = 0; k < p.top_k; ++k) {
    unsigned long long best = 0;
    for (uint32_t i = t; i < p.cols; i += kThreads) {
      const unsigned long long key = key_of(load1<BF16>(grow, i), i);
      if (key < last && key > best) best = key;
    }
    last = block_reduce(best, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; }, red_key);
    if (t == 0) r.write_top(p, row, k, last);
  }
}

struct LogprobGradParams {
  const void *logits;
  const int32_t *targets;
  const float *lse, *entropy, *grad_logp, *grad_entropy;
  void *d_logits;
  unsigned long long stride, d_stride;
  uint32_t rows, cols, chunks;
  float scale;
};

// A CTA takes kGradGroups groups a thread of one row, all loaded before the first is worked on. SAME_PHASE: gradient rows lie at the same place between
// 16-byte boundaries as logits rows, so that they are stored in groups too.
constexpr int kGradGroups = 4;
template <bool BF16, bool SAME_PHASE>
__global__ void __launch_bounds__(kThreads) k_token_logprobs_backward(const LogprobGradParams p) {
  ptx::pdl_wait();
  constexpr int E = RowSplit<BF16>::kElements;
  const uint32_t row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const void *grow = row_at<BF16>(p.logits, row, p.stride);
  uint8_t *drow = static_cast<uint8_t *>(p.d_logits) + (size_t)row * p.d_stride * (16 / E);
  const RowSplit<BF16> split(grow, p.cols);
  const uint4 *body = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(grow) + (size_t)split.head * (16 / E));
  const uint32_t g0 = chunk * (kGradGroups * kThreads) + t;
  uint4 v[kGradGroups];
#pragma unroll
  for (int i = 0; i < kGradGroups; ++i)
    if (g0 + i * kThreads < split.groups) v[i] = __ldcs(body + g0 + i * kThreads);
  const int32_t target = __ldg(p.targets + row);
  const bool has = target >= 0 && (uint32_t)target < p.cols;
  const float lse = __ldg(p.lse + row), entropy = __ldg(p.entropy + row);
  const float g = has && p.grad_logp ? __ldg(p.grad_logp + row) : 0.0f, h = p.grad_entropy ? __ldg(p.grad_entropy + row) : 0.0f;
  const float g_all = -p.scale * fmaf(h, entropy, g), h_all = -p.scale * h, g_one = p.scale * g;
  const uint32_t one = has ? (uint32_t)target : 0xffffffffu;
  auto gradient = [&](float x, uint32_t i) {  // -scale p (g + h (log p + entropy)), and scale g at the target; p = 0 has no part (log p = -inf)
    const float y = fmaf(x, p.scale, -lse), prob = ex2_approx(y * kLog2e);
    const float d = prob == 0.0f ? 0.0f : prob * fmaf(h_all, y, g_all);
    return i == one ? d + g_one : d;
  };
  auto put = [&](uint32_t i, float d) {
    if (BF16) reinterpret_cast<uint16_t *>(drow)[i] = to_bf16(d);
    else reinterpret_cast<float *>(drow)[i] = d;
  };
  if (chunk == 0) {
    const uint32_t end = split.body_end();
    if (t < split.head) put(t, gradient(load1<BF16>(grow, t), t));
    if (t >= 32 && t - 32 < p.cols - end) put(end + (t - 32), gradient(load1<BF16>(grow, end + (t - 32)), end + (t - 32)));
  }
#pragma unroll
  for (int i = 0; i < kGradGroups; ++i) {
    const uint32_t group = g0 + i * kThreads, c0 = split.head + group * E;
    if (group >= split.groups) break;
    float d[E];
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = gradient(element<BF16>(v[i], e), c0 + e);
    if (SAME_PHASE) {
      uint4 w;
      if (BF16) {
        uint32_t q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(q[k]) : "f"(d[(2 * k + 1) % E]), "f"(d[(2 * k) % E]));
        w = make_uint4(q[0], q[1], q[2], q[3]);
      } else {
        w = make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3]));
      }
      __stcs(reinterpret_cast<uint4 *>(drow + (size_t)c0 * (16 / E)), w);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) put(c0 + e, d[e]);
    }
  }
}

int finish(int st) {
  note_status(st);
  return st;
}

struct DeviceInfo {
  std::once_flag once;
  bool ok = false;
};

// Shared memory of a whole SM for the longest slices; asked for once per kernel and device.
template <bool BF16>
bool prepare() {
  static DeviceInfo table[64];
  int dev = 0;
  if (check_cuda(cudaGetDevice(&dev)) != DF_OK || dev < 0 || dev >= 64) return false;
  DeviceInfo &d = table[dev];
  std::call_once(d.once, [&]() {
    d.ok = cudaFuncSetAttribute(k_token_logprobs<BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kMost * kThreads * 16)) == cudaSuccess;
  });
  return d.ok;
}

// Slices of a row: as few CTAs as hold it at four to an SM; more while the rows alone do not give every SM two CTAs; beyond eight slices' worth of
// columns the slices grow to an SM each.
template <bool BF16>
int launch_forward(LogprobParams &p, cudaStream_t s) {
  const uint32_t n = p.cols / RowSplit<BF16>::kElements + 1;
  const int n_sm = sm_count();
  if (n_sm == 0 || !prepare<BF16>()) return DF_ERR_CUDA;
  auto groups_of = [&](uint32_t slices) { return (n + slices * kThreads - 1) / (slices * kThreads); };
  uint32_t slices = 1;
  while (slices < kMaxSlices && (groups_of(slices) > kUsual || ((uint64_t)p.rows * slices < 2u * (uint64_t)n_sm && groups_of(slices) > 2))) slices *= 2;
  p.slices = slices;
  p.groups = groups_of(slices);
  int st;
  if (p.groups > kMost || (uint64_t)p.rows * slices > 0x7fffffffull)
    st = check_cuda(launch_kernel(k_token_logprobs_any<BF16>, dim3(p.rows), dim3(kThreads), 0, s, p));
  else
    st = check_cuda(launch_clusters(k_token_logprobs<BF16>, slices, dim3(p.rows * slices), dim3(kThreads), (size_t)p.groups * kThreads * 16, s, p));
  note_launch();
  return st;
}

template <bool BF16>
int launch_backward(LogprobGradParams &p, cudaStream_t s) {
  constexpr uint32_t per = kGradGroups * kThreads * RowSplit<BF16>::kElements;
  p.chunks = (p.cols + per - 1) / per;
  if ((uint64_t)p.rows * p.chunks > 0x7fffffffull) return DF_ERR_UNSUPPORTED;
  const uint64_t elt = BF16 ? 2 : 4;
  const bool same_phase = (((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.d_logits)) | (p.stride * elt ^ p.d_stride * elt)) & 15u) == 0;
  const int st = check_cuda(launch_kernel(same_phase ? k_token_logprobs_backward<BF16, true> : k_token_logprobs_backward<BF16, false>,
                                          dim3(p.rows * p.chunks), dim3(kThreads), 0, s, p));
  note_launch();
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
  LogprobParams p = {logits, targets, logp, entropy, lse, top_logp, top_ids, row_stride, rows, cols, top_k, 1, 0, scale};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return finish(logits_bf16 ? launch_forward<true>(p, s) : launch_forward<false>(p, s));
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
  LogprobGradParams p = {logits, targets, lse, entropy, grad_logp, grad_entropy, d_logits, row_stride, d_row_stride, rows, cols, 0, scale};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return finish(logits_bf16 ? launch_backward<true>(p, s) : launch_backward<false>(p, s));
}

}  // extern "C"
