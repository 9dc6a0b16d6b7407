// token_logprobs.cu - log probabilities of given tokens with entropy and the best alternatives, and their gradient, for B200 (sm_100a).
//
// Per row of logits x, z = scale x, m = max z, S = sum exp(z - m):
//   lse = m + log S      logp = (z_t - m) - log S      entropy = log S - (sum exp(z - m) (z - m)) / S      top k of x, equal ones by index
//   dx = scale (g (onehot - p) - h p (log p + entropy)),  p = exp(z - lse),  g, h the gradients of logp and entropy
// The entropy is formed from differences to the maximum, so that nothing large cancels; a column with exp(z - m) = 0 adds nothing (its z - m
// may be -inf). All sums in fp32.
//
// Both directions are bound by HBM: the forward reads every logit once, the gradient reads and writes it once. In the forward a CTA, or where there are few
// rows a cluster of them, walks a row once, kChunk 16-byte groups a thread at a time, with a running maximum and sums per thread; the CTAs' parts
// (maximum, sums, best keys) meet in the shared memory of the cluster's first. Holding the row in shared memory instead (four CTAs or two of an SM) took
// 50 to 66 us at 1024 x 50257 bf16, 27 this way (3.8 TB/s): loads of one row then ran beside the sums of one other at best. fp32: 40 us, 5.2 TB/s. What is left in
// bf16: all rows are there at once and in the same phase, and looking for alternatives, when memory idles, takes 3 to 5 us of it; the walk takes 24 (floor 15.7), with 60 % of
// the issue slots in use (some 5 instructions an element) and the exponentials' pipe half busy. The gradient, 512 x 50257: fp32 34 us (floor 31.5), bf16 19 (15.7; 80 % of the issue slots).
// Alternatives without sorting a row: each of the 4 (16) warps names its 8 (2) largest lane maxima; the k-th largest of these 32 is a bound that at
// least k elements reach, and for logits in no particular order few others do. A thread also keeps the maxima of up to kParts parts of
// its elements; only parts that reach the bound are read again (out of L2), and what is found is put in a list and ranked by counting (key: the value's
// order, then the lower index). Where more than the list's length reach the bound (equal logits, masked rows) the larger ones are listed and the
// first of the equal ones added in their order.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <float.h>
#include <math.h>

#include "df_common.cuh"
#include "sm100_ptx.cuh"

namespace cg = cooperative_groups;

namespace df {
namespace {

using ptx::ex2_approx;

constexpr int kMaxSlices = 8, kList = 256, kLook = 256, kParts = 16, kTop = DF_LOGPROBS_MAX_TOP;
constexpr int kChunk = 4;  // groups of a thread that are loaded at once

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
template <int kThreads>
struct SliceSmem {
  static constexpr int kWarps = kThreads / 32;
  float most[kParts][kThreads];                // the threads' elements in up to kParts parts: their maxima
  unsigned long long list[kList];
  unsigned long long best[kMaxSlices * kTop];  // (first CTA) every CTA's best, in order
  float4 part[kMaxSlices];                     // (first CTA) maximum, sum, weighted sum, bad
  float red[3][kWarps];
  unsigned long long red_key[kWarps];
  uint32_t bound[32];
  uint32_t look[kLook];  // parts that reach the bound
  uint32_t taken[kWarps];
  uint32_t n_list, n_look;
};

// The k best of `n` keys in `list`, in order, to `out`: a thread's key comes where as many are larger. All keys differ.
template <int kThreads>
__device__ __forceinline__ void rank_list(const unsigned long long *list, uint32_t n, uint32_t k, unsigned long long *out) {
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long key = list[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += list[j] > key ? 1u : 0u;
    if (rank < k) out[rank] = key;
  }
}

// Sums relative to `from` become sums relative to `to` (which is not below it).
__device__ __forceinline__ void rebase(float from, float to, float scale_log2, float &sum, float &weighted) {
  const float down = fmaxf((from - to) * scale_log2, -2000.0f), f = ex2_approx(down);  // from = -inf: sums are 0
  weighted = fmaf(sum, down, weighted) * f;  // y to the old maximum becomes y + down
  sum *= f;
}

// kThreads: 128 where rows fill the machine (1024 rows, seven to an SM, are all there at once, and the CTA's ends take half of what they take with 256), 512
// for few rows.
template <bool BF16, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 8 : 2) k_token_logprobs(const LogprobParams p) {
  ptx::pdl_wait();
  constexpr int kWarps = kThreads / 32, kNamed = 32 / kWarps;
  constexpr int E = RowSplit<BF16>::kElements;
  __shared__ SliceSmem<kThreads> sm;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
  if (p.slices > 1) cluster.barrier_arrive();  // waited for before the first write to another CTA's shared memory
  if (t == 0) sm.n_list = sm.n_look = 0;
  const void *grow = row_at<BF16>(p.logits, row, p.stride);
  const RowSplit<BF16> split(grow, p.cols);
  // this CTA: groups [g0, g1) of the row's body; the first also has its head, the last its tail
  const uint32_t per = p.groups * kThreads, g0 = min(split.groups, slice * per), g1 = min(split.groups, g0 + per);
  const uint4 *body = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(grow) + (size_t)split.head * (16 / E));
  uint32_t extra = p.cols;  // the scalar element of this thread, if any
  if (slice == 0 && t < split.head) extra = t;
  if (slice == p.slices - 1 && t >= 32 && t - 32 < p.cols - split.body_end()) extra = split.body_end() + (t - 32);
  const float scale_log2 = p.scale * kLog2e;
  const float2 scale2 = make_float2(scale_log2, scale_log2);
  auto pair_of = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); };

  // ---- one walk: maximum (NaN apart) and sums of this thread's elements
  const float x_extra = extra < p.cols ? load1<BF16>(grow, extra) : -INFINITY;
  float mine = -INFINITY, sum = 0.0f, weighted = 0.0f;
  constexpr uint32_t kNone = BF16 ? 0xff80ff80u : 0xff800000u;  // -inf
  uint4 ahead[kChunk];  // the next chunk is on its way while one is worked on
  auto load = [&](uint32_t g) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) ahead[i] = g + i * kThreads < g1 ? __ldg(body + g + i * kThreads) : make_uint4(kNone, kNone, kNone, kNone);
  };
  load(g0 + t);
  const uint32_t chunks = (g1 - g0 + kChunk * kThreads - 1) / (kChunk * kThreads), chunks_per_part = (chunks + kParts - 1) / kParts;
  uint32_t at_part = 0, chunk_of_part = 0;
  float part_most = -INFINITY;
  for (uint32_t g = g0 + t; g < g1; g += kChunk * kThreads) {
    uint4 v[kChunk];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = ahead[i];
    load(g + kChunk * kThreads);
    float top = -INFINITY;
    if (BF16) {
      __nv_bfloat162 top2 = pair_of(kNone);
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
        top2 = __hmax2(top2, __hmax2(__hmax2(pair_of(v[i].x), pair_of(v[i].y)), __hmax2(pair_of(v[i].z), pair_of(v[i].w))));
      top = fmaxf(__low2float(top2), __high2float(top2));
    } else {
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, element<BF16>(v[i], e));
    }
    part_most = fmaxf(part_most, top);
    sm.most[at_part][t] = part_most;
    if (++chunk_of_part == chunks_per_part) {
      ++at_part;
      chunk_of_part = 0;
      part_most = -INFINITY;
    }
    if (top > mine) {
      rebase(mine, top, scale_log2, sum, weighted);
      mine = top;
    }
    const float2 minus_top = mine == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-mine, -mine);
    Sums2 sums;  // a chunk by itself first: a thread's sums are then of some dozens of terms, not hundreds
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
#pragma unroll
      for (int e = 0; e < E; e += 2) sums.add(element<BF16>(v[i], e), element<BF16>(v[i], e + 1), scale2, minus_top);
    sum += sums.sum.x + sums.sum.y;
    weighted += sums.weighted.x + sums.weighted.y;
  }
  const bool any = g0 + t < g1;                     // groups for this thread
  const float body_most = mine;
  const bool nan_here = any && isnan(sum);          // a NaN or +inf among them
  if (extra < p.cols) {
    const float top = fmaxf(mine, x_extra);
    rebase(mine, top, scale_log2, sum, weighted);
    mine = top;
    Sums2 one;
    one.add(x_extra, -INFINITY, scale2, mine == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(-mine, -mine));
    sum += one.sum.x;
    weighted += one.weighted.x;
  }
  // ---- the CTA's
  float top = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sm.red[0][warp] = top;
  const uint32_t full_warps = min((g1 - g0) / 32, (uint32_t)kWarps);  // every lane of them has a maximum
  const uint32_t named = full_warps == 0 ? 0u : full_warps == kWarps ? (uint32_t)kNamed : (p.top_k + full_warps - 1) / full_warps;
  if (p.top_k && warp < full_warps) {  // this warp's largest lane maxima
    uint32_t left = order_of(body_most), bound = 0;  // no value's order is 0: a lane that is out
    for (uint32_t n = 0; n < named; ++n) {
      bound = __reduce_max_sync(0xffffffffu, left);
      const uint32_t holds = __ballot_sync(0xffffffffu, left == bound);
      if (lane == __ffs(holds) - 1) left = 0;
      if (lane == 0 && n < kNamed) sm.bound[n * kWarps + warp] = bound;
    }
    if (lane == 0 && full_warps < kWarps) sm.bound[warp] = bound;
  }
  __syncthreads();
  top = sm.red[0][lane % kWarps];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (mine != top && top != -INFINITY) rebase(mine, top, scale_log2, sum, weighted);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    weighted += __shfl_xor_sync(0xffffffffu, weighted, o);
  }
  if (lane == 0) { sm.red[1][warp] = sum; sm.red[2][warp] = weighted; }

  // ---- the slice's best: which parts of which threads reach the bound
  float bound = -INFINITY;  // fewer than 32 groups: everything
  if (p.top_k) {
    if (full_warps == kWarps) {  // the k-th largest of 32: the smallest that fewer than k are above
      const uint32_t order = sm.bound[lane];
      uint32_t above = 0;
#pragma unroll 8
      for (int j = 0; j < 32; ++j) above += sm.bound[j] > order ? 1u : 0u;
      bound = value_of(__reduce_min_sync(0xffffffffu, above < p.top_k ? order : 0xffffffffu));
    } else if (full_warps) {  // at least k lanes have a maximum that reaches the smallest of these
      bound = value_of(__reduce_min_sync(0xffffffffu, lane < full_warps ? sm.bound[lane] : 0xffffffffu));
    }
    if (any && (body_most >= bound || nan_here)) {
      const uint32_t my_parts = at_part + (chunk_of_part ? 1 : 0);
      for (uint32_t i = 0; i < my_parts; ++i) {
        if (!(sm.most[i][t] >= bound) && !nan_here) continue;
        const uint32_t at = atomicAdd(&sm.n_look, 1u);
        if (at < kLook) sm.look[at] = i << 16 | t;
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
  SliceSmem<kThreads> *first = &sm;
  if (p.slices > 1) {
    cluster.barrier_wait();
    first = cluster.map_shared_rank(&sm, 0);
  }
  if (t == 0) first->part[slice] = make_float4(top, sum, weighted, bad ? 1.0f : 0.0f);
  unsigned long long *best = first->best + slice * p.top_k;
  if (p.top_k) {
    auto note = [&](float x, uint32_t i) {
      const uint32_t at = atomicAdd(&sm.n_list, 1u);
      if (at < kList) sm.list[at] = key_of(x, i);
    };
    const uint32_t n_look = sm.n_look, per_part = chunks_per_part * kChunk;
    if (n_look <= kLook) {
      if (extra < p.cols && !(x_extra < bound)) note(x_extra, extra);  // a NaN is nobody's maximum, but comes first
      for (uint32_t i = t; i < n_look * per_part; i += kThreads) {
        const uint32_t n = i / per_part, what = sm.look[n], g = g0 + (what & 0xffffu) + ((what >> 16) * per_part + (i - n * per_part)) * kThreads;
        if (g >= g1) continue;
        const uint4 v = __ldg(body + g);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!(element<BF16>(v, e) < bound)) note(element<BF16>(v, e), split.head + g * E + e);
      }
    }
    __syncthreads();
    uint32_t n = sm.n_list;
    if (n_look > kLook || n > kList) {
      // Many equal the bound (equal logits, columns masked out): the larger ones, and of the equal ones the first, in their order.
      __syncthreads();
      if (t == 0) sm.n_list = 0;
      __syncthreads();
      if (extra < p.cols && !(x_extra <= bound)) note(x_extra, extra);
      for (uint32_t g = g0 + t; g < g1; g += kThreads) {
        const uint4 v = __ldg(body + g);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!(element<BF16>(v, e) <= bound)) note(element<BF16>(v, e), split.head + g * E + e);
      }
      __syncthreads();
      n = sm.n_list;
      auto take = [&](uint32_t mine, auto &&value_at) {  // this thread's `mine` equal elements stand behind those of the threads before it
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= (uint32_t)o) upto += x;
        }
        if (lane == 31) sm.taken[warp] = upto;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (int w = 0; w < kWarps; ++w) {
          if (w < (int)warp) before += sm.taken[w];
          all += sm.taken[w];
        }
        for (uint32_t i = 0, at = n + before + upto - mine; i < mine && at < p.top_k; ++i, ++at) sm.list[at] = value_at(i);
        __syncthreads();
        n = min(n + all, max(n, p.top_k));
      };
      if (n < p.top_k) {
        const bool in_head = extra < split.head;
        take(in_head && x_extra == bound ? 1u : 0u, [&](uint32_t) { return key_of(x_extra, extra); });
        for (uint32_t gb = g0; gb < g1 && n < p.top_k; gb += kThreads) {
          const uint32_t g = gb + t;
          uint32_t equal = 0;
          if (g < g1) {
            const uint4 v = __ldg(body + g);
#pragma unroll
            for (int e = 0; e < E; ++e) equal |= element<BF16>(v, e) == bound ? 1u << e : 0u;
          }
          take(__popc(equal), [&](uint32_t i) { return key_of(bound, split.head + g * E + __fns(equal, 0, i + 1)); });
        }
        if (n < p.top_k) take(!in_head && extra < p.cols && x_extra == bound ? 1u : 0u, [&](uint32_t) { return key_of(x_extra, extra); });
      }
    }
    if (n <= kList) {
      for (uint32_t k = n + t; k < p.top_k; k += kThreads) best[k] = 0;  // a slice with fewer elements than k
      rank_list<kThreads>(sm.list, n, p.top_k, best);
    } else {  // more than the list holds are larger than the bound: one after another
      unsigned long long last = ~0ull;
      for (uint32_t k = 0; k < p.top_k; ++k) {
        unsigned long long most = 0;
        auto consider = [&](float x, uint32_t i) {
          const unsigned long long key = key_of(x, i);
          if (key < last && key > most) most = key;
        };
        if (extra < p.cols) consider(x_extra, extra);
        for (uint32_t g = g0 + t; g < g1; g += kThreads) {
          const uint4 v = __ldg(body + g);
#pragma unroll
          for (int e = 0; e < E; ++e) consider(element<BF16>(v, e), split.head + g * E + e);
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
  RowResult r = {-INFINITY, 0.0f, 0.0f, false};
  for (uint32_t s = 0; s < p.slices; ++s) {
    r.top = fmaxf(r.top, sm.part[s].x);
    r.bad |= sm.part[s].w != 0.0f;
  }
  for (uint32_t s = 0; s < p.slices; ++s) {
    const float4 q = sm.part[s];
    if (q.x == -INFINITY) continue;  // nothing of this slice can come
    float sum_s = q.y, weighted_s = q.z;
    rebase(q.x, r.top, scale_log2, sum_s, weighted_s);
    r.sum += sum_s;
    r.weighted += weighted_s;
  }
  if (t == 0) r.write<BF16>(p, row, grow);
  if (p.top_k) {
    if (p.slices == 1) {
      if (t < p.top_k) r.write_top(p, row, t, sm.best[t]);
    } else {  // keys that are not there are 0 and differ from each other in nothing: they are never among the k best, which exist
      const uint32_t n = p.slices * p.top_k;
      for (uint32_t i = t; i < n; i += kThreads) {
        const unsigned long long key = sm.best[i];
        uint32_t rank = key ? 0u : n;
        for (uint32_t j = 0; j < n; ++j) rank += sm.best[j] > key ? 1u : 0u;
        if (rank < p.top_k) r.write_top(p, row, rank, key);
      }
    }
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
constexpr int kGradGroups = 4, kGradThreads = 256;
template <bool BF16, bool SAME_PHASE>
__global__ void __launch_bounds__(kGradThreads) k_token_logprobs_backward(const LogprobGradParams p) {
  ptx::pdl_wait();
  constexpr int E = RowSplit<BF16>::kElements;
  const uint32_t row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks, t = threadIdx.x;
  const void *grow = row_at<BF16>(p.logits, row, p.stride);
  uint8_t *drow = static_cast<uint8_t *>(p.d_logits) + (size_t)row * p.d_stride * (16 / E);
  const RowSplit<BF16> split(grow, p.cols);
  const uint4 *body = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(grow) + (size_t)split.head * (16 / E));
  const uint32_t g0 = chunk * (kGradGroups * kGradThreads) + t;
  uint4 v[kGradGroups];
#pragma unroll
  for (int i = 0; i < kGradGroups; ++i)
    if (g0 + i * kGradThreads < split.groups) v[i] = __ldcs(body + g0 + i * kGradThreads);
  const int32_t target = __ldg(p.targets + row);
  // A row that nothing can come of (lse -inf) has no part of anything: p = 0 throughout, as if lse were +inf, and no target.
  const float lse_row = __ldg(p.lse + row), entropy = __ldg(p.entropy + row);
  const float lse = lse_row == -INFINITY ? INFINITY : lse_row;
  const bool has = target >= 0 && (uint32_t)target < p.cols && lse_row != -INFINITY;
  const float g = has && p.grad_logp ? __ldg(p.grad_logp + row) : 0.0f, h = p.grad_entropy ? __ldg(p.grad_entropy + row) : 0.0f;
  const float g_all = -p.scale * fmaf(h, entropy, g), h_all = -p.scale * h, g_one = p.scale * g;
  const uint32_t one = has ? (uint32_t)target : 0xffffffffu;
  auto gradient = [&](float x, uint32_t i) {  // -scale p (g + h (log p + entropy)), and scale g at the target; p = 0 has no part (log p = -inf)
    // log p is at most 0: the rounding of an lse of 10^30 (a row masked with the type's lowest value) must not become an exponent. NaN stays NaN.
    float y = fmaf(x, p.scale, -lse);
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(0.0f));
    const float prob = ex2_approx(y * kLog2e);
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
    const uint32_t group = g0 + i * kGradThreads, c0 = split.head + group * E;
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

// Rows that give every SM three CTAs of 128 threads get one each, and so do rows that give it one where they are short; fewer or longer ones are cut among up to eight of
// 512 while a CTA still has a chunk. Measured, 128 threads to 512, us: 50257 fp32 columns 74 rows 12.8 to 13.5, 148 16.7 to 11.3, 296 24.5 to 15.9, 400 25.9
// to 25.2, 592 29.5 to 29.9, 1024 39.7 to 53.5; bf16 296 13.6 to 11.8, 400 16.7 to 18.9, 1024 27.5 to 38.2. 4000 groups of 16 bytes: 8 rows 6.9 to 6.0, 64 rows 7.2 to
// 6.3, 148 7.3 to 8.0, 300 8.5 to 11.8; 1100 groups: 8 rows 5.4 to 5.0, 300 6.0 to 10.0.
template <bool BF16>
int launch_forward(LogprobParams &p, cudaStream_t s) {
  const uint32_t n = p.cols / RowSplit<BF16>::kElements + 1;
  const int n_sm = sm_count();
  if (n_sm == 0) return DF_ERR_CUDA;
  const bool many = p.rows >= 3u * (uint32_t)n_sm || (p.rows >= (uint32_t)n_sm && n <= 4096) || n <= kChunk * 128;
  const uint32_t threads = many ? 128 : 512;
  p.slices = 1;
  while (!many && p.slices < kMaxSlices && (uint64_t)p.rows * p.slices < 2u * (uint64_t)n_sm && n > p.slices * (kChunk * threads)) p.slices *= 2;
  p.groups = (n + p.slices * threads - 1) / (p.slices * threads);
  const int st = check_cuda(launch_clusters(many ? k_token_logprobs<BF16, 128> : k_token_logprobs<BF16, 512>, p.slices, dim3(p.rows * p.slices),
                                            dim3(threads), 0, s, p));
  note_launch();
  return st;
}

template <bool BF16>
int launch_backward(LogprobGradParams &p, cudaStream_t s) {
  constexpr uint32_t per = kGradGroups * kGradThreads * RowSplit<BF16>::kElements;
  p.chunks = (p.cols + per - 1) / per;
  if ((uint64_t)p.rows * p.chunks > 0x7fffffffull) return DF_ERR_UNSUPPORTED;
  const uint64_t elt = BF16 ? 2 : 4;
  const bool same_phase = (((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.d_logits)) | (p.stride * elt ^ p.d_stride * elt)) & 15u) == 0;
  const int st = check_cuda(launch_kernel(same_phase ? k_token_logprobs_backward<BF16, true> : k_token_logprobs_backward<BF16, false>,
                                          dim3(p.rows * p.chunks), dim3(kGradThreads), 0, s, p));
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
