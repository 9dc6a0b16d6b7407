// linear_ce.cu — softmax cross entropy from hidden states and the output weight, without keeping the logits (sm_100a):
//   z = scale * x w^T [R, V],  lse_r = log sum_v exp z_rv,  loss_r = lse_r - z_r,target
//   G = exp(z - lse) - onehot,  d_x = (grad * scale) G w,  d_w = G^T (grad * scale) x
// Rows whose target is outside 0 .. V - 1 are left out: loss, lse and gradients 0, whatever x holds there.
//
// Forward: one product with an epilogue that keeps of every row and 128 columns the largest logit and the sum of exponentials, and
// the target's logit; a second kernel joins them. bf16 operands enter as they are (products exact, sums fp32). fp32 operands are cut
// into two fp16 parts (product_sm100.cuh), both scaled row by row.
// Backward, per piece of the vocabulary: the logits again with an epilogue that writes G in fp16 (one part for bf16 calls: 11 bits, where a
// bf16 result has 8; two for fp32 calls: 22), then d_w = G^T x' with x' = grad * x, complete for its piece, and d_x += G w in fp32, its
// contraction split where there are few tiles. w and x' are contracted row by row there, so that each has one scale for all of it. grad is not in G, so that a row's G keeps its bits however small its weight is.
#include <math.h>

#include "product_sm100.cuh"

namespace df {
namespace {

using namespace ptx;

// G is stored times 2^15, the most that fp16 holds of 1: one part (bf16 calls) has 11 bits for probabilities down to 2^-29 and steps of 2^-39 below, two have 22 bits down to 2^-28 and
// steps of 2^-50. Columns that are unlikely in every row have nothing else in their row of d_w.
constexpr float kGScale = 32768.0f, kGScaleLog2 = 15.0f;
constexpr uint64_t kPieceBytes = 256ull << 20;  // of G, or of a piece's weight in parts

int finish(int st) {
  note_status(st);
  return st;
}

struct Words {  // at the head of the workspace
  uint32_t largest_w, largest_x;  // bits of the largest finite |w|, and |grad x| over the rows that count
};

__device__ __forceinline__ float load_f(const void *p, bool bf16, size_t i) {
  return bf16 ? __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16) : static_cast<const float *>(p)[i];
}
__device__ __forceinline__ float at_most_0(float x) {  // NaN where x is
  float y;
  asm("min.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// What a product is times for the logit: the call's scale and, for fp32 calls, the scale of the row's parts and, where the weight has one for all of it, the weight's.
__device__ __forceinline__ float logit_factor(float scale, const float *row_factor, const uint32_t *largest_w, uint32_t row, bool in) {
  float inv = 1.0f;
  if (largest_w) part_scale(*largest_w, &inv);
  return (row_factor && in ? scale * row_factor[row] : scale) * inv;
}

// The same for the exponent of 2, above 0 also where operands are so small that it vanishes: -inf, the largest of no columns, times it stays -inf.
__device__ __forceinline__ float exponent_factor(float c) { return fmaxf(c * kLog2e, 1.17549435e-38f); }

// Elements k .. k + 3 of a row that begins at element `at`, 0 behind its end: together where wide (16 bytes fp32, 8 bf16), else one by one.
__device__ __forceinline__ float4 load_four(const void *base, bool bf16, size_t at, uint32_t k, uint32_t width, bool wide) {
  if (wide && k + 4 <= width) {
    if (!bf16) return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at + k);
    const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + at + k);
    return make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u));
  }
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (k < width) v.x = load_f(base, bf16, at + k);
  if (k + 1 < width) v.y = load_f(base, bf16, at + k + 1);
  if (k + 2 < width) v.z = load_f(base, bf16, at + k + 2);
  if (k + 3 < width) v.w = load_f(base, bf16, at + k + 3);
  return v;
}

// Four values of a row at element `at`, of which `left` are in the row: together where wide (16 bytes fp32, 8 bf16), else one by one.
__device__ __forceinline__ void write_four(void *out, size_t at, float4 v, uint32_t left, bool bf16, bool wide) {
  if (wide && left >= 4) {
    if (bf16) {
      uint2 b;
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.x) : "f"(v.y), "f"(v.x));
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.y) : "f"(v.w), "f"(v.z));
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + at) = b;
    } else {
      *reinterpret_cast<float4 *>(static_cast<float *>(out) + at) = v;
    }
    return;
  }
  const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (uint32_t x = 0; x < 4; ++x) {
    if (x >= left) break;
    if (bf16) {
      uint32_t b;
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(0.0f), "f"(w[x]));
      static_cast<uint16_t *>(out)[at + x] = (uint16_t)b;
    } else {
      static_cast<float *>(out)[at + x] = w[x];
    }
  }
}

// ---------------------------------------------------------------- epilogues
struct LseEpi {
  struct Params {
    const int32_t *targets;
    const float *row_factor, *col_factor;  // fp32 calls: 1 / scale of a row's parts, of x and of the weight
    float2 *parts;               // [slots][rows_pad]: largest logit (as the product has it), sum of e^(z - largest)
    float *picked;               // [rows]: the target's logit (as the product has it)
    float scale;
    uint32_t rows, cols, rows_pad, col_base, slot_base, slot_cols;  // col_base: first column of the piece; cols: of the piece; slot_cols: of a warp
  };
  const Params &p;
  float c, m, s;
  uint32_t row, col0;
  int target;
  bool in;
  __device__ __forceinline__ LseEpi(const Params &q, uint8_t *, int) : p(q) {}
  __device__ __forceinline__ void begin(const ProductTile &, uint32_t r, uint32_t c0) {
    row = r;
    col0 = c0;
    in = r < p.rows;
    target = in ? p.targets[r] - (int)p.col_base : -1;
    c = exponent_factor(logit_factor(p.scale, p.row_factor, nullptr, r, in));
    m = -INFINITY;
    s = 0.0f;
  }
  // Differences are formed before they are scaled: the target's logit and the largest may agree in most of their bits.
  __device__ __forceinline__ void block(int cg, float (&v)[32]) {
    const uint32_t first = col0 + cg * 32;
    if (first >= p.cols) return;
    if (p.col_factor) {
#pragma unroll
      for (int x = 0; x < 32; x += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4 *>(p.col_factor + first + x));  // the same for all lanes
        v[x] *= q.x;
        v[x + 1] *= q.y;
        v[x + 2] *= q.z;
        v[x + 3] *= q.w;
      }
    }
    const uint32_t at = (uint32_t)target - first;
    if (__any_sync(0xffffffffu, at < 32u)) {
      float z = 0.0f;
#pragma unroll
      for (int x = 0; x < 32; ++x) z = at == (uint32_t)x ? v[x] : z;
      if (in && at < 32u && (uint32_t)target < p.cols) p.picked[row] = z;
    }
    if (first + 32 > p.cols) {
#pragma unroll
      for (int x = 0; x < 32; ++x) v[x] = first + x < p.cols ? v[x] : -INFINITY;
    }
    float top = v[0];
#pragma unroll
    for (int x = 1; x < 32; ++x) top = fmaxf(top, v[x]);
    top = fmaxf(m, top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float2 add = make_float2(0.0f, 0.0f);
    const float2 minus = make_float2(-ref, -ref), cc = make_float2(c, c);
#pragma unroll
    for (int x = 0; x < 32; x += 2) {
      const float2 d = mul2(add2(make_float2(v[x], v[x + 1]), minus), cc);
      add = add2(add, make_float2(ex2_approx(d.x), ex2_approx(d.y)));
    }
    s = s * ex2_approx((m - ref) * c) + (add.x + add.y);
    m = top;
  }
  __device__ __forceinline__ void end() {
    if (in && col0 < p.cols) p.parts[(size_t)(p.slot_base + col0 / p.slot_cols) * p.rows_pad + row] = make_float2(m, s);
  }
};

template <int PARTS>
struct GradEpi {
  struct Params {
    const int32_t *targets;
    const float *lse, *row_factor;
    const float *picked;  // logarithm of the targets' probabilities
    const uint32_t *largest_w;
    __half *g, *g_lo;  // [rows][pitch]
    float scale;
    uint32_t rows, cols, pitch, col_base, all_cols;
  };
  const Params &p;
  uint4 *slab;
  int lane;
  float c, off;
  uint32_t row, col0;
  int target;
  bool counts;
  __device__ __forceinline__ GradEpi(const Params &q, uint8_t *sl, int l) : p(q), slab(reinterpret_cast<uint4 *>(sl)), lane(l) {}
  __device__ __forceinline__ void begin(const ProductTile &, uint32_t r, uint32_t c0) {
    row = r;
    col0 = c0;
    const bool in = r < p.rows;
    const int t = in ? p.targets[r] : -1;
    counts = (uint32_t)t < p.all_cols;
    target = counts ? t - (int)p.col_base : -1;
    c = logit_factor(p.scale, p.row_factor, p.row_factor ? p.largest_w : nullptr, r, in);
    off = counts ? p.lse[r] : 0.0f;
  }
  // 64 bytes of a row a lane: turned over in halves of the slab, then 8 rows of 64 bytes at a time
  __device__ __forceinline__ void store(__half *dst, uint32_t first, const uint32_t (&h)[16], int half) {
    uint4 *sl = slab + half * 128;
#pragma unroll
    for (int x = 0; x < 4; ++x) sl[lane * 4 + (x ^ ((lane >> 1) & 3))] = make_uint4(h[4 * x], h[4 * x + 1], h[4 * x + 2], h[4 * x + 3]);
    __syncwarp();
    const uint32_t row0 = row - lane;
    const int lrow = lane >> 2, chunk = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = 8 * i + lrow;
      const uint4 q = sl[rr * 4 + (chunk ^ ((rr >> 1) & 3))];
      if (row0 + rr < p.rows) *reinterpret_cast<uint4 *>(dst + (size_t)(row0 + rr) * p.pitch + first + 8 * chunk) = q;
    }
  }
  __device__ __forceinline__ void block(int cg, float (&v)[32]) {
    const uint32_t first = col0 + cg * 32;
    if (first >= p.cols) return;  // the pitch is a multiple of 32, so a block that begins inside may be written whole
    const uint32_t at = (uint32_t)target - first;
    // the logarithm of the probability first: where it is near 0 it has all its bits, and p - 1 at the target is e^log p - 1
    const bool here = __any_sync(0xffffffffu, at < 32u);
    float one = 0.0f;
#pragma unroll
    for (int x = 0; x < 32; ++x) v[x] = at_most_0(fmaf(v[x], c, -off));  // a probability is at most 1, also under an lse that is rounded; a NaN stays
    if (here) {
      // the tensor cores cut sums off, which a sum of terms of one sign feels most, and p - 1 of a target of high probability: 40 rows of 1000 in bf16 whose targets
      // have a logit of 16 and 1 - p of 5e-5 had p - 1 off by a third of itself (the median), with it by 2e-4
      one = expm1f(at < 32u ? at_most_0(p.picked[row]) : 0.0f) * kGScale;
    }
#pragma unroll
    for (int x = 0; x < 32; ++x) v[x] = ex2_approx(fmaf(v[x], kLog2e, kGScaleLog2));
    if (here) {
#pragma unroll
      for (int x = 0; x < 32; ++x) v[x] = at == (uint32_t)x ? one : v[x];
    }
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      if constexpr (PARTS == 2) {
        split_half2<kProdLowUp>(v[2 * x], v[2 * x + 1], hi[x], lo[x]);
        lo[x] = counts ? lo[x] : 0u;
      } else {
        hi[x] = pack_half2(v[2 * x], v[2 * x + 1]);
      }
      hi[x] = counts ? hi[x] : 0u;  // whatever such a row holds
    }
    __syncwarp();
    store(p.g, first, hi, 0);
    if constexpr (PARTS == 2) store(p.g_lo, first, lo, 1);
  }
  __device__ __forceinline__ void end() {}
};

// Sums into fp32 planes, one per slice of the contraction (d_x), or results of a whole contraction in the caller's type (d_w).
struct OutEpi {
  struct Params {
    float *planes;              // d_x: [splits][rows][plane_pitch]
    uint64_t plane_rows;
    uint32_t plane_pitch;
    int add;                    // the planes hold the pieces before this one
    void *out;                  // d_w (planes null): row r of the product is row row_base + r of out
    uint64_t out_stride;
    uint32_t out_bf16, vec;     // vec: rows can be written 16 bytes (fp32) or 8 (bf16) at a time
    const uint32_t *largest_x;  // d_w: its factor is scale / (2^15 s_x)
    float scale;
    uint32_t rows, cols;
  };
  const Params &p;
  float4 *slab;
  int lane;
  float f, inv;  // inv, a power of two, by itself: where x is near the smallest numbers their product leaves fp32
  float *plane;
  uint32_t row0, col0;
  __device__ __forceinline__ OutEpi(const Params &q, uint8_t *sl, int l) : p(q), slab(reinterpret_cast<float4 *>(sl)), lane(l) {}
  __device__ __forceinline__ void begin(const ProductTile &t, uint32_t r, uint32_t c0) {
    row0 = r - lane;
    col0 = c0;
    if (p.planes) {
      plane = p.planes + (size_t)t.split * p.plane_rows * p.plane_pitch;
    } else {
      part_scale(*p.largest_x, &inv);
      f = p.scale / kGScale;
    }
  }
  __device__ __forceinline__ void block(int cg, float (&v)[32]) {
    const uint32_t first = col0 + cg * 32;
    if (first >= p.cols) return;
    float4 q[8];
    turn_over(slab, lane, v, q);
    const uint32_t col = first + 4 * (lane & 7);
    if (col >= p.cols) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t r = row0 + 4 * i + (lane >> 3);
      if (r >= p.rows) continue;
      if (p.planes) {
        float4 *at = reinterpret_cast<float4 *>(plane + (size_t)r * p.plane_pitch + col);
        if (p.add)  // at L2, nobody else adds to it in this launch; read, added and written here it is 40 us more for 8192 rows of 768
          asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(q[i].x), "f"(q[i].y), "f"(q[i].z), "f"(q[i].w) : "memory");
        else
          *at = q[i];
        continue;
      }
      write_four(p.out, (size_t)r * p.out_stride + col, make_float4(q[i].x * f * inv, q[i].y * f * inv, q[i].z * f * inv, q[i].w * f * inv), p.cols - col, p.out_bf16, p.vec);
    }
  }
  __device__ __forceinline__ void end() {}
};

// ---------------------------------------------------------------- around the products
// The largest finite magnitude of w (first `w_blocks` blocks) and of grad * x over the rows that count (the others), a warp a row.
struct RangeParams {
  const void *w, *x;
  const float *grad;
  const int32_t *targets;
  Words *words;
  uint64_t w_stride, x_stride;
  uint32_t vocab, rows, width, w_blocks, bf16;
};
__global__ void __launch_bounds__(256) k_ranges(const RangeParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool is_w = blockIdx.x < p.w_blocks;
  const uint32_t n = is_w ? p.vocab : p.rows, step = (is_w ? p.w_blocks : gridDim.x - p.w_blocks) * 8;
  const void *src = is_w ? p.w : p.x;
  const uint64_t stride = is_w ? p.w_stride : p.x_stride;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(src) | (stride * (p.bf16 ? 2 : 4));
  uint32_t top = 0;
  for (uint32_t r = (is_w ? blockIdx.x : blockIdx.x - p.w_blocks) * 8 + warp; r < n; r += step) {
    float g = 1.0f;
    if (!is_w) {
      if ((uint32_t)p.targets[r] >= p.vocab) continue;
      g = p.grad ? p.grad[r] : 1.0f;
    }
    const size_t at = (size_t)r * stride;
    uint32_t k = 0;
    if ((bits & 15u) == 0) {
      const uint32_t per = p.bf16 ? 8 : 4, n16 = p.width / per;
      const uint4 *row = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(src) + at * (p.bf16 ? 2 : 4));
#pragma unroll 4
      for (uint32_t i = lane; i < n16; i += 32) {
        const uint4 q = row[i];
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (p.bf16) {
            top = max(top, finite_bits(__uint_as_float(u[x] << 16) * g));
            top = max(top, finite_bits(__uint_as_float(u[x] & 0xffff0000u) * g));
          } else {
            top = max(top, finite_bits(__uint_as_float(u[x]) * g));
          }
        }
      }
      k = n16 * per;
    }
    for (k += lane; k < p.width; k += 32) top = max(top, finite_bits(load_f(src, p.bf16, at + k) * g));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  __shared__ uint32_t tops[8];
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) top = max(top, tops[i]);
    atomicMax(is_w ? &p.words->largest_w : &p.words->largest_x, top);  // a maximum does not depend on the order
  }
}

// Rows cut into parts (or, for bf16 calls, copied): a warp a row. scale_from: the word that the whole tensor's scale follows from; null: every
// row its own, its inverse written to row_factor. grad: rows times grad, rows that do not count as zeros. hi null: only `picked` is wanted.
struct PackParams {
  const void *src;
  const uint32_t *scale_from;
  float *row_factor;
  const float *grad;
  const int32_t *targets;  // null: every row counts
  const void *other;         // with the rows of `other` that `picks` names, `picked` becomes scale * product - lse, in double and rounded once
  const float *lse;
  const int32_t *picks;
  float *picked;
  uint64_t other_stride;
  float scale;
  uint16_t *hi, *lo;       // lo null: one part; raw: bf16 as they are (operands that cannot be copied in place)
  uint64_t stride;
  uint32_t rows, width, pitch, vocab, bf16, raw;
};
__global__ void __launch_bounds__(256) k_pack(const PackParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= p.rows) return;
  const bool counts = !p.targets || (uint32_t)p.targets[r] < p.vocab;
  const float g = p.grad && counts ? p.grad[r] : 1.0f;
  const size_t at = (size_t)r * p.stride, to = (size_t)r * p.pitch;
  const bool wide = ((reinterpret_cast<uintptr_t>(p.src) | (p.stride * (p.bf16 ? 2 : 4))) & 15u) == 0;
  if (p.picked) {
    const uint32_t t = (uint32_t)p.picks[r];
    if (t < p.vocab) {
      const bool wide_w = ((reinterpret_cast<uintptr_t>(p.other) | (p.other_stride * (p.bf16 ? 2 : 4))) & 15u) == 0;
      double sum = 0.0;
#pragma unroll 4
      for (uint32_t k = lane * 4; k < p.width; k += 128) {
        const float4 x = load_four(p.src, p.bf16, at, k, p.width, wide), w = load_four(p.other, p.bf16, (size_t)t * p.other_stride, k, p.width, wide_w);
        sum = fma((double)x.x, (double)w.x, fma((double)x.y, (double)w.y, fma((double)x.z, (double)w.z, fma((double)x.w, (double)w.w, sum))));
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == 0) p.picked[r] = (float)((double)p.scale * sum - (double)p.lse[r]);
    }
  }
  if (!p.hi) return;
  // four elements at a time, zeros behind the end (the pitch is a multiple of 64)
  auto four = [&](uint32_t k) {
    if (!counts) return make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v = load_four(p.src, p.bf16, at, k, p.width, wide);
    if (p.grad) v = make_float4(v.x * g, v.y * g, v.z * g, v.w * g);
    return v;
  };
  float s = 1.0f, inv;
  if (!p.raw) {
    uint32_t top = 0;
    if (p.scale_from) {
      top = *p.scale_from;
    } else {
#pragma unroll 4
      for (uint32_t k = lane * 4; k < p.width; k += 128) {
        const float4 v = four(k);
        top = max(max(top, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
      }
      top = __reduce_max_sync(0xffffffffu, top);
    }
    s = part_scale(top, &inv);
    if (p.row_factor && lane == 0) p.row_factor[r] = inv;
  }
#pragma unroll 4
  for (uint32_t k = lane * 4; k < p.width; k += 128) {
    const float4 v = four(k);
    uint2 hi, lo;
    if (p.raw) {
      hi = make_uint2((__float_as_uint(v.x) >> 16) | (__float_as_uint(v.y) & 0xffff0000u), (__float_as_uint(v.z) >> 16) | (__float_as_uint(v.w) & 0xffff0000u));
    } else {
      split_half2<kProdLowUp>(v.x * s, v.y * s, hi.x, lo.x);
      split_half2<kProdLowUp>(v.z * s, v.w * s, hi.y, lo.y);
    }
    *reinterpret_cast<uint2 *>(p.hi + to + k) = hi;
    if (p.lo) *reinterpret_cast<uint2 *>(p.lo + to + k) = lo;
  }
}

// loss and lse of `group` rows a block, 32 / group lanes of each of 32 warps and row: they share the slots, then a warp a row joins what the warps have. It also takes a row's target again, in sums that are rounded: the tensor
// cores cut the sum of a whole row off at each 16 of it, which a target's logit, a sum of terms of one sign where the model has learned something, feels most (4096
// rows of 768 in bf16: the loss 1.0e-6 off 64 bits without; 75 rows over 364 columns of 256 in fp32, the gradient from such an lse 2.8e-6). With d what the logit lacks, sum e^z grows by p (e^d - 1) of itself.
struct JoinParams {
  const float2 *parts;
  const float *picked, *row_factor;
  const int32_t *targets;
  const uint16_t *x, *w;    // bf16 calls
  const float *x32, *w32;   // fp32 calls on the tensor cores
  uint64_t x_stride, w_stride;
  float *loss, *lse;
  uint32_t rows, cols, rows_pad, slots, width, group;  // group: a power of two, at most 32
  float scale;
};
__global__ void __launch_bounds__(1024) k_join(const JoinParams p) {
  pdl_wait();
  __shared__ float2 s_part[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY, s = 0.0f, c;
  auto join = [&](float2 q) {
    const float top = fmaxf(m, q.x), ref = top == -INFINITY ? 0.0f : top;
    s = s * ex2_approx((m - ref) * c) + q.y * ex2_approx((q.x - ref) * c);
    m = top;
  };
  auto join_lanes = [&](uint32_t from) {
#pragma unroll 1
    for (uint32_t d = from; d < 32; d <<= 1) join(make_float2(__shfl_xor_sync(0xffffffffu, m, d), __shfl_xor_sync(0xffffffffu, s, d)));
  };
  {
    const uint32_t r = lane & (p.group - 1), first = blockIdx.x * p.group + r, lanes = 32 / p.group;
    c = exponent_factor(logit_factor(p.scale, p.row_factor, nullptr, first, first < p.rows));
    if (first < p.rows) {
#pragma unroll 4
      for (uint32_t i = warp * lanes + lane / p.group; i < p.slots; i += 32 * lanes) join(p.parts[(size_t)i * p.rows_pad + first]);
    }
    join_lanes(p.group);
    if (lane == r) s_part[warp][r] = make_float2(m, s);
  }
  const uint32_t row = blockIdx.x * p.group + warp;
  const bool mine = warp < (int)p.group && row < p.rows;
  float again = 0.0f;
  if (p.x && mine) {
    const uint32_t t = (uint32_t)p.targets[row];
    float sum = 0.0f;
    if (t < p.cols) {
      const uint16_t *x = p.x + (size_t)row * p.x_stride, *w = p.w + (size_t)t * p.w_stride;
      uint32_t done = 0;
      if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15u) == 0) {
        float other = 0.0f;
        done = p.width & ~7u;
#pragma unroll 4
        for (uint32_t k = lane * 8; k < done; k += 256) {
          const uint4 a = *reinterpret_cast<const uint4 *>(x + k), b = *reinterpret_cast<const uint4 *>(w + k);
          const uint32_t aa[4] = {a.x, a.y, a.z, a.w}, bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sum = fmaf(__uint_as_float(aa[i] << 16), __uint_as_float(bb[i] << 16), sum);
            other = fmaf(__uint_as_float(aa[i] & 0xffff0000u), __uint_as_float(bb[i] & 0xffff0000u), other);
          }
        }
        sum += other;
      }
#pragma unroll 4
      for (uint32_t k = done + lane; k < p.width; k += 32) sum = fmaf(load_f(x, true, k), load_f(w, true, k), sum);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    again = sum;
  } else if (p.x32 && mine) {  // in double, and in the unit that the product's row has
    const uint32_t t = (uint32_t)p.targets[row];
    double sum = 0.0;
    if (t < p.cols) {
      const float *x = p.x32 + (size_t)row * p.x_stride, *w = p.w32 + (size_t)t * p.w_stride;
#pragma unroll 8
      for (uint32_t k = lane; k < p.width; k += 32) sum = fma((double)x[k], (double)w[k], sum);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    again = (float)(sum / (double)p.row_factor[row]);
  }
  __syncthreads();
  if (!mine) return;
  const float cn = logit_factor(p.scale, p.row_factor, nullptr, row, true);
  c = exponent_factor(cn);
  m = s_part[lane][warp].x;
  s = s_part[lane][warp].y;
  join_lanes(1);
  if (lane != 0) return;
  if ((uint32_t)p.targets[row] >= p.cols) {
    p.lse[row] = 0.0f;
    p.loss[row] = 0.0f;
    return;
  }
  float target = p.picked[row], l = logf(s);
  if (p.x || p.x32) {
    const float d = (again - target) * cn;
    if (fabsf(d) < 1.0f) {  // above, all of it is rounding of logits of 2^20 and more: what was computed stays together. A NaN stays as well.
      l += log1pf(expf((target - m) * cn - l) * expm1f(d));
      target = again;
    }
  }
  p.lse[row] = fmaf(m, cn, l);
  p.loss[row] = fmaf(m - target, cn, l);
}

}  // namespace
}  // namespace df

#include "linear_ce_few.cuh"

namespace df {
namespace {

// d_x = factor * sum of the planes, in the caller's type; rows that do not count get zeros. A CTA has 32 groups of four elements, and eight warps share the planes,
// added in the order of the warps.
struct SumParams {
  const float *planes, *grad;
  const int32_t *targets;
  const uint32_t *largest_w;
  void *out;
  uint64_t out_stride, plane_size;
  uint32_t rows, width, pitch, splits, vocab, out_bf16, vec;
  float scale;
};
__global__ void __launch_bounds__(256) k_sum_planes(const SumParams p) {
  pdl_wait();
  __shared__ float4 s_sum[8][32];
  const uint32_t per_row = (p.width + 3) / 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t i = (uint64_t)blockIdx.x * 32 + lane;
  const bool in = i < (uint64_t)per_row * p.rows;
  const uint32_t r = (uint32_t)(i / per_row), col = (uint32_t)(i % per_row) * 4;
  const bool counts = in && (uint32_t)p.targets[r] < p.vocab;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (counts) {
    const float *at = p.planes + (size_t)r * p.pitch + col;
#pragma unroll 4
    for (uint32_t k = warp; k < p.splits; k += 8) {
      const float4 a = *reinterpret_cast<const float4 *>(at + k * p.plane_size);
      v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
    }
  }
  s_sum[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || !in) return;
  for (int k = 1; k < 8; ++k) {
    const float4 a = s_sum[k][lane];
    v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
  }
  if (counts) {
    float f = p.scale, inv = 1.0f;  // one after the other: their product may leave fp32
    if (p.largest_w) {
      part_scale(*p.largest_w, &inv);
      f /= kGScale;
    }
    const float g = p.grad[r];
    v.x = v.x * f * g * inv; v.y = v.y * f * g * inv; v.z = v.z * f * g * inv; v.w = v.w * f * g * inv;
  }
  write_four(p.out, (size_t)r * p.out_stride + col, v, p.width - col, p.out_bf16, p.vec);
}

// ---------------------------------------------------------------- sizes
uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// What a call uses of its workspace, in bytes from its start (all of it multiples of 256).
struct Layout {
  uint64_t row_factor, col_factor, x_parts, x_grad, w_parts, w_raw, parts, picked, g, planes, total;
  uint32_t pitch;           // of rows of `width` 16-bit elements or floats
  uint32_t piece, n_pieces; // columns of the vocabulary at a time
  uint32_t slots, rows_pad;
  int splits;               // of d_x's contraction
  bool few;                 // linear_ce_few.cuh
};

constexpr int kMaxSplits = 16;
constexpr uint64_t kPairs = 74;  // of SMs

bool in_place(const void *p, uint64_t stride) { return ((reinterpret_cast<uintptr_t>(p) | (stride * 2)) & 15u) == 0; }

// Time of a backward piece of t tiles of 256 columns in units of 64 of a contraction on every pair of SMs (about 512 cycles and part), with `splits` slices of d_x:
// waves of tiles times their blocks, for the three products, and what a piece costs besides (four launches, w cut into parts).
struct Tiles {
  uint64_t m, k;              // tiles of 256 rows and of 256 of the width
  uint64_t rows64, width64;   // blocks of 64
  double besides;
  double piece(uint64_t t, uint64_t splits) const {
    auto waves = [](uint64_t n) { return (n + kPairs - 1) / kPairs; };
    return (double)(waves(m * t) * (width64 + 3) + waves(t * k) * (rows64 + 3) + waves(m * k * splits) * ((4 * t + splits - 1) / splits + 3)) + besides;
  }
};

constexpr uint32_t kFewBlocks = 592;

// Whether the weight is better read as it is (linear_ce_few.cuh) than through the tensor cores. In us, 50257 columns of 768 in fp32, weights out of cache: the loss of 1 row 44 against
// 151, 8 rows 60 and 126, 16 rows 108 and 133, 24 rows 189 (on the same weight again) and 133; 130000 columns of 2000: 16 rows 560 and 876. The gradient of 1 row 112 and 283, 8 rows 155
// and 258. bf16 needs no parts: the loss of 8 rows 58 and 27; the gradient of 8 rows of 50257 x 768 234 and 168 (the same weight again), but 34 and 49 with 3000 columns of 512, where launches
// count (3 against 8), and 56 and 63 with 5000 of 1024.
bool few_rows(uint32_t rows, uint32_t vocab, uint32_t width, bool bf16, bool backward) {
  if (kFewMost * up(width, 128) * 4 > kFewSmem) return false;
  if (!backward) return !bf16 && rows <= kFewMost;
  return rows <= kFewGradMost && (uint64_t)rows * vocab <= (64u << 20) && (!bf16 || (uint64_t)vocab * width <= (8u << 20));
}

Layout layout(uint32_t rows, uint32_t vocab, uint32_t width, bool bf16, bool backward) {
  Layout l = {};
  const uint64_t parts = bf16 ? 1 : 2;
  l.pitch = (uint32_t)up(width, 64);
  l.rows_pad = (uint32_t)up(rows, 32);
  uint64_t at = 256;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  if (few_rows(rows, vocab, width, bf16, backward)) {
    l.few = true;
    l.slots = (vocab + 31) / 32 < kFewBlocks ? (vocab + 31) / 32 : kFewBlocks;  // CTAs of the logits
    if (backward) {
      l.piece = (vocab + kFewRanges - 1) / kFewRanges;  // rows of the weight of a range
      l.splits = (int)((vocab + l.piece - 1) / l.piece);
      l.g = take((uint64_t)rows * vocab * 4);
      l.planes = take((uint64_t)l.splits * rows * l.pitch * 4);
    } else {
      l.parts = take((uint64_t)l.slots * l.rows_pad * 8);
      l.picked = take((uint64_t)rows * 4);
    }
    l.total = at;
    return l;
  }
  uint64_t per_col = (uint64_t)l.pitch * 2 * parts;
  if (backward && (uint64_t)rows * 2 * parts > per_col) per_col = (uint64_t)rows * 2 * parts;
  const uint64_t all = (vocab + 255) / 256;  // tiles of the vocabulary
  uint64_t most = kPieceBytes / per_col / 256, piece = all;
  if (most < 1) most = 1;
  if (!backward) {
    const uint64_t n = (all + most - 1) / most;
    piece = (all + n - 1) / n;
  }
  l.splits = 1;
  if (backward) {
    const Tiles c = {((uint64_t)rows + 255) / 256, ((uint64_t)width + 255) / 256, ((uint64_t)rows + 63) / 64, ((uint64_t)width + 63) / 64, bf16 ? 24.0 : 12.0};
    if (most > all) most = all;
    double best = 1e300;
    const uint64_t least = most > 3 ? most / 3 : 1, step = (most - least) / 48 + 1;
    for (uint64_t t = least; t <= most; t += step) {
      const uint64_t tail = all % t;
      // as many slices as there are pairs for, and the fewer the better: each is a plane of sums
      uint64_t few = 1;
      for (uint64_t k = 2; k <= (uint64_t)kMaxSplits && k <= 4 * t; ++k)
        if (c.piece(t, k) < 0.97 * c.piece(t, few)) few = k;
      const double cost = (double)(all / t) * c.piece(t, few) + (tail ? c.piece(tail, few) : 0.0);
      if (cost < best) {
        best = cost;
        piece = t;
        l.splits = (int)few;
      }
    }
  }
  l.piece = (uint32_t)piece * 256;
  l.n_pieces = (uint32_t)((all + piece - 1) / piece);
  l.row_factor = take((uint64_t)rows * 4);
  l.x_parts = take((uint64_t)rows * l.pitch * 2 * parts);
  l.w_parts = take((uint64_t)l.piece * l.pitch * 2 * parts);
  if (!backward) {
    l.col_factor = take((uint64_t)l.piece * 4);
    l.slots = (vocab + 63) / 64 + l.n_pieces;
    l.parts = take((uint64_t)l.slots * l.rows_pad * 8);
    l.picked = take((uint64_t)rows * 4);
  } else {
    l.x_grad = take((uint64_t)rows * l.pitch * 2 * parts);
    if (bf16) l.w_raw = take((uint64_t)l.piece * l.pitch * 2);
    l.picked = take((uint64_t)rows * 4);
    l.g = take((uint64_t)rows * l.piece * 2 * parts);
    l.planes = take((uint64_t)l.splits * rows * l.pitch * 4);
  }
  l.total = at;
  return l;
}

bool sizes_ok(uint32_t rows, uint32_t vocab, uint32_t width) {
  return vocab > 0 && width > 0 && vocab < (1u << 30) && width < (1u << 24) && rows < (1u << 30);
}

// How many slices have blocks when n are cut into `wanted` of the same length. Asked again with the answer and no more blocks, it is no more.
int slices(uint32_t n, int wanted) {
  const uint32_t each = (n + (uint32_t)wanted - 1) / (uint32_t)wanted;
  return (int)((n + each - 1) / each);
}

// Time in us of waves of tiles of parts with n blocks of 64 of the contraction each. A pair of CTAs writes its results while no sums are added up; one CTA takes the time
// that its operands' bytes take, and writes results meanwhile.
double tile_time(bool pair, uint64_t tiles, uint64_t n) {
  const double each = pair ? 1.2 * (double)n + 4.0 : n > 2 ? (double)n : 2.5;
  return (double)((tiles + (pair ? kPairs : 2 * kPairs) - 1) / (pair ? kPairs : 2 * kPairs)) * each;
}

// Which tiles (times on the same inputs again; new ones cost more, 4096 x 50257 250). bf16: always pairs (1000 x 5000 rows of 768: 19 us and 21, 4096 x 50257: 204 and 304, the gradient 63
// and 64, 8192 x 50257: 1739 and 2178). Parts: by the
// estimate (777 x 10007 rows of 330, gradient: pairs 157 us, single CTAs 122; 2048 x 50257 of 768: 415 and 487).
bool pairs(int parts, uint32_t M, uint32_t N, uint32_t K, int splits) {
  if (parts == 1) return true;
  const uint32_t n_kb = (K + kProdK - 1) / kProdK, each = (n_kb + splits - 1) / splits;
  auto tiles = [&](uint64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t) * (uint64_t)slices(n_kb, splits); };
  return tile_time(true, tiles(256), each) < tile_time(false, tiles(128), each);
}

template <bool A_MN, bool B_MN, int PARTS, class Epi>
int product(const Operand &a, const Operand &b, uint32_t M, uint32_t N, uint32_t K, int splits, bool bf16, const typename Epi::Params &e, cudaStream_t s) {
  ProductParams p = {};
  p.M = M;
  p.N = N;
  p.n_kb = (int)((K + kProdK - 1) / kProdK);
  p.splits = slices(p.n_kb, splits);
  p.kb_per_split = (p.n_kb + splits - 1) / splits;
  p.fmt = bf16 ? (uint32_t)kFmtBF16 : (uint32_t)kFmtF16;
  if constexpr (PARTS == 2)
    if (!pairs(PARTS, M, N, K, splits)) return launch_product<ProdCfg<false, A_MN, B_MN, PARTS>, Epi>(a, b, p, e, s);
  return launch_product<ProdCfg<true, A_MN, B_MN, PARTS>, Epi>(a, b, p, e, s);
}

struct HeadCall {
  const void *x, *w;
  const int32_t *targets;
  uint64_t x_stride, w_stride;
  uint32_t rows, vocab, width;
  bool bf16;
  float scale;
  uint8_t *ws;
  Layout l;
  cudaStream_t s;

  const uint8_t *row_of_w(uint32_t v) const { return static_cast<const uint8_t *>(w) + (size_t)v * w_stride * (bf16 ? 2 : 4); }
  uint16_t *at16(uint64_t offset) const { return reinterpret_cast<uint16_t *>(ws + offset); }

  // to 0: only the targets' log probabilities are wanted
  int pack(const void *src, uint64_t stride, uint32_t n, uint64_t to, bool raw, const uint32_t *scale_from, float *row_factor, const float *grad,
           const int32_t *which, float *picked = nullptr, const float *lse = nullptr) const {
    PackParams p = {};
    p.other = w;
    p.other_stride = w_stride;
    p.picks = targets;
    p.picked = picked;
    p.lse = lse;
    p.scale = scale;
    p.src = src;
    p.scale_from = scale_from;
    p.row_factor = row_factor;
    p.grad = grad;
    p.targets = which;
    p.hi = to ? at16(to) : nullptr;
    p.lo = bf16 ? nullptr : at16(to) + (size_t)n * l.pitch;
    p.stride = stride;
    p.rows = n;
    p.width = width;
    p.pitch = l.pitch;
    p.vocab = vocab;
    p.bf16 = bf16;
    p.raw = raw;
    const int st = check_cuda(launch_kernel(k_pack, dim3((n + 7) / 8), dim3(256), 0, s, p));
    note_launch();
    return st;
  }
  Operand packed(uint64_t at, uint32_t n, bool is_bf16) const {
    return {at16(at), at16(at) + (size_t)n * l.pitch, is_bf16, n, width, l.pitch};
  }
  int ranges(const float *grad, bool of_x) const {
    RangeParams p = {w, x, grad, targets, reinterpret_cast<Words *>(ws), w_stride, x_stride, vocab, rows, width, 0, bf16};
    const uint32_t n_sm = (uint32_t)sm_count();
    p.w_blocks = (vocab + 7) / 8 < 8 * n_sm ? (vocab + 7) / 8 : 8 * n_sm;
    const uint32_t x_blocks = !of_x ? 0 : ((rows + 7) / 8 < 2 * n_sm ? (rows + 7) / 8 : 2 * n_sm);
    int st = check_cuda(cudaMemsetAsync(ws, 0, sizeof(Words), s));
    if (st != DF_OK) return st;
    st = check_cuda(launch_kernel(k_ranges, dim3(p.w_blocks + x_blocks), dim3(256), 0, s, p));
    note_launch();
    return st;
  }
  // operands of the logits: bf16 in place where a copy can start there, else copied; fp32 in parts (x once, w piece by piece)
  int logits_x(Operand *o, float *picked = nullptr, const float *lse = nullptr) const {
    if (bf16 && in_place(x, x_stride)) {
      *o = {x, x, true, rows, width, x_stride};
      return DF_OK;
    }
    *o = packed(l.x_parts, rows, bf16);
    return pack(x, x_stride, rows, l.x_parts, bf16, nullptr, bf16 ? nullptr : reinterpret_cast<float *>(ws + l.row_factor), nullptr, nullptr, picked, lse);
  }

  int join(float *loss, float *lse, uint32_t slots, bool again) const {  // again: targets' logits in rounded sums
    JoinParams j = {};
    j.parts = reinterpret_cast<const float2 *>(ws + l.parts);
    j.picked = reinterpret_cast<const float *>(ws + l.picked);
    j.row_factor = bf16 || l.few ? nullptr : reinterpret_cast<const float *>(ws + l.row_factor);
    j.targets = targets;
    j.x = again && bf16 ? static_cast<const uint16_t *>(x) : nullptr;
    j.w = static_cast<const uint16_t *>(w);
    j.x32 = again && !bf16 ? static_cast<const float *>(x) : nullptr;
    j.w32 = static_cast<const float *>(w);
    j.x_stride = x_stride;
    j.w_stride = w_stride;
    j.loss = loss;
    j.lse = lse;
    j.rows = rows;
    j.cols = vocab;
    j.rows_pad = l.rows_pad;
    j.slots = slots;
    j.width = width;
    j.scale = scale;
    j.group = 1;  // as many blocks as there are SMs, while there are rows for them
    while (j.group < 32 && (uint64_t)j.group * (uint64_t)sm_count() < rows) j.group *= 2;
    const int st = check_cuda(launch_kernel(k_join, dim3((rows + j.group - 1) / j.group), dim3(1024), 0, s, j));
    note_launch();
    return st;
  }
  int sum_planes(const float *grad, void *d_x, uint64_t dx_stride, int splits, const uint32_t *largest_w) const {
    const uint32_t elt = bf16 ? 2 : 4, wide = bf16 ? 7 : 15;
    SumParams q = {};
    q.planes = reinterpret_cast<const float *>(ws + l.planes);
    q.grad = grad;
    q.targets = targets;
    q.largest_w = largest_w;
    q.out = d_x;
    q.out_stride = dx_stride;
    q.plane_size = (uint64_t)rows * l.pitch;
    q.rows = rows;
    q.width = width;
    q.pitch = l.pitch;
    q.splits = (uint32_t)splits;
    q.vocab = vocab;
    q.out_bf16 = bf16;
    q.vec = ((reinterpret_cast<uintptr_t>(d_x) | (dx_stride * elt)) & wide) == 0;
    q.scale = scale;
    const int st = check_cuda(launch_kernel(k_sum_planes, dim3((unsigned)(((uint64_t)rows * ((width + 3) / 4) + 31) / 32)), dim3(256), 0, s, q));
    note_launch();
    return st;
  }

  FewParams few() const {
    FewParams p = {};
    p.x = x;
    p.w = w;
    p.targets = targets;
    p.x_stride = x_stride;
    p.w_stride = w_stride;
    p.rows = rows;
    p.vocab = vocab;
    p.width = width;
    p.padded = (uint32_t)up(width, 128);
    p.rows_pad = l.rows_pad;
    const uint64_t elt = bf16 ? 2 : 4;
    p.wide = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | (x_stride * elt) | (w_stride * elt)) & (bf16 ? 7u : 15u)) == 0;
    p.scale = scale;
    return p;
  }
  int forward_few(float *loss, float *lse) const {
    FewParams p = few();
    p.parts = reinterpret_cast<float2 *>(ws + l.parts);
    p.picked = reinterpret_cast<float *>(ws + l.picked);
    const int st = bf16 ? launch_few_logits<true, false>(p, l.slots, s) : launch_few_logits<false, false>(p, l.slots, s);
    return st != DF_OK ? st : join(loss, lse, l.slots, false);
  }
  int backward_few(const float *lse, const float *grad, void *d_x, uint64_t dx_stride, void *d_w, uint64_t dw_stride) const {
    FewParams p = few();
    p.lse = lse;
    p.g = reinterpret_cast<float *>(ws + l.g);
    int st = bf16 ? launch_few_logits<true, true>(p, l.slots, s) : launch_few_logits<false, true>(p, l.slots, s);
    if (st != DF_OK) return st;
    FewGradParams q = {};
    q.x = x;
    q.w = w;
    q.targets = targets;
    q.g = p.g;
    q.grad = grad;
    q.d_w = d_w;
    q.planes = d_x ? reinterpret_cast<float *>(ws + l.planes) : nullptr;
    q.x_stride = x_stride;
    q.w_stride = w_stride;
    q.dw_stride = dw_stride;
    q.rows = rows;
    q.vocab = vocab;
    q.width = width;
    q.pitch = l.pitch;
    q.range = l.piece;
    q.wide = p.wide;
    q.dw_wide = ((reinterpret_cast<uintptr_t>(d_w) | (dw_stride * (bf16 ? 2 : 4))) & (bf16 ? 7u : 15u)) == 0;
    q.scale = scale;
    st = bf16 ? launch_few_gradients<true>(q, s) : launch_few_gradients<false>(q, s);
    return st != DF_OK || !d_x ? st : sum_planes(grad, d_x, dx_stride, l.splits, nullptr);
  }

  int forward(float *loss, float *lse) const {
    if (l.few) return forward_few(loss, lse);
    int st = DF_OK;
    Operand a;
    if (st == DF_OK) st = logits_x(&a);
    uint32_t slots = 0;
    const bool as_it_is = bf16 && in_place(w, w_stride);  // then all of it at a time
    const uint32_t piece = as_it_is ? vocab : l.piece;
    for (uint32_t c0 = 0; st == DF_OK && c0 < vocab; c0 += piece) {
      const uint32_t n = vocab - c0 < piece ? vocab - c0 : piece;
      Operand b = {row_of_w(c0), nullptr, true, n, width, w_stride};
      if (!as_it_is) {
        st = pack(row_of_w(c0), w_stride, n, l.w_parts, bf16, nullptr, bf16 ? nullptr : reinterpret_cast<float *>(ws + l.col_factor), nullptr, nullptr);
        b = packed(l.w_parts, n, bf16);
      }
      LseEpi::Params e = {};
      e.targets = targets;
      e.row_factor = bf16 ? nullptr : reinterpret_cast<const float *>(ws + l.row_factor);
      e.col_factor = bf16 ? nullptr : reinterpret_cast<const float *>(ws + l.col_factor);
      e.parts = reinterpret_cast<float2 *>(ws + l.parts);
      e.picked = reinterpret_cast<float *>(ws + l.picked);
      e.scale = scale;
      e.rows = rows;
      e.cols = n;
      e.rows_pad = l.rows_pad;
      e.col_base = c0;
      e.slot_base = slots;
      e.slot_cols = pairs(bf16 ? 1 : 2, rows, n, width, 1) ? 128 : 64;
      slots += (n + e.slot_cols - 1) / e.slot_cols;
      if (st == DF_OK)
        st = bf16 ? product<false, false, 1, LseEpi>(a, b, rows, n, width, 1, true, e, s) : product<false, false, 2, LseEpi>(a, b, rows, n, width, 1, false, e, s);
    }
    if (st != DF_OK) return st;
    return join(loss, lse, slots, true);
  }

  template <int PARTS>
  int backward(const float *lse, const float *grad, void *d_x, uint64_t dx_stride, void *d_w, uint64_t dw_stride) const {
    if (l.few) return backward_few(lse, grad, d_x, dx_stride, d_w, dw_stride);
    const Words *words = reinterpret_cast<const Words *>(ws);
    const uint32_t elt = bf16 ? 2 : 4, wide = bf16 ? 7 : 15;
    int st = ranges(grad, d_w != nullptr);
    Operand a;
    // the targets' log probabilities come with the pass over x that there is: its parts (fp32), grad x, or one of its own
    float *picked = reinterpret_cast<float *>(ws + l.picked), *in_parts = bf16 ? nullptr : picked, *in_grad = bf16 ? picked : nullptr;
    if (st == DF_OK) st = logits_x(&a, in_parts, lse);
    if (st == DF_OK && d_w) st = pack(x, x_stride, rows, l.x_grad, false, &words->largest_x, nullptr, grad, targets, in_grad, lse);
    if (st == DF_OK && !d_w && bf16) st = pack(x, x_stride, rows, 0, false, nullptr, nullptr, nullptr, nullptr, picked, lse);
    int splits = l.splits;
    for (uint32_t c0 = 0; st == DF_OK && c0 < vocab; c0 += l.piece) {
      const uint32_t n = vocab - c0 < l.piece ? vocab - c0 : l.piece;
      // w in fp16 parts, for d_x and for the logits of fp32 calls
      st = pack(row_of_w(c0), w_stride, n, l.w_parts, false, &words->largest_w, nullptr, nullptr, nullptr);
      const Operand wp = packed(l.w_parts, n, false);
      Operand b = wp;
      if (bf16) {
        b = {row_of_w(c0), nullptr, true, n, width, w_stride};
        if (!in_place(w, w_stride)) {
          if (st == DF_OK) st = pack(row_of_w(c0), w_stride, n, l.w_raw, true, nullptr, nullptr, nullptr, nullptr);
          b = packed(l.w_raw, n, true);
        }
      }
      typename GradEpi<PARTS>::Params e = {};
      e.targets = targets;
      e.lse = lse;
      e.row_factor = bf16 ? nullptr : reinterpret_cast<const float *>(ws + l.row_factor);
      e.largest_w = &words->largest_w;
      e.picked = picked;
      e.g = reinterpret_cast<__half *>(ws + l.g);
      e.g_lo = e.g + (size_t)rows * l.piece;
      e.scale = scale;
      e.rows = rows;
      e.cols = n;
      e.pitch = l.piece;
      e.col_base = c0;
      e.all_cols = vocab;
      if (st == DF_OK) st = product<false, false, PARTS, GradEpi<PARTS>>(a, b, rows, n, width, 1, bf16, e, s);
      const Operand g = {e.g, e.g_lo, false, rows, n, l.piece};
      if (st == DF_OK && d_x) {
        if (c0 == 0) splits = slices((n + kProdK - 1) / kProdK, splits);
        OutEpi::Params o = {};
        o.planes = reinterpret_cast<float *>(ws + l.planes);
        o.plane_rows = rows;
        o.plane_pitch = l.pitch;
        o.add = c0 > 0;
        o.rows = rows;
        o.cols = width;
        st = product<false, true, PARTS, OutEpi>(g, wp, rows, width, n, splits, false, o, s);
      }
      if (st == DF_OK && d_w) {
        OutEpi::Params o = {};
        o.out = static_cast<uint8_t *>(d_w) + (size_t)c0 * dw_stride * elt;
        o.out_stride = dw_stride;
        o.out_bf16 = bf16;
        o.vec = ((reinterpret_cast<uintptr_t>(o.out) | (dw_stride * elt)) & wide) == 0;
        o.largest_x = &words->largest_x;
        o.scale = scale;
        o.rows = n;
        o.cols = width;
        st = product<true, true, PARTS, OutEpi>(g, packed(l.x_grad, rows, false), n, width, rows, 1, false, o, s);
      }
    }
    return st != DF_OK || !d_x ? st : sum_planes(grad, d_x, dx_stride, splits, &words->largest_w);
  }
};

// Memory of a call: [rows] of width elements, stride apart; null: none.
struct Span {
  uintptr_t from = 0, to = 0;
  Span(const void *p, uint64_t rows, uint64_t stride, uint64_t width, uint64_t elt) {
    if (!p) return;
    from = reinterpret_cast<uintptr_t>(p);
    to = from + ((rows - 1) * stride + width) * elt;
  }
  Span(const void *p, uint64_t bytes) : Span(p, 1, 0, bytes, 1) {}
  bool meets(const Span &o) const { return from < o.to && o.from < to; }
};
// Whether one of the first `written` shares memory with another.
bool overlap(const Span *spans, int n, int written) {
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < n; ++j)
      if (spans[i].meets(spans[j])) return true;
  return false;
}

int check_call(const void *x, const void *w, const int32_t *targets, uint32_t rows, uint32_t vocab, uint32_t width, uint64_t x_stride, uint64_t w_stride,
               float scale) {
  if (!sizes_ok(rows, vocab, width) || !(scale > 0.0f) || !isfinite(scale)) return DF_ERR_INVALID_ARG;
  if ((rows > 1 && x_stride < width) || (vocab > 1 && w_stride < width) || x_stride >= (1ull << 32) || w_stride >= (1ull << 32)) return DF_ERR_INVALID_ARG;
  if (rows && (!x || !targets)) return DF_ERR_INVALID_ARG;
  return w ? DF_OK : DF_ERR_INVALID_ARG;
}

}  // namespace
}  // namespace df

using namespace df;

extern "C" {

uint64_t df_linear_cross_entropy_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t width, uint32_t bf16, uint32_t backward) {
  if (rows == 0 || !sizes_ok(rows, vocab, width)) return 0;
  const uint64_t forward = layout(rows, vocab, width, bf16 != 0, false).total;
  if (!backward) return forward;
  // enough for both, so that a program asks once: the forward holds a weight that it has to copy, or cuts into parts, in larger pieces where rows are few
  const uint64_t both = layout(rows, vocab, width, bf16 != 0, true).total;
  return both > forward ? both : forward;
}

int df_linear_cross_entropy(const void *x, const void *weight, const int32_t *targets, float *loss, float *lse, void *workspace, uint64_t workspace_bytes,
                            uint32_t rows, uint32_t vocab, uint32_t width, uint64_t x_stride, uint64_t weight_stride, float scale, uint32_t bf16,
                            void *stream) {
  DF_RANGE("df_linear_cross_entropy");
  int st = check_call(x, weight, targets, rows, vocab, width, x_stride, weight_stride, scale);
  if (st != DF_OK) return finish(st);
  if (rows == 0) return DF_OK;
  if (!loss || !lse) return finish(DF_ERR_INVALID_ARG);
  const Layout l = layout(rows, vocab, width, bf16 != 0, false);
  if (!workspace || workspace_bytes < l.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return finish(DF_ERR_WORKSPACE);
  const uint64_t elt = bf16 ? 2 : 4;
  const Span all[] = {Span(loss, 4ull * rows), Span(lse, 4ull * rows), Span(workspace, l.total), Span(x, rows, x_stride, width, elt),
                      Span(weight, vocab, weight_stride, width, elt), Span(targets, 4ull * rows)};
  if (overlap(all, 6, 3)) return finish(DF_ERR_INVALID_ARG);
  const HeadCall call = {x, weight, targets, rows > 1 ? x_stride : up(width, 8), vocab > 1 ? weight_stride : up(width, 8), rows, vocab, width, bf16 != 0, scale,
                         static_cast<uint8_t *>(workspace), l, static_cast<cudaStream_t>(stream)};
  return finish(call.forward(loss, lse));
}

int df_linear_cross_entropy_backward(const void *x, const void *weight, const int32_t *targets, const float *lse, const float *grad_loss, void *d_x,
                                     void *d_weight, void *workspace, uint64_t workspace_bytes, uint32_t rows, uint32_t vocab, uint32_t width,
                                     uint64_t x_stride, uint64_t weight_stride, uint64_t dx_stride, uint64_t dw_stride, float scale, uint32_t bf16,
                                     void *stream) {
  DF_RANGE("df_linear_cross_entropy_backward");
  int st = check_call(x, weight, targets, rows, vocab, width, x_stride, weight_stride, scale);
  if (st != DF_OK) return finish(st);
  if ((d_x && rows > 1 && dx_stride < width) || (d_weight && vocab > 1 && dw_stride < width) || dx_stride >= (1ull << 32) || dw_stride >= (1ull << 32))
    return finish(DF_ERR_INVALID_ARG);
  const uint64_t elt = bf16 ? 2 : 4;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {  // a sum over no rows
    if (Span(d_weight, vocab, dw_stride, width, elt).meets(Span(weight, vocab, weight_stride, width, elt))) return finish(DF_ERR_INVALID_ARG);
    if (d_weight) st = check_cuda(cudaMemset2DAsync(d_weight, (vocab > 1 ? dw_stride : width) * elt, 0, width * elt, vocab, s));
    return finish(st);
  }
  if (!lse || !grad_loss) return finish(DF_ERR_INVALID_ARG);
  if (!d_x && !d_weight) return DF_OK;
  const Layout l = layout(rows, vocab, width, bf16 != 0, true);
  if (!workspace || workspace_bytes < l.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return finish(DF_ERR_WORKSPACE);
  const Span all[] = {Span(d_x, rows, dx_stride, width, elt), Span(d_weight, vocab, dw_stride, width, elt), Span(workspace, l.total), Span(x, rows, x_stride, width, elt),
                      Span(weight, vocab, weight_stride, width, elt), Span(targets, 4ull * rows), Span(lse, 4ull * rows), Span(grad_loss, 4ull * rows)};
  if (overlap(all, 8, 3)) return finish(DF_ERR_INVALID_ARG);
  const HeadCall call = {x, weight, targets, rows > 1 ? x_stride : up(width, 8), vocab > 1 ? weight_stride : up(width, 8), rows, vocab, width, bf16 != 0, scale,
                         static_cast<uint8_t *>(workspace), l, s};
  return finish(bf16 ? call.backward<1>(lse, grad_loss, d_x, dx_stride, d_weight, dw_stride) : call.backward<2>(lse, grad_loss, d_x, dx_stride, d_weight, dw_stride));
}

}  // extern "C"
