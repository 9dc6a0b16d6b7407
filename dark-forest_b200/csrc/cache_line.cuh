// cache_line.cuh - what the kernels that attend to the 8-bit paged cache share: how a step's work is dealt out to CTAs, rows of q and results in memory, widened
// codes, partial results.
//
// The whole step is one line of units: 64 tokens (a stage) of one head and row tile of one request, request after request. The grid's CTAs take equal parts
// of it, whatever the requests' lengths. A segment (request, row tile, head) that is cut leaves partial (m, l, out) states in the workspace, and the CTA
// that finishes its last part adds them in their order. Every CTA forms the sums over the requests itself.
#pragma once

#include <float.h>
#include <math.h>

#include "cache_codes.cuh"
#include "sm100_ptx.cuh"

namespace df {

constexpr uint32_t kStageTokens = 64;
constexpr uint32_t kMaxGrid = 640;
constexpr uint32_t kCounterBytes = 4096;  // a counter per CTA, at the workspace's beginning
static_assert(kMaxGrid * 4 <= kCounterBytes, "a counter for each CTA");

struct AttendParams {
  const void *q;
  const float *k_scale, *v_scale;
  const int32_t *table, *lens, *starts;
  void *out;
  float *lse;
  unsigned int *counters;
  float *partial;
  unsigned int *status;
  unsigned long long q_stride;
  uint32_t n_requests, n_tokens, heads, kv_heads, group, D, P, n_pages, width;
  uint32_t q_aligned, out_aligned;  // 16-byte boundaries
  uint32_t whole;  // the line would be too long in units
  float scale_log2;
};

// A kernel's way of working, W: kRows (of a warp, or of the CTA), kDeal (row tiles of one, two or four warps, by the request's rows), kSegmentUnits (what a
// segment costs besides its stages: its rows of q, sums over warps, its results; counted at its beginning), kThreads.
struct Request {
  uint32_t first, rows, q_len, len, tiles, row_tiles;
  uint32_t weight_log2;  // warps that the rows of a tile are dealt to (1, 2, 4; the tokens to the others): units of a stage
};

template <class W>
__device__ __forceinline__ Request request_of(const AttendParams &p, uint32_t r) {
  Request q;
  const long long most = (long long)p.width * p.P;
  q.len = (uint32_t)min((long long)max(__ldg(p.lens + r), 0), most);
  const int b = max(0, min(__ldg(p.starts + r), (int)p.n_tokens)), e = max(b, min(__ldg(p.starts + r + 1), (int)p.n_tokens));
  q.first = (uint32_t)b;
  q.q_len = (uint32_t)(e - b);
  q.rows = q.q_len * p.group;
  q.weight_log2 = !W::kDeal || q.rows <= W::kRows ? 0u : q.rows <= 2 * W::kRows ? 1u : 2u;
  q.row_tiles = (q.rows + (W::kRows << q.weight_log2) - 1) / W::kRows >> q.weight_log2;
  q.tiles = max(1u, (q.len + kStageTokens - 1) / kStageTokens);
  return q;
}

// What a CTA does of one segment.
struct Part {
  Request rq;
  uint32_t r, h, row0;           // K/V head; first row of the row tile
  uint32_t t0, t1;               // stages [t0, t1)
  uint32_t limit;                // tokens that the tile's last row sees
  uint32_t parts, first_cta;     // of the whole segment
};

template <class W>
__device__ __forceinline__ uint32_t span_of(const Request &q) { return (q.tiles << q.weight_log2) + W::kSegmentUnits; }
template <class W>
__device__ __forceinline__ uint32_t tile_at(const Request &q, uint32_t x) {  // stages of a segment in front of its unit x
  return x <= W::kSegmentUnits ? 0u : (x - W::kSegmentUnits) >> q.weight_log2;
}

// The line of units (or, where no segment is cut, of segments) and this CTA's place on it. Its length is below 2^31 (the launcher sees to
// it), so that its divisions are of 32 bits: those of 64 took a part's first microseconds.
struct Line {
  uint32_t at, end, base;  // base: of request r
  uint32_t per_cta, r;
  bool whole;  // counted in segments
};

template <class W>
__device__ __forceinline__ bool next_part(const AttendParams &p, Line &line, Part &part) {
  while (line.at < line.end) {
    Request q = request_of<W>(p, line.r);
    uint32_t span = line.whole ? 1u : span_of<W>(q);
    while (line.at >= line.base + span * q.row_tiles * p.kv_heads) {  // on to the request that holds line.at (it is below the line's end)
      line.base += span * q.row_tiles * p.kv_heads;
      q = request_of<W>(p, ++line.r);
      span = line.whole ? 1u : span_of<W>(q);
    }
    const uint32_t idx = line.whole ? line.at - line.base : (line.at - line.base) / span;
    const uint32_t s0 = line.base + idx * span, s1 = s0 + span;
    const uint32_t row_tile = q.row_tiles == 1 ? 0u : idx / p.kv_heads;
    part.rq = q;
    part.r = line.r;
    part.h = idx - row_tile * p.kv_heads;
    part.row0 = row_tile * (W::kRows << q.weight_log2);
    part.parts = 1;
    part.first_cta = blockIdx.x;
    part.t0 = 0;
    part.t1 = q.tiles;
    const uint32_t from = line.at, stop = min(s1, line.end);
    line.at = stop;
    if (from != s0 || stop != s1) {  // cut
      part.t0 = tile_at<W>(q, from - s0);
      if (stop < s1) part.t1 = tile_at<W>(q, stop - s0);
      // A boundary between CTAs counts down to whole stages; so the first CTA that a segment reaches may have none of it, every other one has
      // some (a CTA has at least four units more than a segment's beginning takes).
      uint32_t c0 = s0 / line.per_cta;
      const uint32_t c1 = (s1 - 1) / line.per_cta;
      if (tile_at<W>(q, (c0 + 1) * line.per_cta - s0) == 0) ++c0;
      part.first_cta = c0;
      part.parts = c1 - c0 + 1;
      if (part.t1 <= part.t0) continue;
    }
    const uint32_t last_row = min(q.rows, part.row0 + (W::kRows << q.weight_log2)) - 1;
    const int see = (int)q.len - (int)q.q_len + (int)(p.group == 1 ? last_row : last_row / p.group) + 1;
    part.limit = (uint32_t)max(0, min(see, (int)q.len));
    part.t1 = max(part.t0, min(part.t1, (part.limit + kStageTokens - 1) / kStageTokens));
    return true;
  }
  return false;
}

// Sums over the requests, in shared memory, and this CTA's place on the line. All threads of the CTA call it; false: nothing is left for this CTA. The barrier in
// it is the only one. Starts that fall somewhere let rows belong to several requests: their units could pass what the line counts to, so nothing is done then.
constexpr uint32_t kFalls = 0xffffffffu;  // in the place of the longest segment's units (below 2^31)
template <class W>
struct LineSmem {
  uint32_t units[W::kThreads], segments[W::kThreads], most[W::kThreads / 32];
};
template <class W>
__device__ __forceinline__ bool begin_line(const AttendParams &p, LineSmem<W> &sm, Line &line) {
  const uint32_t t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const uint32_t per = (p.n_requests + W::kThreads - 1) / W::kThreads, r0 = min(p.n_requests, t * per), r1 = min(p.n_requests, r0 + per);
  uint32_t units = 0, segments = 0, most = 0;
  for (uint32_t r = r0; r < r1; ++r) {
    const Request q = request_of<W>(p, r);
    const uint32_t n = q.row_tiles * p.kv_heads;
    segments += n;
    units += n * span_of<W>(q);
    if (n) most = max(most, span_of<W>(q));
    if (__ldg(p.starts + r + 1) < __ldg(p.starts + r)) most = kFalls;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, units, o), b = __shfl_up_sync(0xffffffffu, segments, o);
    if (lane >= (uint32_t)o) { units += a; segments += b; }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  sm.units[t] = units;
  sm.segments[t] = segments;
  if (lane == 0) sm.most[warp] = most;
  __syncthreads();
  uint32_t all_units = 0, all_segments = 0;
  most = 0;
#pragma unroll
  for (uint32_t w = 0; w < W::kThreads / 32; ++w) {
    all_units += sm.units[32 * w + 31];
    all_segments += sm.segments[32 * w + 31];
    most = max(most, sm.most[w]);
  }
  if (most == kFalls) {
    if (blockIdx.x == 0 && t == 0 && p.status) atomicOr(p.status, DEV_STATUS_BOUNDS);
    return false;
  }
  const uint32_t G = gridDim.x, seg_per = (all_segments + G - 1) / G, unit_per = max(W::kSegmentUnits + 8u, (all_units + G - 1) / G);
  line.whole = p.whole || (unsigned long long)seg_per * most <= unit_per + W::kSegmentUnits;  // cutting costs another end
  line.per_cta = line.whole ? seg_per : unit_per;
  const uint32_t total = line.whole ? all_segments : all_units;
  if ((unsigned long long)line.per_cta * blockIdx.x >= total) return false;  // (the whole CTA)
  line.at = line.per_cta * blockIdx.x;
  line.end = min(total, line.at + line.per_cta);
  // the warp, then the lane, then the request of those lane's that line.at falls to: every warp looks for itself
  {
    const uint32_t *sums = line.whole ? sm.segments : sm.units;
    uint32_t base = 0, w = 0;
    while (line.at >= base + sums[32 * w + 31]) base += sums[32 * w++ + 31];
    const uint32_t mine = base + sums[32 * w + lane];
    const uint32_t owner = __ffs(__ballot_sync(0xffffffffu, line.at < mine)) - 1;
    const uint32_t before = __shfl_sync(0xffffffffu, mine, max(owner, 1u) - 1);
    line.base = owner == 0 ? base : before;
    line.r = (32 * w + owner) * per;  // next_part goes on to the request
  }
  return true;
}

// ---------------------------------------------------------------- widening codes to pairs of halves
// int8: 1024 + (code + 128) is a half with the code in its last bits. e4m3: an instruction.
__device__ __forceinline__ uint32_t half_of_biased(uint32_t biased) {  // two halves 1024 + (code + 128)
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
  const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&biased), bias);
  return *reinterpret_cast<const uint32_t *>(&x);
}
__device__ __forceinline__ void halves_of_e4m3(uint32_t w, uint32_t &low, uint32_t &high) {  // bytes (0, 1) and (2, 3)
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(low), "=r"(high) : "r"(w));
}
// The four codes of a word as two pairs: bytes (0, 1) and (2, 3).
template <int FORMAT>
__device__ __forceinline__ void widen_word(uint32_t w, uint32_t &first, uint32_t &second) {
  if (FORMAT == DF_CACHE_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    first = half_of_biased(__byte_perm(u, 0x64646464u, 0x4140));
    second = half_of_biased(__byte_perm(u, 0x64646464u, 0x4342));
  } else {
    halves_of_e4m3(w, first, second);
  }
}
// Byte i of two words each, for the four i: pair[i] = (a.byte i, b.byte i).
template <int FORMAT>
__device__ __forceinline__ void widen_pairs(uint32_t a, uint32_t b, uint32_t (&pair)[4]) {
  const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);  // a0 b0 a1 b1, a2 b2 a3 b3
  widen_word<FORMAT>(lo, pair[0], pair[1]);
  widen_word<FORMAT>(hi, pair[2], pair[3]);
}

__device__ __forceinline__ uint32_t halves(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// a pair of floats as halves and what they leave
__device__ __forceinline__ void split_halves(float x, float y, uint32_t &first, uint32_t &second) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h), rest = ptx::fma2(f, make_float2(-1.0f, -1.0f), make_float2(x, y));
  first = *reinterpret_cast<const uint32_t *>(&h);
  second = halves(rest.x, rest.y);
}

// Four elements of a row of q, as they lie there.
template <bool BF16>
struct Raw4 {
  uint32_t w[BF16 ? 2 : 4];
  __device__ __forceinline__ void load(const void *q, unsigned long long e, bool aligned) {
    if constexpr (BF16) {
      const uint16_t *p = static_cast<const uint16_t *>(q) + e;
      if (aligned) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = v.x; w[1] = v.y;
      } else {
        w[0] = __ldg(p) | ((uint32_t)__ldg(p + 1) << 16);
        w[1] = __ldg(p + 2) | ((uint32_t)__ldg(p + 3) << 16);
      }
    } else {
      const uint32_t *p = static_cast<const uint32_t *>(q) + e;
      if (aligned) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __ldg(p + i);
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t &x : w) x = 0u;
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (BF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __uint_as_float(w[i]);
  }
};

template <bool BF16>
__device__ __forceinline__ void store_row4(void *out, size_t e, bool aligned, const float (&x)[4]) {
  if (BF16) {
    uint32_t w[2];
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[0]) : "f"(x[1]), "f"(x[0]));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[1]) : "f"(x[3]), "f"(x[2]));
    uint16_t *p = static_cast<uint16_t *>(out) + e;
    if (aligned) {
      *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    }
  } else {
    float *p = static_cast<float *>(out) + e;
    if (aligned) {
      *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = x[i];
    }
  }
}

// Weights of V. Pages have scales of their own, so the largest weight exp(s - m) need not belong to the largest part of the result; half-precision weights
// must reach down from that part, and nothing that a row does not see may move them. So a row keeps, besides its maximum m,
//   d = max (s - m) + log2 v_scale   over the tokens that it sees (units of log 2),
// and its output in units of 2^e, e the whole number next to d: a weight is exp(s - m) * (v_scale 2^-e), at most 2^(1/2), exact in all bits that exp(s - m)
// has where scales are powers of two. The logarithm is bounded, so that 2^e and 2^-e are numbers; a row that has seen nothing has the lowest d.
constexpr float kLeastExcess = -126.0f;
__device__ __forceinline__ float scale_log(float v_scale) { return fminf(fmaxf(__log2f(v_scale), kLeastExcess), 126.0f); }
__device__ __forceinline__ float unit_exponent(float d) { return (d + 12582912.0f) - 12582912.0f; }  // 1.5 * 2^23: rounds to a whole number
// v_scale 2^-e, given 2^-e. Bounded, so that a weight of zero stays one beside any scale; NaN stays NaN.
__device__ __forceinline__ float share_of(float v_scale, float units) {
  float share;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(share) : "f"(v_scale * units), "f"(0x1p126f));
  return share;
}

// Sums (m, l, o[4]) states one after another.
struct Running {
  float m = -FLT_MAX, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  __device__ __forceinline__ void add(float m2, float l2, const float4 &o2) {
    const float top = fmaxf(m, m2), a = ptx::ex2_approx(m - top), b = ptx::ex2_approx(m2 - top);
    m = top;
    l = l * a + l2 * b;
    o[0] = o[0] * a + o2.x * b;
    o[1] = o[1] * a + o2.y * b;
    o[2] = o[2] * a + o2.z * b;
    o[3] = o[3] * a + o2.w * b;
  }
};


// Four dims of a finished row.
template <bool BF16>
__device__ __forceinline__ void finish_row4(const AttendParams &p, size_t row, uint32_t dim, const float4 &x, float m, float l, float weight_bits) {
  const bool none = l == 0.0f;  // a row that sees nothing
  const float inv = 1.0f / l;
  const float y[4] = {none ? 0.0f : x.x * inv, none ? 0.0f : x.y * inv, none ? 0.0f : x.z * inv, none ? 0.0f : x.w * inv};
  if (dim < p.D) store_row4<BF16>(p.out, row * p.D + dim, p.out_aligned, y);
  if (dim == 0 && p.lse) p.lse[row] = l == 0.0f ? -INFINITY : (m - weight_bits + log2f(l)) * kLn2;
}

// The pool as lines of 128 bytes: a slice (page, head) is P * D / 128 of them, 16 tokens D / 8.
inline bool encode_pool_map(CUtensorMap *map, const void *pool, const AttendParams &p) {
  PFN_encodeTiled encode = get_encode_tiled();
  if (!encode) return false;
  const cuuint64_t lines = (cuuint64_t)p.P * p.D / 128;
  const cuuint64_t dims[3] = {128, lines, (cuuint64_t)p.n_pages * p.kv_heads};
  const cuuint64_t strides[2] = {128, lines * 128};
  const cuuint32_t box[3] = {128, p.D / 8, 1}, step[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query rows of many tokens per request, on tcgen05 (cache_attention_many.cu).
int cache_attention_many(AttendParams &p, const void *k_cache, const void *v_cache, bool bf16, uint32_t format, cudaStream_t s);

}  // namespace df
