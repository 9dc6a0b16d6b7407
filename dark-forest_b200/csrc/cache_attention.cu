// cache_attention.cu - attention of ragged queries over an 8-bit paged cache, for B200 (sm_100a).
//
// For query row (token j of request r, head h), with kv = h / (n_heads / n_kv_heads) and last = lens[r] - q_len + j:
//   s_t = scale * k_scale[page(t), kv] * (q . k_code_t),  t = 0 .. last        m = max s, l = sum exp(s_t - m)
//   out = sum exp(s_t - m) / l * v_scale[page(t), kv] * v_code_t               lse = m + log l
// One pass over the cache with a running maximum and sum per row; nothing but codes leaves HBM.
//
// What bounds it. With few query rows, HBM: a token of a head costs 2 d bytes and (rows) * 4 d operations. At 8 bits an SM gets 23 codes a cycle,
// more than its fp32 lanes could widen and multiply one by one, so both products run on the tensor cores, on codes widened to half
// precision in registers (every code is a half exactly). m16n8k16 instructions take it: their operand layouts leave the order of the contracted
// index free, so that a lane reads whole 16-byte pieces of rows and no element is moved between lanes:
//   scores   A = 16 rows of q, B = 8 tokens: lane (g, c) = (lane / 4, lane % 4) holds the dims c * DP/4 ... of token g; k-step kt is its word kt.
//   output   A = weights, in the accumulators' own layout, B = 16 tokens x 8 dims: lane (g, c) holds the dims g * DP/8 ... of its four tokens;
//            n-tile i is its byte i. The accumulators of lane (g, c) are then row g's dims c * DP/4 ..., like its part of q.
// Precision. An fp32 query row, times a power of two that brings its largest element to 1 .. 2, enters as two halves (22 bits), and so do the
// weights exp(s - m) * 2^15: the 16 rows of an instruction are then 8 rows and their second parts, and the two accumulators are added. A bf16 row
// fits one half, its weights are rounded to 11 bits (the result has 8): 16 rows. The products of 16 tokens, which share one v_scale, are
// added to the row's fp32 sums.
//
// Work. A CTA is one warp that loads (tensor-map copies of 16 tokens, 128-byte swizzle: the reads above are then free of bank conflicts at
// head sizes 64 and 128) and four that compute, over a ring of stages of 64 tokens. A request with no more rows (query tokens times heads per K/V head)
// than a warp takes is computed with its tokens dealt to the four warps; one with more has its rows dealt to them, and every warp goes over
// all tokens. The whole step is one line of units (64 tokens of one head and row tile; four units where rows are dealt, which takes four times as
// long); the grid's CTAs take equal parts of it, whatever the requests' lengths. A segment (request, row tile, head) that is cut leaves partial (m, l, out)
// states in the workspace, and the CTA that finishes its last part adds them in their order. Every CTA forms the sums over the requests itself.
#include <float.h>
#include <math.h>

#include <mutex>
#include <type_traits>

#include "cache_codes.cuh"
#include "sm100_ptx.cuh"

namespace df {
namespace {

using ptx::ex2_approx;

constexpr uint32_t kStageTokens = 64, kComputeWarps = 4, kThreads = 32 * (kComputeWarps + 1);
constexpr float kWeightBits = 15.0f;  // weights are held times 2^15, so that halves reach down to 2^-39 of the largest one
constexpr uint32_t kMaxGrid = 640;
constexpr uint32_t kCounterBytes = 4096;  // a counter per CTA, at the workspace's beginning

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

// How query rows fill the 16 rows of an instruction: 8 fp32 rows and their second parts, or 16 bf16 rows. A warp takes 16 rows (fp32: two instructions' worth,
// which share the widened codes), or, where requests have few, 8: half the accumulators and operands then let more of its work overlap.
enum Mode { kFp32Few, kFp32, kBf16Few, kBf16 };
// Rows that one warp takes, and the size of a partial state.
template <Mode MODE>
constexpr uint32_t kRows = MODE == kBf16 || MODE == kFp32 ? 16 : 8;
template <Mode MODE, int DP>
constexpr uint32_t kPartialFloats = kComputeWarps * kRows<MODE> * (DP + 2);

struct Request {
  uint32_t first, rows, q_len, len, tiles, row_tiles;
  uint32_t weight_log2;  // warps that the rows of a tile are dealt to (1, 2, 4; the tokens to the others): units of a stage
};

template <uint32_t ROWS>
__device__ __forceinline__ Request request_of(const AttendParams &p, uint32_t r) {
  Request q;
  const long long most = (long long)p.width * p.P;
  q.len = (uint32_t)min((long long)max(__ldg(p.lens + r), 0), most);
  const int b = max(0, min(__ldg(p.starts + r), (int)p.n_tokens)), e = max(b, min(__ldg(p.starts + r + 1), (int)p.n_tokens));
  q.first = (uint32_t)b;
  q.q_len = (uint32_t)(e - b);
  q.rows = q.q_len * p.group;
  q.weight_log2 = q.rows <= ROWS ? 0u : q.rows <= 2 * ROWS ? 1u : 2u;
  q.row_tiles = (q.rows + (ROWS << q.weight_log2) - 1) / ROWS >> q.weight_log2;
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

// What a segment costs besides its stages (its rows of q, the sums over warps, its results), in units: 5 to 8 us beside 1.2 us for a stage of 128-byte
// tokens with every SM busy. Counted at the segment's beginning; without it CTAs with several short segments ended 20 us after the others
// (32 ragged requests: 94 us, 77 with it).
template <int DP>
constexpr uint32_t kSegmentUnits = DP == 128 ? 6 : 10;
template <int DP>
__device__ __forceinline__ uint32_t span_of(const Request &q) { return (q.tiles << q.weight_log2) + kSegmentUnits<DP>; }
template <int DP>
__device__ __forceinline__ uint32_t tile_at(const Request &q, uint32_t x) {  // stages of a segment in front of its unit x
  return x <= kSegmentUnits<DP> ? 0u : (x - kSegmentUnits<DP>) >> q.weight_log2;
}

// The line of units (or, where no segment is cut, of segments) and this CTA's place on it. Its length is below 2^31 (the launcher sees to
// it), so that its divisions are of 32 bits: those of 64 took a part's first microseconds.
struct Line {
  uint32_t at, end, base;  // base: of request r
  uint32_t per_cta, r;
  bool whole;  // counted in segments
};

template <uint32_t ROWS, int DP>
__device__ __forceinline__ bool next_part(const AttendParams &p, Line &line, Part &part) {
  while (line.at < line.end) {
    Request q = request_of<ROWS>(p, line.r);
    uint32_t span = line.whole ? 1u : span_of<DP>(q);
    while (line.at >= line.base + span * q.row_tiles * p.kv_heads) {  // on to the request that holds line.at (it is below the line's end)
      line.base += span * q.row_tiles * p.kv_heads;
      q = request_of<ROWS>(p, ++line.r);
      span = line.whole ? 1u : span_of<DP>(q);
    }
    const uint32_t idx = line.whole ? line.at - line.base : (line.at - line.base) / span;
    const uint32_t s0 = line.base + idx * span, s1 = s0 + span;
    const uint32_t row_tile = q.row_tiles == 1 ? 0u : idx / p.kv_heads;
    part.rq = q;
    part.r = line.r;
    part.h = idx - row_tile * p.kv_heads;
    part.row0 = row_tile * (ROWS << q.weight_log2);
    part.parts = 1;
    part.first_cta = blockIdx.x;
    part.t0 = 0;
    part.t1 = q.tiles;
    const uint32_t from = line.at, stop = min(s1, line.end);
    line.at = stop;
    if (from != s0 || stop != s1) {  // cut
      part.t0 = tile_at<DP>(q, from - s0);
      if (stop < s1) part.t1 = tile_at<DP>(q, stop - s0);
      // A boundary between CTAs counts down to whole stages; so the first CTA that a segment reaches may have none of it, every other one has
      // some (a CTA has at least four units more than a segment's beginning takes).
      uint32_t c0 = s0 / line.per_cta;
      const uint32_t c1 = (s1 - 1) / line.per_cta;
      if (tile_at<DP>(q, (c0 + 1) * line.per_cta - s0) == 0) ++c0;
      part.first_cta = c0;
      part.parts = c1 - c0 + 1;
      if (part.t1 <= part.t0) continue;
    }
    const uint32_t last_row = min(q.rows, part.row0 + (ROWS << q.weight_log2)) - 1;
    const int see = (int)q.len - (int)q.q_len + (int)(p.group == 1 ? last_row : last_row / p.group) + 1;
    part.limit = (uint32_t)max(0, min(see, (int)q.len));
    part.t1 = max(part.t0, min(part.t1, (part.limit + kStageTokens - 1) / kStageTokens));
    return true;
  }
  return false;
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

__device__ __forceinline__ void mma_half(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_half_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // onto zeros
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t halves(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// a pair of floats as halves and what they leave
__device__ __forceinline__ void split_halves(float x, float y, uint32_t &first, uint32_t &second) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  first = *reinterpret_cast<const uint32_t *>(&h);
  second = halves(x - f.x, y - f.y);
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

// Sums (m, l, o[4]) states one after another.
struct Running {
  float m = -FLT_MAX, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  __device__ __forceinline__ void add(float m2, float l2, const float4 &o2) {
    const float top = fmaxf(m, m2), a = ex2_approx(m - top), b = ex2_approx(m2 - top);
    m = top;
    l = l * a + l2 * b;
    o[0] = o[0] * a + o2.x * b;
    o[1] = o[1] * a + o2.y * b;
    o[2] = o[2] * a + o2.z * b;
    o[3] = o[3] * a + o2.w * b;
  }
};

__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the compute warps; all of them come to each

template <int DP>
constexpr uint32_t kSubBytes = 16 * DP;  // a box of 16 tokens, or less where D < DP: whole swizzle periods
// CTAs of an SM, by the registers that they need, and stages of the ring, by the shared memory that is left to each.
template <Mode MODE, int DP>
constexpr int kCtas = DP == 64 ? (kRows<MODE> == 8 ? 4 : 3) : MODE == kFp32Few ? 3 : 2;
template <Mode MODE, int DP>
constexpr uint32_t kStagesOf = DP == 64 ? (kRows<MODE> == 8 ? 5 : 6) : MODE == kFp32Few ? 3 : MODE == kFp32 ? 4 : 5;
// A warp's region of shared memory: its rows of q as operands (16 bytes a lane and k-step, for each instruction that shares a code), later 8 rows of sums.
template <Mode MODE>
constexpr uint32_t kTiles = MODE == kFp32 ? 2 : 1;
template <Mode MODE, int DP>
constexpr uint32_t kWarpBytes = kTiles<MODE> * 8 * DP * 4;
template <Mode MODE, int DP>
constexpr uint32_t kRingBytes = kStagesOf<MODE, DP> * 2 * (kStageTokens / 16) * kSubBytes<DP>;
template <Mode MODE, int DP>
constexpr uint32_t kSmemBytes = 1024 + kRingBytes<MODE, DP> + kComputeWarps * kWarpBytes<MODE, DP>;

template <Mode MODE, int FORMAT, int DP>
__global__ void __launch_bounds__(kThreads, kCtas<MODE, DP>)
k_cache_attention(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const AttendParams p) {
  constexpr uint32_t ROWS = kRows<MODE>, kStages = kStagesOf<MODE, DP>;
  constexpr bool BF16 = MODE == kBf16Few || MODE == kBf16;
  constexpr int KT = DP / 16, NT = DP / 8, RW = ROWS / 8, MT = kTiles<MODE>;  // k-steps, n-tiles, rows of a lane
  extern __shared__ uint8_t smem_raw[];
  __shared__ float2 s_scale[kStages][kStageTokens / 16];  // k_scale, v_scale of a stage's boxes
  __shared__ float s_m[kComputeWarps][8], s_l[kComputeWarps][8];
  __shared__ Line s_line[kComputeWarps];
  __shared__ Part s_part[kComputeWarps];
  __shared__ uint64_t s_full[kStages], s_empty[kStages];
  __shared__ uint32_t s_units[kThreads], s_segments[kThreads], s_most[kThreads / 32], s_last, s_abort;
  const uint32_t t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const uint32_t ring = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *ring_bytes = smem_raw + (ring - ptx::smem_u32(smem_raw));
  float *merge = reinterpret_cast<float *>(ring_bytes + kRingBytes<MODE, DP>);  // [warp]: q as operands [k-step][lane][4 words], later a state [8 rows][DP]
  if (t == 0) {
    for (uint32_t s = 0; s < kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&s_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&s_empty[s]), kComputeWarps);
    }
    ptx::mbar_init_fence();
    s_abort = 0;
    ptx::tma_prefetch_desc(&k_map);
    ptx::tma_prefetch_desc(&v_map);
  }
  ptx::pdl_wait();

  // ---- the line: sums over the requests, and the request at which this CTA begins
  const uint32_t per = (p.n_requests + kThreads - 1) / kThreads, r0 = min(p.n_requests, t * per), r1 = min(p.n_requests, r0 + per);
  uint32_t units = 0, segments = 0, most = 0;
  for (uint32_t r = r0; r < r1; ++r) {
    const Request q = request_of<ROWS>(p, r);
    const uint32_t n = q.row_tiles * p.kv_heads;
    segments += n;
    units += n * span_of<DP>(q);
    if (n) most = max(most, span_of<DP>(q));
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, units, o), b = __shfl_up_sync(0xffffffffu, segments, o);
    if (lane >= (uint32_t)o) { units += a; segments += b; }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  s_units[t] = units;
  s_segments[t] = segments;
  if (lane == 0) s_most[warp] = most;
  __syncthreads();
  uint32_t all_units = 0, all_segments = 0;
  most = 0;
#pragma unroll
  for (uint32_t w = 0; w < kThreads / 32; ++w) {
    all_units += s_units[32 * w + 31];
    all_segments += s_segments[32 * w + 31];
    most = max(most, s_most[w]);
  }
  Line line;
  const uint32_t G = gridDim.x, seg_per = (all_segments + G - 1) / G, unit_per = max(kSegmentUnits<DP> + 8u, (all_units + G - 1) / G);
  line.whole = p.whole || (unsigned long long)seg_per * most <= unit_per + kSegmentUnits<DP>;  // cutting costs another end
  line.per_cta = line.whole ? seg_per : unit_per;
  const uint32_t total = line.whole ? all_segments : all_units;
  if ((unsigned long long)line.per_cta * blockIdx.x >= total) return;  // (the whole CTA)
  line.at = line.per_cta * blockIdx.x;
  line.end = min(total, line.at + line.per_cta);
  // the warp, then the lane, then the request of those lane's that line.at falls to: every warp looks for itself
  {
    const uint32_t *sums = line.whole ? s_segments : s_units;
    uint32_t base = 0, w = 0;
    while (line.at >= base + sums[32 * w + 31]) base += sums[32 * w++ + 31];
    const uint32_t mine = base + sums[32 * w + lane];
    const uint32_t owner = __ffs(__ballot_sync(0xffffffffu, line.at < mine)) - 1;
    const uint32_t before = __shfl_sync(0xffffffffu, mine, max(owner, 1u) - 1);
    line.base = owner == 0 ? base : before;
    line.r = (32 * w + owner) * per;  // next_part goes on to the request
  }

  const uint32_t a_full = ptx::smem_u32(&s_full[0]), a_empty = ptx::smem_u32(&s_empty[0]);
  const uint32_t chunks = p.D / 16;  // 16-byte pieces of a row
  uint32_t stage = 0;  // stages so far, this CTA
  if (warp == kComputeWarps) {
    // ---------------------------------------------------------------- the loading warp
    // Eight stages at a time: lane i has the page and scales of box i % 4 of stage i / 4. They are looked up a group ahead: the table's
    // entry before the present group is loaded, the scales behind it.
    struct Group {
      uint32_t stages, slice, line, boxes;  // boxes: a bit per lane that has one
      int32_t page;
      float2 scale;
    } now, then;
    const uint32_t box_bytes = 16 * p.D;
    uint32_t tile = 0, head = 0;
    Part part;
    part.t1 = 0;
    auto look_up = [&](Group &gr) {
      gr.stages = 0;
      if (tile >= part.t1) {
        do {
          if (!next_part<ROWS, DP>(p, line, part)) return;
        } while (part.t0 >= part.t1);  // a part that sees nothing
        tile = part.t0;
      }
      head = part.h;
      const uint32_t token = (tile + lane / 4) * kStageTokens + lane % 4 * 16;
      const bool in = token < part.limit && tile + lane / 4 < part.t1;
      gr.page = in ? __ldg(p.table + (size_t)part.r * p.width + token / p.P) : -1;
      gr.line = token % p.P * p.D / 128;
      gr.boxes = __ballot_sync(0xffffffffu, in);
      gr.stages = min(8u, part.t1 - tile);
      tile += gr.stages;
    };
    auto look_up_scales = [&](Group &gr) {
      const bool in = (uint32_t)gr.page < p.n_pages;
      gr.slice = in ? (uint32_t)gr.page * p.kv_heads + head : p.n_pages * p.kv_heads;  // behind the last slice: zeros
      gr.scale = in ? make_float2(__ldg(p.k_scale + gr.slice), __ldg(p.v_scale + gr.slice)) : make_float2(0.0f, 0.0f);
    };
    uint32_t slot = 0, phase = 1;  // (the phase that a slot's second use waits for is the first, 0: see the flip at the ring's end)
    look_up(now);
    look_up_scales(now);
    while (now.stages) {
      look_up(then);
      for (uint32_t s = 0; s < now.stages; ++s) {
        if (stage >= kStages && !ptx::mbar_wait_warp(a_empty + 8 * slot, phase, &s_abort)) {
          if (lane == 0 && p.status) atomicOr(p.status, DEV_STATUS_WAIT_EXPIRED);
          goto loaded;
        }
        const bool my_turn = lane / 4 == s;
        if (my_turn) s_scale[slot][lane % 4] = now.scale;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_expect_tx(a_full + 8 * slot, 2 * box_bytes * __popc((now.boxes >> (4 * s)) & 15u));
        __syncwarp();
        if (my_turn && (now.boxes >> lane & 1)) {
          const uint32_t dst = ring + (slot * 2 * 4 + lane % 4) * kSubBytes<DP>;
          ptx::tma_load_3d(dst, &k_map, a_full + 8 * slot, 0, (int)now.line, (int)now.slice);
          ptx::tma_load_3d(dst + 4 * kSubBytes<DP>, &v_map, a_full + 8 * slot, 0, (int)now.line, (int)now.slice);
        }
        ++stage;
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1;
        }
      }
      if (then.stages) look_up_scales(then);
      now = then;
    }
  loaded:
    if (s_abort) {  // copies in flight write to this CTA's shared memory: none may be left when it goes
      for (uint32_t s = stage > kStages ? stage - kStages : 0; s < stage; ++s)
        for (uint32_t polls = 0; polls < (1u << 16) && !ptx::mbar_try_wait(a_full + 8 * (s % kStages), (s / kStages) & 1); ++polls) {
        }
    }
    return;
  }

  // ---------------------------------------------------------------- the computing warps
  const uint32_t g = lane >> 2, c = lane & 3;
  bool ok = true;
  uint32_t slot = 0, phase = 0;  // of the next stage
  uint8_t *q_at = ring_bytes + kRingBytes<MODE, DP> + warp * kWarpBytes<MODE, DP> + lane * 16;
  // Tokens of a lane's accumulators: tile j, columns 2c and 2c + 1. With 64-byte rows the order below keeps two rows of a 128-byte
  // line together, which the swizzle then spreads over all banks.
  auto token_of = [&](uint32_t j, uint32_t col) { return DP == 128 ? 8 * j + col : 4 * (col >> 1) + 2 * j + (col & 1); };
  auto piece = [&](uint32_t token, uint32_t chunk) {  // where a box has a 16-byte piece
    const uint32_t x = token * chunks + min(chunk, chunks - 1);
    return (x * 16) ^ ((x & 0x38u) << 1);
  };
  // Behind the row's end (D < DP) its last piece is read again: it meets zeros of q, or makes dims that are not stored.
  uint32_t k_off[2][KT / 4], v_off[4];
#pragma unroll
  for (int k4 = 0; k4 < KT / 4; ++k4) {
    k_off[0][k4] = piece(token_of(0, g), c * (KT / 4) + k4);
    k_off[1][k4] = piece(token_of(1, g), c * (KT / 4) + k4);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) v_off[k] = DP == 128 ? piece(token_of(k >> 1, 2 * c + (k & 1)), g) : piece(token_of(k >> 1, 2 * c + (k & 1)), g >> 1) + 8 * (g & 1);
  // A warp's place on the line and its present part lie in shared memory: registers are for the loop over the tokens.
  if (lane == 0) s_line[warp] = line;
  for (;;) {
    __syncwarp();
    Line next = s_line[warp];
    __syncwarp();
    Part found;
    if (!next_part<ROWS, DP>(p, next, found)) break;
    if (lane == 0) {
      s_line[warp] = next;
      s_part[warp] = found;
    }
    __syncwarp();
    const Part &part = s_part[warp];
    const uint32_t tile0 = found.t0, tile1 = found.t1;
    const uint32_t weight = 1u << part.rq.weight_log2, row_warp = warp & (weight - 1), token_warp = warp >> part.rq.weight_log2;
    const uint32_t warp_row = part.row0 + row_warp * ROWS;
    const int behind = (int)part.rq.len - (int)part.rq.q_len + 1, most_seen = (int)part.rq.len;
    auto see_of = [&](uint32_t j) { return (uint32_t)max(0, min(behind + (int)j, most_seen)); };  // tokens that query token j sees
    // rows of this lane
    uint32_t see[RW];
    bool valid[RW];
    float norm[RW], m[RW], l[RW];
    float2 o[RW][NT];  // columns 2c, 2c + 1 of n-tile n: dims 2c * DP/8 + n and (2c + 1) * DP/8 + n
    __syncwarp();  // the region below was read as a merge buffer by this warp's lanes alone, behind a barrier
    Raw4<BF16> raw[RW][KT];  // all loads first: they come from DRAM
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const uint32_t row = warp_row + g + 8 * i;
      valid[i] = row < part.rq.rows;
      const uint32_t j = p.group == 1 ? row : row / p.group, head = part.h * p.group + row - j * p.group;
      see[i] = valid[i] ? see_of(j) : 0u;
      const unsigned long long e = (unsigned long long)(part.rq.first + j) * p.q_stride + (unsigned long long)head * p.D + c * (DP / 4);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if (valid[i] && c * (DP / 4) + kt * 4 < p.D) raw[i][kt].load(p.q, e + kt * 4, p.q_aligned);
        else raw[i][kt].zero();
      }
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      float top = 0.0f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, fabsf(raw[i][kt].at(k)));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the largest element to 1 .. 2 (an infinity or zero stays)
      const uint32_t exponent = min(max(__float_as_uint(top) >> 23, 1u), 253u);
      const bool keep = top == 0.0f || top == INFINITY;
      const float down = keep ? 1.0f : __uint_as_float((254u - exponent) << 23);
      norm[i] = (keep ? 1.0f : __uint_as_float(exponent << 23)) * p.scale_log2;  // the scale after the product: q itself fits its halves
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint32_t a[2][2];
        if (BF16) {  // this row's two of the four operand words
          a[0][0] = halves(raw[i][kt].at(0) * down, raw[i][kt].at(1) * down);
          a[0][1] = halves(raw[i][kt].at(2) * down, raw[i][kt].at(3) * down);
          if (MODE == kBf16Few) {
            *reinterpret_cast<uint2 *>(q_at + kt * 512) = make_uint2(a[0][0], a[0][1]);
          } else {
            *reinterpret_cast<uint32_t *>(q_at + kt * 512 + 4 * i) = a[0][0];
            *reinterpret_cast<uint32_t *>(q_at + kt * 512 + 4 * (2 + i)) = a[0][1];
          }
        } else {
          split_halves(raw[i][kt].at(0) * down, raw[i][kt].at(1) * down, a[0][0], a[0][1]);
          split_halves(raw[i][kt].at(2) * down, raw[i][kt].at(3) * down, a[1][0], a[1][1]);
          *reinterpret_cast<uint4 *>(q_at + (kt * MT + i) * 512) = make_uint4(a[0][0], a[0][1], a[1][0], a[1][1]);
        }
      }
      m[i] = -FLT_MAX;
      l[i] = 0.0f;
#pragma unroll
      for (int n2 = 0; n2 < NT; ++n2) o[i][n2] = make_float2(0.0f, 0.0f);
    }
    // what the warp's rows see, at least and at most: rows are in the order of their tokens
    const uint32_t last_row = min(part.rq.rows, warp_row + ROWS) - 1;
    const uint32_t see_all = see_of(p.group == 1 ? warp_row : warp_row / p.group);
    const uint32_t see_any = warp_row < part.rq.rows ? see_of(p.group == 1 ? last_row : last_row / p.group) : 0u;
    const bool second_rows = RW == 2 && warp_row + 8 < part.rq.rows;  // whether rows 8 .. 15 of the warp are there

    // Two boxes, 32 tokens, at a time. Where tokens are dealt to four warps, two of them share a stage and the pairs take turns; to two, each
    // takes a half. Every warp waits for every stage and gives it back, also one that has nothing to do with it: a wait names its phase by a
    // parity, and a warp that had passed over a stage of a slot would take that stage for the next one.
    const uint32_t pair0 = weight == kComputeWarps ? 0u : token_warp & 1, pair1 = weight == kComputeWarps ? 2u : pair0 + 1;
    bool idle = weight == 1 && token_warp >> 1 != 0;
    for (uint32_t tile = tile0; ok && tile < tile1; ++tile) {
      ok = ptx::mbar_wait_warp(a_full + 8 * slot, phase, &s_abort);
      const uint32_t here = slot;
      if (++slot == kStages) {
        slot = 0;
        phase ^= 1;
      }
      auto give_back = [&]() {
        if (lane == 0) ptx::mbar_arrive(a_empty + 8 * here);
      };
      if (idle || !ok) {
        if (ok) give_back();
        idle = false;
        continue;
      }
      idle = weight == 1;
      const uint8_t *stage_at = ring_bytes + here * 2 * 4 * kSubBytes<DP>;
      bool given_back = false;
      for (uint32_t pair = pair0; pair < pair1; ++pair) {
        const uint32_t token0 = tile * kStageTokens + pair * 32;
        if (token0 >= see_any) break;
        const float2 scale[2] = {s_scale[here][2 * pair], s_scale[here][2 * pair + 1]};
        const uint8_t *k_at = stage_at + 2 * pair * kSubBytes<DP>, *v_at = k_at + 4 * kSubBytes<DP>;
        // ---- scores
        float acc[MT][4][4];
#pragma unroll
        for (int k4 = 0; k4 < KT / 4; ++k4) {
          uint32_t w[4][4];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            const uint4 v = *reinterpret_cast<const uint4 *>(k_at + (nt >> 1) * kSubBytes<DP> + k_off[nt & 1][k4]);
            w[nt][0] = v.x; w[nt][1] = v.y; w[nt][2] = v.z; w[nt][3] = v.w;
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            uint32_t a[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              if (MODE == kBf16Few) {
                const uint2 q2 = *reinterpret_cast<const uint2 *>(q_at + (k4 * 4 + kk) * 512);
                a[mt][0] = q2.x; a[mt][1] = 0u; a[mt][2] = q2.y; a[mt][3] = 0u;
              } else {
                const uint4 q4 = *reinterpret_cast<const uint4 *>(q_at + ((k4 * 4 + kk) * MT + mt) * 512);
                a[mt][0] = q4.x; a[mt][1] = q4.y; a[mt][2] = q4.z; a[mt][3] = q4.w;
              }
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
              uint32_t b0, b1;
              widen_word<FORMAT>(w[nt][kk], b0, b1);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                if (k4 == 0 && kk == 0) mma_half_first(acc[mt][nt], a[mt], b0, b1);
                else mma_half(acc[mt][nt], a[mt], b0, b1);
              }
            }
          }
        }
        // ---- V's bytes. Where registers allow (kEarly) all of them now, so that the stage is given back before the longer half of the work on
        // it; else two words of a lane's piece at a time, when they are used.
        const bool masked = token0 + 32 > see_all;
        constexpr bool kEarly = RW == 1;
        constexpr int kWords = kEarly ? NT / 4 : 2;
        uint32_t w[2][4][kWords];
        auto load_v = [&](int part) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint8_t *at = v_at + b * kSubBytes<DP> + v_off[k] + 8 * part;
              if constexpr (kWords == 4) {
                const uint4 v = *reinterpret_cast<const uint4 *>(at);
                w[b][k][0] = v.x; w[b][k][1] = v.y; w[b][k][2] = v.z; w[b][k][3] = v.w;
              } else {
                const uint2 v = *reinterpret_cast<const uint2 *>(at);
                w[b][k][0] = v.x; w[b][k][1] = v.y;
              }
            }
          if (FORMAT == DF_CACHE_E4M3 && masked) {  // behind the last token that a row sees a box may hold any bytes, and an 8-bit float may be NaN
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const bool behind_all = token0 + 16 * b + token_of(k >> 1, 2 * c + (k & 1)) >= see_any;
#pragma unroll
                for (int i = 0; i < kWords; ++i) w[b][k][i] = behind_all ? 0u : w[b][k][i];
              }
          }
        };
        if (kEarly) {
          load_v(0);
          if (pair + 1 == pair1) {
            __syncwarp();
            give_back();
            given_back = true;
          }
        }
        // ---- weights
        // The two boxes' weights meet one scale of V, the larger one; a row that sees none of a box's tokens takes nothing of
        // it, whatever its scale is (it may be NaN).
        const float v_scale = fmaxf(scale[0].y, scale[1].y);
        const bool v_alike = scale[0].y == scale[1].y && !masked;
        uint32_t pa[MT][2][4];
        float v_row[RW], before[RW];
        bool grew = false;
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          before[i] = m[i];
          v_row[i] = 0.0f;
          if (MODE == kBf16Few || (BF16 && i == 1 && !second_rows)) pa[0][0][1] = pa[0][0][3] = pa[0][1][1] = pa[0][1][3] = 0u;
          if (i == 1 && !second_rows) {
            if (!BF16) {
#pragma unroll
              for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) pa[MT - 1][b][k] = 0u;
            }
            continue;
          }
          const float f[2] = {scale[0].x * norm[i], scale[1].x * norm[i]};
          float s[4][2];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) s[nt][k] = (BF16 ? acc[0][nt][2 * i + k] : acc[i % MT][nt][k] + acc[i % MT][nt][2 + k]) * f[nt >> 1];
          if (masked) {
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (token0 + 16 * (nt >> 1) + token_of(nt & 1, 2 * c + k) >= see[i]) s[nt][k] = -INFINITY;
          }
          float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), fmaxf(fmaxf(s[2][0], s[2][1]), fmaxf(s[3][0], s[3][1])));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          grew |= top > m[i];
          m[i] = fmaxf(m[i], top);
          const float shift = m[i] - kWeightBits;
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) s[nt][k] = ex2_approx(s[nt][k] - shift);
          l[i] = fmaf(l[i], ex2_approx(before[i] - m[i]), ((s[0][0] + s[0][1]) + (s[1][0] + s[1][1])) + ((s[2][0] + s[2][1]) + (s[3][0] + s[3][1])));
          v_row[i] = token0 < see[i] ? v_scale : 0.0f;
          if (!v_alike) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const float share = token0 + 16 * b < see[i] && v_scale != 0.0f ? __fdividef(scale[b].y, v_scale) : 0.0f;
#pragma unroll
              for (int nt = 2 * b; nt < 2 * b + 2; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k) s[nt][k] *= share;
            }
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (BF16) {
              pa[0][b][i] = halves(s[2 * b][0], s[2 * b][1]);
              pa[0][b][2 + i] = halves(s[2 * b + 1][0], s[2 * b + 1][1]);
            } else {
              split_halves(s[2 * b][0], s[2 * b][1], pa[i % MT][b][0], pa[i % MT][b][1]);
              split_halves(s[2 * b + 1][0], s[2 * b + 1][1], pa[i % MT][b][2], pa[i % MT][b][3]);
            }
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            const float f = ex2_approx(before[i] - m[i]);
#pragma unroll
            for (int n = 0; n < NT; ++n) o[i][n] = make_float2(o[i][n].x * f, o[i][n].y * f);
          }
        }
        // ---- output
#pragma unroll
        for (int n4 = 0; n4 < NT / 4; ++n4) {
          if (!kEarly && n4 % 2 == 0) load_v(n4 / 2);
          const int i4 = kEarly ? n4 : n4 % 2;
          uint32_t b0[2][4], b1[2][4];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            widen_pairs<FORMAT>(w[b][0][i4], w[b][1][i4], b0[b]);
            widen_pairs<FORMAT>(w[b][2][i4], w[b][3][i4], b1[b]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int n = n4 * 4 + k;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float d[4];
              mma_half_first(d, pa[mt][0], b0[0][k], b1[0][k]);
              mma_half(d, pa[mt][1], b0[1][k], b1[1][k]);
              if (BF16) {
                o[0][n] = ptx::fma2(make_float2(v_row[0], v_row[0]), make_float2(d[0], d[1]), o[0][n]);
                if (RW == 2) o[RW - 1][n] = ptx::fma2(make_float2(v_row[RW - 1], v_row[RW - 1]), make_float2(d[2], d[3]), o[RW - 1][n]);
              } else {
                o[mt][n] = ptx::fma2(make_float2(v_row[mt], v_row[mt]), ptx::add2(make_float2(d[0], d[1]), make_float2(d[2], d[3])), o[mt][n]);
              }
            }
          }
        }
      }
      if (!given_back) {
        __syncwarp();
        give_back();
      }
    }
    if (!ok && lane == 0 && p.status) atomicOr(p.status, DEV_STATUS_WAIT_EXPIRED);
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // four of the lane's DP / 4 dims of row i, from the n-th on
    auto four = [&](int i, int n) {
      return n < NT ? make_float4(o[i][n].x, o[i][n + 1].x, o[i][n + 2].x, o[i][n + 3].x)
                    : make_float4(o[i][n - NT].y, o[i][n - NT + 1].y, o[i][n - NT + 2].y, o[i][n - NT + 3].y);
    };

    // ---- the result, or this part of it
    const bool split = part.parts > 1;
    const uint32_t rows = min(part.rq.rows - part.row0, weight * ROWS);
    auto state_of = [&](uint32_t cta) {  // the first CTA of a segment has it last, every other one first
      return p.partial + (size_t)(2 * cta + (cta == part.first_cta ? 1 : 0)) * kPartialFloats<MODE, DP>;
    };
    auto finish_row = [&](size_t row, uint32_t dim, const float4 &x, float mm, float ll) {  // four dims of a finished row
      const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
      const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
      if (dim < p.D) store_row4<BF16>(p.out, row * p.D + dim, p.out_aligned, y);
      if (dim == 0 && p.lse) p.lse[row] = ll == 0.0f ? -INFINITY : (mm - kWeightBits + log2f(ll)) * kLn2;
    };
    auto global_row = [&](uint32_t row) {
      const uint32_t rr = part.row0 + row;
      const uint32_t j = p.group == 1 ? rr : rr / p.group;
      return (size_t)(part.rq.first + j) * p.heads + part.h * p.group + rr - j * p.group;
    };
    float *mine_state = state_of(blockIdx.x), *mine_o = mine_state + 2 * kComputeWarps * ROWS;
    if (weight == kComputeWarps) {
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        if (!valid[i]) continue;
        const uint32_t row = warp * ROWS + g + 8 * i;
#pragma unroll
        for (int n = 0; n < DP / 4; n += 4) {
          const uint32_t dim = c * (DP / 4) + n;
          if (split) *reinterpret_cast<float4 *>(mine_o + row * DP + dim) = four(i, n);
          else finish_row(global_row(row), dim, four(i, n), m[i], l[i]);
        }
        if (split && c == 0) *reinterpret_cast<float2 *>(mine_state + 2 * row) = make_float2(m[i], l[i]);
      }
    } else {
      // Four dims of a row, at a place that keeps the lanes of a store in different banks.
      auto spread = [&](uint32_t row, uint32_t d4) { return d4 ^ (((d4 >> (DP == 128 ? 3 : 2)) ^ (row << 2)) & (DP / 16 - 1)); };
      // the states of the warps that shared the tokens, eight rows of a warp at a time; a warp's is where its part of q was
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        if (8u * i >= rows) break;
        if (valid[i]) {
          if (c == 0) { s_m[warp][g] = m[i]; s_l[warp][g] = l[i]; }
#pragma unroll
          for (int n = 0; n < DP / 16; ++n) *reinterpret_cast<float4 *>(merge + warp * (kWarpBytes<MODE, DP> / 4) + g * DP + 4 * spread(g, c * (DP / 16) + n)) = four(i, 4 * n);
        }
        compute_barrier();
        for (uint32_t e = t; e < weight * 8 * (DP / 4); e += 32 * kComputeWarps) {
          const uint32_t w0 = e / (8 * (DP / 4)), r8 = e / (DP / 4) % 8, row = w0 * ROWS + r8 + 8 * i, dim = e % (DP / 4) * 4;
          if (row >= rows) break;
          Running sum;
          for (uint32_t w = w0; w < kComputeWarps; w += weight)
            sum.add(s_m[w][r8], s_l[w][r8], *reinterpret_cast<const float4 *>(merge + w * (kWarpBytes<MODE, DP> / 4) + r8 * DP + 4 * spread(r8, dim / 4)));
          const float4 x = make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
          if (!split) {
            finish_row(global_row(row), dim, x, sum.m, sum.l);
          } else {
            *reinterpret_cast<float4 *>(mine_o + row * DP + dim) = x;
            if (dim == 0) *reinterpret_cast<float2 *>(mine_state + 2 * row) = make_float2(sum.m, sum.l);
          }
        }
        if (i + 1 < RW) compute_barrier();
      }
    }
    if (split) {
      compute_barrier();
      if (t == 0) {  // releases what the barrier has gathered, and acquires what the CTAs before have released
        unsigned int arrived;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(arrived) : "l"(p.counters + part.first_cta) : "memory");
        s_last = arrived + 1 == part.parts;
        if (s_last) p.counters[part.first_cta] = 0;  // ready for the next call
      }
      compute_barrier();
      if (s_last) {
        const uint32_t elements = rows * (DP / 4), ways = max(1u, 32 * kComputeWarps / elements);
        // thread: four dims of a row, and every `ways`-th part where there are fewer of them than threads
        const uint32_t e0 = ways > 1 ? t % elements : t, way = ways > 1 ? t / elements : 0;
        for (uint32_t e = e0; e < elements && way < ways; e += 32 * kComputeWarps) {
          const uint32_t row = e / (DP / 4), dim = e % (DP / 4) * 4;
          Running sum;
#pragma unroll 4
          for (uint32_t i = way; i < part.parts; i += ways) {
            const float *state = state_of(part.first_cta + i);
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(state + 2 * row));
            sum.add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4 *>(state + 2 * kComputeWarps * ROWS + row * DP + dim)));
          }
          if (ways == 1) {
            finish_row(global_row(row), dim, make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]), sum.m, sum.l);
          } else {  // elements * ways <= 128 threads, six floats each
            float *at = merge + (way * elements + e) * 8;
            *reinterpret_cast<float4 *>(at) = make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
            at[4] = sum.m;
            at[5] = sum.l;
          }
        }
        if (ways > 1) {
          compute_barrier();
          if (t < elements) {
            Running sum;
            for (uint32_t w = 0; w < ways; ++w) {
              const float *at = merge + (w * elements + t) * 8;
              sum.add(at[4], at[5], *reinterpret_cast<const float4 *>(at));
            }
            finish_row(global_row(t / (DP / 4)), t % (DP / 4) * 4, make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]), sum.m, sum.l);
          }
        }
      }
    }
    compute_barrier();  // the merge buffer and s_last are free again
  }
}

struct DeviceInfo {
  std::once_flag once;
  uint32_t grid = 0;
};

// CTAs that the device keeps resident, asked once per kernel and device.
template <Mode MODE, int FORMAT, int DP>
uint32_t resident_ctas() {
  static DeviceInfo table[64];
  int dev = 0;
  if (check_cuda(cudaGetDevice(&dev)) != DF_OK || dev < 0 || dev >= 64) return 0;
  DeviceInfo &d = table[dev];
  std::call_once(d.once, [&]() {
    auto kernel = k_cache_attention<MODE, FORMAT, DP>;
    int per_sm = 0, n_sm = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes<MODE, DP>) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, (int)kThreads, kSmemBytes<MODE, DP>) != cudaSuccess ||
        cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return;
    d.grid = (uint32_t)(per_sm * n_sm);
  });
  return d.grid;
}

// The pool as lines of 128 bytes: a slice (page, head) is P * D / 128 of them, 16 tokens D / 8.
bool encode_pool_map(CUtensorMap *map, const void *pool, const AttendParams &p) {
  PFN_encodeTiled encode = get_encode_tiled();
  if (!encode) return false;
  const cuuint64_t lines = (cuuint64_t)p.P * p.D / 128;
  const cuuint64_t dims[3] = {128, lines, (cuuint64_t)p.n_pages * p.kv_heads};
  const cuuint64_t strides[2] = {128, lines * 128};
  const cuuint32_t box[3] = {128, p.D / 8, 1}, step[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <Mode MODE, int FORMAT, int DP>
int launch(AttendParams &p, const void *k_cache, const void *v_cache, cudaStream_t s) {
  constexpr uint32_t kFits = (DF_CACHE_WORKSPACE_BYTES - kCounterBytes) / (2 * kPartialFloats<MODE, DP> * 4);
  static_assert(kFits >= 2 * 148 && kMaxGrid * 4 <= kCounterBytes, "workspace");
  uint32_t grid = resident_ctas<MODE, FORMAT, DP>();
  if (grid == 0) return DF_ERR_CUDA;
  grid = grid < kFits ? grid : kFits;
  grid = grid < kMaxGrid ? grid : kMaxGrid;
  CUtensorMap k_map, v_map;
  if (!encode_pool_map(&k_map, k_cache, p) || !encode_pool_map(&v_map, v_cache, p)) return DF_ERR_CUDA;
  const int st = check_cuda(launch_kernel(k_cache_attention<MODE, FORMAT, DP>, dim3(grid), dim3(kThreads), kSmemBytes<MODE, DP>, s, k_map, v_map, p));
  note_launch();
  return st;
}

template <Mode MODE, int FORMAT>
int launch_for_head(AttendParams &p, const void *k_cache, const void *v_cache, cudaStream_t s) {
  return p.D <= 64 ? launch<MODE, FORMAT, 64>(p, k_cache, v_cache, s) : launch<MODE, FORMAT, 128>(p, k_cache, v_cache, s);
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
  if (!cache_shape_valid(n_kv_heads, d_head, page_size, n_pages) || (uint64_t)n_requests * n_kv_heads >= (1ull << 30))
    return finish(DF_ERR_INVALID_ARG);
  if (format != DF_CACHE_INT8 && format != DF_CACHE_E4M3) return finish(DF_ERR_INVALID_ARG);
  if (n_heads == 0 || n_heads % n_kv_heads != 0 || !isfinite(scale) || (uint64_t)n_tokens * n_heads >= (1ull << 31)) return finish(DF_ERR_INVALID_ARG);
  if (n_tokens > 1 && q_row_stride < (uint64_t)n_heads * d_head) return finish(DF_ERR_INVALID_ARG);
  if (!cache_shape_supported(d_head, page_size)) return finish(DF_ERR_UNSUPPORTED);
  if (n_tokens == 0 || n_requests == 0) return DF_OK;
  if (!q || !lens || !starts || !out || n_pages == 0 || !k_cache || !v_cache || !k_scale || !v_scale || (table_width && !block_table))
    return finish(DF_ERR_INVALID_ARG);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return finish(DF_ERR_INVALID_ARG);
  if (workspace_bytes < DF_CACHE_WORKSPACE_BYTES) return finish(DF_ERR_WORKSPACE);
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15u) != 0) return finish(DF_ERR_UNSUPPORTED);
  AttendParams p = {};
  p.q = q;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.table = block_table;
  p.lens = lens;
  p.starts = starts;
  p.out = out;
  p.lse = lse;
  p.counters = static_cast<unsigned int *>(workspace);
  p.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kCounterBytes);
  p.status = device_status_ptr();
  p.q_stride = q_row_stride;
  p.n_requests = n_requests;
  p.n_tokens = n_tokens;
  p.heads = n_heads;
  p.kv_heads = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.D = d_head;
  p.P = page_size;
  p.n_pages = n_pages;
  p.width = table_width;
  // what the line's units can add up to: segments (row tiles of at least eight rows, times K/V heads) of at most the table's width
  const uint64_t longest = ((uint64_t)table_width * page_size + kStageTokens - 1) / kStageTokens * kComputeWarps;
  p.whole = ((uint64_t)n_tokens * p.group / 8 + n_requests) * n_kv_heads * (longest + 16) >= (1ull << 31);
  p.q_aligned = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(q_row_stride * (q_bf16 ? 2 : 4))) & 15u) == 0;
  p.out_aligned = (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  p.scale_log2 = scale * kLog2e;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Eight rows to a warp while requests have no more on average.
  const bool few = (uint64_t)n_tokens * p.group <= 8ull * n_requests;
  auto run = [&](auto format_constant) {
    constexpr int FORMAT = decltype(format_constant)::value;
    if (!q_bf16) return few ? launch_for_head<kFp32Few, FORMAT>(p, k_cache, v_cache, s) : launch_for_head<kFp32, FORMAT>(p, k_cache, v_cache, s);
    return few ? launch_for_head<kBf16Few, FORMAT>(p, k_cache, v_cache, s) : launch_for_head<kBf16, FORMAT>(p, k_cache, v_cache, s);
  };
  return finish(format == DF_CACHE_INT8 ? run(std::integral_constant<int, DF_CACHE_INT8>{}) : run(std::integral_constant<int, DF_CACHE_E4M3>{}));
}
