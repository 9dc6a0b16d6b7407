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
// fits one half; its weights are two as well: in tiles of 8 rows the second halves take the other 8 (as zeros they cost registers: 2 CTAs an SM, and 72
// us instead of 69 at 32 requests of bf16), in tiles of 16 they are multiplied behind the first ones (16 requests of 20 rows, 8 heads of 128:
// 54 to 59 us; with weights rounded to 11 bits a result of 8 bits comes out as its neighbour now and then, 6e-4 of it in the 2-norm). V's scales enter the weights as
// cache_line.cuh says (unit_exponent; 59 to 63 us there, 1 to 2 % with few rows). The products of 32 tokens are added to the row's fp32 sums.
//
// Work. A CTA is one warp that loads (tensor-map copies of 16 tokens, 128-byte swizzle: the reads above are then free of bank conflicts at
// head sizes 64 and 128) and four that compute, over a ring of stages of 64 tokens. Of a request with no more rows (query tokens times heads per K/V
// head) than a warp takes, the tokens are dealt to the four warps; with up to twice as many, the rows to two pairs of warps and the tokens to the two of a
// pair; with more, the rows to all four, and every warp goes over all tokens. A stage then counts one, two or four units of the line on which work is dealt out (cache_line.cuh),
// since it takes a warp as much longer. Calls of many rows go to cache_attention_many.cu.
//
// What it reaches. 32 requests of 200 to 16000 tokens, one new each, 32 heads on 8 of 128, bf16 and e4m3: 66 us for 342 MB, 5.2 TB/s, 79 % of a copy's rate. One request of
// 131073 tokens, 16 heads of 128, fp32 and int8: 107 us for 537 MB, 5.0 TB/s. One of 300 tokens, 12 heads of 64: 7.2 us, of which 2.4 are a launch. The copies
// alone (no arithmetic) took 92 us of the second. What is left is latency with few warps to hide it: twelve computing warps an SM, 3.5 warps a scheduler of which 0.75 (first case) and 0.98 (second)
// can issue, 47 and 55 % of the issue slots in use; for each slot that a warp issues in it waits 2.3 and 1.7 for fixed latencies, 1.2 and 0.7 for memory; the ALU pipe,
// which widens, is 42 and 48 % busy, the tensor pipe a third. 735 instructions per 32 tokens (waits and the loading warp's included), 325 of them in the ALU pipe, 64
// products. A segment's beginning, its end and the addition of its parts take 8 to 10 us. 16 rows a warp: two CTAs an SM, 2.3 warps a scheduler, 0.43 of them able to issue, 35 % of the slots.
#include <float.h>
#include <math.h>

#include <mutex>
#include <type_traits>

#include "cache_line.cuh"
#include "sm100_ptx.cuh"

namespace df {
namespace {

using ptx::ex2_approx;

constexpr uint32_t kComputeWarps = 4, kThreads = 32 * (kComputeWarps + 1);
constexpr float kWeightBits = 15.0f;  // weights are held times 2^15, so that halves reach down to 2^-39 of the largest one

// How query rows fill the 16 rows of an instruction: 8 fp32 rows and their second parts, or 16 bf16 rows. A warp takes 16 rows (fp32: two instructions' worth,
// which share the widened codes), or, where requests have few, 8: half the accumulators and operands then let more of its work overlap.
enum Mode { kFp32Few, kFp32, kBf16Few, kBf16 };
// Rows that one warp takes, and the size of a partial state.
template <Mode MODE>
constexpr uint32_t kRows = MODE == kBf16 || MODE == kFp32 ? 16 : 8;
// What a segment costs besides its stages: 5 to 8 us beside 1.2 us for a stage of 128-byte tokens with every SM busy. Without it CTAs with several short
// segments ended 20 us after the others (32 ragged requests: 94 us, 77 with it).
template <Mode MODE, int DP>
struct Work {
  static constexpr uint32_t kRows = df::kRows<MODE>, kSegmentUnits = DP == 128 ? 6 : 10, kThreads = df::kThreads;
  static constexpr bool kDeal = true;
};
template <Mode MODE, int DP>
constexpr uint32_t kPartialFloats = kComputeWarps * kRows<MODE> * (DP + 2);

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

__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the compute warps; all of them come to each

template <int DP>
constexpr uint32_t kSubBytes = 16 * DP;  // a box of 16 tokens, or less where D < DP: whole swizzle periods
// CTAs of an SM, by the registers that they need, and stages of the ring, by the shared memory that is left to each.
template <Mode MODE, int DP>
constexpr int kCtas = DP == 64 ? (kRows<MODE> == 8 ? 4 : 3) : kRows<MODE> == 8 ? 3 : 2;
template <Mode MODE, int DP>
constexpr uint32_t kStagesOf = DP == 64 ? (kRows<MODE> == 8 ? 5 : 6) : kRows<MODE> == 8 ? 3 : MODE == kFp32 ? 4 : 5;
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
  using W = Work<MODE, DP>;
  constexpr uint32_t ROWS = kRows<MODE>, kStages = kStagesOf<MODE, DP>;
  constexpr bool BF16 = MODE == kBf16Few || MODE == kBf16;
  constexpr int KT = DP / 16, NT = DP / 8, RW = ROWS / 8, MT = kTiles<MODE>;  // k-steps, n-tiles, rows of a lane
  constexpr int PT = RW;  // operands that a box's weights fill: two where 16 rows have two halves each
  extern __shared__ uint8_t smem_raw[];
  __shared__ float2 s_scale[kStages][kStageTokens / 16];  // k_scale, v_scale of a stage's boxes
  __shared__ float s_m[kComputeWarps][8], s_l[kComputeWarps][8];
  __shared__ Line s_line[kComputeWarps];
  __shared__ Part s_part[kComputeWarps];
  __shared__ uint64_t s_full[kStages], s_empty[kStages];
  __shared__ LineSmem<W> s_sums;
  __shared__ uint32_t s_last, s_abort;
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

  Line line;
  if (!begin_line<W>(p, s_sums, line)) return;

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
          if (!next_part<W>(p, line, part)) return;
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
    if (!next_part<W>(p, next, found)) break;
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
    float norm[RW], m[RW], l[RW], excess[RW];  // (excess: d of unit_exponent)
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
            *reinterpret_cast<uint4 *>(q_at + kt * 512) = make_uint4(a[0][0], 0u, a[0][1], 0u);  // with the zeros of rows 8 .. 15: read as an operand's four words
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
      excess[i] = kLeastExcess;
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
              const uint4 q4 = *reinterpret_cast<const uint4 *>(q_at + ((k4 * 4 + kk) * MT + mt) * 512);
              a[mt][0] = q4.x; a[mt][1] = q4.y; a[mt][2] = q4.z; a[mt][3] = q4.w;
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
        const bool v_alike = scale[0].y == scale[1].y;
        const float v_log[2] = {scale_log(scale[0].y), scale_log(scale[1].y)};
        uint32_t pa[PT][2][4];
        float down[RW];
        bool grew = false;
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          down[i] = 1.0f;
          if (i == 1 && !second_rows) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                if (BF16) pa[0][b][2 * k + 1] = pa[PT - 1][b][2 * k + 1] = 0u;
                else pa[PT - 1][b][2 * k] = pa[PT - 1][b][2 * k + 1] = 0u;
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
          float tops[2];  // of the boxes
#pragma unroll
          for (int b = 0; b < 2; ++b) tops[b] = fmaxf(fmaxf(s[2 * b][0], s[2 * b][1]), fmaxf(s[2 * b + 1][0], s[2 * b + 1][1]));
          if (v_alike) tops[0] = tops[1] = fmaxf(tops[0], tops[1]);
          tops[0] = fmaxf(tops[0], __shfl_xor_sync(0xffffffffu, tops[0], 1));
          tops[0] = fmaxf(tops[0], __shfl_xor_sync(0xffffffffu, tops[0], 2));
          if (v_alike) {
            tops[1] = tops[0];
          } else {
            tops[1] = fmaxf(tops[1], __shfl_xor_sync(0xffffffffu, tops[1], 1));
            tops[1] = fmaxf(tops[1], __shfl_xor_sync(0xffffffffu, tops[1], 2));
          }
          const float before = m[i], e_before = unit_exponent(excess[i]);
          m[i] = fmaxf(before, fmaxf(tops[0], tops[1]));
          excess[i] = fmaxf(excess[i] + (before - m[i]), fmaxf(tops[0] - m[i] + v_log[0], tops[1] - m[i] + v_log[1]));
          const float e_now = unit_exponent(excess[i]), units = ex2_approx(-e_now);
          grew |= m[i] > before || e_now != e_before;
          down[i] = ex2_approx((before - m[i]) + (e_before - e_now));
          const float shift = m[i] - kWeightBits;
#pragma unroll
          for (int nt = 0; nt < 4; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) s[nt][k] = ex2_approx(s[nt][k] - shift);
          l[i] = fmaf(l[i], ex2_approx(before - m[i]), ((s[0][0] + s[0][1]) + (s[1][0] + s[1][1])) + ((s[2][0] + s[2][1]) + (s[3][0] + s[3][1])));
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            // a row that sees none of a box's tokens takes nothing of it, whatever its scale is (it may be NaN)
            const float share = masked && token0 + 16 * b >= see[i] ? 0.0f : share_of(scale[b].y, units);
#pragma unroll
            for (int nt = 2 * b; nt < 2 * b + 2; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k) s[nt][k] *= share;
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (BF16 && RW == 2) {  // first halves of 16 rows, then their second ones
              split_halves(s[2 * b][0], s[2 * b][1], pa[0][b][i], pa[PT - 1][b][i]);
              split_halves(s[2 * b + 1][0], s[2 * b + 1][1], pa[0][b][2 + i], pa[PT - 1][b][2 + i]);
            } else {
              split_halves(s[2 * b][0], s[2 * b][1], pa[i % MT][b][0], pa[i % MT][b][1]);
              split_halves(s[2 * b + 1][0], s[2 * b + 1][1], pa[i % MT][b][2], pa[i % MT][b][3]);
            }
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int i = 0; i < RW; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) o[i][n] = make_float2(o[i][n].x * down[i], o[i][n].y * down[i]);
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
              if (BF16 && RW == 2) {
                mma_half(d, pa[PT - 1][0], b0[0][k], b1[0][k]);
                mma_half(d, pa[PT - 1][1], b0[1][k], b1[1][k]);
                o[0][n] = ptx::add2(make_float2(d[0], d[1]), o[0][n]);
                o[RW - 1][n] = ptx::add2(make_float2(d[2], d[3]), o[RW - 1][n]);
              } else {
                o[mt][n] = ptx::add2(ptx::add2(make_float2(d[0], d[1]), make_float2(d[2], d[3])), o[mt][n]);
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
      const float unit = ex2_approx(unit_exponent(excess[i]));
#pragma unroll
      for (int n = 0; n < NT; ++n) o[i][n] = make_float2(o[i][n].x * unit, o[i][n].y * unit);
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
    auto finish_row = [&](size_t row, uint32_t dim, const float4 &x, float mm, float ll) { finish_row4<BF16>(p, row, dim, x, mm, ll, kWeightBits); };
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

template <Mode MODE, int FORMAT, int DP>
int launch(AttendParams &p, const void *k_cache, const void *v_cache, cudaStream_t s) {
  constexpr uint32_t kFits = (DF_CACHE_WORKSPACE_BYTES - kCounterBytes) / (2 * kPartialFloats<MODE, DP> * 4);
  static_assert(kFits >= 2 * 148, "workspace");
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
  // How many rows requests have on average decides who multiplies. Up to 8: a warp's few. Up to 32: 16 rows a warp. Above: tiles of 128 rows on tcgen05, which
  // take the same time for 9 rows as for 32. Measured over 3000 to 6000 cached tokens, mma.sync to tcgen05, us, bf16 and fp32: 16 requests of 12 heads of
  // 64, 16 rows 47 to 100, 54 to 101; 32 rows 74 to 100, 84 to 102; 64 rows 129 to 100, 148 to 103. 16 requests of 8 heads of 128, 20 rows 89 to 88, 102 to
  // 96; 32 rows 96 to 89, 111 to 97; 64 rows 171 to 91, 195 to 102. One request of 12 heads of 64, 24 rows 30 to 26, 32 to 27; 40 rows 58 to 27, 60 to 28.
  // These are requests alike. The mean decides for the whole call, so requests unlike each other cost more together than apart: 31 single tokens beside
  // a piece of 500 tokens, 12 heads of 64 in fp32, 134 us (49 and 40 by themselves); 24 beside 8 pieces of 128, 32 heads on 8 of 128 in bf16, 232 (43 and 138).
  const uint64_t rows = (uint64_t)n_tokens * p.group;
  if (rows > 32ull * n_requests) return finish(cache_attention_many(p, k_cache, v_cache, q_bf16 != 0, format, s));
  const bool few = rows <= 8ull * n_requests;
  auto run = [&](auto format_constant) {
    constexpr int FORMAT = decltype(format_constant)::value;
    if (!q_bf16) return few ? launch_for_head<kFp32Few, FORMAT>(p, k_cache, v_cache, s) : launch_for_head<kFp32, FORMAT>(p, k_cache, v_cache, s);
    return few ? launch_for_head<kBf16Few, FORMAT>(p, k_cache, v_cache, s) : launch_for_head<kBf16, FORMAT>(p, k_cache, v_cache, s);
  };
  return finish(format == DF_CACHE_INT8 ? run(std::integral_constant<int, DF_CACHE_INT8>{}) : run(std::integral_constant<int, DF_CACHE_E4M3>{}));
}
