// cache_attention_many.cu - attention over the 8-bit paged cache for requests of many query rows (pieces of prompts, drafted tokens), on tcgen05, for
// B200 (sm_100a). The mathematics is that of cache_attention.cu, the dealing out of work that of cache_line.cuh.
//
// With few rows the codes bound the kernel, with many the products: 4 d operations a row and token. So codes are widened to halves once for 128 rows, by
// warps of their own, into shared memory tiles that tcgen05.mma (kind::f16) reads, instead of once for every 8 or 16 rows in the registers of the
// warps that multiply. One CTA per SM, fourteen warps, stages of 64 tokens of one head against a tile of 128 rows (query token, head of the group):
//   warps 0-7   a thread per row: scores from tensor memory, running maximum, weights back as halves. Warps 0-3 take the even stages, 4-7 the odd ones, each
//               with a maximum, a sum and an output of its own (as if the tokens were cut in two); at a part's end they are added
//   warps 8-11  codes -> halves: K [token][dim] (K-major), V [token][dim] (MN-major), 128-byte swizzled slabs of 64 dims, two buffers each
//   warp 12     copies of the codes, 16 tokens a box, and the scales of their pages
//   warp 13     issues: scores of stage j + 2 ahead of the output product of stage j
// Precision: as there. An fp32 row is two halves (two K-steps for one, into the same accumulators), a bf16 row one; weights are two either way, and are held
// times 2^7; what they refer to (the maximum m, and the unit 2^(m + e) of cache_line.cuh that V's scales need) is moved when a row's own weights have grown by 2^8 (the
// accumulators are then rescaled by the row's thread), so that they stay in the halves' range either way.
// What bounds it. Two requests of 500 tokens over 6000 to 9000 cached ones, 12 heads of 64, fp32, int8: 100 us, 250 TFLOP/s of the formula's operations (twice as
// many are done). A stage takes 1.1 us; of that the tensor pipe works a quarter, and the issuing warp is busy for 1300 cycles (waits apart; one
// instruction of 64 columns costs it 70), nearly as long as a row's warp is (2500 cycles for every second stage, with two of them and a
// widening warp on each scheduler: 53 % of the issue slots, 0.8 of 3.5 warps able to issue). One request of 2000 tokens over 8000, 32 heads on 8 of 128: 485 us in bf16, 605 us in fp32.
// What it came from: row tiles on mma.sync 244 us; four row warps 152; eight, each with every second stage 133; a score's factor and the shift of its exponent in one
// operation 125; one branch around the products of a stage 114; masks and rescaling in tensor memory, without spilling the scores 108; scores two stages
// ahead 99; outputs added up every 16 stages, which all precision above 5.9e-6 needs, 106, with states that a warp reads and writes side by side 99; V's scales by what a
// row sees 100. Measured and left out: more registers for the row warps by setmaxnreg (more spills in all), segments counted as 2 or 4 stages more (the
// same, and 7 % more where CTAs have two), keys widened one stage ahead only (113).
#include "cache_line.cuh"

#include <mutex>

namespace df {
namespace {

using namespace ptx;

constexpr uint32_t kRowWarps = 8, kLoadWarp = 12, kMmaWarp = 13;  // (warps 8 to 11 widen)
constexpr uint32_t kTileRows = 128;
constexpr float kManyWeightBits = 7.0f, kRescale = 8.0f, kRescaleV = 7.0f;  // (room for the rounding of s + log2 v_scale)
constexpr uint32_t kTmemColumns = 512, kScoreColumn = 0, kWeightColumn = 128, kOutColumn = 256;  // scores 2 x 64, weights 2 x (32 + 32), outputs 2 x DP
// Stages whose output products add up in place. The tensor cores cut their sums off, they do not round them, at every step of 16 tokens: 9000 tokens one after another
// left an error of 6e-6 where fp32 sums leave 2e-6. So a row's thread adds an fp32 output up, rounded, every 16 stages (8 of its half), in tensor memory where there is room
// (heads of up to 64 dims), else in the workspace. bf16 results have 8 bits: all stages.
template <bool BF16>
constexpr uint32_t kChunk = BF16 ? 0x40000000u : 16u;
template <bool BF16, int DP>
constexpr bool kSumsOutside = !BF16 && DP == 128;

template <int DP>
struct ManyWork {
  static constexpr uint32_t kRows = kTileRows, kSegmentUnits = 8, kThreads = 448;
  static constexpr bool kDeal = false;
};
template <int DP>
constexpr uint32_t kManyPartialFloats = kTileRows * (DP + 2);
template <bool BF16, int DP>
constexpr uint32_t kManyCtaFloats = 2 * kManyPartialFloats<DP> + (kSumsOutside<BF16, DP> ? kTileRows * DP : 0);  // two states; sums of the second half

template <bool BF16, int DP>
struct ManySmem {
  static constexpr uint32_t kStages = DP == 128 ? 4 : 8, kParts = BF16 ? 1 : 2, kSlabs = DP / 64;  // kParts: of q (weights have two)
  static constexpr uint32_t kBoxBytes = 16 * DP, kStageBytes = 8 * kBoxBytes;         // codes: K boxes, V boxes
  static constexpr uint32_t kTileBytes = kSlabs * 64 * 128, kQBytes = kSlabs * 128 * 128;  // 64 tokens, 128 rows of halves
  static constexpr uint32_t kK = kStages * kStageBytes, kV = kK + 2 * kTileBytes, kQ = kV + 2 * kTileBytes;
  static constexpr uint32_t kTotal = kQ + kParts * kQBytes + 1024;
};

enum Bar { FULL = 0, EMPTY = 8, K_FULL = 16, K_FREE = 18, V_FULL = 20, PV_DONE = 22, S_FULL = 24, S_FREE = 26, P_FULL = 28, Q_FULL = 30, O_FREE = 31, DRAIN = 32, NUM_BARS = 33 };

__device__ __forceinline__ void row_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }  // the row warps; all of them come to each

template <bool BF16, int FORMAT, int DP>
__global__ void __launch_bounds__(ManyWork<DP>::kThreads, 1)
k_cache_attention_many(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const AttendParams p) {
  using W = ManyWork<DP>;
  using M = ManySmem<BF16, DP>;
  constexpr uint32_t kStages = M::kStages, kParts = M::kParts;
  extern __shared__ uint8_t smem_raw[];
  __shared__ LineSmem<W> s_sums;
  __shared__ float2 s_box_scale[kStages][4];  // k_scale, v_scale of the boxes in the ring
  __shared__ float4 s_scale[4][4];            // and of the last four stages widened, with log2 v_scale
  __shared__ uint64_t s_bars[NUM_BARS];
  __shared__ float s_top[2][kTileRows];       // largest elements of the halves of q's rows; no other use: a half without stages may be at its state already
  __shared__ float s_state[2][4][kTileRows];  // of the two halves' rows: maximum, sum, units of the output in place and of that added up before
  __shared__ Line s_line[kRowWarps];
  __shared__ Part s_part[kRowWarps];
  __shared__ uint32_t s_last, s_abort, s_tmem;
  const uint32_t t = threadIdx.x, warp = t >> 5, lane = t & 31;
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t a_smem = smem_u32(smem);
  auto bar = [&](uint32_t id) { return smem_u32(&s_bars[id]); };
  if (t == 0) {
    for (uint32_t i = 0; i < NUM_BARS; ++i) {
      const bool warps = (i >= EMPTY && i < EMPTY + 8) || i == K_FULL || i == K_FULL + 1 || i == V_FULL || i == V_FULL + 1 || i == S_FREE || i == S_FREE + 1 ||
                         i == P_FULL || i == P_FULL + 1;
      mbar_init(bar(i), i == Q_FULL || i == O_FREE ? 8 : warps ? 4 : 1);
    }
    mbar_init_fence();
    s_abort = 0;
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  pdl_wait();
  Line line;
  if (!begin_line<W>(p, s_sums, line)) return;  // its barrier also stands between the set-up and the first wait
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&s_tmem), kTmemColumns);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  const uint32_t chunks = p.D / 16;  // 16-byte pieces of a row of codes
  Part part;

  if (warp == kLoadWarp) {
    // ---------------------------------------------------------------- copies
    struct Group {
      uint32_t stages, slice, line, boxes;
      int32_t page;
      float2 scale;
    } now, then;
    const uint32_t box_bytes = 16 * p.D;
    uint32_t tile = 0, head = 0, slot = 0, phase = 1, stage = 0;
    part.t1 = 0;
    auto look_up = [&](Group &gr) {
      gr.stages = 0;
      if (tile >= part.t1) {
        do {
          if (!next_part<W>(p, line, part)) return;
        } while (part.t0 >= part.t1);
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
    bool ok = true;
    look_up(now);
    look_up_scales(now);
    while (ok && now.stages) {
      look_up(then);
      for (uint32_t s = 0; s < now.stages; ++s) {
        if (stage >= kStages && !mbar_wait_warp(bar(EMPTY + slot), phase, &s_abort)) {
          ok = false;
          break;
        }
        const bool my_turn = lane / 4 == s;
        if (my_turn) s_box_scale[slot][lane % 4] = now.scale;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bar(FULL + slot), 2 * box_bytes * __popc((now.boxes >> (4 * s)) & 15u));
        __syncwarp();
        if (my_turn && (now.boxes >> lane & 1)) {
          const uint32_t dst = a_smem + slot * M::kStageBytes + lane % 4 * M::kBoxBytes;
          tma_load_3d(dst, &k_map, bar(FULL + slot), 0, (int)now.line, (int)now.slice);
          tma_load_3d(dst + 4 * M::kBoxBytes, &v_map, bar(FULL + slot), 0, (int)now.line, (int)now.slice);
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
    if (s_abort) {  // copies in flight write to this CTA's shared memory: none may be left when it goes
      for (uint32_t s = stage > kStages ? stage - kStages : 0; s < stage; ++s)
        for (uint32_t polls = 0; polls < (1u << 16) && !mbar_try_wait(bar(FULL + s % kStages), (s / kStages) & 1); ++polls) {
        }
    }
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- products
    const uint32_t idesc_s = make_idesc(kFmtF16, 128, 64, 0, 0), idesc_o = make_idesc(kFmtF16, 128, DP, 0, 1);
    const uint64_t d_q = make_smem_desc(a_smem + M::kQ, 16, 1024, kSwz128), d_k = make_smem_desc(a_smem + M::kK, 16, 1024, kSwz128);
    const uint64_t d_v = make_smem_desc(a_smem + M::kV, 64 * 128, 1024, kSwz128);
    uint32_t stage = 0, n_part = 0;  // stages and parts with stages so far
    bool ok = true;
    auto scores = [&](uint32_t j) {
      const uint32_t b = j & 1;
      if (!mbar_wait_warp(bar(K_FULL + b), (j >> 1) & 1, &s_abort)) return false;
      if (j >= 2 && !mbar_wait_warp(bar(S_FREE + b), ((j >> 1) - 1) & 1, &s_abort)) return false;
      tc_fence_after_sync();
      if (elect_one()) {  // one election for all products of a stage: one for each cost 114 us where this takes 108
#pragma unroll
        for (uint32_t part_of_q = 0; part_of_q < kParts; ++part_of_q)
#pragma unroll
          for (uint32_t kk = 0; kk < DP / 16; ++kk) {
            const uint64_t qa = d_q + ((part_of_q * M::kQBytes + (kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4);
            const uint64_t kb = d_k + ((b * M::kTileBytes + (kk >> 2) * (64 * 128) + (kk & 3) * 32) >> 4);
            mma_f16_ss(tmem + kScoreColumn + b * 64, qa, kb, idesc_s, part_of_q > 0 || kk > 0);
          }
        mma_commit(bar(S_FULL + b));
        mma_commit(bar(K_FREE + b));
      }
      __syncwarp();
      return true;
    };
    auto output = [&](uint32_t j, uint32_t i) {  // stage j, the i-th of its part
      const uint32_t b = j & 1;
      const bool first = i % kChunk<BF16> < 2;  // of its half of a chunk
      if (!mbar_wait_warp(bar(V_FULL + b), (j >> 1) & 1, &s_abort)) return false;
      if (!mbar_wait_warp(bar(P_FULL + b), (j >> 1) & 1, &s_abort)) return false;
      if (i == 0 && n_part > 0 && !mbar_wait_warp(bar(O_FREE), (n_part - 1) & 1, &s_abort)) return false;
      tc_fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (uint32_t part_of_w = 0; part_of_w < 2; ++part_of_w)
#pragma unroll
          for (uint32_t kk = 0; kk < 4; ++kk)
            mma_f16_ts(tmem + kOutColumn + b * DP, tmem + kWeightColumn + b * 64 + part_of_w * 32 + kk * 8, d_v + ((b * M::kTileBytes + kk * 2048) >> 4), idesc_o,
                       !first || part_of_w > 0 || kk > 0);
        mma_commit(bar(PV_DONE + b));
      }
      __syncwarp();
      return true;
    };
    while (ok && next_part<W>(p, line, part)) {
      const uint32_t n = part.t1 - part.t0;
      if (n == 0) continue;
      ok = mbar_wait_warp(bar(Q_FULL), n_part & 1, &s_abort) && scores(stage) && (n == 1 || scores(stage + 1));
      for (uint32_t j = 0; ok && j < n; ++j) {
        if (j + 2 < n) ok = scores(stage + j + 2);  // before the wait for the weights of stage j: a row's next scores are there when it has written them
        ok = ok && output(stage + j, j);
      }
      stage += n;
      ++n_part;
    }
    commit_elected(bar(DRAIN));  // nothing of this CTA's may be under way when its memory goes, also where a wait has run out
    for (uint32_t polls = 0; polls < (1u << 16) && !__all_sync(0xffffffffu, mbar_try_wait(bar(DRAIN), 0)); ++polls) {
    }
  } else if (warp >= kRowWarps) {
    // ---------------------------------------------------------------- codes to halves
    const uint32_t wt = t - 32 * kRowWarps;  // 0 .. 127
    uint32_t stage = 0;
    bool ok = true;
    auto widen = [&](const uint8_t *from, uint8_t *to, uint32_t token_limit) {
#pragma unroll
      for (uint32_t i = 0; i < 64 * (DP / 16) / 128; ++i) {
        const uint32_t piece = i * 128 + wt, token = piece / (DP / 16), chunk = piece % (DP / 16);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);  // (a code of zero is zero in both formats)
        if (chunk < chunks && token < token_limit) {
          const uint32_t x = (token & 15) * chunks + chunk;
          v = *reinterpret_cast<const uint4 *>(from + (token >> 4) * M::kBoxBytes + ((x * 16) ^ ((x & 0x38u) << 1)));
        }
        uint32_t h[8];
        widen_word<FORMAT>(v.x, h[0], h[1]);
        widen_word<FORMAT>(v.y, h[2], h[3]);
        widen_word<FORMAT>(v.z, h[4], h[5]);
        widen_word<FORMAT>(v.w, h[6], h[7]);
        uint8_t *row = to + (chunk >> 2) * (64 * 128) + token * 128;
        const uint32_t at = (chunk & 3) * 2, swap = token & 7;
        *reinterpret_cast<uint4 *>(row + ((at ^ swap) * 16)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(row + (((at + 1) ^ swap) * 16)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    auto keys = [&](uint32_t j) {
      const uint32_t b = j & 1, slot = j % kStages;
      if (!mbar_wait_warp(bar(FULL + slot), (j / kStages) & 1, &s_abort)) return false;
      if (j >= 2 && !mbar_wait_warp(bar(K_FREE + b), ((j >> 1) - 1) & 1, &s_abort)) return false;
      if (wt < 4) {
        const float2 scale = s_box_scale[slot][wt];
        s_scale[j & 3][wt] = make_float4(scale.x, scale.y, scale_log(scale.y), 0.0f);
      }
      widen(smem + slot * M::kStageBytes, smem + M::kK + b * M::kTileBytes, 64);
      if (lane == 0) mbar_arrive(bar(K_FULL + b));
      return true;
    };
    auto values = [&](uint32_t j, uint32_t token_limit) {
      const uint32_t b = j & 1, slot = j % kStages;
      if (j >= 2 && !mbar_wait_warp(bar(PV_DONE + b), ((j >> 1) - 1) & 1, &s_abort)) return false;
      // what lies behind the last token that a row sees may be any bytes; its weights are 0, but an 8-bit float may be NaN
      widen(smem + slot * M::kStageBytes + 4 * M::kBoxBytes, smem + M::kV + b * M::kTileBytes, token_limit);
      if (lane == 0) {
        mbar_arrive(bar(V_FULL + b));
        mbar_arrive(bar(EMPTY + slot));
      }
      return true;
    };
    // As the products need them: the keys of a stage ahead of the values of two stages before.
    while (ok && next_part<W>(p, line, part)) {
      for (uint32_t j = 0; ok && j < 2 && part.t0 + j < part.t1; ++j) ok = keys(stage + j);
      for (uint32_t tile = part.t0; ok && tile < part.t1; ++tile, ++stage) {
        if (tile + 2 < part.t1) ok = keys(stage + 2);
        ok = ok && values(stage, part.limit - tile * kStageTokens);
      }
    }
  } else {
    // ---------------------------------------------------------------- rows
    const uint32_t b = warp >> 2, row = t & 127, lane_base = ((warp & 3) * 32) << 16;  // half (of the stages), row
    const uint32_t t_out = tmem + kOutColumn + b * DP + lane_base;
    uint32_t stage = 0;
    bool ok = true;
    // A part's description is read from shared memory where it is used: in registers it would cost the loop over its stages some.
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
      const uint32_t rr = part.row0 + row, rows = min(part.rq.rows - part.row0, kTileRows), n = found.t1 - found.t0, t0 = found.t0;
      const bool valid = row < rows, any_rows = (warp & 3) * 32 < rows;  // of this warp
      const int behind = (int)part.rq.len - (int)part.rq.q_len + 1, most_seen = (int)part.rq.len;
      auto see_of = [&](uint32_t r) { return (uint32_t)max(0, min(behind + (int)(p.group == 1 ? r : r / p.group), most_seen)); };
      auto global_row = [&](uint32_t r) {
        const uint32_t x = part.row0 + r, j = p.group == 1 ? x : x / p.group;
        return (size_t)(part.rq.first + j) * p.heads + part.h * p.group + x - j * p.group;
      };
      const uint32_t see = valid ? see_of(rr) : 0u, see_first = any_rows ? see_of(part.row0 + (warp & 3) * 32) : 0u;  // rows are in the order of their tokens
      // ---- q, scaled to 1 .. 2, as halves
      float norm = 0.0f;
      if (n > 0) {
        const uint32_t j = p.group == 1 ? rr : rr / p.group, head = part.h * p.group + rr - j * p.group;
        const unsigned long long e = (unsigned long long)(part.rq.first + j) * p.q_stride + (unsigned long long)head * p.D;
        Raw4<BF16> x[DP / 8];  // half of the row in each of its two threads
        float top = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < DP / 8; ++i) {
          const uint32_t d = b * (DP / 2) + 4 * i;
          if (valid && d < p.D) x[i].load(p.q, e + d, p.q_aligned);
          else x[i].zero();
        }
#pragma unroll
        for (uint32_t i = 0; i < DP / 8; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) top = fmaxf(top, fabsf(x[i].at(k)));
        s_top[b][row] = top;
        row_barrier();
        top = fmaxf(top, s_top[1 - b][row]);
        const uint32_t exponent = min(max(__float_as_uint(top) >> 23, 1u), 253u);
        const bool keep = top == 0.0f || top == INFINITY;
        // (the scale's sign goes into q: what multiplies a score is then not negative, and a maximum stays one)
        const float down = copysignf(keep ? 1.0f : __uint_as_float((254u - exponent) << 23), p.scale_log2);
        norm = (keep ? 1.0f : __uint_as_float(exponent << 23)) * fabsf(p.scale_log2);
#pragma unroll
        for (uint32_t i = 0; i < DP / 8; i += 2) {  // 16 bytes of halves
          uint32_t first[4], second[4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const Raw4<BF16> &y = x[i + half];
            if (BF16) {
              first[2 * half] = halves(y.at(0) * down, y.at(1) * down);
              first[2 * half + 1] = halves(y.at(2) * down, y.at(3) * down);
            } else {
              split_halves(y.at(0) * down, y.at(1) * down, first[2 * half], second[2 * half]);
              split_halves(y.at(2) * down, y.at(3) * down, first[2 * half + 1], second[2 * half + 1]);
            }
          }
          const uint32_t d = b * (DP / 2) + 4 * i;
          uint8_t *at = smem + M::kQ + (d >> 6) * (128 * 128) + row * 128 + ((((d >> 3) & 7) ^ (row & 7)) * 16);
          *reinterpret_cast<uint4 *>(at) = make_uint4(first[0], first[1], first[2], first[3]);
          if (!BF16) *reinterpret_cast<uint4 *>(at + M::kQBytes) = make_uint4(second[0], second[1], second[2], second[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(Q_FULL));
      }
      // The maximum that the weights refer to, and d and e of unit_exponent with it: the output is in units of 2^(m + e).
      float m = -FLT_MAX, l = 0.0f, excess = kLeastExcess, e = kLeastExcess;
      bool started = false, had_sum = false;  // this half has had a stage; chunks before this one
      float m_sum = -FLT_MAX, e_sum = 0.0f;   // m and e of what those add up to
      const bool split = part.parts > 1;
      auto state_of = [&](uint32_t cta) { return p.partial + (size_t)(2 * cta + (cta == part.first_cta ? 1 : 0)) * kManyPartialFloats<DP>; };
      float *mine = state_of(blockIdx.x);  // (of no other segment while this one lasts, cut or not)
      // A state's outputs lie as [dim / 4][row][4]: a warp's rows side by side. Where halves add up outside: the first in the segment's own state.
      auto at_dim = [&](float *outputs, uint32_t d) { return reinterpret_cast<float4 *>(outputs) + d / 4 * kTileRows + row; };
      auto sums_of = [&](uint32_t half) {
        return half == 0 ? mine + 2 * kTileRows : p.partial + (size_t)gridDim.x * 2 * kManyPartialFloats<DP> + (size_t)blockIdx.x * kTileRows * DP;
      };
      const uint32_t first_stage = stage;
      for (; ok && stage < first_stage + n; ++stage) {
        if ((stage & 1) != b) continue;
        const uint32_t use = stage >> 1, token0 = (t0 + stage - first_stage) * kStageTokens;
        ok = mbar_wait_warp(bar(S_FULL + b), use & 1, &s_abort);
        if (!ok) break;
        if (!any_rows) {  // whatever these lanes' weights are, nobody reads their outputs
          if (lane == 0) mbar_arrive(bar(S_FREE + b));
          if (stage >= 2) {
            ok = mbar_wait_warp(bar(PV_DONE + b), (use - 1) & 1, &s_abort);
            if (!ok) break;
          }
          if (lane == 0) mbar_arrive(bar(P_FULL + b));
          started = true;
          continue;
        }
        tc_fence_after_sync();
        const int seen = (int)see - (int)token0;  // of this stage's tokens (0 or less: none)
        if (token0 + 64 > see_first) {            // masked where they lie: beside all 64 in registers there is no room for it
#pragma unroll 1
          for (int c = 0; c < 64; c += 16) {
            uint32_t x[16];
            tmem_ld16(tmem + kScoreColumn + b * 64 + c + lane_base, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (c + k >= seen) x[k] = 0xff800000u;  // -inf
            tmem_st16(tmem + kScoreColumn + b * 64 + c + lane_base, x);
          }
          tmem_wait_st();
        }
        uint32_t s[64];
        {
          uint32_t (&s0)[32] = *reinterpret_cast<uint32_t (*)[32]>(&s[0]), (&s1)[32] = *reinterpret_cast<uint32_t (*)[32]>(&s[32]);
          tmem_ld32(tmem + kScoreColumn + b * 64 + lane_base, s0);
          tmem_ld32(tmem + kScoreColumn + b * 64 + 32 + lane_base, s1);
          tmem_wait_ld();
        }
        float v_scale[4], f[4], v_log[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 scale = s_scale[stage & 3][i];
          f[i] = scale.x * norm;
          v_scale[i] = scale.y;
          v_log[i] = scale.z;
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S_FREE + b));  // scores and scales are in registers
        float top = -INFINITY, top_v = -INFINITY;  // of the scores, and with log2 v_scale
        // f: what a box's scores are multiplied by; above 0 (or NaN, for rows that see the box), so that -inf stays -inf
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (f[i] < 0x1p-120f || 16 * i >= seen) f[i] = 0x1p-120f;
          float most[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            most[k] = fmaxf(fmaxf(__uint_as_float(s[16 * i + 4 * k]), __uint_as_float(s[16 * i + 4 * k + 1])),
                            fmaxf(__uint_as_float(s[16 * i + 4 * k + 2]), __uint_as_float(s[16 * i + 4 * k + 3])));
          const float top_i = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * f[i];
          top = fmaxf(top, top_i);
          top_v = fmaxf(top_v, top_i + v_log[i]);
        }
        // the product of two stages ago has read the weights' buffer and written this half's output
        if (stage >= 2) {
          ok = mbar_wait_warp(bar(PV_DONE + b), (use - 1) & 1, &s_abort);
          if (!ok) break;
          tc_fence_after_sync();
        }
        const bool fresh = started && (stage - first_stage) % kChunk<BF16> < 2;  // a chunk's first of this half: what is there is added up
        const bool add_sum = had_sum;
        const float factor = ex2_approx((m_sum - m) + (e_sum - e));
        if (fresh) {
          m_sum = m;
          e_sum = e;
          had_sum = true;
        }
        const bool grow_m = top > m + kRescale, grow = grow_m || top_v - m > e + kRescaleV;  // (also the first that a row sees)
        const bool rescale = started && !fresh && __any_sync(0xffffffffu, grow);
        float down_out = 1.0f;
        if (grow || fresh || !started) {  // (a row for itself: what others see changes nothing of it)
          const float to = grow_m || fresh || !started ? fmaxf(m, top) : m, before = e;  // (V has no part in the sum of the weights)
          excess = fmaxf(excess + (m - to), top_v - to);
          e = unit_exponent(excess);
          down_out = ex2_approx((m - to) + (before - e));
          l *= ex2_approx(m - to);
          m = to;
        }
        started = true;
        const float minus_shift = kManyWeightBits - m, units = ex2_approx(-e);
        float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // 32 tokens at a time: fewer registers
          uint32_t first[16], second[16];
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            const int i = 2 * half + x / 16;
            const float share = 16 * i < seen ? share_of(v_scale[i], units) : 0.0f;  // a row takes nothing of a box that it sees nothing of
            float2 w = fma2(as_float2(s[32 * half + x], s[32 * half + x + 1]), make_float2(f[i], f[i]), make_float2(minus_shift, minus_shift));
            w = make_float2(ex2_approx(w.x), ex2_approx(w.y));
            sums[x / 2 & 1] = add2(sums[x / 2 & 1], w);
            w = mul2(w, make_float2(share, share));
            split_halves(w.x, w.y, first[x / 2], second[x / 2]);
          }
          tmem_st16(tmem + kWeightColumn + b * 64 + 16 * half + lane_base, first);
          tmem_st16(tmem + kWeightColumn + b * 64 + 32 + 16 * half + lane_base, second);
        }
        sums[0] = add2(sums[0], sums[1]);
        l += sums[0].x + sums[0].y;
        if (!BF16 && fresh) {
          float *outside = sums_of(b);
#pragma unroll 1
          for (uint32_t d = 0; d < DP; d += 16) {
            uint32_t o[16];
            tmem_ld16(t_out + d, o);
            if (kSumsOutside<BF16, DP>) {
              float4 *at = at_dim(outside, d);
              float4 before[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) before[x] = add_sum ? at[x * kTileRows] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 4; ++x)
                at[x * kTileRows] = make_float4(fmaf(before[x].x, factor, __uint_as_float(o[4 * x])), fmaf(before[x].y, factor, __uint_as_float(o[4 * x + 1])),
                                    fmaf(before[x].z, factor, __uint_as_float(o[4 * x + 2])), fmaf(before[x].w, factor, __uint_as_float(o[4 * x + 3])));
            } else {
              uint32_t before[16];
              if (add_sum) tmem_ld16(t_out + 2 * DP + d, before);
              tmem_wait_ld();
              if (add_sum) {
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(fmaf(__uint_as_float(before[x]), factor, __uint_as_float(o[x])));
              }
              tmem_st16(t_out + 2 * DP + d, o);
            }
          }
        }
        if (rescale) {
#pragma unroll 1
          for (uint32_t d = 0; d < DP; d += 16) {
            uint32_t o[16];
            tmem_ld16(t_out + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * down_out);
            tmem_st16(t_out + d, o);
          }
        }
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL + b));
      }
      stage = first_stage + n;
      // ---- results: this half's last product, then the other's by the barrier
      if (started && ok) {
        const uint32_t last = stage - 1 - ((stage - 1 - b) & 1);
        ok = mbar_wait_warp(bar(PV_DONE + b), (last >> 1) & 1, &s_abort);
      }
      s_state[b][0][row] = m;
      s_state[b][1][row] = l;
      s_state[b][2][row] = started && ok ? ex2_approx(e) : -1.0f;  // below 0: there is no output
      s_state[b][3][row] = had_sum ? ex2_approx((m_sum - m) + e_sum) : -1.0f;
      tc_fence_before_sync();
      row_barrier();
      tc_fence_after_sync();
      const float m_all = fmaxf(s_state[0][0][row], s_state[1][0][row]);
      const float w0 = ex2_approx(s_state[0][0][row] - m_all), w1 = ex2_approx(s_state[1][0][row] - m_all);
      const float l_all = s_state[0][1][row] * w0 + s_state[1][1][row] * w1, u0 = s_state[0][2][row], u1 = s_state[1][2][row];
      const float g0 = s_state[0][3][row], g1 = s_state[1][3][row];
      const bool has0 = !(u0 < 0.0f), has1 = !(u1 < 0.0f), sum0 = !BF16 && !(g0 < 0.0f), sum1 = !BF16 && !(g1 < 0.0f);  // the same in all rows
      const size_t out_row = valid ? global_row(row) : 0;
#pragma unroll 1
      for (uint32_t d = b * (DP / 2); d < (b + 1) * (DP / 2); d += 16) {  // half of the dims each
        float y[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) y[x] = 0.0f;
        auto add = [&](uint32_t column, float f) {
          uint32_t o[16];
          tmem_ld16(tmem + column + d + lane_base, o);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 16; ++x) y[x] = fmaf(__uint_as_float(o[x]), f, y[x]);
        };
        auto add_outside = [&](float *sums, float f) {
#pragma unroll
          for (int x = 0; x < 16; x += 4) {
            const float4 o = *at_dim(sums, d + x);
            y[x] = fmaf(o.x, f, y[x]);
            y[x + 1] = fmaf(o.y, f, y[x + 1]);
            y[x + 2] = fmaf(o.z, f, y[x + 2]);
            y[x + 3] = fmaf(o.w, f, y[x + 3]);
          }
        };
        if (has0) add(kOutColumn, w0 * u0);
        if (has1) add(kOutColumn + DP, w1 * u1);
        if (kSumsOutside<BF16, DP>) {
          if (sum0) add_outside(sums_of(0), w0 * g0);
          if (sum1) add_outside(sums_of(1), w1 * g1);
        } else {
          if (sum0) add(kOutColumn + 2 * DP, w0 * g0);
          if (sum1) add(kOutColumn + 3 * DP, w1 * g1);
        }
        if (valid) {
#pragma unroll
          for (int x = 0; x < 16; x += 4) {
            const float4 v = make_float4(y[x], y[x + 1], y[x + 2], y[x + 3]);
            if (split) *at_dim(mine + 2 * kTileRows, d + x) = v;
            else finish_row4<BF16>(p, out_row, d + x, v, m_all, l_all, kManyWeightBits);
          }
        }
        __syncwarp();
      }
      if (n > 0) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(O_FREE));
      }
      if (split) {
        if (valid && b == 0) *reinterpret_cast<float2 *>(mine + 2 * row) = make_float2(m_all, l_all);
        row_barrier();
        if (t == 0) {  // releases what the barrier has gathered, and acquires what the CTAs before have released
          unsigned int arrived;
          asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(arrived) : "l"(p.counters + part.first_cta) : "memory");
          s_last = arrived + 1 == part.parts;
          if (s_last) p.counters[part.first_cta] = 0;  // ready for the next call
        }
        row_barrier();
        if (s_last) {
          constexpr uint32_t kAtOnce = 4, kPieces = DP / 4;
          for (uint32_t e = t; e < rows * kPieces; e += 32 * kRowWarps * kAtOnce) {
            Running sum[kAtOnce];
            for (uint32_t i = 0; i < part.parts; ++i) {
              const float *state = state_of(part.first_cta + i);
              float2 ml[kAtOnce];
              float4 o[kAtOnce];
#pragma unroll
              for (uint32_t k = 0; k < kAtOnce; ++k) {
                const uint32_t at = min(e + k * 32 * kRowWarps, rows * kPieces - 1), piece = at / rows, r = at - piece * rows;
                ml[k] = __ldcg(reinterpret_cast<const float2 *>(state + 2 * r));
                o[k] = __ldcg(reinterpret_cast<const float4 *>(state + 2 * kTileRows) + piece * kTileRows + r);
              }
#pragma unroll
              for (uint32_t k = 0; k < kAtOnce; ++k) sum[k].add(ml[k].x, ml[k].y, o[k]);
            }
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
              const uint32_t at = e + k * 32 * kRowWarps, piece = at / rows, r = at - piece * rows;
              if (piece < kPieces)
                finish_row4<BF16>(p, global_row(r), piece * 4, make_float4(sum[k].o[0], sum[k].o[1], sum[k].o[2], sum[k].o[3]), sum[k].m, sum[k].l,
                                  kManyWeightBits);
            }
          }
        }
      }
      row_barrier();  // s_last, s_top and s_state are free again
    }
  }
  // ---- teardown: every role comes here, also when a wait has run out
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (t == 0 && s_abort && p.status) atomicOr(p.status, DEV_STATUS_WAIT_EXPIRED);
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemColumns);
}

struct DeviceInfo {
  std::once_flag once;
  uint32_t grid = 0;
};

template <bool BF16, int FORMAT, int DP>
int launch(AttendParams &p, const void *k_cache, const void *v_cache, cudaStream_t s) {
  static DeviceInfo table[64];
  constexpr uint32_t smem = ManySmem<BF16, DP>::kTotal;
  constexpr uint32_t kFits = (DF_CACHE_WORKSPACE_BYTES - kCounterBytes) / (kManyCtaFloats<BF16, DP> * 4);
  static_assert(kFits >= 160, "workspace");
  auto kernel = k_cache_attention_many<BF16, FORMAT, DP>;
  int dev = 0;
  if (check_cuda(cudaGetDevice(&dev)) != DF_OK || dev < 0 || dev >= 64) return DF_ERR_CUDA;
  DeviceInfo &d = table[dev];
  std::call_once(d.once, [&]() {
    int n_sm = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess &&
        cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
      d.grid = n_sm < (int)kFits ? (uint32_t)n_sm : kFits;
  });
  if (d.grid == 0) return DF_ERR_CUDA;
  CUtensorMap k_map, v_map;
  if (!encode_pool_map(&k_map, k_cache, p) || !encode_pool_map(&v_map, v_cache, p)) return DF_ERR_CUDA;
  const int st = check_cuda(launch_kernel(kernel, dim3(d.grid), dim3(ManyWork<DP>::kThreads), smem, s, k_map, v_map, p));
  note_launch();
  return st;
}

template <bool BF16, int FORMAT>
int launch_for_head(AttendParams &p, const void *k_cache, const void *v_cache, cudaStream_t s) {
  return p.D <= 64 ? launch<BF16, FORMAT, 64>(p, k_cache, v_cache, s) : launch<BF16, FORMAT, 128>(p, k_cache, v_cache, s);
}

}  // namespace

int cache_attention_many(AttendParams &p, const void *k_cache, const void *v_cache, bool bf16, uint32_t format, cudaStream_t s) {
  if (bf16)
    return format == DF_CACHE_INT8 ? launch_for_head<true, DF_CACHE_INT8>(p, k_cache, v_cache, s) : launch_for_head<true, DF_CACHE_E4M3>(p, k_cache, v_cache, s);
  return format == DF_CACHE_INT8 ? launch_for_head<false, DF_CACHE_INT8>(p, k_cache, v_cache, s) : launch_for_head<false, DF_CACHE_E4M3>(p, k_cache, v_cache, s);
}

}  // namespace df
