// product_sm100.cuh — batched matrix products of 16-bit operands on tcgen05 with an epilogue of the caller's:
//   acc[m][n] = sum_k A[m][k] B[n][k]
// Operands lie in global memory with either side contiguous (K-major: rows of k; MN-major: rows of m or n), bf16 or fp16. With
// PARTS = 2 a value is two fp16 numbers, hi = fp16(s x) and lo = fp16(2^11 (s x - hi)) for a power of two s that the caller undoes: 22 bits
// where |x| is within 2^27 of the largest that s was chosen for (2^14 .. 2^15 after it), and nothing below 2^-50 of that one: without the 2^11, lo would leave fp16 that much earlier,
// and a probability of 1e-9 among ones near 1 would have 9 bits. Then
//   A B = 2^-11 (A_lo B_hi + A_hi B_lo) + A_hi B_hi      (A_lo B_lo, 2^-22 of it at most, is left out)
// is three products in that order: the tensor cores cut sums off instead of rounding them, and a large sum is cut off at each of its
// additions, so the small terms come first (the first large one scales their sum down by 2^11 as it adds to it) and every 128 of the contraction the sum is taken out to registers and added up rounded. (More often costs time: a
// tile's sums are 128 KB a CTA, which tensor memory gives out in about 2000 cycles, and 64 of the contraction are 1536 cycles of products.)
//
// One persistent kernel, at most one CTA an SM, 384 threads:
//   warp 0       copies: a ring of slots, each 64 of the contraction: 128 rows of A and this CTA's rows of B (PARTS = 2: of the low parts, of the high parts, in
//                turn), 128-byte swizzle;
//   warp 1       issues the products into one of two accumulators in tensor memory;
//   warps 4-11   the epilogue of one tile under the products of the next: a warp has the 32 rows of its quarter of tensor memory, a row
//                a lane, and half of the tile's columns, 32 at a time. With PARTS = 2 its sums are 128 registers a thread, which it takes over from warps 0-3.
// The tile is 256 x 256 over a pair of CTAs (cta_group::2: 32 KB a CTA and part for 512 cycles of products), or 128 x 128 of one.
// Tiles that run at the same time share the operand with the more rows (K-major B: the output weight, by the tiles of all rows; MN-major B: the gradient of the
// logits, by the tiles of the width): it is read from HBM once.
// The contraction can be split: tile z * tiles + t is slice z of tile t, and the epilogue is told z.
#pragma once

#include <cuda_fp16.h>
#include <math.h>

#include <atomic>

#include "df_common.cuh"
#include "sm100_ptx.cuh"

namespace df {

struct ProductParams {
  uint32_t M, N;
  int m_tiles, n_tiles;     // tiles of this form along M and N
  int splits;
  int n_kb, kb_per_split;   // blocks of 64 of the contraction: all, and of one slice
  long long tiles;
  uint32_t fmt;             // kFmtF16 or kFmtBF16
  unsigned int *status;
};

// One tile's place, as the epilogue sees it.
struct ProductTile {
  int m_tile, n_tile, split;
};

constexpr int kProdEpiWarps = 8, kProdThreads = 384, kProdK = 64;
constexpr int kProdChunk = 2;  // products of parts: blocks of 64 between takings out of the sums
constexpr int kProdLowUp = 11;  // low parts are held times 2^11
constexpr uint32_t kProdSlabBytes = 32 * 128;  // a warp's staging slab: 32 rows of 128 bytes
// Sums in registers: the launch gives 168 registers to each thread of three warpgroups; the two of the epilogue take over 48 from each thread of the first.
constexpr int kProdLaunchRegs = 168, kProdEpiRegs = 216, kProdOtherRegs = 72;
static_assert(2 * kProdEpiRegs + kProdOtherRegs <= 3 * kProdLaunchRegs, "setmaxnreg waits for registers that the block was not launched with");
template <int N> __device__ __forceinline__ void prod_regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void prod_regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// The waits of sm100_ptx.cuh with their polling loop in place: a kernel that moves registers between its warps cannot be compiled with calls.
__device__ __forceinline__ bool prod_wait(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag) {
  using namespace ptx;
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
#pragma unroll 1
  for (uint32_t polls = 1; polls < kWaitMaxPolls; ++polls) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((polls & 255u) == 0u && (*abort_flag != 0u || global_timer_ns() - t0 > kWaitBudgetNs)) break;
  }
  *abort_flag = 1u;
  return false;
}
__device__ __forceinline__ bool prod_wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag) {
  using namespace ptx;
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, prod_wait(bar, parity, abort_flag)) != 0;
}

// PAIR: tiles of 256 x 256 over two CTAs, else 128 x 128 of one: twice the operands' bytes for the same products, but a quarter of the tile, and with half the sums a
// thread four accumulators, so that results are written under the next tile's products.
template <bool PAIR_, bool A_MN_, bool B_MN_, int PARTS_>
struct ProdCfg {
  static constexpr bool PAIR = PAIR_, A_MN = A_MN_, B_MN = B_MN_;
  static constexpr int PARTS = PARTS_, kCtas = PAIR ? 2 : 1, T = PAIR ? 256 : 128;
  static constexpr bool kSums = PARTS == 2;  // sums in registers
  static constexpr int kChunk = kSums ? kProdChunk : 0x40000000;
  static constexpr uint32_t kTileBytes = 128 * kProdK * 2, kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = 6;
  static constexpr uint32_t kSmemStaging = kStages * kStageBytes;
  static constexpr uint32_t kSmemBars = kSmemStaging + kProdEpiWarps * kProdSlabBytes;
  static constexpr uint32_t kSmemTotal = kSmemBars + 256 + 1024;
  static constexpr int kAccs = 512 / T;
  static constexpr int FULL = 0, EMPTY = FULL + kStages, ACC_FULL = EMPTY + kStages, ACC_EMPTY = ACC_FULL + kAccs, DRAIN = ACC_EMPTY + kAccs, NUM_BARS = DRAIN + 1;
  static_assert(NUM_BARS * 8 <= 192 && kSmemTotal <= 227 * 1024, "shared memory");
};

// Epi: struct Params; begin(tile, row, col0) for this lane's row and the first of this warp's TN / 2 columns; block(cg, v): columns
// col0 + 32 cg ..; end(). All of it warp-uniform in control flow apart from guarded accesses to memory.
template <class C, class Epi>
__global__ void __launch_bounds__(kProdThreads, 1)
k_product(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA_lo, const __grid_constant__ CUtensorMap tmB,
          const __grid_constant__ CUtensorMap tmB_lo, const __grid_constant__ ProductParams p, const __grid_constant__ typename Epi::Params e) {
  using namespace ptx;
  constexpr int kStages = C::kStages, T = C::T;
  constexpr bool PAIR = C::PAIR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t a0 = smem_u32(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kSmemBars);
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + C::kSmemBars + 192);
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(smem + C::kSmemBars + 196);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  auto bar = [&](int id) { return smem_u32(&bars[id]); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::NUM_BARS; ++i) mbar_init(bar(i), i >= C::ACC_EMPTY && i < C::DRAIN ? C::kCtas * kProdEpiWarps : 1);
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_holder), 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_holder), 512);
      tmem_relinquish();
    }
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  tc_fence_before_sync();
  if (PAIR) cluster_sync();
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();
  const long long first_tile = blockIdx.x / C::kCtas, tile_step = gridDim.x / C::kCtas;

  auto decode = [&](long long id, int *kb0, int *kb1) {
    ProductTile t;
    const int per_split = p.m_tiles * p.n_tiles, r = (int)(id % per_split);
    t.split = (int)(id / per_split);
    t.m_tile = C::B_MN ? r / p.n_tiles : r % p.m_tiles;
    t.n_tile = C::B_MN ? r % p.n_tiles : r / p.m_tiles;
    *kb0 = t.split * p.kb_per_split;
    *kb1 = *kb0 + p.kb_per_split < p.n_kb ? *kb0 + p.kb_per_split : p.n_kb;
    return t;
  };

  if (warp < 4) {
    if constexpr (C::kSums) prod_regs_less<kProdOtherRegs>();
    if (warp == 0) {
      // ---------------------------------------------------------- copies: each CTA its own rows
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (long long id = first_tile; ok && id < p.tiles; id += tile_step) {
          int kb0, kb1;
          const ProductTile t = decode(id, &kb0, &kb1);
          const int row_a = t.m_tile * T + (int)rank * 128, row_b = t.n_tile * T + (int)rank * 128;
          for (int kb = kb0; ok && kb < kb1; ++kb) {
#pragma unroll
            for (int lo = C::PARTS - 1; lo >= 0; --lo, ++it) {
              const uint32_t s = it % kStages, use = it / kStages;
              if (use > 0 && !prod_wait(bar(C::EMPTY + s), (use - 1) & 1, abort_flag)) { ok = false; break; }
              const uint32_t sa = a0 + s * C::kStageBytes;
              // in a pair both CTAs' copies count on the even CTA's barrier, which expects the bytes of both
              const uint32_t full = PAIR ? map_to_rank(bar(C::FULL + s), 0) : bar(C::FULL + s);
              if (rank == 0) mbar_arrive_expect_tx(bar(C::FULL + s), C::kCtas * C::kStageBytes);
              auto copy = [&](uint32_t dst, const CUtensorMap *m, int x, int y) {
                if (PAIR) tma_load_2d_pair(dst, m, full, x, y);
                else tma_load_2d(dst, m, full, x, y);
              };
              auto load = [&](uint32_t dst, const CUtensorMap *m, bool mn, int row) {
                if (mn) {
                  copy(dst, m, row, kb * kProdK);
                  copy(dst + 8192, m, row + 64, kb * kProdK);
                } else {
                  copy(dst, m, kb * kProdK, row);
                }
              };
              load(sa, lo ? &tmA_lo : &tmA, C::A_MN, row_a);
              load(sa + C::kTileBytes, lo ? &tmB_lo : &tmB, C::B_MN, row_b);
            }
          }
        }
      }
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- products: in a pair the even CTA issues for both
      const uint32_t idesc = make_idesc(p.fmt, T, T, C::A_MN ? 1 : 0, C::B_MN ? 1 : 0);
      uint32_t it = 0, j = 0;
      bool ok = true;
      // K-major: 16 of k are 32 bytes of a swizzled row; MN-major: 16 rows of 128 bytes, the next 64 of m or n 8192 bytes on
      // fresh: the sum begins; down: it holds the small terms, 2^11 too large
      auto issue = [&](uint32_t d, uint32_t sa, uint32_t sb, bool fresh, bool down = false) {
        const uint64_t da = make_smem_desc(sa, C::A_MN ? 8192 : 16, 1024, kSwz128), db = make_smem_desc(sb, C::B_MN ? 8192 : 16, 1024, kSwz128);
#pragma unroll
        for (int k = 0; k < kProdK / 16; ++k) {
          const uint64_t oa = (uint64_t)((k * (C::A_MN ? 2048 : 32)) >> 4), ob = (uint64_t)((k * (C::B_MN ? 2048 : 32)) >> 4);
          if (C::PARTS == 2 && down && k == 0) mma_f16_ss_down<kProdLowUp, PAIR>(d, da, db, idesc);
          else if (PAIR) mma_f16_ss_pair(d, da + oa, db + ob, idesc, fresh && k == 0 ? 0u : 1u);
          else mma_f16_ss(d, da + oa, db + ob, idesc, fresh && k == 0 ? 0u : 1u);
        }
      };
      auto commit = [&](int id) {
        if (PAIR) mma_commit_pair(bar(id));
        else mma_commit(bar(id));
      };
      for (long long id = first_tile; ok && id < p.tiles; id += tile_step) {
        int kb0, kb1;
        decode(id, &kb0, &kb1);
        for (int kb = kb0; ok && kb < kb1;) {
          const uint32_t acc = j % C::kAccs, d = tmem + acc * T;
          const int n = kb1 - kb < C::kChunk ? kb1 - kb : C::kChunk;
          if (j >= C::kAccs && !prod_wait_warp(bar(C::ACC_EMPTY + acc), (j / C::kAccs - 1) & 1, abort_flag)) { ok = false; break; }
          if constexpr (C::PARTS == 2) {
            // the small terms of the chunk's blocks, then the large ones
            for (int i = 0; ok && i < n; ++i) {
              const uint32_t t = it + 2 * i, s_lo = t % kStages, s_hi = (t + 1) % kStages;
              if (!prod_wait_warp(bar(C::FULL + s_lo), (t / kStages) & 1, abort_flag) ||
                  !prod_wait_warp(bar(C::FULL + s_hi), ((t + 1) / kStages) & 1, abort_flag)) { ok = false; break; }
              tc_fence_after_sync();
              if (elect_one()) {
                const uint32_t lo = a0 + s_lo * C::kStageBytes, hi = a0 + s_hi * C::kStageBytes;
                issue(d, lo, hi + C::kTileBytes, i == 0);
                issue(d, hi, lo + C::kTileBytes, false);
                commit(C::EMPTY + s_lo);
              }
              __syncwarp();
            }
            if (ok && elect_one()) {
              for (int i = 0; i < n; ++i) {
                const uint32_t s_hi = (it + 2 * i + 1) % kStages, hi = a0 + s_hi * C::kStageBytes;
                issue(d, hi, hi + C::kTileBytes, false, i == 0);
                commit(C::EMPTY + s_hi);
              }
              commit(C::ACC_FULL + acc);
            }
            __syncwarp();
            it += 2 * n;
          } else {
            for (int i = 0; i < n; ++i, ++it) {
              const uint32_t s = it % kStages, sa = a0 + s * C::kStageBytes;
              if (!prod_wait_warp(bar(C::FULL + s), (it / kStages) & 1, abort_flag)) { ok = false; break; }
              tc_fence_after_sync();
              if (elect_one()) {
                issue(d, sa, sa + C::kTileBytes, i == 0);
                commit(C::EMPTY + s);
                if (i + 1 == n) commit(C::ACC_FULL + acc);
              }
              __syncwarp();
            }
          }
          kb += n;
          ++j;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    if constexpr (C::kSums) prod_regs_more<kProdEpiRegs>();
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    constexpr int kGroups = T / 64;  // 32-column blocks of this warp
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + half * (T / 2);
    Epi epi(e, smem + C::kSmemStaging + (warp - 4) * kProdSlabBytes, lane);
    auto release = [&](uint32_t acc) {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(map_to_rank(bar(C::ACC_EMPTY + acc), 0));
        else mbar_arrive(bar(C::ACC_EMPTY + acc));
      }
    };
    uint32_t j = 0;
    bool ok = true;
    for (long long id = first_tile; ok && id < p.tiles; id += tile_step) {
      int kb0, kb1;
      const ProductTile t = decode(id, &kb0, &kb1);
      const uint32_t row = (uint32_t)(t.m_tile * T + (int)rank * 128 + quarter * 32 + lane), col0 = (uint32_t)(t.n_tile * T + half * (T / 2));
      epi.begin(t, row, col0);
      if constexpr (!C::kSums) {
        const uint32_t acc = j % C::kAccs;
        if (!prod_wait_warp(bar(C::ACC_FULL + acc), (j / C::kAccs) & 1, abort_flag)) break;
        tc_fence_after_sync();
#pragma unroll 1
        for (int cg = 0; cg < kGroups; ++cg) {
          uint32_t r[32];
          tmem_ld32(lane_base + acc * T + cg * 32, r);
          tmem_wait_ld();
          if (cg == kGroups - 1) release(acc);
          float v[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(r[x]);
          epi.block(cg, v);
        }
        ++j;
      } else {
        float sum[kGroups][32];
#pragma unroll
        for (int cg = 0; cg < kGroups; ++cg)
#pragma unroll
          for (int x = 0; x < 32; ++x) sum[cg][x] = 0.0f;
#pragma unroll 1
        for (int kb = kb0; kb < kb1; kb += C::kChunk, ++j) {
          const uint32_t acc = j % C::kAccs;
          if (!prod_wait_warp(bar(C::ACC_FULL + acc), (j / C::kAccs) & 1, abort_flag)) { ok = false; break; }
          tc_fence_after_sync();
#pragma unroll
          for (int cg = 0; cg < kGroups; ++cg) {
            uint32_t r[32];
            tmem_ld32(lane_base + acc * T + cg * 32, r);
            tmem_wait_ld();
            if (cg == kGroups - 1) release(acc);
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const float2 q = add2(make_float2(sum[cg][x], sum[cg][x + 1]), as_float2(r[x], r[x + 1]));
              sum[cg][x] = q.x;
              sum[cg][x + 1] = q.y;
            }
          }
        }
        if (!ok) break;
#pragma unroll
        for (int cg = 0; cg < kGroups; ++cg) epi.block(cg, sum[cg]);
      }
      epi.end();
    }
  }

  // ---------------------------------------------------------------- teardown (all roles), as in linear_sm100.cu
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {
    if (warp == 1 && rank == 0) {
      if (elect_one()) {
        if (PAIR) mma_commit_pair(bar(C::DRAIN));
        else mma_commit(bar(C::DRAIN));
      }
      __syncwarp();
      for (int n = 0; n < (1 << 16) && !mbar_try_wait(bar(C::DRAIN), 0); ++n) {
      }
    }
    if (warp == 0 && lane == 0) {
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 2000000ull) {
      }
    }
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, DEV_STATUS_WAIT_EXPIRED);
    __syncthreads();
  }
  if (PAIR) cluster_sync();
  if (warp == 1) {
    tc_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// Two values as two fp16 parts each, packed: hi and lo of (x, y), lo times 2^UP.
template <int UP>
__device__ __forceinline__ void split_half2(float x, float y, uint32_t &hi, uint32_t &lo) {
  constexpr float up = (float)(1 << UP);
  const __half2 h = __floats2half2_rn(x, y);
  const float2 back = __half22float2(h);
  const __half2 l = __floats2half2_rn((x - back.x) * up, (y - back.y) * up);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ uint32_t pack_half2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// The power of two that brings the largest magnitude (as the bits of a float, 0 where there is none) to 2^14 .. 2^15, and its inverse.
__device__ __forceinline__ float part_scale(uint32_t largest_bits, float *inverse) {
  const int exponent = (int)(largest_bits >> 23) - 127;
  int shift = largest_bits == 0u ? 0 : 14 - exponent;
  shift = shift > 126 ? 126 : shift;
  *inverse = __uint_as_float((uint32_t)(127 - shift) << 23);
  return __uint_as_float((uint32_t)(127 + shift) << 23);
}

// Turns a warp's 32 x 32 block over in its slab: a lane comes with the values of its row and leaves with 16-byte chunk lane % 8 of rows
// 4 i + lane / 8, i = 0 .. 7, so that memory moves in whole 128-byte lines.
__device__ __forceinline__ void turn_over(float4 *slab, int lane, const float (&v)[32], float4 (&out)[8]) {
  __syncwarp();
#pragma unroll
  for (int x = 0; x < 8; ++x) slab[lane * 8 + (x ^ (lane & 7))] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
  __syncwarp();
  const int lrow = lane >> 3, chunk = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = slab[(4 * i + lrow) * 8 + (chunk ^ ((4 * i + lrow) & 7))];
}

// ---------------------------------------------------------------- host
// A 16-bit matrix [rows][cols] (row pitch in elements, a multiple of 8) as an operand: K-major boxes are 64 columns x 128 rows, MN-major ones
// 64 x 64. Outside of it a copy gives zeros.
inline bool operand_map(CUtensorMap *m, const void *base, bool bf16, uint64_t rows, uint64_t cols, uint64_t pitch, bool mn_major) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {pitch * 2};
  const cuuint32_t box[2] = {64, mn_major ? 64u : 128u};
  const cuuint32_t estr[2] = {1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// An operand as the launcher needs it: its parts (lo only with two).
struct Operand {
  const void *hi, *lo;
  bool bf16;
  uint64_t rows, cols, pitch;
};

// How many clusters of a kernel run at once on the current device, its attributes set; asked for once per kernel and device. 0: it cannot be launched
// (a build with other register counts than its hand-over of registers needs would wait for ever).
template <auto Kernel>
int cluster_slots(uint32_t ctas, uint32_t smem, int regs) {
  static std::atomic<int> slots_of[64];
  int dev = 0;
  if (check_cuda(cudaGetDevice(&dev)) != DF_OK || dev < 0 || dev >= 64) return 0;
  int slots = slots_of[dev].load(std::memory_order_acquire);
  if (slots != 0) return slots;
  cudaFuncAttributes have;
  if (check_cuda(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != DF_OK ||
      check_cuda(cudaFuncGetAttributes(&have, Kernel)) != DF_OK || (regs != 0 && have.numRegs != regs))
    return 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(64 * ctas);
  cfg.blockDim = dim3(kProdThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (check_cuda(cudaOccupancyMaxActiveClusters(&slots, Kernel, &cfg)) != DF_OK || slots <= 0) return 0;
  slots_of[dev].store(slots, std::memory_order_release);
  return slots;
}

template <class C, class Epi>
int launch_product(const Operand &a, const Operand &b, ProductParams p, const typename Epi::Params &e, cudaStream_t s) {
  static_assert(sizeof(ProductParams) + sizeof(typename Epi::Params) + 4 * sizeof(CUtensorMap) < 4000, "kernel parameters");
  const int slots = cluster_slots<k_product<C, Epi>>(C::kCtas, C::kSmemTotal, C::kSums ? kProdLaunchRegs : 0);
  if (slots == 0) return DF_ERR_CUDA;
  p.m_tiles = (int)((p.M + C::T - 1) / C::T);
  p.n_tiles = (int)((p.N + C::T - 1) / C::T);
  p.tiles = (long long)p.m_tiles * p.n_tiles * p.splits;
  p.status = device_status_ptr();
  CUtensorMap ma, ma_lo, mb, mb_lo;
  bool ok = operand_map(&ma, a.hi, a.bf16, a.rows, a.cols, a.pitch, C::A_MN) && operand_map(&mb, b.hi, b.bf16, b.rows, b.cols, b.pitch, C::B_MN);
  ma_lo = ma;
  mb_lo = mb;
  if (C::PARTS == 2) ok = ok && operand_map(&ma_lo, a.lo, a.bf16, a.rows, a.cols, a.pitch, C::A_MN) && operand_map(&mb_lo, b.lo, b.bf16, b.rows, b.cols, b.pitch, C::B_MN);
  if (!ok) {
    note_status(DF_ERR_CUDA);
    return DF_ERR_CUDA;
  }
  const long long grid = (p.tiles < slots ? p.tiles : slots) * C::kCtas;
  const int st = check_cuda(launch_clusters(k_product<C, Epi>, C::PAIR ? 2 : 0, dim3((unsigned)grid), dim3(kProdThreads), C::kSmemTotal, s, ma, ma_lo, mb, mb_lo, p, e));
  note_launch();
  return st;
}

}  // namespace df
