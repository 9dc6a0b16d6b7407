// muon.cu — matrices orthogonalised by Newton-Schulz products, and the optimiser step that applies them (sm_100a):
//   X = U / (|U|_F + eps);  `steps` times:  G = X X^T (rows <= cols; else X^T X),  B = b G + c G G,  X <- a X + B X (else a X + X B)
// Each singular value goes through s -> a s + b s^3 + c s^5 by itself; with the usual coefficients five steps bring those that are not
// tiny near 1. G and B are symmetric: only tiles on and right of the diagonal are computed, and written twice.
// A singular value far below the largest grows by a factor of up to a^steps (485), and so does whatever a rounding put beside it: all
// factors are held in two fp16 parts (22 bits; product_sm100.cuh) times 2^12, which suits values up to 15, and sums leave the tensor cores every
// 64 of the contraction. a X is added to the sums that have left them, in fp32: as a I in B it would be the largest term of sums that the tensor cores cut off (36 x 59: 1.7e-6
// off 64 bits with it there, 1.3e-6 so; 768 x 768: 1.5e-6 and 0.9e-6).
//
// All products of all steps are one cooperative launch. Its tiles are numbered step by step, product by product, matrix by matrix, and dealt out
// to the CTAs in turn; a tile waits until the tiles of the product before it, of the same matrix, are written (a counter per matrix). What it waits for has
// a lower number, and every CTA takes its tiles in their order, so the lowest unfinished tile never waits.
#include <math.h>

#include <algorithm>

#include "product_sm100.cuh"

namespace df {
namespace {

using namespace ptx;

constexpr float kPartScale = 4096.0f, kPartInverse = 1.0f / 4096.0f;
constexpr int kMostMatrices = 64;               // of a group: what the kernels' tables of pointers hold
constexpr uint64_t kGroupBytes = 192ull << 20;  // of workspace, beyond one matrix: what L2 loses between products is read again
constexpr int kNormBlocks = 256;                // partial sums of squares per matrix, at most
constexpr uint32_t kMostTensors = 1024;         // of an optimiser step

int finish(int st) {
  note_status(st);
  return st;
}
uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

__device__ __forceinline__ float load_f(const void *p, bool bf16, size_t i) {
  return bf16 ? __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16) : static_cast<const float *>(p)[i];
}

struct Table {
  const void *source[kMostMatrices];   // the update, or the gradient
  float *momentum[kMostMatrices];      // null: no optimiser step
};
struct Targets {
  void *out[kMostMatrices];  // where the result goes: the caller's matrix, or the parameter
};

// ---------------------------------------------------------------- before the products
struct UpdateParams {
  Table t;
  double *sums;    // [matrices][kNormBlocks]
  uint32_t *done;  // [matrices]: set to 0 here
  uint16_t *hi, *lo;
  uint64_t row_stride, matrix;  // of the source; elements of a matrix in parts
  uint32_t rows, cols, pitch, bf16, nesterov, vec;  // vec: four elements of a row at a time
  float beta, eps;
};

__device__ __forceinline__ float4 load_four(const void *p, bool bf16, size_t i) {
  if (!bf16) return *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
  const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
  return make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u));
}

// Moves the momentum, and adds up the squares of U: a warp a row, or all of a matrix that lies in one piece by 128 elements a warp. Squares in double: a
// gradient of 1e-30 is none of 0.
__global__ void __launch_bounds__(256) k_update(const __grid_constant__ UpdateParams p) {
  pdl_wait();
  const int m = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const void *source = p.t.source[m];
  float *momentum = p.t.momentum[m];
  const bool flat = p.rows == 1 || p.row_stride == p.cols;  // rows * cols below 2^31
  const uint32_t rows = flat ? 1 : p.rows, cols = flat ? p.rows * p.cols : p.cols;
  const uint32_t workers = gridDim.x * 8, me = blockIdx.x * 8 + warp;
  double sum = 0.0;
  for (uint32_t r = flat ? 0 : me; r < rows; r += flat ? 1 : workers) {
    const size_t at = (size_t)r * p.row_stride, at_m = (size_t)r * p.cols;
    const uint32_t whole = p.vec ? cols & ~3u : 0, step = flat ? workers : 1;
#pragma unroll 4
    for (uint32_t c = ((flat ? me : 0) * 32 + lane) * 4; c < whole; c += step * 128) {
      float4 u = load_four(source, p.bf16, at + c);
      if (momentum) {
        float4 v = *reinterpret_cast<const float4 *>(momentum + at_m + c);
        v = make_float4(fmaf(p.beta, v.x, u.x), fmaf(p.beta, v.y, u.y), fmaf(p.beta, v.z, u.z), fmaf(p.beta, v.w, u.w));
        *reinterpret_cast<float4 *>(momentum + at_m + c) = v;
        u = p.nesterov ? make_float4(fmaf(p.beta, v.x, u.x), fmaf(p.beta, v.y, u.y), fmaf(p.beta, v.z, u.z), fmaf(p.beta, v.w, u.w)) : v;
      }
      sum += ((double)u.x * u.x + (double)u.y * u.y) + ((double)u.z * u.z + (double)u.w * u.w);
    }
    for (uint32_t c = whole + (flat ? me : 0) * 32 + lane; c < cols; c += step * 32) {
      float u = load_f(source, p.bf16, at + c);
      if (momentum) {
        const float v = fmaf(p.beta, momentum[at_m + c], u);
        momentum[at_m + c] = v;
        u = p.nesterov ? fmaf(p.beta, v, u) : v;
      }
      sum += (double)u * u;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  __shared__ double part[8];
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) sum += part[i];
    p.sums[m * kNormBlocks + blockIdx.x] = sum;
    if (blockIdx.x == 0) p.done[m] = 0;
  }
}

// What brings a matrix's elements to its X times 2^12: multiplied by `first`, a power of two that is 1 for all but the smallest and largest norms, then by the result. A
// norm below 2^-116 has a factor that fp32 does not hold (eps = 0, or as small), one above 2^138 one with fewer bits. A norm of 0 gives infinity, and 0 times that NaN.
__device__ __forceinline__ float norm_factor(double sum_of_squares, float eps, float *first) {
  const double f = (double)kPartScale / (sqrt(sum_of_squares) + (double)eps);
  *first = f > 0x1p100 ? 0x1p64f : f < 0x1p-100 ? 0x1p-64f : 1.0f;
  return (float)(f / (double)*first);
}

// X in parts, a warp a row
__global__ void __launch_bounds__(256) k_normalise(const __grid_constant__ UpdateParams p, int blocks) {
  pdl_wait();
  const int m = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0.0;
  for (int i = lane; i < blocks; i += 32) sum += p.sums[m * kNormBlocks + i];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  float first;
  const float f = norm_factor(sum, p.eps, &first);
  const void *source = p.t.source[m];
  const float *momentum = p.t.momentum[m];
  for (uint32_t r = blockIdx.x * 8 + warp; r < p.rows; r += gridDim.x * 8) {
    const size_t at = (size_t)r * p.row_stride, at_m = (size_t)r * p.cols, to = (size_t)m * p.matrix + (size_t)r * p.pitch;
#pragma unroll 2
    for (uint32_t c = lane * 4; c < p.pitch; c += 128) {
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (p.vec && c + 4 <= p.cols) {
        const float4 u = load_four(source, p.bf16, at + c);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        if (momentum) {
          const float4 q = *reinterpret_cast<const float4 *>(momentum + at_m + c);
          const float g[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = p.nesterov ? fmaf(p.beta, g[x], v[x]) : g[x];
        }
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (c + x >= p.cols) continue;
          v[x] = load_f(source, p.bf16, at + c + x);
          if (momentum) v[x] = p.nesterov ? fmaf(p.beta, momentum[at_m + c + x], v[x]) : momentum[at_m + c + x];
        }
      }
      uint2 hi, lo;
      split_half2<0>(v[0] * first * f, v[1] * first * f, hi.x, lo.x);
      split_half2<0>(v[2] * first * f, v[3] * first * f, hi.y, lo.y);
      *reinterpret_cast<uint2 *>(p.hi + to + c) = hi;
      *reinterpret_cast<uint2 *>(p.lo + to + c) = lo;
    }
  }
}

// ---------------------------------------------------------------- the products
// Tiles of 128 x 128, the contraction cut among KS CTAs of a cluster. (Tiles of 256 x 256 over a pair of CTAs, whose operands are half the bytes, took 119 us for
// 64 x 64 where these take 79, 371 and 242 for 768 x 768, 1839 and 1923 for 48 of them: a tile's 128 sums a thread leave no room to write one tile's results
// while the next is added up.)
template <int KS_>
struct NsCfg {
  static constexpr int KS = KS_, T = 128;
  static constexpr int kOwned = T / KS, W = kOwned / 2 < 32 ? kOwned / 2 : 32, kGroups = kOwned / 2 / W;  // columns of a CTA's results; of a warp, W at a time
  static constexpr uint32_t kTileBytes = 128 * kProdK * 2, kSlotBytes = 2 * kTileBytes;  // a slot: A and B, low or high parts, in turn
  static constexpr int kSlots = KS > 1 ? 5 : 6;
  // the other half of shared memory: slabs of the epilogue's warps, or the partial sums [KS][128][kOwned] of the columns that this CTA owns
  static constexpr uint32_t kSmemStaging = kSlots * kSlotBytes, kStagingBytes = KS > 1 ? 128 * 128 * 4 : kProdEpiWarps * kProdSlabBytes;
  static constexpr uint32_t kSmemBars = kSmemStaging + kStagingBytes;
  static constexpr uint32_t kSmemTotal = kSmemBars + 256 + 1024;
  static constexpr int kAccs = 4;  // accumulators of 128 columns: so many blocks of the next tile run while results of this one are written
  static constexpr int FULL = 0, EMPTY = FULL + kSlots, ACC_FULL = EMPTY + kSlots, ACC_EMPTY = ACC_FULL + kAccs, RED_FULL = ACC_EMPTY + kAccs, RED_FREE = RED_FULL + 1,
                       DRAIN = RED_FREE + 1, NUM_BARS = DRAIN + 1;
  static_assert(NUM_BARS * 8 <= 240 && kSmemTotal <= 227 * 1024, "shared memory");
};

struct NsParams {
  // [buffer][hi, lo]: X with k along its rows or its columns, G, B
  CUtensorMap x_k[2][2], x_mn[2][2], g[2], b[2];
  uint32_t *done;             // [matrices]: epilogue warps that are through with their tile
  uint16_t *x[2][2], *gp[2], *bp[2];
  uint64_t x_matrix, g_matrix;
  uint32_t rows, cols, side, x_pitch, g_pitch;
  int wide, n, steps;
  int from, to;               // units of this launch
  int ordered;                // 1: what a unit needs was written by launches before this one
  int side_tiles, x_m_tiles, x_n_tiles, g_units, x_units;  // tiles: along the side, of X; of a symmetric product, of X's
  float a, b_, c;             // of the polynomial, times the parts' scales
  Targets t;
  uint64_t out_stride;
  uint32_t out_bf16, vec, apply;
  float keep, step;
  unsigned int *status;
};

enum Product { kGram, kPolynomial, kNext };
struct Unit {
  int step, batch, m, n, blocks;
  Product product;
  uint32_t after;  // tiles of this matrix that have to be written before
};
__device__ __forceinline__ Unit unit_of(const NsParams &p, int u) {
  Unit w;
  const int per_step = p.n * (2 * p.g_units + p.x_units);
  w.step = u / per_step;
  int r = u % per_step;
  w.after = (uint32_t)w.step * (uint32_t)(2 * p.g_units + p.x_units);
  const int g_all = p.n * p.g_units;
  w.product = r < g_all ? kGram : (r < 2 * g_all ? kPolynomial : kNext);
  if (w.product == kNext) {
    r -= 2 * g_all;
    w.after += 2 * p.g_units;
    w.batch = r / p.x_units;
    r %= p.x_units;
    w.m = r / p.x_n_tiles;
    w.n = r % p.x_n_tiles;
    w.blocks = (int)(p.side + kProdK - 1) / kProdK;
    return w;
  }
  if (w.product == kPolynomial) {
    r -= g_all;
    w.after += p.g_units;
  }
  w.batch = r / p.g_units;
  r %= p.g_units;
  w.m = 0;
  while (r >= p.side_tiles - w.m) {  // the tiles with n >= m, row after row
    r -= p.side_tiles - w.m;
    ++w.m;
  }
  w.n = w.m + r;
  w.blocks = (int)((w.product == kPolynomial ? p.side : (p.wide ? p.cols : p.rows)) + kProdK - 1) / kProdK;
  return w;
}

// W columns of a row in two parts
template <int W>
__device__ __forceinline__ void write_parts(uint16_t *hi, uint16_t *lo, size_t at, const float (&v)[W]) {
#pragma unroll
  for (int x = 0; x < W; x += 8) {
    uint4 h, l;
    split_half2<0>(v[x], v[x + 1], h.x, l.x);
    split_half2<0>(v[x + 2], v[x + 3], h.y, l.y);
    split_half2<0>(v[x + 4], v[x + 5], h.z, l.z);
    split_half2<0>(v[x + 6], v[x + 7], h.w, l.w);
    *reinterpret_cast<uint4 *>(hi + at + x) = h;
    *reinterpret_cast<uint4 *>(lo + at + x) = l;
  }
}

// v += factor * (hi + lo), W columns of a row. Written by other SMs of this launch: not through L1.
template <int W>
__device__ __forceinline__ void add_parts(const uint16_t *hi, const uint16_t *lo, size_t at, float factor, float (&v)[W]) {
#pragma unroll
  for (int x = 0; x < W; x += 8) {
    const uint4 h = __ldcg(reinterpret_cast<const uint4 *>(hi + at + x)), l = __ldcg(reinterpret_cast<const uint4 *>(lo + at + x));
    const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float2 q = __half22float2(*reinterpret_cast<const __half2 *>(&hh[y])), r = __half22float2(*reinterpret_cast<const __half2 *>(&ll[y]));
      v[x + 2 * y] = fmaf(factor, q.x + r.x, v[x + 2 * y]);
      v[x + 2 * y + 1] = fmaf(factor, q.y + r.y, v[x + 2 * y + 1]);
    }
  }
}

// G = X X^T, or B = b G + c G G: symmetric, in parts, each tile in its place and in the mirrored one
template <int W>
__device__ __forceinline__ void symmetric_block(const NsParams &p, const Unit &w, uint32_t row, uint32_t first, float (&v)[W]) {
  if (first >= p.side || row >= p.side) return;  // the pitch is a multiple of 64: a block that begins inside may be written whole
  const size_t base = (size_t)w.batch * p.g_matrix, at = base + (size_t)row * p.g_pitch + first;
  uint16_t *hi, *lo;
  if (w.product == kPolynomial) {
    hi = p.bp[0];
    lo = p.bp[1];
#pragma unroll
    for (int x = 0; x < W; ++x) v[x] *= p.c;
    add_parts<W>(p.gp[0], p.gp[1], at, p.b_, v);
  } else {
    hi = p.gp[0];
    lo = p.gp[1];
#pragma unroll
    for (int x = 0; x < W; ++x) v[x] *= kPartInverse;
  }
  write_parts<W>(hi, lo, at, v);
  if (w.m == w.n) return;
  // the mirrored tile: a column's 32 rows lie together across the warp's lanes
#pragma unroll
  for (int x = 0; x < W; ++x) {
    if (first + x >= p.side) break;
    const size_t to = base + (size_t)(first + x) * p.g_pitch + row;
    const __half h = __float2half_rn(v[x]);
    *reinterpret_cast<__half *>(hi + to) = h;
    *reinterpret_cast<__half *>(lo + to) = __float2half_rn(v[x] - __half2float(h));
  }
}

// Four columns of X of the last step: written in the caller's type, or applied to the parameter: P <- keep P - step X
__device__ __forceinline__ void last_four(const NsParams &p, void *out, uint32_t r, uint32_t col, float4 q) {
  constexpr float scale = kPartInverse * kPartInverse;
  float y[4] = {q.x * scale, q.y * scale, q.z * scale, q.w * scale};
  const size_t at = (size_t)r * p.out_stride + col;
  if (p.vec && col + 4 <= p.cols) {
    if (p.out_bf16) {
      uint2 b;
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.x) : "f"(y[1]), "f"(y[0]));
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.y) : "f"(y[3]), "f"(y[2]));
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + at) = b;
    } else {
      float4 *to = reinterpret_cast<float4 *>(static_cast<float *>(out) + at);
      if (p.apply) {
        const float4 old = *to;
        y[0] = fmaf(p.keep, old.x, -p.step * y[0]);
        y[1] = fmaf(p.keep, old.y, -p.step * y[1]);
        y[2] = fmaf(p.keep, old.z, -p.step * y[2]);
        y[3] = fmaf(p.keep, old.w, -p.step * y[3]);
      }
      *to = make_float4(y[0], y[1], y[2], y[3]);
    }
    return;
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (col + x >= p.cols) break;
    if (p.out_bf16) {
      uint32_t b;
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(0.0f), "f"(y[x]));
      static_cast<uint16_t *>(out)[at + x] = (uint16_t)b;
    } else {
      float *to = static_cast<float *>(out) + at + x;
      *to = p.apply ? fmaf(p.keep, *to, -p.step * y[x]) : y[x];
    }
  }
}
// 32 columns of a warp's rows, turned over so that memory moves in whole lines
__device__ __forceinline__ void last_block(const NsParams &p, const Unit &w, float4 *slab, int lane, uint32_t row0, uint32_t first, const float (&v)[32]) {
  if (first >= p.cols) return;
  float4 q[8];
  turn_over(slab, lane, v, q);
  const uint32_t col = first + 4 * (lane & 7);
  if (col >= p.cols) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t r = row0 + 4 * i + (lane >> 3);
    if (r < p.rows) last_four(p, p.t.out[w.batch], r, col, q[i]);
  }
}

// Blocks of 32 rows x 64 columns of a warp, v[0 .. 63] a lane's row: they go through the warp's slab, so that global memory moves in whole lines (a lane's own
// row as it is: 32 lines an instruction, 8 us for a tile's 128 x 256; turned over 4).
__device__ __forceinline__ void store_block(uint4 *slab, int lane, uint16_t *dst, size_t pitch, uint32_t rows, const uint4 (&q)[8]) {
  __syncwarp();
#pragma unroll
  for (int x = 0; x < 8; ++x) slab[lane * 8 + (x ^ (lane & 7))] = q[x];
  __syncwarp();
  const int lrow = lane >> 3, chunk = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 v = slab[(4 * i + lrow) * 8 + (chunk ^ ((4 * i + lrow) & 7))];
    if ((uint32_t)(4 * i + lrow) < rows) *reinterpret_cast<uint4 *>(dst + (size_t)(4 * i + lrow) * pitch + 8 * chunk) = v;
  }
}
__device__ __forceinline__ void split_block(const float (&v)[64], uint4 (&q)[8], bool low) {
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) split_half2<0>(v[8 * x + 2 * y], v[8 * x + 2 * y + 1], h[y], l[y]);
    q[x] = low ? make_uint4(l[0], l[1], l[2], l[3]) : make_uint4(h[0], h[1], h[2], h[3]);
  }
}
// `rows`: how many of the warp's 32 are in the matrix
__device__ __forceinline__ void next_block(uint16_t *const (&dst)[2], size_t at, uint32_t pitch, uint4 *slab, int lane, uint32_t rows, float (&v)[64]) {
#pragma unroll
  for (int low = 0; low < 2; ++low) {
    uint4 q[8];
    split_block(v, q, low != 0);
    store_block(slab, lane, dst[low] + at, pitch, rows, q);
  }
}
// v += factor * (hi + lo) of such a block, which other SMs of this launch have written: not through L1
__device__ __forceinline__ void add_block(uint16_t *const (&src)[2], size_t at, uint32_t pitch, uint4 *slab, int lane, uint32_t rows, float factor, float (&v)[64]) {
  const int lrow = lane >> 3, chunk = lane & 7;
#pragma unroll
  for (int low = 0; low < 2; ++low) {
    uint4 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[i] = (uint32_t)(4 * i + lrow) < rows ? __ldcg(reinterpret_cast<const uint4 *>(src[low] + at + (size_t)(4 * i + lrow) * pitch + 8 * chunk)) : make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) slab[(4 * i + lrow) * 8 + (chunk ^ ((4 * i + lrow) & 7))] = q[i];
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint4 g = slab[lane * 8 + (x ^ (lane & 7))];
      const uint32_t gg[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&gg[y]));
        v[8 * x + 2 * y] = fmaf(factor, f.x, v[8 * x + 2 * y]);
        v[8 * x + 2 * y + 1] = fmaf(factor, f.y, v[8 * x + 2 * y + 1]);
      }
    }
  }
}
__device__ __forceinline__ void symmetric_64(const NsParams &p, const Unit &w, uint4 *slab, int lane, uint32_t row0, uint32_t first, float (&v)[64]) {
  if (first >= p.side || row0 >= p.side) return;
  const size_t base = (size_t)w.batch * p.g_matrix, at = base + (size_t)row0 * p.g_pitch + first;
  const uint32_t rows = p.side - row0;
  if (w.product == kPolynomial) {
#pragma unroll
    for (int x = 0; x < 64; ++x) v[x] *= p.c;
    add_block(p.gp, at, p.g_pitch, slab, lane, rows, p.b_, v);
  } else {
#pragma unroll
    for (int x = 0; x < 64; ++x) v[x] *= kPartInverse;
  }
  uint16_t *const(&dst)[2] = w.product == kPolynomial ? p.bp : p.gp;
  next_block(dst, at, p.g_pitch, slab, lane, rows, v);
  if (w.m == w.n) return;
  // the mirrored tile: column x of the block is row first + x, 32 elements from row0 on. Two lanes make a pair of rows of a column each.
  const uint32_t columns = p.side - first;
#pragma unroll
  for (int low = 0; low < 2; ++low) {
    uint32_t *words = reinterpret_cast<uint32_t *>(slab);
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 64; x += 2) {
      uint32_t h, l;
      split_half2<0>(v[x], v[x + 1], h, l);
      const uint32_t mine = low ? l : h, other = __shfl_xor_sync(0xffffffffu, mine, 1);
      words[(x + (lane & 1)) * 16 + (lane >> 1)] = lane & 1 ? __byte_perm(other, mine, 0x7632) : __byte_perm(mine, other, 0x5410);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t c = 8 * i + (lane >> 2);
      const uint4 q = slab[c * 4 + (lane & 3)];
      if (c < columns) *reinterpret_cast<uint4 *>(dst[low] + base + (size_t)(first + c) * p.g_pitch + row0 + 8 * (lane & 3)) = q;
    }
  }
}

__device__ __forceinline__ uint32_t load_acquire(const uint32_t *p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Writes by ordinary stores become visible to the copy engines of other SMs: a fence between the two ways to memory at both ends.
__device__ __forceinline__ void fence_proxies() { asm volatile("fence.proxy.async;" ::: "memory"); }

// As prod_wait_warp, for a barrier on which other CTAs of the cluster arrive behind their writes to this one's shared memory.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag) {
  auto there = [&]() {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
  };
  bool done = there();
  if (!done) {
    const uint64_t t0 = global_timer_ns();
#pragma unroll 1
    for (uint32_t polls = 1; !done && polls < kWaitMaxPolls; ++polls) {
      done = there();
      if ((polls & 255u) == 0u && (*abort_flag != 0u || global_timer_ns() - t0 > kWaitBudgetNs)) break;
    }
    if (!done) *abort_flag = 1u;
  }
  return __all_sync(0xffffffffu, done) != 0;
}

template <class C>
__global__ void __launch_bounds__(kProdThreads, 1) k_newton_schulz(const __grid_constant__ NsParams p) {
  constexpr int kSlots = C::kSlots, T = C::T, KS = C::KS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t a0 = smem_u32(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kSmemBars);
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + C::kSmemBars + 240);
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(smem + C::kSmemBars + 244);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t part = KS > 1 ? cluster_rank() : 0;
  auto bar = [&](int id) { return smem_u32(&bars[id]); };
  auto first_block = [&](int blocks) { return (int)part * blocks / KS; };
  auto my_blocks = [&](int blocks) { return ((int)part + 1) * blocks / KS - (int)part * blocks / KS; };

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::NUM_BARS; ++i)
      mbar_init(bar(i), i >= C::ACC_EMPTY && i < C::RED_FULL ? kProdEpiWarps
                        : i == C::RED_FULL || i == C::RED_FREE     ? KS * kProdEpiWarps
                                                                   : 1);
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  if (KS > 1) cluster_sync();
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();
  const int first = p.from + blockIdx.x / KS, apart = gridDim.x / KS, units = p.to;

  if (warp < 4) {
    prod_regs_less<kProdOtherRegs>();
    if (warp == 0) {
      // ---------------------------------------------------------- copies
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int u = first; ok && u < units; u += apart) {
          const Unit w = unit_of(p, u);
          const uint32_t need = p.ordered ? 0 : w.after * (KS * kProdEpiWarps);
          if (load_acquire(p.done + w.batch) < need) {
            const uint64_t t0 = global_timer_ns();
#pragma unroll 1
            for (uint32_t polls = 1; load_acquire(p.done + w.batch) < need; ++polls) {
              if ((polls & 63u) == 0u && (*abort_flag != 0u || polls >= kWaitMaxPolls || global_timer_ns() - t0 > kWaitBudgetNs)) { ok = false; break; }
            }
            if (!ok) {
              *abort_flag = 1u;
              break;
            }
          }
          fence_proxies();
          const int cur = w.step & 1;
          const bool x_product = w.product == kNext;
          // G: X X^T (k along rows) or X^T X (k along columns); B: G G; X: B X or X B
          const bool mn_a = w.product == kGram && !p.wide, mn_b = mn_a || (x_product && p.wide);
          const CUtensorMap *a, *b;
          if (w.product == kGram) a = b = p.wide ? p.x_k[cur] : p.x_mn[cur];
          else if (w.product == kPolynomial) a = b = p.g;
          else if (p.wide) { a = p.b; b = p.x_mn[cur]; }
          else { a = p.x_k[cur]; b = p.b; }
          const int row_a = w.m * T, row_b = w.n * T;
          const int kb0 = first_block(w.blocks), kb1 = kb0 + my_blocks(w.blocks);
          for (int kb = kb0; ok && kb < kb1; ++kb) {
#pragma unroll
            for (int lo = 1; lo >= 0; --lo, ++it) {
              const uint32_t s = it % kSlots, use = it / kSlots;
              if (use > 0 && !prod_wait(bar(C::EMPTY + s), (use - 1) & 1, abort_flag)) { ok = false; break; }
              const uint32_t sa = a0 + s * C::kSlotBytes, full = bar(C::FULL + s);
              mbar_arrive_expect_tx(full, C::kSlotBytes);
              auto copy = [&](uint32_t dst, const CUtensorMap *m, int x, int y) { tma_load_3d(dst, m, full, x, y, w.batch); };
              auto load = [&](uint32_t dst, const CUtensorMap *m, bool mn, int row) {
                if (mn) {
                  copy(dst, m, row, kb * kProdK);
                  copy(dst + 8192, m, row + 64, kb * kProdK);
                } else {
                  copy(dst, m, kb * kProdK, row);
                }
              };
              load(sa, a + lo, mn_a, row_a);
              load(sa + C::kTileBytes, b + lo, mn_b, row_b);
            }
          }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- products
      uint32_t it = 0;
      bool ok = true;
      for (int u = first; ok && u < units; u += apart) {
        const Unit w = unit_of(p, u);
        const bool mn_a = w.product == kGram && !p.wide, mn_b = mn_a || (w.product == kNext && p.wide);
        const uint32_t idesc = make_idesc(kFmtF16, T, T, mn_a ? 1 : 0, mn_b ? 1 : 0);
        const uint32_t lbo_a = mn_a ? 8192 : 16, lbo_b = mn_b ? 8192 : 16;
        const uint64_t step_a = mn_a ? 2048 >> 4 : 32 >> 4, step_b = mn_b ? 2048 >> 4 : 32 >> 4;
        auto issue = [&](uint32_t d, uint32_t sa, uint32_t sb, bool fresh) {
          const uint64_t da = make_smem_desc(sa, lbo_a, 1024, kSwz128), db = make_smem_desc(sb, lbo_b, 1024, kSwz128);
#pragma unroll
          for (int k = 0; k < kProdK / 16; ++k) mma_f16_ss(d, da + k * step_a, db + k * step_b, idesc, fresh && k == 0 ? 0u : 1u);
        };
        const int blocks = my_blocks(w.blocks);
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          const uint32_t acc = it % C::kAccs, d = tmem + acc * T, s_lo = (2 * it) % kSlots, s_hi = (2 * it + 1) % kSlots;
          const uint32_t lo = a0 + s_lo * C::kSlotBytes, hi = a0 + s_hi * C::kSlotBytes;
          if (it >= C::kAccs && !prod_wait_warp(bar(C::ACC_EMPTY + acc), (it / C::kAccs - 1) & 1, abort_flag)) { ok = false; break; }
          if (!prod_wait_warp(bar(C::FULL + s_lo), ((2 * it) / kSlots) & 1, abort_flag) ||
              !prod_wait_warp(bar(C::FULL + s_hi), ((2 * it + 1) / kSlots) & 1, abort_flag)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            issue(d, lo, hi + C::kTileBytes, true);
            issue(d, hi, lo + C::kTileBytes, false);
            mma_commit(bar(C::EMPTY + s_lo));
            issue(d, hi, hi + C::kTileBytes, false);
            mma_commit(bar(C::EMPTY + s_hi));
            mma_commit(bar(C::ACC_FULL + acc));
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ------------------------------------------------------------ sums and results
    prod_regs_more<kProdEpiRegs>();
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    constexpr int kSums = T / 64, W = C::W, kGroups = C::kGroups;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + half * (T / 2);
    float4 *slab = reinterpret_cast<float4 *>(smem + C::kSmemStaging + (KS > 1 ? 0 : (warp - 4) * kProdSlabBytes));
    const int local = quarter * 32 + lane;  // row of the tile's 128
    uint32_t j = 0, turn = 0;
    bool ok = true;
    for (int u = first; ok && u < units; u += apart, ++turn) {
      const Unit w = unit_of(p, u);
      float sum[kSums][32];
#pragma unroll
      for (int cg = 0; cg < kSums; ++cg)
#pragma unroll
        for (int x = 0; x < 32; ++x) sum[cg][x] = 0.0f;
      const int blocks = my_blocks(w.blocks);
#pragma unroll 1
      for (int kb = 0; kb < blocks; ++kb, ++j) {
        const uint32_t acc = j % C::kAccs;
        if (!prod_wait_warp(bar(C::ACC_FULL + acc), (j / C::kAccs) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after_sync();
#pragma unroll
        for (int cg = 0; cg < kSums; ++cg) {
          uint32_t r[32];
          tmem_ld32(lane_base + acc * T + cg * 32, r);
          tmem_wait_ld();
          if (cg == kSums - 1) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::ACC_EMPTY + acc));
          }
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            const float2 q = add2(make_float2(sum[cg][x], sum[cg][x + 1]), as_float2(r[x], r[x + 1]));
            sum[cg][x] = q.x;
            sum[cg][x + 1] = q.y;
          }
        }
      }
      if (!ok) break;
      if constexpr (KS > 1) {
        // ---------------------------------------------------------- partial sums meet at the CTAs that own their columns, and are added in the order of the slices
        constexpr int OW = C::kOwned, kQuads = OW / 4;
        auto place = [&](int slice, int quad) {  // of 16 bytes; 8 lanes' places fall into different banks
          const int s = OW >= 32 ? (local & 7) : ((local >> 1) & 3);
          return (slice * 128 + local) * kQuads + (quad ^ s);
        };
        const uint32_t in_rows = (w.product == kNext ? p.rows : p.side) - (uint32_t)(w.m * T), in_cols = (w.product == kNext ? p.cols : p.side) - (uint32_t)(w.n * T);
        if (turn > 0 && !wait_cluster(bar(C::RED_FREE), (turn - 1) & 1, abort_flag)) { ok = false; break; }
#pragma unroll
        for (int cg = 0; cg < kSums; ++cg)
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            const int c = half * (T / 2) + cg * 32 + x, owner = c / OW;
            if ((uint32_t)local >= in_rows || (uint32_t)c >= in_cols) continue;  // zeros that nobody writes
            const uint32_t dst = map_to_rank(a0 + C::kSmemStaging + place((int)part, (c - owner * OW) / 4) * 16, (uint32_t)owner);
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(sum[cg][x]), "f"(sum[cg][x + 1]), "f"(sum[cg][x + 2]), "f"(sum[cg][x + 3])
                         : "memory");
          }
        __syncwarp();
        if (lane < KS) mbar_arrive_cluster(map_to_rank(bar(C::RED_FULL), lane));
        if (!wait_cluster(bar(C::RED_FULL), turn & 1, abort_flag)) { ok = false; break; }
#pragma unroll
        for (int cg = 0; cg < kGroups; ++cg)
#pragma unroll
          for (int x = 0; x < W; x += 4) {
            const int quad = (half * (OW / 2) + cg * W + x) / 4;
            float4 v = slab[place(0, quad)];
#pragma unroll
            for (int k = 1; k < KS; ++k) {
              const float4 q = slab[place(k, quad)];
              v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
            }
            sum[cg][x] = v.x;
            sum[cg][x + 1] = v.y;
            sum[cg][x + 2] = v.z;
            sum[cg][x + 3] = v.w;
          }
        __syncwarp();
        if (lane < KS) mbar_arrive_cluster(map_to_rank(bar(C::RED_FREE), lane));
      }
      const uint32_t row0 = (uint32_t)(w.m * T + quarter * 32), row = row0 + lane;
      const uint32_t col0 = (uint32_t)(w.n * T + (int)part * C::kOwned + half * (C::kOwned / 2));
      if (w.product != kGram) {  // what it reads of G or X: the copies have been waited for, these loads as well
        (void)load_acquire(p.done + w.batch);
        __syncwarp();
      }
      const bool last = w.product == kNext && w.step + 1 == p.steps;
      const int next = (w.step + 1) & 1;
      if constexpr (KS == 1) {
        uint4 *slab16 = reinterpret_cast<uint4 *>(slab);
#pragma unroll
        for (int cg = 0; cg < kGroups; cg += 2) {
          const uint32_t c = col0 + cg * W;
          float(&v)[64] = reinterpret_cast<float(&)[64]>(sum[cg]);
          if (w.product != kNext) {
            symmetric_64(p, w, slab16, lane, row0, c, v);
          } else if (c < p.cols && row0 < p.rows) {
            const size_t at = (size_t)w.batch * p.x_matrix + (size_t)row0 * p.x_pitch + c;
            add_block(p.x[w.step & 1], at, p.x_pitch, slab16, lane, p.rows - row0, p.a, v);
            if (!last) {
#pragma unroll
              for (int x = 0; x < 64; ++x) v[x] *= kPartInverse;
              next_block(p.x[next], at, p.x_pitch, slab16, lane, p.rows - row0, v);
            } else {
              last_block(p, w, slab, lane, row0, c, sum[cg]);
              last_block(p, w, slab, lane, row0, c + W, sum[cg + 1]);
            }
          }
        }
      } else {
        float(&v)[W] = reinterpret_cast<float(&)[W]>(sum[0]);
        if (w.product != kNext) {
          symmetric_block<W>(p, w, row, col0, v);
        } else if (col0 < p.cols && row < p.rows) {
          const size_t at = (size_t)w.batch * p.x_matrix + (size_t)row * p.x_pitch + col0;
          add_parts<W>(p.x[w.step & 1][0], p.x[w.step & 1][1], at, p.a, v);
          if (!last) {
#pragma unroll
            for (int x = 0; x < W; ++x) v[x] *= kPartInverse;
            write_parts<W>(p.x[next][0], p.x[next][1], at, v);
          } else {
#pragma unroll
            for (int x = 0; x < W; x += 4)
              if (col0 + x < p.cols) last_four(p, p.t.out[w.batch], row, col0 + x, make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]));
          }
        }
      }
      fence_proxies();
      __syncwarp();
      if (lane == 0) asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(p.done + w.batch), "r"(1u) : "memory");
    }
  }

  // ---------------------------------------------------------------- teardown (all roles), as in linear_sm100.cu
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {
    if (warp == 1) {
      if (elect_one()) mma_commit(bar(C::DRAIN));
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
  if (KS > 1) cluster_sync();  // no CTA leaves while another may still signal its barriers or write to its shared memory
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- matrices with a small side, a CTA or a cluster each
// A matrix of at most 128 rows (its smaller side; a taller one is turned over on the way in and out) stays in shared memory as two fp16 parts from its first product to
// its last, up to 256 columns in a CTA, up to 2048 in a cluster of up to eight: G, B and the new X go from tensor memory through registers to where the next product
// reads them. In a cluster every CTA adds up G from all CTAs' parts of it, which lie in global memory between two cluster barriers, and the rest is its own columns'.
// Nothing else between products leaves the SM (64 x 64: 33 us, where tiles that wait for a counter in global memory take 79; 128 x 128: 59 and 116).
// Slabs of 64 columns, 128 bytes a row, 128-byte swizzle: K-major for the products over columns, and the same bytes MN-major for B X, which contracts X's rows.
constexpr uint32_t kSmallRows = 128, kSmallCols = 256, kSmallCtas = 8;
constexpr uint32_t kSlab = 128 * 128;                                       // bytes: 128 rows x 64 columns of one part
constexpr uint32_t kSmallX = 0, kSmallG = 8 * kSlab, kSmallBars = 12 * kSlab;  // X: 4 slabs high, 4 low; G, then B: 2 high, 2 low
constexpr uint32_t kSmallSmem = kSmallBars + 128 + 1024;
constexpr uint32_t kSmallPitch = kSmallCols + 1;  // of the result in fp32, over all of it
static_assert(kSmallRows * kSmallPitch * 4 <= kSmallBars, "the result does not fit");

struct SmallParams {
  Table t;
  Targets o;
  uint64_t source_stride, out_stride;
  uint32_t rows, cols, bf16, nesterov, apply, steps, ctas, share;  // share: columns of a CTA
  float beta, eps, a, b, c, keep, step;
  double *sums;   // [matrices][ctas]
  float4 *grams;  // [matrices][2][ctas][32][128]: four columns of a row each, for odd and even steps
  unsigned int *status;
};

__device__ __forceinline__ uint32_t small_at(uint32_t row, uint32_t col) {  // byte of an element in its part
  return (col >> 6) * kSlab + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}
// 64 columns of a row in parts: a slab's row
__device__ __forceinline__ void small_store(uint8_t *hi, uint8_t *lo, uint32_t row, const float (&v)[64]) {
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    uint4 h, l;
    split_half2<0>(v[8 * x], v[8 * x + 1], h.x, l.x);
    split_half2<0>(v[8 * x + 2], v[8 * x + 3], h.y, l.y);
    split_half2<0>(v[8 * x + 4], v[8 * x + 5], h.z, l.z);
    split_half2<0>(v[8 * x + 6], v[8 * x + 7], h.w, l.w);
    const uint32_t at = row * 128 + ((x ^ (row & 7)) << 4);
    *reinterpret_cast<uint4 *>(hi + at) = h;
    *reinterpret_cast<uint4 *>(lo + at) = l;
  }
}

// v += factor * (hi + lo) of such a row
__device__ __forceinline__ void small_add(const uint8_t *hi, const uint8_t *lo, uint32_t row, float factor, float (&v)[64]) {
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const uint32_t at = row * 128 + ((x ^ (row & 7)) << 4);
    const uint4 h = *reinterpret_cast<const uint4 *>(hi + at), l = *reinterpret_cast<const uint4 *>(lo + at);
    const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float2 q = __half22float2(*reinterpret_cast<const __half2 *>(&hh[y])), r = __half22float2(*reinterpret_cast<const __half2 *>(&ll[y]));
      v[8 * x + 2 * y] = fmaf(factor, q.x + r.x, v[8 * x + 2 * y]);
      v[8 * x + 2 * y + 1] = fmaf(factor, q.y + r.y, v[8 * x + 2 * y + 1]);
    }
  }
}

__global__ void __launch_bounds__(256, 1) k_newton_schulz_small(const __grid_constant__ SmallParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t a0 = smem_u32(smem);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kSmallBars);
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + kSmallBars + 40);
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(smem + kSmallBars + 44);
  __shared__ double part[8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(bar(i), 1);
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  const int m = blockIdx.x / p.ctas, rank = blockIdx.x % p.ctas;
  const bool wide = p.rows <= p.cols;
  const uint32_t side = wide ? p.rows : p.cols, all = wide ? p.cols : p.rows, off = rank * p.share, large = all - off < p.share ? all - off : p.share;
  const uint32_t slabs = (large + 63) / 64, side_blocks = (side + 63) / 64, halves = (large + 127) / 128;
  // this CTA's part of the source
  const uint32_t rows = wide ? p.rows : large, cols = wide ? large : p.cols, row_off = wide ? 0 : off, col_off = wide ? off : 0;
  for (uint32_t i = tid; i < 8 * kSlab / 16; i += 256) reinterpret_cast<uint4 *>(smem + kSmallX)[i] = make_uint4(0u, 0u, 0u, 0u);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();
  const void *source = p.t.source[m];
  float *momentum = p.t.momentum[m];

  // ---------------------------------------------------------------- U, its norm, X. A warp a row of the source, its lanes the columns, the same ones in both passes.
  double sum = 0.0;
  for (uint32_t r = row_off + warp; r < row_off + rows; r += 8) {
#pragma unroll 4
    for (uint32_t c = col_off + lane; c < col_off + cols; c += 32) {
      float u = load_f(source, p.bf16, (size_t)r * p.source_stride + c);
      if (momentum) {
        const float v = fmaf(p.beta, momentum[r * p.cols + c], u);
        momentum[r * p.cols + c] = v;
        u = p.nesterov ? fmaf(p.beta, v, u) : v;
      }
      sum += (double)u * u;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < 8; ++i) sum += part[i];
  if (p.ctas > 1) {
    if (tid == 0) p.sums[blockIdx.x] = sum;
    cluster_sync();
    sum = 0.0;
    for (uint32_t i = 0; i < p.ctas; ++i) sum += __ldcg(p.sums + m * p.ctas + i);
  }
  float first;
  const float f = norm_factor(sum, p.eps, &first);
  for (uint32_t r = row_off + warp; r < row_off + rows; r += 8) {
#pragma unroll 4
    for (uint32_t c = col_off + lane; c < col_off + cols; c += 32) {
      float u = load_f(source, p.bf16, (size_t)r * p.source_stride + c);
      if (momentum) {
        const float v = momentum[r * p.cols + c];
        u = p.nesterov ? fmaf(p.beta, v, u) : v;
      }
      u = u * first * f;
      const __half h = __float2half_rn(u);
      const uint32_t at = wide ? small_at(r, c - off) : small_at(c, r - off);
      *reinterpret_cast<__half *>(smem + kSmallX + at) = h;
      *reinterpret_cast<__half *>(smem + kSmallX + 4 * kSlab + at) = __float2half_rn(u - __half2float(h));
    }
  }

  // ---------------------------------------------------------------- the products: block i of 64 of a contraction into accumulator i, its end on barrier i
  uint32_t phases = 0;  // bit i: the phase of barrier i that ends next
  bool ok = true;
  const int quarter = warp & 3, half = warp >> 2;
  const uint32_t row = quarter * 32 + lane, lanes = tmem + ((uint32_t)(quarter * 32) << 16) + half * 64;
  // block `acc`: A's slab at a (K-major), B at b: K-major slab, or MN-major rows with the next 64 columns a slab further
  auto issue = [&](int acc, uint32_t a, uint32_t a_lo, uint32_t b, uint32_t b_lo, bool b_mn) {
    const uint32_t idesc = make_idesc(kFmtF16, 128, 128, 0, b_mn ? 1 : 0);
    auto product = [&](uint32_t x, uint32_t y, bool fresh) {
      const uint64_t dx = make_smem_desc(a0 + x, 16, 1024, kSwz128), dy = make_smem_desc(a0 + y, b_mn ? kSlab : 16, 1024, kSwz128);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mma_f16_ss(tmem + acc * 128, dx + (uint64_t)(k * 32 >> 4), dy + (uint64_t)(k * (b_mn ? 2048 : 32) >> 4), idesc, fresh && k == 0 ? 0u : 1u);
    };
    if (elect_one()) {
      product(a_lo, b, true);
      product(a, b_lo, false);
      product(a, b, false);
      mma_commit(bar(acc));
    }
    __syncwarp();
  };
  auto take = [&](int acc, float (&v)[64]) {  // adds this lane's 64 columns
    if (!ok || !mbar_wait_warp(bar(acc), (phases >> acc) & 1, abort_flag)) {
      ok = false;
      return;
    }
    phases ^= 1u << acc;
    tc_fence_after_sync();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t r[32];
      tmem_ld32(lanes + acc * 128 + g * 32, r);
      tmem_wait_ld();
#pragma unroll
      for (int x = 0; x < 32; ++x) v[32 * g + x] += __uint_as_float(r[x]);
    }
  };
  auto meet = [&]() {  // what was written to shared memory is there for the tensor cores, and their results have been read
    fence_proxy_async_smem();
    tc_fence_before_sync();
    const bool stop = __syncthreads_or(!ok) != 0;
    tc_fence_after_sync();
    return !stop;
  };
  auto clear = [](float (&v)[64]) {
#pragma unroll
    for (int x = 0; x < 64; ++x) v[x] = 0.0f;
  };
  bool go = meet();
  for (uint32_t step = 0; step < p.steps; ++step) {  // to the end also where a wait has run out: the cluster's barriers are met by all
    float g[64], v[64];
    clear(g);
    if (go) {
      if (warp == 0)
        for (uint32_t c = 0; c < slabs; ++c) issue((int)c, kSmallX + c * kSlab, kSmallX + (4 + c) * kSlab, kSmallX + c * kSlab, kSmallX + (4 + c) * kSlab, false);
      for (uint32_t c = 0; c < slabs; ++c) take((int)c, g);
    }
    if (p.ctas > 1) {
      // a part of step s is written when every CTA has read those of step s - 2: it has been at the barrier of step s - 1 since
      float4 *parts = p.grams + (size_t)(m * 2 + (step & 1)) * p.ctas * 4096 + (half * 16) * 128 + row;
#pragma unroll
      for (int q = 0; q < 16; ++q) parts[(size_t)rank * 4096 + q * 128] = make_float4(g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3]);
      cluster_sync();
      clear(g);
      for (uint32_t k = 0; k < p.ctas; ++k) {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float4 x = __ldcg(parts + (size_t)k * 4096 + q * 128);
          g[4 * q] += x.x;
          g[4 * q + 1] += x.y;
          g[4 * q + 2] += x.z;
          g[4 * q + 3] += x.w;
        }
      }
    }
    if (!go) continue;
#pragma unroll
    for (int x = 0; x < 64; ++x) g[x] *= kPartInverse;
    small_store(smem + kSmallG + half * kSlab, smem + kSmallG + (2 + half) * kSlab, row, g);
    if (!(go = meet())) continue;
    if (warp == 0)
      for (uint32_t c = 0; c < side_blocks; ++c) issue((int)c, kSmallG + c * kSlab, kSmallG + (2 + c) * kSlab, kSmallG + c * kSlab, kSmallG + (2 + c) * kSlab, false);
    clear(v);
    for (uint32_t c = 0; c < side_blocks; ++c) take((int)c, v);
#pragma unroll
    for (int x = 0; x < 64; ++x) v[x] = fmaf(p.c, v[x], p.b * g[x]);
    small_store(smem + kSmallG + half * kSlab, smem + kSmallG + (2 + half) * kSlab, row, v);
    if (!(go = meet())) continue;
    if (warp == 0)
      for (uint32_t h = 0; h < halves; ++h)
        for (uint32_t c = 0; c < side_blocks; ++c)
          issue((int)(2 * h + c), kSmallG + c * kSlab, kSmallG + (2 + c) * kSlab, kSmallX + 2 * h * kSlab + c * 8192, kSmallX + (4 + 2 * h) * kSlab + c * 8192, true);
    if (step + 1 < p.steps) {
      for (uint32_t h = 0; h < halves; ++h) {
        clear(v);
        for (uint32_t c = 0; c < side_blocks; ++c) take((int)(2 * h + c), v);
        small_add(smem + kSmallX + (2 * h + half) * kSlab, smem + kSmallX + (4 + 2 * h + half) * kSlab, row, p.a, v);
#pragma unroll
        for (int x = 0; x < 64; ++x) v[x] *= kPartInverse;
        // only the products that have just ended read these slabs of X
        small_store(smem + kSmallX + (2 * h + half) * kSlab, smem + kSmallX + (4 + 2 * h + half) * kSlab, row, v);
      }
      go = meet();
      continue;
    }
    // the last: in fp32 over everything in shared memory, once no product reads it
    clear(g);
    clear(v);
    for (uint32_t c = 0; c < side_blocks; ++c) take((int)c, g);
    small_add(smem + kSmallX + half * kSlab, smem + kSmallX + (4 + half) * kSlab, row, p.a, g);
    if (halves > 1) {
      for (uint32_t c = 0; c < side_blocks; ++c) take((int)(2 + c), v);
      small_add(smem + kSmallX + (2 + half) * kSlab, smem + kSmallX + (6 + half) * kSlab, row, p.a, v);
    }
    if (!(go = meet())) continue;
    float *x = reinterpret_cast<float *>(smem) + row * kSmallPitch + half * 64;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      x[i] = g[i] * (kPartInverse * kPartInverse);
      x[128 + i] = v[i] * (kPartInverse * kPartInverse);
    }
  }
  __syncthreads();
  if (go) {
    const float *x = reinterpret_cast<const float *>(smem);
    for (uint32_t r = row_off + warp; r < row_off + rows; r += 8) {
#pragma unroll 4
      for (uint32_t c = col_off + lane; c < col_off + cols; c += 32) {
        const float y = wide ? x[r * kSmallPitch + c - off] : x[c * kSmallPitch + r - off];
        const size_t at = (size_t)r * p.out_stride + c;
        if (p.bf16) {
          uint32_t b;
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(0.0f), "f"(y));
          static_cast<uint16_t *>(p.o.out[m])[at] = (uint16_t)b;
        } else {
          float *to = static_cast<float *>(p.o.out[m]) + at;
          *to = p.apply ? fmaf(p.keep, *to, -p.step * y) : y;
        }
      }
    }
  } else if (tid == 0 && p.status) {  // a wait ran out: the products in flight are given time to end before the memory goes
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) {
    }
    atomicOr(p.status, DEV_STATUS_WAIT_EXPIRED);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- host
struct Layout {
  uint64_t done, x, x_next, g, b, total;  // offsets: parts hi, then lo, of all matrices of a group
  uint64_t x_matrix, g_matrix;      // elements of a matrix
  uint32_t x_pitch, g_pitch, side, group;
  bool small;            // k_newton_schulz_small,
  uint32_t ctas, share;  // on so many CTAs a matrix, with so many columns each
};
Layout layout(uint32_t n, uint32_t rows, uint32_t cols) {
  Layout l = {};
  l.side = rows < cols ? rows : cols;
  const uint32_t larger = rows < cols ? cols : rows;
  l.small = l.side <= kSmallRows && larger <= kSmallCtas * kSmallCols;
  if (l.small) {
    l.ctas = (larger + kSmallCols - 1) / kSmallCols;
    l.share = (uint32_t)up((larger + l.ctas - 1) / l.ctas, 64);
    l.ctas = (larger + l.share - 1) / l.share;
    l.group = n < (uint32_t)kMostMatrices ? n : (uint32_t)kMostMatrices;
    l.g = up((uint64_t)l.group * l.ctas * 8, 256);
    l.total = l.g + (l.ctas > 1 ? (uint64_t)l.group * 2 * l.ctas * 65536 : 0);
    return l;
  }
  l.x_pitch = (uint32_t)up(cols, 64);
  l.g_pitch = (uint32_t)up(l.side, 64);
  l.x_matrix = up((uint64_t)rows * l.x_pitch, 128);
  l.g_matrix = up((uint64_t)l.side * l.g_pitch, 128);
  const uint64_t each = 8 * l.x_matrix + 8 * l.g_matrix;
  uint64_t group = kGroupBytes / each;
  if (group > (uint64_t)kMostMatrices) group = kMostMatrices;
  if (group < 1) group = 1;
  l.group = n < group ? n : (uint32_t)group;
  l.done = (uint64_t)kMostMatrices * kNormBlocks * 8;
  uint64_t at = l.done + kMostMatrices * 4;
  auto take = [&](uint64_t elements) {
    const uint64_t here = at;
    at += elements * l.group * 4;
    return here;
  };
  l.x = take(l.x_matrix);
  l.x_next = take(l.x_matrix);
  l.g = take(l.g_matrix);
  l.b = take(l.g_matrix);
  l.total = at;
  return l;
}

bool sizes_ok(uint32_t n, uint32_t rows, uint32_t cols) {
  return rows > 0 && cols > 0 && n < (1u << 24) && rows <= 65536u && cols <= 65536u && (uint64_t)rows * cols < (1ull << 31);
}

// A matrix of parts in a batch as an operand, as operand_map
bool batch_map(CUtensorMap *m, const void *base, uint64_t rows, uint64_t cols, uint64_t pitch, uint64_t n, uint64_t matrix, bool mn_major) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[3] = {cols, rows, n};
  const cuuint64_t strides[2] = {pitch * 2, matrix * 2};
  const cuuint32_t box[3] = {64, mn_major ? 64u : 128u, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
  uint32_t rows, cols, steps;
  float a, b, c, eps;
  uint8_t *ws;
  Layout l;
  cudaStream_t s;

  // All products of all steps in one launch (step < 0), or one product of a step.
  template <class C>
  int products(uint32_t n, NsParams &p, int step, Product which) const {
    auto tiles = [](uint32_t v) { return (int)((v + C::T - 1) / C::T); };
    p.side_tiles = tiles(l.side);
    p.x_m_tiles = tiles(rows);
    p.x_n_tiles = tiles(cols);
    p.g_units = p.side_tiles * (p.side_tiles + 1) / 2;
    p.x_units = p.x_m_tiles * p.x_n_tiles;
    const int slots = cluster_slots<k_newton_schulz<C>>(C::KS, C::kSmemTotal, kProdLaunchRegs);
    if (slots == 0) return DF_ERR_CUDA;
    const int per_step = (int)n * (2 * p.g_units + p.x_units);
    long long most = (long long)n * (p.g_units > p.x_units ? p.g_units : p.x_units);
    p.from = 0;
    p.to = (int)steps * per_step;
    p.ordered = step >= 0;
    if (step >= 0) {
      p.from = step * per_step + (which == kGram ? 0 : which == kPolynomial ? 1 : 2) * (int)n * p.g_units;
      p.to = p.from + (int)n * (which == kNext ? p.x_units : p.g_units);
      most = p.to - p.from;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C::KS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    if (step < 0) {
      attr[1].id = cudaLaunchAttributeCooperative;
      attr[1].val.cooperative = 1;
    } else {
      attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[1].val.programmaticStreamSerializationAllowed = option(DF_OPT_PDL) != 0;
    }
    cfg.gridDim = dim3((unsigned)((most < slots ? most : slots) * C::KS));
    cfg.blockDim = dim3(kProdThreads);
    cfg.dynamicSmemBytes = C::kSmemTotal;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const int st = check_cuda(cudaLaunchKernelEx(&cfg, k_newton_schulz<C>, p));
    note_launch();
    return st;
  }
  int products(int form, uint32_t n, NsParams &p, int step, Product which) const {
    switch (form) {
      case 0: return products<NsCfg<1>>(n, p, step, which);
      case 1: return products<NsCfg<2>>(n, p, step, which);
      default: return products<NsCfg<4>>(n, p, step, which);
    }
  }

  // Time of a product in us with its contraction cut in 1 << form, without what comes between products: 64 of the contraction, 64 KB of operands a CTA,
  // take about 1 us; results take 3, the exchange of partial sums 5.
  double estimate(uint32_t n, int form, Product which) const {
    const uint64_t ks = 1ull << form, slots = 148 / ks, m = (l.side + 127) / 128, x = (uint64_t)((rows + 127) / 128) * ((cols + 127) / 128), g = m * (m + 1) / 2;
    const uint64_t k = which == kGram ? (rows > cols ? rows : cols) : l.side, blocks = ((k + 63) / 64 + ks - 1) / ks;
    return (double)(((which == kNext ? x : g) * n + slots - 1) / slots) * ((double)blocks + (form > 0 ? 5.0 : 1.0));
  }

  int small(uint32_t n, const UpdateParams &u, const NsParams &q) const {
    static std::atomic<bool> ready[64];
    int dev = 0;
    if (check_cuda(cudaGetDevice(&dev)) != DF_OK || dev < 0 || dev >= 64) return DF_ERR_CUDA;
    if (!ready[dev].load(std::memory_order_acquire)) {
      if (check_cuda(cudaFuncSetAttribute(k_newton_schulz_small, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmallSmem)) != DF_OK) return DF_ERR_CUDA;
      ready[dev].store(true, std::memory_order_release);
    }
    SmallParams p = {};
    p.t = u.t;
    p.o = q.t;
    p.source_stride = u.row_stride;
    p.out_stride = q.out_stride;
    p.rows = rows;
    p.cols = cols;
    p.bf16 = u.bf16;
    p.nesterov = u.nesterov;
    p.apply = q.apply;
    p.steps = steps;
    p.beta = u.beta;
    p.eps = eps;
    p.a = a * kPartScale;
    p.b = b;
    p.c = c * kPartInverse;
    p.keep = q.keep;
    p.step = q.step;
    p.ctas = l.ctas;
    p.share = l.share;
    p.sums = reinterpret_cast<double *>(ws);
    p.grams = reinterpret_cast<float4 *>(ws + l.g);
    p.status = device_status_ptr();
    const int st = check_cuda(launch_clusters(k_newton_schulz_small, l.ctas > 1 ? l.ctas : 0, dim3(n * l.ctas), dim3(256), kSmallSmem, s, p));
    note_launch();
    return st;
  }

  int run(uint32_t n, UpdateParams u, NsParams p) const {
    if (l.small) return small(n, u, p);
    auto part = [&](uint64_t at, uint64_t matrix, int lo) { return reinterpret_cast<uint16_t *>(ws + at) + lo * matrix * l.group; };
    bool ok = true;
    for (int i = 0; i < 2; ++i) {
      for (int j = 0; j < 2; ++j) {
        p.x[j][i] = part(j ? l.x_next : l.x, l.x_matrix, i);
        ok = ok && batch_map(&p.x_k[j][i], p.x[j][i], rows, cols, l.x_pitch, n, l.x_matrix, false) &&
             batch_map(&p.x_mn[j][i], p.x[j][i], rows, cols, l.x_pitch, n, l.x_matrix, true);
      }
      p.gp[i] = part(l.g, l.g_matrix, i);
      p.bp[i] = part(l.b, l.g_matrix, i);
      ok = ok && batch_map(&p.g[i], p.gp[i], l.side, l.side, l.g_pitch, n, l.g_matrix, false) &&
           batch_map(&p.b[i], p.bp[i], l.side, l.side, l.g_pitch, n, l.g_matrix, false);
    }
    if (!ok) return DF_ERR_CUDA;
    u.sums = reinterpret_cast<double *>(ws);
    u.done = p.done = reinterpret_cast<uint32_t *>(ws + l.done);
    u.hi = p.x[0][0];
    u.lo = p.x[0][1];
    u.matrix = l.x_matrix;
    u.rows = rows;
    u.cols = cols;
    u.pitch = l.x_pitch;
    u.eps = eps;
    const uint32_t each = (uint32_t)(1184 / n), quarter = (uint32_t)(((uint64_t)rows * cols + 4095) / 4096), sums = quarter < each ? quarter : each;
    const uint32_t blocks = sums < 1 ? 1 : (sums < (uint32_t)kNormBlocks ? sums : (uint32_t)kNormBlocks);
    int st = check_cuda(launch_kernel(k_update, dim3(blocks, n), dim3(256), 0, s, u));
    if (st != DF_OK) return st;
    st = check_cuda(launch_kernel(k_normalise, dim3((rows + 7) / 8 < 4 * each ? (rows + 7) / 8 : 4 * each, n), dim3(256), 0, s, u, (int)blocks));
    note_launch(2);
    if (st != DF_OK) return st;
    p.x_matrix = l.x_matrix;
    p.g_matrix = l.g_matrix;
    p.rows = rows;
    p.cols = cols;
    p.side = l.side;
    p.x_pitch = l.x_pitch;
    p.g_pitch = l.g_pitch;
    p.wide = rows <= cols;
    p.n = (int)n;
    p.steps = (int)steps;
    p.a = a * kPartScale;  // parts are times 2^12, their product 2^24
    p.b_ = b;
    p.c = c * kPartInverse;
    p.status = device_status_ptr();
    // One launch with one form for everything, about 5 us between products (fences, a counter, first copies), or a launch a product with the form that suits
    // each, about 7 between (1200 x 3000: one launch 527 at best, three a step 446; 64 x 64: 79 and 101).
    const Product all[3] = {kGram, kPolynomial, kNext};
    double one = 1e300, own = 0.0;
    int one_form = 0, own_form[3] = {0, 0, 0};
    for (int f = 0; f < 3; ++f) {
      double t = 0.0;
      for (Product q : all) t += estimate(n, f, q) + 5.0;
      if (t < one) {
        one = t;
        one_form = f;
      }
    }
    for (int i = 0; i < 3; ++i) {
      double best = 1e300;
      for (int f = 0; f < 3; ++f) {
        const double t = estimate(n, f, all[i]) + 7.0;
        if (t < best) {
          best = t;
          own_form[i] = f;
        }
      }
      own += best;
    }
    if (one <= own) return products(one_form, n, p, -1, kGram);
    for (uint32_t i = 0; st == DF_OK && i < steps; ++i)
      for (int q = 0; st == DF_OK && q < 3; ++q) st = products(own_form[q], n, p, (int)i, all[q]);
    return st;
  }
};

int check_call(uint32_t n, uint32_t rows, uint32_t cols, uint32_t steps, float a, float b, float c, float eps) {
  if (!sizes_ok(n, rows, cols) || steps < 1 || steps > 64) return DF_ERR_INVALID_ARG;
  if (!isfinite(a) || !isfinite(b) || !isfinite(c) || !isfinite(eps) || eps < 0.0f) return DF_ERR_INVALID_ARG;
  // the parts hold values up to 15; |B|, and X after a step, are at most this for singular values up to 1. What later steps bring follows from the data.
  return fabsf(a) + fabsf(b) + fabsf(c) < 15.0f ? DF_OK : DF_ERR_UNSUPPORTED;
}

bool meet(const void *x, uint64_t x_bytes, const void *y, uint64_t y_bytes) {  // whether they share memory
  const uintptr_t u = reinterpret_cast<uintptr_t>(x), v = reinterpret_cast<uintptr_t>(y);
  return u < v + y_bytes && v < u + x_bytes;
}
// Whether a parameter or a momentum, which are written, shares memory with anything else of the table. All are of the same size, so of two in order of their
// addresses that meet, the first meets its successor and the second its predecessor.
bool tensors_meet(const df_muon_tensor_t *t, uint32_t n, uint64_t bytes) {
  struct Held {
    uintptr_t at;
    bool written;
  } all[3 * kMostTensors];
  uint32_t k = 0;
  for (uint32_t i = 0; i < n; ++i) {
    all[k++] = {reinterpret_cast<uintptr_t>(t[i].parameter), true};
    all[k++] = {reinterpret_cast<uintptr_t>(t[i].momentum), true};
    all[k++] = {reinterpret_cast<uintptr_t>(t[i].gradient), false};
  }
  std::sort(all, all + k, [](const Held &x, const Held &y) { return x.at < y.at; });
  for (uint32_t i = 1; i < k; ++i)
    if ((all[i].written || all[i - 1].written) && all[i].at - all[i - 1].at < bytes) return true;
  return false;
}

bool aligned(const void *p, uint64_t row_bytes, uint64_t to) { return ((reinterpret_cast<uintptr_t>(p) | row_bytes) & (to - 1)) == 0; }

}  // namespace
}  // namespace df

using namespace df;

extern "C" {

uint64_t df_orthogonalize_workspace_bytes(uint32_t n, uint32_t rows, uint32_t cols) {
  return n == 0 || !sizes_ok(n, rows, cols) ? 0 : layout(n, rows, cols).total;
}

int df_orthogonalize(const void *update, void *out, void *workspace, uint64_t workspace_bytes, uint32_t n, uint32_t rows, uint32_t cols,
                     uint64_t update_matrix_stride, uint64_t update_row_stride, uint64_t out_matrix_stride, uint64_t out_row_stride, uint32_t steps, float a,
                     float b, float c, float eps, uint32_t bf16, void *stream) {
  DF_RANGE("df_orthogonalize");
  int st = check_call(n, rows, cols, steps, a, b, c, eps);
  if (st != DF_OK) return finish(st);
  if (n == 0) return DF_OK;
  if (!update || !out) return finish(DF_ERR_INVALID_ARG);
  const uint64_t most = 1ull << 40;
  if (update_matrix_stride >= most || update_row_stride >= most || out_matrix_stride >= most || out_row_stride >= most) return finish(DF_ERR_INVALID_ARG);
  if (rows > 1 && (update_row_stride < cols || out_row_stride < cols)) return finish(DF_ERR_INVALID_ARG);
  // results lie apart: one matrix behind the other, or row by row of all of them
  if (n > 1 && out_matrix_stride < (uint64_t)(rows - 1) * out_row_stride + cols &&
      (out_matrix_stride < cols || (rows > 1 && out_row_stride < (uint64_t)(n - 1) * out_matrix_stride + cols)))
    return finish(DF_ERR_INVALID_ARG);
  // out is the update, element by element, or shares nothing with it
  const uint64_t in_elt = bf16 ? 2 : 4, in_bytes = ((uint64_t)(n - 1) * update_matrix_stride + (uint64_t)(rows - 1) * update_row_stride + cols) * in_elt;
  const uint64_t out_bytes = ((uint64_t)(n - 1) * out_matrix_stride + (uint64_t)(rows - 1) * out_row_stride + cols) * in_elt;
  const bool same = update == out && (rows == 1 || update_row_stride == out_row_stride) && (n == 1 || update_matrix_stride == out_matrix_stride);
  if (!same && meet(update, in_bytes, out, out_bytes)) return finish(DF_ERR_INVALID_ARG);
  const Layout l = layout(n, rows, cols);
  if (!workspace || workspace_bytes < l.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return finish(DF_ERR_WORKSPACE);
  if (meet(update, in_bytes, workspace, l.total) || meet(out, out_bytes, workspace, l.total)) return finish(DF_ERR_INVALID_ARG);
  const Plan plan = {rows, cols, steps, a, b, c, eps, static_cast<uint8_t *>(workspace), l, static_cast<cudaStream_t>(stream)};
  const uint64_t elt = bf16 ? 2 : 4;
  for (uint32_t i0 = 0; st == DF_OK && i0 < n; i0 += l.group) {
    const uint32_t k = n - i0 < l.group ? n - i0 : l.group;
    UpdateParams u = {};
    NsParams last = {};
    u.row_stride = update_row_stride;
    u.bf16 = bf16 != 0;
    u.vec = 1;
    last.out_stride = out_row_stride;
    last.out_bf16 = bf16 != 0;
    last.vec = 1;
    for (uint32_t i = 0; i < k; ++i) {
      u.t.source[i] = static_cast<const uint8_t *>(update) + (i0 + i) * update_matrix_stride * elt;
      last.t.out[i] = static_cast<uint8_t *>(out) + (i0 + i) * out_matrix_stride * elt;
      if (!aligned(last.t.out[i], rows > 1 ? out_row_stride * elt : 0, bf16 ? 8 : 16)) last.vec = 0;
      if (!aligned(u.t.source[i], rows > 1 ? update_row_stride * elt : 0, bf16 ? 8 : 16)) u.vec = 0;
    }
    st = plan.run(k, u, last);
  }
  return finish(st);
}

int df_muon_update(const void *tensors, uint32_t n, uint32_t rows, uint32_t cols, float lr, float momentum, float weight_decay, uint32_t nesterov,
                   float update_scale, uint32_t steps, float a, float b, float c, float eps, void *workspace, uint64_t workspace_bytes, void *stream) {
  DF_RANGE("df_muon_update");
  int st = check_call(n, rows, cols, steps, a, b, c, eps);
  if (st != DF_OK) return finish(st);
  if (!isfinite(lr) || !isfinite(momentum) || !isfinite(weight_decay) || !isfinite(update_scale)) return finish(DF_ERR_INVALID_ARG);
  if (n == 0) return DF_OK;
  if (!tensors) return finish(DF_ERR_INVALID_ARG);
  const df_muon_tensor_t *t = static_cast<const df_muon_tensor_t *>(tensors);
  if (n > kMostTensors) return finish(DF_ERR_UNSUPPORTED);
  for (uint32_t i = 0; i < n; ++i)
    if (!t[i].parameter || !t[i].momentum || !t[i].gradient) return finish(DF_ERR_INVALID_ARG);
  if (tensors_meet(t, n, (uint64_t)rows * cols * 4)) return finish(DF_ERR_INVALID_ARG);
  const Layout l = layout(n, rows, cols);
  if (!workspace || workspace_bytes < l.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return finish(DF_ERR_WORKSPACE);
  for (uint32_t i = 0; i < n; ++i)
    for (const void *p : {static_cast<const void *>(t[i].parameter), static_cast<const void *>(t[i].momentum), static_cast<const void *>(t[i].gradient)})
      if (meet(p, (uint64_t)rows * cols * 4, workspace, l.total)) return finish(DF_ERR_INVALID_ARG);
  const Plan plan = {rows, cols, steps, a, b, c, eps, static_cast<uint8_t *>(workspace), l, static_cast<cudaStream_t>(stream)};
  for (uint32_t i0 = 0; st == DF_OK && i0 < n; i0 += l.group) {
    const uint32_t k = n - i0 < l.group ? n - i0 : l.group;
    UpdateParams u = {};
    NsParams last = {};
    u.row_stride = cols;
    u.vec = 1;
    u.beta = momentum;
    u.nesterov = nesterov != 0;
    last.out_stride = cols;
    last.vec = 1;
    last.apply = 1;
    last.keep = (float)(1.0 - (double)lr * (double)weight_decay);
    last.step = lr * update_scale;
    for (uint32_t i = 0; i < k; ++i) {
      u.t.source[i] = t[i0 + i].gradient;
      u.t.momentum[i] = t[i0 + i].momentum;
      last.t.out[i] = t[i0 + i].parameter;
      if (!aligned(last.t.out[i], rows > 1 ? (uint64_t)cols * 4 : 0, 16)) last.vec = 0;
      if (!aligned(u.t.source[i], 0, 16) || !aligned(u.t.momentum[i], 0, 16)) u.vec = 0;
      if (rows > 1 && cols % 4 != 0) u.vec = 0;
    }
    st = plan.run(k, u, last);
  }
  return finish(st);
}

}  // extern "C"
