// muon.cu — matrices orthogonalised by Newton-Schulz products, and the optimiser step that applies them (sm_100a):
//   X = U / (|U|_F + eps);  `steps` times:  G = X X^T (rows <= cols; else X^T X),  B = a I + b G + c G G,  X <- B X (else X B)
// Each singular value goes through s -> a s + b s^3 + c s^5 by itself; with the usual coefficients five steps bring those that are not
// tiny near 1. G and B are symmetric: only tiles on and right of the diagonal are computed, and written twice.
// A singular value far below the largest grows by a factor of up to a^steps (485), and so does whatever a rounding put beside it: all
// factors are held in two fp16 parts (22 bits; product_sm100.cuh) times 2^12, which suits values up to 15, and sums leave the tensor cores every
// 768 of the contraction. a is on the diagonal of B, so that X's new value is one product.
#include <math.h>

#include "product_sm100.cuh"

namespace df {
namespace {

using namespace ptx;

constexpr float kPartScale = 4096.0f, kPartInverse = 1.0f / 4096.0f;
constexpr int kMostMatrices = 64;               // of a group: what the kernels' tables of pointers hold
constexpr uint64_t kGroupBytes = 512ull << 20;  // of workspace, beyond one matrix
constexpr int kNormBlocks = 64;                 // partial sums of squares per matrix
constexpr int kChunk = 1;
constexpr uint32_t kMostTensors = 1024;         // of an optimiser step: every pair is checked for overlap

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
  double *sums;  // [matrices][kNormBlocks]
  uint16_t *hi, *lo;
  uint64_t row_stride, matrix;  // of the source; elements of a matrix in parts
  uint32_t rows, cols, pitch, bf16, nesterov;
  float beta, eps;
};

// U at (row, col): the source itself, or the momentum with or without a look ahead (the momentum has been moved already)
__device__ __forceinline__ float update_at(const UpdateParams &p, int m, uint32_t r, uint32_t c) {
  const float g = load_f(p.t.source[m], p.bf16, (size_t)r * p.row_stride + c);
  if (!p.t.momentum[m]) return g;
  const float v = p.t.momentum[m][(size_t)r * p.cols + c];
  return p.nesterov ? fmaf(p.beta, v, g) : v;
}

// Moves the momentum, and adds up squares: blocks of a matrix take rows in turn. Squares in double: a gradient of 1e-30 is none of 0.
__global__ void __launch_bounds__(256) k_update(const __grid_constant__ UpdateParams p) {
  pdl_wait();
  const int m = blockIdx.y;
  double sum = 0.0;
  const uint64_t n = (uint64_t)p.rows * p.cols;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)kNormBlocks * 256) {
    const uint32_t r = (uint32_t)(i / p.cols), c = (uint32_t)(i % p.cols);
    if (p.t.momentum[m]) p.t.momentum[m][i] = fmaf(p.beta, p.t.momentum[m][i], load_f(p.t.source[m], p.bf16, (size_t)r * p.row_stride + c));
    const double u = update_at(p, m, r, c);
    sum += u * u;
  }
  __shared__ double part[256];
  part[threadIdx.x] = sum;
  __syncthreads();
  for (int half = 128; half > 0; half >>= 1) {
    if ((int)threadIdx.x < half) part[threadIdx.x] += part[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.sums[m * kNormBlocks + blockIdx.x] = part[0];
}

// X in parts
__global__ void __launch_bounds__(256) k_normalise(const __grid_constant__ UpdateParams p) {
  pdl_wait();
  const int m = blockIdx.y;
  __shared__ float factor;
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int i = 0; i < kNormBlocks; ++i) sum += p.sums[m * kNormBlocks + i];
    factor = (float)((double)kPartScale / (sqrt(sum) + (double)p.eps));
  }
  __syncthreads();
  const float f = factor;
  const uint32_t quads = p.pitch / 4;
  const uint64_t n = (uint64_t)p.rows * quads;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
    const uint32_t r = (uint32_t)(i / quads), c = (uint32_t)(i % quads) * 4;
    float v[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = c + x < p.cols ? update_at(p, m, r, c + x) * f : 0.0f;
    uint2 hi, lo;
    split_half2(v[0], v[1], hi.x, lo.x);
    split_half2(v[2], v[3], hi.y, lo.y);
    const size_t to = (size_t)m * p.matrix + (size_t)r * p.pitch + c;
    *reinterpret_cast<uint2 *>(p.hi + to) = hi;
    *reinterpret_cast<uint2 *>(p.lo + to) = lo;
  }
}

// ---------------------------------------------------------------- epilogues
// A row's 32 columns of two parts, 64 bytes each
__device__ __forceinline__ void write_parts(uint16_t *hi, uint16_t *lo, size_t at, const float (&v)[32]) {
#pragma unroll
  for (int x = 0; x < 32; x += 8) {
    uint4 h, l;
    split_half2(v[x], v[x + 1], h.x, l.x);
    split_half2(v[x + 2], v[x + 3], h.y, l.y);
    split_half2(v[x + 4], v[x + 5], h.z, l.z);
    split_half2(v[x + 6], v[x + 7], h.w, l.w);
    *reinterpret_cast<uint4 *>(hi + at + x) = h;
    *reinterpret_cast<uint4 *>(lo + at + x) = l;
  }
}
__device__ __forceinline__ float one_part(const uint16_t *hi, const uint16_t *lo, size_t i) {
  return __half2float(*reinterpret_cast<const __half *>(hi + i)) + __half2float(*reinterpret_cast<const __half *>(lo + i));
}

// G = X X^T, or B = a I + b G + c G G: symmetric, in parts, each tile in its place and in the mirrored one
struct SymmetricEpi {
  struct Params {
    uint16_t *hi, *lo;              // [matrices][side][pitch]
    const uint16_t *g_hi, *g_lo;    // null: G itself
    uint64_t matrix;
    uint32_t side, pitch;
    float a, b, c;                  // of B, times the parts' scales
  };
  const Params &p;
  uint32_t row, col0;
  size_t base;
  bool mirror;
  __device__ __forceinline__ SymmetricEpi(const Params &q, uint8_t *, int) : p(q) {}
  __device__ __forceinline__ void begin(const ProductTile &t, uint32_t r, uint32_t c0) {
    row = r;
    col0 = c0;
    base = (size_t)t.batch * p.matrix;
    mirror = t.m_tile != t.n_tile;
  }
  __device__ __forceinline__ void block(int cg, float (&v)[32]) {
    const uint32_t first = col0 + cg * 32;
    if (first >= p.side || row >= p.side) return;  // the pitch is a multiple of 64: a block that begins inside may be written whole
    const size_t at = base + (size_t)row * p.pitch + first;
    if (p.g_hi) {
#pragma unroll
      for (int x = 0; x < 32; x += 8) {
        const uint4 h = *reinterpret_cast<const uint4 *>(p.g_hi + at + x), l = *reinterpret_cast<const uint4 *>(p.g_lo + at + x);
        const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float2 u = __half22float2(*reinterpret_cast<const __half2 *>(&hh[y])), w = __half22float2(*reinterpret_cast<const __half2 *>(&ll[y]));
          v[x + 2 * y] = fmaf(p.c, v[x + 2 * y], p.b * (u.x + w.x));
          v[x + 2 * y + 1] = fmaf(p.c, v[x + 2 * y + 1], p.b * (u.y + w.y));
        }
      }
#pragma unroll
      for (int x = 0; x < 32; ++x) v[x] += first + x == row ? p.a : 0.0f;
    } else {
#pragma unroll
      for (int x = 0; x < 32; ++x) v[x] *= p.c;
    }
    write_parts(p.hi, p.lo, at, v);
    if (!mirror) return;
    // the mirrored tile: a column's 32 rows lie together across the warp's lanes
#pragma unroll
    for (int x = 0; x < 32; ++x) {
      if (first + x >= p.side) break;
      const size_t to = base + (size_t)(first + x) * p.pitch + row;
      const __half h = __float2half_rn(v[x]);
      *reinterpret_cast<__half *>(p.hi + to) = h;
      *reinterpret_cast<__half *>(p.lo + to) = __float2half_rn(v[x] - __half2float(h));
    }
  }
  __device__ __forceinline__ void end() {}
};

// X of the next step, in parts
struct NextEpi {
  struct Params {
    uint16_t *hi, *lo;
    uint64_t matrix;
    uint32_t rows, cols, pitch;
    float scale;
  };
  const Params &p;
  uint32_t row, col0;
  size_t base;
  __device__ __forceinline__ NextEpi(const Params &q, uint8_t *, int) : p(q) {}
  __device__ __forceinline__ void begin(const ProductTile &t, uint32_t r, uint32_t c0) {
    row = r;
    col0 = c0;
    base = (size_t)t.batch * p.matrix;
  }
  __device__ __forceinline__ void block(int cg, float (&v)[32]) {
    const uint32_t first = col0 + cg * 32;
    if (first >= p.cols || row >= p.rows) return;
#pragma unroll
    for (int x = 0; x < 32; ++x) v[x] *= p.scale;
    write_parts(p.hi, p.lo, base + (size_t)row * p.pitch + first, v);
  }
  __device__ __forceinline__ void end() {}
};

// X of the last step: written in the caller's type, or applied to the parameter: P <- keep P - step X
struct LastEpi {
  struct Params {
    Targets t;
    uint64_t row_stride;
    uint32_t rows, cols, bf16, vec, apply;
    float scale, keep, step;
  };
  const Params &p;
  float4 *slab;
  int lane;
  uint32_t row0, col0;
  void *out;
  __device__ __forceinline__ LastEpi(const Params &q, uint8_t *sl, int l) : p(q), slab(reinterpret_cast<float4 *>(sl)), lane(l) {}
  __device__ __forceinline__ void begin(const ProductTile &t, uint32_t r, uint32_t c0) {
    row0 = r - lane;
    col0 = c0;
    out = p.t.out[t.batch];
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
      float w[4] = {q[i].x * p.scale, q[i].y * p.scale, q[i].z * p.scale, q[i].w * p.scale};
      const size_t at = (size_t)r * p.row_stride + col;
      if (p.vec && col + 4 <= p.cols) {
        if (p.bf16) {
          uint2 b;
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.x) : "f"(w[1]), "f"(w[0]));
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b.y) : "f"(w[3]), "f"(w[2]));
          *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + at) = b;
        } else {
          float4 *to = reinterpret_cast<float4 *>(static_cast<float *>(out) + at);
          if (p.apply) {
            const float4 old = *to;
            w[0] = fmaf(p.keep, old.x, -p.step * w[0]);
            w[1] = fmaf(p.keep, old.y, -p.step * w[1]);
            w[2] = fmaf(p.keep, old.z, -p.step * w[2]);
            w[3] = fmaf(p.keep, old.w, -p.step * w[3]);
          }
          *to = make_float4(w[0], w[1], w[2], w[3]);
        }
        continue;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (col + x >= p.cols) break;
        if (p.bf16) {
          uint32_t b;
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(0.0f), "f"(w[x]));
          static_cast<uint16_t *>(out)[at + x] = (uint16_t)b;
        } else {
          float *to = static_cast<float *>(out) + at + x;
          *to = p.apply ? fmaf(p.keep, *to, -p.step * w[x]) : w[x];
        }
      }
    }
  }
  __device__ __forceinline__ void end() {}
};

// ---------------------------------------------------------------- host
struct Layout {
  uint64_t x, x_next, g, b, total;  // offsets: parts hi, then lo, of all matrices of a group
  uint64_t x_matrix, g_matrix;      // elements of a matrix
  uint32_t x_pitch, g_pitch, side, group;
};
Layout layout(uint32_t n, uint32_t rows, uint32_t cols) {
  Layout l = {};
  l.side = rows < cols ? rows : cols;
  l.x_pitch = (uint32_t)up(cols, 64);
  l.g_pitch = (uint32_t)up(l.side, 64);
  l.x_matrix = up((uint64_t)rows * l.x_pitch, 128);
  l.g_matrix = up((uint64_t)l.side * l.g_pitch, 128);
  const uint64_t each = 8 * l.x_matrix + 8 * l.g_matrix;
  uint64_t group = kGroupBytes / each;
  if (group > (uint64_t)kMostMatrices) group = kMostMatrices;
  if (group < 1) group = 1;
  l.group = n < group ? n : (uint32_t)group;
  uint64_t at = (uint64_t)kMostMatrices * kNormBlocks * 8;
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

template <bool A_MN, bool B_MN, class Epi>
int product(const Operand &a, const Operand &b, uint32_t M, uint32_t N, uint32_t K, uint32_t batch, bool symmetric, const typename Epi::Params &e, cudaStream_t s) {
  ProductParams p = {};
  p.M = M;
  p.N = N;
  p.batch = (int)batch;
  p.symmetric = symmetric;
  p.n_kb = (int)((K + kProdK - 1) / kProdK);
  p.kb_per_split = p.n_kb;
  p.splits = 1;
  p.chunk = kChunk;
  p.fmt = (uint32_t)kFmtF16;
  // A pair's tile is four of a single CTA's; it takes about as long as two of them (its operands are shared), on twice the SMs.
  auto tiles = [&](uint32_t t) {
    const uint64_t m = (M + t - 1) / t, q = (N + t - 1) / t;
    return (symmetric ? m * (m + 1) / 2 : m * q) * batch;
  };
  const uint64_t n_sm = (uint64_t)sm_count();
  if (n_sm < 2) return DF_ERR_CUDA;
  const uint64_t wide = (tiles(256) + n_sm / 2 - 1) / (n_sm / 2) * 12, narrow = (tiles(128) + n_sm - 1) / n_sm * 10;
  if (wide < narrow) return launch_product<ProdCfg<true, A_MN, B_MN, 2>, Epi>(a, b, p, e, s);
  return launch_product<ProdCfg<false, A_MN, B_MN, 2>, Epi>(a, b, p, e, s);
}

struct Plan {
  uint32_t rows, cols, steps;
  float a, b, c, eps;
  uint8_t *ws;
  Layout l;
  cudaStream_t s;

  Operand parts(uint64_t at, uint64_t rows_, uint64_t cols_, uint64_t pitch, uint64_t matrix) const {
    uint16_t *hi = reinterpret_cast<uint16_t *>(ws + at);
    return {hi, hi + matrix * l.group, false, rows_, cols_, pitch, matrix};
  }

  int run(uint32_t n, UpdateParams u, LastEpi::Params last) const {
    Operand x = parts(l.x, rows, cols, l.x_pitch, l.x_matrix), next = parts(l.x_next, rows, cols, l.x_pitch, l.x_matrix);
    const Operand g = parts(l.g, l.side, l.side, l.g_pitch, l.g_matrix), bb = parts(l.b, l.side, l.side, l.g_pitch, l.g_matrix);
    u.sums = reinterpret_cast<double *>(ws);
    u.hi = static_cast<uint16_t *>(const_cast<void *>(x.hi));
    u.lo = static_cast<uint16_t *>(const_cast<void *>(x.lo));
    u.matrix = l.x_matrix;
    u.rows = rows;
    u.cols = cols;
    u.pitch = l.x_pitch;
    u.eps = eps;
    int st = check_cuda(launch_kernel(k_update, dim3(kNormBlocks, n), dim3(256), 0, s, u));
    if (st != DF_OK) return st;
    const uint64_t quads = (uint64_t)rows * (l.x_pitch / 4);
    const uint32_t blocks = (uint32_t)((quads + 255) / 256 < 512 ? (quads + 255) / 256 : 512);
    st = check_cuda(launch_kernel(k_normalise, dim3(blocks, n), dim3(256), 0, s, u));
    note_launch(2);
    const bool wide = rows <= cols;
    for (uint32_t i = 0; st == DF_OK && i < steps; ++i) {
      SymmetricEpi::Params e = {};
      e.hi = static_cast<uint16_t *>(const_cast<void *>(g.hi));
      e.lo = static_cast<uint16_t *>(const_cast<void *>(g.lo));
      e.matrix = l.g_matrix;
      e.side = l.side;
      e.pitch = l.g_pitch;
      e.c = kPartInverse;  // parts are times 2^12, their product 2^24
      st = wide ? product<false, false, SymmetricEpi>(x, x, l.side, l.side, cols, n, true, e, s)
                : product<true, true, SymmetricEpi>(x, x, l.side, l.side, rows, n, true, e, s);
      if (st != DF_OK) break;
      e.hi = static_cast<uint16_t *>(const_cast<void *>(bb.hi));
      e.lo = static_cast<uint16_t *>(const_cast<void *>(bb.lo));
      e.g_hi = static_cast<const uint16_t *>(g.hi);
      e.g_lo = static_cast<const uint16_t *>(g.lo);
      e.a = a * kPartScale;
      e.b = b;
      e.c = c * kPartInverse;
      st = product<false, false, SymmetricEpi>(g, g, l.side, l.side, l.side, n, true, e, s);
      if (st != DF_OK) break;
      if (i + 1 == steps) {
        last.rows = rows;
        last.cols = cols;
        last.scale = kPartInverse * kPartInverse;
        st = wide ? product<false, true, LastEpi>(bb, x, rows, cols, rows, n, false, last, s) : product<false, false, LastEpi>(x, bb, rows, cols, cols, n, false, last, s);
        break;
      }
      NextEpi::Params f = {};
      f.hi = static_cast<uint16_t *>(const_cast<void *>(next.hi));
      f.lo = static_cast<uint16_t *>(const_cast<void *>(next.lo));
      f.matrix = l.x_matrix;
      f.rows = rows;
      f.cols = cols;
      f.pitch = l.x_pitch;
      f.scale = kPartInverse;
      st = wide ? product<false, true, NextEpi>(bb, x, rows, cols, rows, n, false, f, s) : product<false, false, NextEpi>(x, bb, rows, cols, cols, n, false, f, s);
      const Operand t = x;
      x = next;
      next = t;
    }
    return st;
  }
};

int check_call(uint32_t n, uint32_t rows, uint32_t cols, uint32_t steps, float a, float b, float c, float eps) {
  if (!sizes_ok(n, rows, cols) || steps < 1 || steps > 64) return DF_ERR_INVALID_ARG;
  if (!isfinite(a) || !isfinite(b) || !isfinite(c) || !isfinite(eps) || eps < 0.0f) return DF_ERR_INVALID_ARG;
  // the parts hold values up to 15; |B| is at most this for singular values up to 1
  return fabsf(a) + fabsf(b) + fabsf(c) < 15.0f ? DF_OK : DF_ERR_UNSUPPORTED;
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
  if (n > 1 && out_matrix_stride < (uint64_t)(rows - 1) * out_row_stride + cols) return finish(DF_ERR_INVALID_ARG);
  const Layout l = layout(n, rows, cols);
  if (!workspace || workspace_bytes < l.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return finish(DF_ERR_WORKSPACE);
  const Plan plan = {rows, cols, steps, a, b, c, eps, static_cast<uint8_t *>(workspace), l, static_cast<cudaStream_t>(stream)};
  const uint64_t elt = bf16 ? 2 : 4;
  for (uint32_t i0 = 0; st == DF_OK && i0 < n; i0 += l.group) {
    const uint32_t k = n - i0 < l.group ? n - i0 : l.group;
    UpdateParams u = {};
    LastEpi::Params last = {};
    u.row_stride = update_row_stride;
    u.bf16 = bf16 != 0;
    last.row_stride = out_row_stride;
    last.bf16 = bf16 != 0;
    last.vec = 1;
    for (uint32_t i = 0; i < k; ++i) {
      u.t.source[i] = static_cast<const uint8_t *>(update) + (i0 + i) * update_matrix_stride * elt;
      last.t.out[i] = static_cast<uint8_t *>(out) + (i0 + i) * out_matrix_stride * elt;
      if (!aligned(last.t.out[i], out_row_stride * elt, bf16 ? 8 : 16)) last.vec = 0;
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
  const uint64_t bytes = (uint64_t)rows * cols * 4;
  auto meet = [&](const void *x, const void *y) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(x), v = reinterpret_cast<uintptr_t>(y);
    return u < v + bytes && v < u + bytes;
  };
  for (uint32_t i = 0; i < n; ++i) {  // what is written may not be anything else of the call
    for (uint32_t j = 0; j < n; ++j)
      if (meet(t[i].parameter, t[j].momentum) || meet(t[i].parameter, t[j].gradient) || meet(t[i].momentum, t[j].gradient) ||
          (i < j && (meet(t[i].parameter, t[j].parameter) || meet(t[i].momentum, t[j].momentum))))
        return finish(DF_ERR_INVALID_ARG);
  }
  const Layout l = layout(n, rows, cols);
  if (!workspace || workspace_bytes < l.total || (reinterpret_cast<uintptr_t>(workspace) & 255u)) return finish(DF_ERR_WORKSPACE);
  const Plan plan = {rows, cols, steps, a, b, c, eps, static_cast<uint8_t *>(workspace), l, static_cast<cudaStream_t>(stream)};
  for (uint32_t i0 = 0; st == DF_OK && i0 < n; i0 += l.group) {
    const uint32_t k = n - i0 < l.group ? n - i0 : l.group;
    UpdateParams u = {};
    LastEpi::Params last = {};
    u.row_stride = cols;
    u.beta = momentum;
    u.nesterov = nesterov != 0;
    last.row_stride = cols;
    last.vec = 1;
    last.apply = 1;
    last.keep = (float)(1.0 - (double)lr * (double)weight_decay);
    last.step = lr * update_scale;
    for (uint32_t i = 0; i < k; ++i) {
      u.t.source[i] = t[i0 + i].gradient;
      u.t.momentum[i] = t[i0 + i].momentum;
      last.t.out[i] = t[i0 + i].parameter;
      if (!aligned(last.t.out[i], (uint64_t)cols * 4, 16)) last.vec = 0;
    }
    st = plan.run(k, u, last);
  }
  return finish(st);
}

}  // extern "C"
