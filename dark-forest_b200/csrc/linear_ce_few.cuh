// linear_ce_few.cuh — the loss from hidden states and its gradient for few rows (linear_ce.cu chooses). Then reading the weight, and writing its gradient, is all there is
// to do: products are fp32 multiply-adds on the weight as it lies in memory, no tensor cores and no copies.
//   k_few_logits     a warp takes four rows of the weight at a time, its lanes four columns each, against up to 16 rows of x in shared memory (four rows, so that a
//                    value of x is read once for four products). 4 R sums a lane become whole sums by halving: a lane gives away half of what it has left at each of
//                    five exchanges. Forward: the largest logit and the sum of exponentials of every row and CTA, for k_join; backward: G in fp32, [rows][vocab].
//   k_few_gradients  a thread has four columns: down a range of the weight's rows it adds up d_x = G w (a plane of sums per range) and forms d_w = G^T x'.
#pragma once

namespace df {
namespace {

constexpr uint32_t kFewMost = 16, kFewGradMost = 8;  // rows of x, in either direction
constexpr uint32_t kFewRanges = 128;       // planes of d_x
constexpr uint32_t kFewSmem = 200 * 1024;  // of x

struct FewParams {
  const void *x, *w;
  const int32_t *targets;
  uint64_t x_stride, w_stride;
  uint32_t rows, vocab, width, padded, rows_pad, wide;  // padded: width up to a multiple of 128; wide: four elements of a row at a time
  float scale;
  float2 *parts;     // forward
  float *picked;
  const float *lse;  // backward
  float *g;
};

template <bool BF16>
__device__ __forceinline__ float4 few_load(const void *base, size_t row, uint32_t k, uint32_t width, bool wide) {
  if (wide && k + 4 <= width) {
    if constexpr (BF16) {
      const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + row + k);
      return make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u));
    } else {
      return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + row + k);
    }
  }
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (k < width) v.x = load_f(base, BF16, row + k);
  if (k + 1 < width) v.y = load_f(base, BF16, row + k + 1);
  if (k + 2 < width) v.z = load_f(base, BF16, row + k + 2);
  if (k + 3 < width) v.w = load_f(base, BF16, row + k + 3);
  return v;
}

template <bool BF16, int R, bool GRAD>
__global__ void __launch_bounds__(256) k_few_logits(const FewParams p) {
  pdl_wait();
  extern __shared__ float xs[];  // [R][padded]
  __shared__ float2 s_part[8][R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row0 = blockIdx.y * R;
  for (uint32_t i = threadIdx.x; i < R * (p.padded / 4); i += 256) {
    const uint32_t r = i / (p.padded / 4), k = i % (p.padded / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row0 + r < p.rows && (uint32_t)p.targets[row0 + r] < p.vocab) v = few_load<BF16>(p.x, (size_t)(row0 + r) * p.x_stride, k, p.width, p.wide);
    *reinterpret_cast<float4 *>(xs + (size_t)r * p.padded + k) = v;
  }
  // whole sums: this lane's are of weight row lane / 8 of the four, and of x's rows first .. first + kOwn - 1
  constexpr int N = 4 * R, kOwn = R > 8 ? R / 8 : 1;
  const int j = lane >> 3, first = (lane & 7) * R / 8;
  const bool mine = R >= 8 || (lane & (8 / (R < 8 ? R : 8) - 1)) == 0;
  int target[kOwn];
  float off[kOwn], m[kOwn], s[kOwn];
  const float c = exponent_factor(p.scale);
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const uint32_t r = row0 + first + o;
    target[o] = r < p.rows ? p.targets[r] : -1;
    off[o] = GRAD && (uint32_t)target[o] < p.vocab ? p.lse[r] : 0.0f;
    m[o] = -INFINITY;
    s[o] = 0.0f;
  }
  __syncthreads();
  for (uint32_t v0 = (blockIdx.x * 8 + warp) * 4; v0 < p.vocab; v0 += gridDim.x * 32) {
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.0f;
#pragma unroll 2
    for (uint32_t k = lane * 4; k < p.padded; k += 128) {
      float4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = v0 + i < p.vocab ? few_load<BF16>(p.w, (size_t)(v0 + i) * p.w_stride, k, p.width, p.wide) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 x = *reinterpret_cast<const float4 *>(xs + (size_t)r * p.padded + k);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i * R + r] = fmaf(w[i].x, x.x, fmaf(w[i].y, x.y, fmaf(w[i].z, x.z, fmaf(w[i].w, x.w, acc[i * R + r]))));
      }
    }
    int n = N;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      if (n > 1) {
        n /= 2;
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
          if (i < n) {
            const bool high = (lane & d) != 0;
            const float give = high ? acc[i] : acc[i + n], keep = high ? acc[i + n] : acc[i];
            acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
          }
      } else {
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], d);
      }
    }
    const uint32_t v = v0 + j;
    if (v >= p.vocab || !mine) continue;
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      const uint32_t r = row0 + first + o;
      if (r >= p.rows) continue;
      if constexpr (GRAD) {
        const float t = at_most_0(fmaf(acc[o], p.scale, -off[o]));  // as in linear_ce.cu
        const float e = (uint32_t)target[o] == v ? expm1f(t) : ex2_approx(t * kLog2e);
        p.g[(size_t)r * p.vocab + v] = (uint32_t)target[o] < p.vocab ? e : 0.0f;
      } else {
        const float top = fmaxf(m[o], acc[o]), ref = top == -INFINITY ? 0.0f : top;
        s[o] = s[o] * ex2_approx((m[o] - ref) * c) + ex2_approx((acc[o] - ref) * c);
        m[o] = top;
        if ((uint32_t)target[o] == v) p.picked[r] = acc[o];
      }
    }
  }
  if constexpr (!GRAD) {
    auto join = [&](float &ma, float &sa, float mb, float sb) {
      const float top = fmaxf(ma, mb), ref = top == -INFINITY ? 0.0f : top;
      sa = sa * ex2_approx((ma - ref) * c) + sb * ex2_approx((mb - ref) * c);
      ma = top;
    };
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
#pragma unroll
      for (int d = 8; d <= 16; d <<= 1) {
        const float mb = __shfl_xor_sync(0xffffffffu, m[o], d), sb = __shfl_xor_sync(0xffffffffu, s[o], d);
        join(m[o], s[o], mb, sb);
      }
      if (j == 0 && mine) s_part[warp][first + o] = make_float2(m[o], s[o]);
    }
    __syncthreads();
    if (threadIdx.x < R && row0 + threadIdx.x < p.rows) {
      float ma = -INFINITY, sa = 0.0f;
      for (int i = 0; i < 8; ++i) join(ma, sa, s_part[i][threadIdx.x].x, s_part[i][threadIdx.x].y);
      p.parts[(size_t)blockIdx.x * p.rows_pad + row0 + threadIdx.x] = make_float2(ma, sa);
    }
  }
}

struct FewGradParams {
  const void *x, *w;
  const int32_t *targets;
  const float *g, *grad;
  void *d_w;      // null: not wanted
  float *planes;  // [ranges][rows][pitch]; null: not wanted
  uint64_t x_stride, w_stride, dw_stride;
  uint32_t rows, vocab, width, pitch, range, wide, dw_wide;
  float scale;
};

// A CTA has 256 columns, a thread four of them (16 bytes of the weight at a time), and its four pairs of warps every fourth row of the range.
template <bool BF16, int R>
__global__ void __launch_bounds__(256) k_few_gradients(const FewGradParams p) {
  pdl_wait();
  constexpr uint32_t kAt = 128, kAhead = 8;  // rows of the weight whose G lies in shared memory; that a thread has under way
  __shared__ __align__(16) float gs[kAt][R];
  __shared__ __align__(16) float part[R][256];  // the sums of the other pairs of warps
  const uint32_t sub = threadIdx.x >> 6, mine = (threadIdx.x & 63) * 4, col = blockIdx.y * 256 + mine;
  const uint32_t from = blockIdx.x * p.range, to = from + p.range < p.vocab ? from + p.range : p.vocab;
  float4 xr[R], acc[R];  // x' = scale grad x
#pragma unroll
  for (int r = 0; r < R; ++r) {
    acc[r] = xr[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    if ((uint32_t)r < p.rows && (uint32_t)p.targets[r] < p.vocab && col < p.width) {
      const float4 x = few_load<BF16>(p.x, (size_t)r * p.x_stride, col, p.width, p.wide);
      const float g = p.grad[r] * p.scale;
      xr[r] = make_float4(x.x * g, x.y * g, x.z * g, x.w * g);
    }
  }
  for (uint32_t v0 = from; v0 < to; v0 += kAt) {
    const uint32_t n = to - v0 < kAt ? to - v0 : kAt;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < R * kAt; i += 256) {
      const uint32_t r = i / kAt, v = i % kAt;
      gs[v][r] = r < p.rows && v < n ? p.g[(size_t)r * p.vocab + v0 + v] : 0.0f;
    }
    __syncthreads();
    if (col >= p.width) continue;
    for (uint32_t v1 = sub; v1 < n; v1 += 4 * kAhead) {
      float4 w[kAhead];  // before any store: the compiler cannot know that d_w is elsewhere
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i)
        w[i] = p.planes && v1 + 4 * i < n ? few_load<BF16>(p.w, (size_t)(v0 + v1 + 4 * i) * p.w_stride, col, p.width, p.wide) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        const uint32_t v = v1 + 4 * i;
        if (v >= n) break;
        float4 d = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float g = gs[v][r];
          acc[r] = make_float4(fmaf(g, w[i].x, acc[r].x), fmaf(g, w[i].y, acc[r].y), fmaf(g, w[i].z, acc[r].z), fmaf(g, w[i].w, acc[r].w));
          d = make_float4(fmaf(g, xr[r].x, d.x), fmaf(g, xr[r].y, d.y), fmaf(g, xr[r].z, d.z), fmaf(g, xr[r].w, d.w));
        }
        if (p.d_w) write_four(p.d_w, (size_t)(v0 + v) * p.dw_stride + col, d, p.width - col, BF16, p.dw_wide);
      }
    }
  }
  if (!p.planes) return;
  for (uint32_t other = 1; other < 4; ++other) {  // the four parts in their order
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (sub == other) *reinterpret_cast<float4 *>(&part[r][mine]) = acc[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float4 x = *reinterpret_cast<const float4 *>(&part[r][mine]);
      if (sub == 0) acc[r] = make_float4(acc[r].x + x.x, acc[r].y + x.y, acc[r].z + x.z, acc[r].w + x.w);
    }
  }
  if (sub != 0 || col >= p.width) return;
#pragma unroll
  for (int r = 0; r < R; ++r)  // the pitch is a multiple of 64
    if ((uint32_t)r < p.rows) *reinterpret_cast<float4 *>(p.planes + ((size_t)blockIdx.x * p.rows + r) * p.pitch + col) = acc[r];
}

template <auto Kernel>
int launch_few(const FewParams &p, dim3 grid, uint32_t smem, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (check_cuda(cudaGetDevice(&dev)) != DF_OK || dev < 0 || dev >= 64) return DF_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (check_cuda(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewSmem)) != DF_OK) return DF_ERR_CUDA;
    ready[dev].store(true, std::memory_order_release);
  }
  const int st = check_cuda(launch_kernel(Kernel, grid, dim3(256), smem, s, p));
  note_launch();
  return st;
}
template <bool BF16, bool GRAD>
int launch_few_logits(const FewParams &p, uint32_t blocks, cudaStream_t s) {
  const uint32_t r = p.rows <= 1 ? 1 : p.rows <= 2 ? 2 : p.rows <= 4 ? 4 : p.rows <= 8 ? 8 : 16, smem = r * p.padded * 4;
  const dim3 grid(blocks, (p.rows + r - 1) / r);
  switch (r) {
    case 1: return launch_few<k_few_logits<BF16, 1, GRAD>>(p, grid, smem, s);
    case 2: return launch_few<k_few_logits<BF16, 2, GRAD>>(p, grid, smem, s);
    case 4: return launch_few<k_few_logits<BF16, 4, GRAD>>(p, grid, smem, s);
    case 8: return launch_few<k_few_logits<BF16, 8, GRAD>>(p, grid, smem, s);
    default: return launch_few<k_few_logits<BF16, 16, GRAD>>(p, grid, smem, s);
  }
}
template <bool BF16>
int launch_few_gradients(const FewGradParams &p, cudaStream_t s) {
  const dim3 grid((p.vocab + p.range - 1) / p.range, (p.width + 255) / 256);
  const int st = check_cuda(p.rows <= 4 ? launch_kernel(k_few_gradients<BF16, 4>, grid, dim3(256), 0, s, p)
                            : launch_kernel(k_few_gradients<BF16, 8>, grid, dim3(256), 0, s, p));
  note_launch();
  return st;
}

}  // namespace
}  // namespace df
