// cache_append.cu - K and V rows of new tokens into the 8-bit paged cache, for B200 (sm_100a).
//
// Per page and head, over all tokens that the page has by now:
//   need = 2^e, the smallest e >= -126 with amax <= Q 2^e   (Q = 127: int8, 448: e4m3)      scale = max(need, the scale that the page has)
//   code = round_to_even(x / scale)                          older codes of a page whose scale grew: round_to_even(c * old / scale)
// A power of two makes every step exact but the one rounding to the code: dividing by it changes no bit of the fraction, and a code that
// is rounded again when the scale doubles lands within half a step of the new scale; over any number of doublings the errors add to less than one
// step (1/2 + 1/4 + ...). A scale of amax / Q would be up to a factor of two finer but would round every older code again with almost every
// new largest element.
//
// The tokens of one page form a run of the slot map (row, row + 1, ... of one page). A warp takes a run, one head, and K or V, so that everything that
// shares a scale is one warp's and nothing is exchanged; its first slot says how many rows the page had. Rows are read once (up to
// kHeld rows' elements stay in registers between the maximum and the rounding), codes written once: 8205 tokens of 12 heads of 64, fp32 to int8, 63 MB in 18 us, 3.5
// TB/s (53 % of a copy's rate). What is missing is the second round: 6168 warps of which 24 an SM are there at once are 1.7 rounds of a chain slots ->
// rows -> maximum -> codes (56 % of the issue slots in use, an instruction waits for loads three times as long as for its slot). bf16: 1.3 rounds, the same time for
// 38 MB. A page whose scale grows has its older codes rounded again, word after word of a lane: 4096 single tokens of 8 heads of 128 take 25 us (floor 4), 130 if all
// of their pages' scales grow in the same call.
#include <math.h>

#include "cache_codes.cuh"
#include "sm100_ptx.cuh"

namespace df {
namespace {

constexpr int kAppendThreads = 128;

struct AppendParams {
  const void *src[2];  // k, v
  uint8_t *cache[2];
  float *scale[2];
  const int32_t *slots;
  unsigned long long stride[2];
  uint32_t n_tokens, H, D, P, n_pages;
  uint32_t per_warp;   // slots that a warp looks through for the beginnings of runs
  uint32_t aligned[2]; // rows start on boundaries of four elements
};

// Four elements of a row, as they lie there (half the registers for bf16) and as numbers.
template <bool BF16>
struct Raw4 {
  uint32_t w[BF16 ? 2 : 4];
};
template <bool BF16>
__device__ __forceinline__ Raw4<BF16> load4(const void *base, unsigned long long e, bool aligned) {
  Raw4<BF16> r;
  if constexpr (BF16) {
    const uint16_t *p = static_cast<const uint16_t *>(base) + e;
    if (aligned) {
      const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
      r.w[0] = v.x; r.w[1] = v.y;
    } else {
      r.w[0] = __ldg(p) | ((uint32_t)__ldg(p + 1) << 16);
      r.w[1] = __ldg(p + 2) | ((uint32_t)__ldg(p + 3) << 16);
    }
  } else {
    const uint32_t *p = static_cast<const uint32_t *>(base) + e;
    if (aligned) {
      const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
      r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = __ldg(p + i);
    }
  }
  return r;
}
template <bool BF16>
__device__ __forceinline__ float4 numbers(const Raw4<BF16> &r) {
  if constexpr (BF16)
    return make_float4(__uint_as_float(r.w[0] << 16), __uint_as_float(r.w[0] & 0xffff0000u), __uint_as_float(r.w[1] << 16), __uint_as_float(r.w[1] & 0xffff0000u));
  else
    return make_float4(__uint_as_float(r.w[0]), __uint_as_float(r.w[1]), __uint_as_float(r.w[2]), __uint_as_float(r.w[3]));
}

__device__ __forceinline__ uint32_t largest(uint32_t m, const float4 &x) {  // of the magnitudes, as bits: infinities and NaN come out on top
  m = max(m, max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu));
  return max(m, max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
}

// the smallest power of two that holds amax (its bits); NaN for infinities and NaN
template <int FORMAT>
__device__ __forceinline__ float scale_for(uint32_t amax) {
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  constexpr uint32_t kFraction = FORMAT == DF_CACHE_INT8 ? 0x7e0000u : 0x600000u;  // 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
  constexpr int kExponent = FORMAT == DF_CACHE_INT8 ? 6 : 8;
  const int e = (int)(amax >> 23) - kExponent + ((amax & 0x7fffffu) > kFraction ? 1 : 0);  // biased by 127
  return __uint_as_float((uint32_t)(e < 1 ? 1 : e) << 23);
}

// four values, already divided by their scale
template <int FORMAT>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  if (FORMAT == DF_CACHE_INT8) {
    auto code = [](float x) { return (uint32_t)(__float2int_rn(fminf(fmaxf(x, -127.0f), 127.0f)) & 0xff); };
    return code(a) | (code(b) << 8) | (code(c) << 16) | (code(d) << 24);
  }
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// kHeld: turns of the warp whose elements stay in registers: those of 16 tokens (two to a turn up to 64 dims, one beyond).
template <bool BF16, int FORMAT, int kHeld>
__global__ void __launch_bounds__(kAppendThreads, BF16 ? (kHeld == 8 ? 8 : 6) : (kHeld == 8 ? 6 : 4)) k_cache_append(const AppendParams p) {
  ptx::pdl_wait();
  const uint32_t lane = threadIdx.x & 31;
  const unsigned long long warp = (unsigned long long)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const uint32_t which = (uint32_t)(warp % (2 * p.H)), h = which >> 1, kv = which & 1;
  const unsigned long long first = warp / (2 * p.H) * p.per_warp;
  if (first >= p.n_tokens) return;
  const uint32_t t_end = (uint32_t)min((unsigned long long)p.n_tokens, first + p.per_warp);
  // a row takes D / 4 lanes, rounded up to a power of two
  uint32_t lanes = 4;
  while (lanes * 4 < p.D) lanes *= 2;
  const uint32_t turn = 32 / lanes, sub = lane / lanes, x = lane % lanes * 4;
  const bool in_row = x < p.D;
  const long long n_slots = (long long)p.n_pages * p.P;
  const void *src = kv ? p.src[1] : p.src[0];  // (no indexed access: it would put the parameters on the stack)
  uint8_t *cache = kv ? p.cache[1] : p.cache[0];
  float *scales = kv ? p.scale[1] : p.scale[0];
  const unsigned long long stride = kv ? p.stride[1] : p.stride[0];
  const bool aligned = (kv ? p.aligned[1] : p.aligned[0]) != 0;
  // the warp's window of slots, one to a lane, and the beginnings of runs in it
  const uint32_t t0 = (uint32_t)first, window = t_end - t0;
  const bool in_window = lane < window;
  const int32_t my_slot = in_window ? __ldg(p.slots + t0 + lane) : -1;
  int32_t before = __shfl_up_sync(0xffffffffu, my_slot, 1);
  if (lane == 0) before = t0 > 0 ? __ldg(p.slots + t0 - 1) : -2;
  const bool valid = my_slot >= 0 && my_slot < n_slots;
  const uint32_t my_page = (uint32_t)my_slot / p.P, my_row = (uint32_t)my_slot - my_page * p.P;
  const bool goes_on = valid && my_row > 0 && before == my_slot - 1;
  const uint32_t going_on = __ballot_sync(0xffffffffu, goes_on);
  // A run's first turn and the scale that its page has are loaded while the run before it is worked on: a decode step's runs are of
  // one token each, and their loads would otherwise follow one another (4096 tokens of 8 heads of 128: 57 us, 25 this way).
  struct Run {
    uint32_t at, page, row, n;
    int32_t slot;
    float old;
    Raw4<BF16> first;
  };
  const unsigned long long e0 = (unsigned long long)h * p.D + x;
  auto begin = [&](uint32_t at) {
    Run r;
    r.at = at;
    r.slot = __shfl_sync(0xffffffffu, my_slot, at);
    r.page = __shfl_sync(0xffffffffu, my_page, at);
    r.row = __shfl_sync(0xffffffffu, my_row, at);
    r.n = 1 + (at == 31 ? 0u : __ffs(~(going_on >> (at + 1))) - 1);  // (bits above the window are 0)
    r.old = r.row > 0 ? scales[(size_t)r.page * p.H + h] : 0.0f;
    r.first = Raw4<BF16>{};
    if (in_row && sub < r.n) r.first = load4<BF16>(src, (unsigned long long)(t0 + at + sub) * stride + e0, aligned);
    return r;
  };
  uint32_t begins = __ballot_sync(0xffffffffu, valid && !goes_on);
  if (!begins) return;
  Run next = begin(__ffs(begins) - 1);
  while (begins) {
    const Run run = next;
    begins &= begins - 1;
    if (begins) next = begin(__ffs(begins) - 1);
    const uint32_t at = run.at, t = t0 + at, page = run.page, row = run.row;
    const int32_t slot = run.slot;
    uint32_t n = run.n;
    while (at + n >= window) {  // the run may go on behind the window
      const uint32_t i = n + lane;
      const bool in = row + i < p.P && t + i < p.n_tokens && __ldg(p.slots + t + i) == slot + (int32_t)i;
      const uint32_t together = __ballot_sync(0xffffffffu, in);
      if (together != 0xffffffffu) {
        n += __ffs(~together) - 1;
        break;
      }
      n += 32;
    }
    auto element = [&](uint32_t i) { return (unsigned long long)(t + i) * stride + e0; };
    Raw4<BF16> held[kHeld];
    held[0] = run.first;
    if (sub >= run.n && sub < n && in_row) held[0] = load4<BF16>(src, element(sub), aligned);
    uint32_t amax = 0;
    if (n > turn) {
#pragma unroll
      for (int i = 1; i < kHeld; ++i) {
        const uint32_t r = i * turn + sub;
        if (in_row && r < n) held[i] = load4<BF16>(src, element(r), aligned);
        else held[i] = Raw4<BF16>{};
      }
#pragma unroll
      for (int i = 1; i < kHeld; ++i) amax = largest(amax, numbers(held[i]));
    }
    amax = largest(amax, numbers(held[0]));
    for (uint32_t r = kHeld * turn + sub; r < n; r += turn)
      if (in_row) amax = largest(amax, numbers(load4<BF16>(src, element(r), aligned)));
    amax = __reduce_max_sync(0xffffffffu, amax);
    float *scale_at = scales + (size_t)page * p.H + h;
    uint8_t *slice = cache + ((size_t)page * p.H + h) * p.P * p.D;
    float scale = scale_for<FORMAT>(amax);
    if (row > 0) {
      const float old = run.old;
      if (!(old <= scale)) scale = isnan(scale) ? scale : old;  // larger already, or NaN
      if (old < scale) {                                        // the older rows' codes, in steps of the new scale
        const float ratio = old / scale;
        uint32_t *words = reinterpret_cast<uint32_t *>(slice);
        for (uint32_t i = lane; i < row * p.D / 4; i += 32) {
          const uint32_t w = words[i];
          words[i] = to_codes<FORMAT>(cache_value<FORMAT>(w & 0xff) * ratio, cache_value<FORMAT>((w >> 8) & 0xff) * ratio,
                                      cache_value<FORMAT>((w >> 16) & 0xff) * ratio, cache_value<FORMAT>(w >> 24) * ratio);
        }
      }
    }
    if (lane == 0) *scale_at = scale;
    const bool poisoned = isnan(scale);
    // Dividing by a power of two is multiplying by its inverse; a scale of the caller's own may be another number.
    const uint32_t scale_bits = __float_as_uint(scale);
    const bool power = (scale_bits & 0x7fffffu) == 0 && scale_bits >= 0x00800000u && scale_bits < 0x7f000000u;
    const float inverse = __uint_as_float(0x7f000000u - scale_bits);
    auto put = [&](uint32_t r, const float4 &v) {
      uint32_t w = 0u;
      if (power) w = to_codes<FORMAT>(v.x * inverse, v.y * inverse, v.z * inverse, v.w * inverse);
      else if (!poisoned) w = to_codes<FORMAT>(v.x / scale, v.y / scale, v.z / scale, v.w / scale);
      *reinterpret_cast<uint32_t *>(slice + (size_t)(row + r) * p.D + x) = w;
    };
    if (in_row && sub < n) put(sub, numbers(held[0]));
    if (n > turn) {
#pragma unroll
      for (int i = 1; i < kHeld; ++i)
        if (in_row && i * turn + sub < n) put(i * turn + sub, numbers(held[i]));
    }
    for (uint32_t r = kHeld * turn + sub; r < n; r += turn)
      if (in_row) put(r, numbers(load4<BF16>(src, element(r), aligned)));
  }
}

int finish(int st) {
  note_status(st);
  return st;
}

template <bool BF16, int FORMAT>
int launch(AppendParams &p, cudaStream_t s) {
  // A slot to a warp while that leaves no more than 32 warps an SM (16 to 32 of them are there at once, by the variant's registers), else windows of up to 32 slots: in a
  // prompt only every 16th slot or so begins a run, and warps that find none cost more than the others' work (8205 tokens of 12 heads: 110 us with a slot
  // to a warp, 18 with windows). 64 tokens of 8 heads, a warp each: 3.4 us, of which 2.4 are a launch.
  const int n_sm = sm_count();
  if (n_sm == 0) return DF_ERR_CUDA;
  const unsigned long long all = (unsigned long long)p.n_tokens * 2 * p.H, two_rounds = 32ull * (unsigned)n_sm;
  p.per_warp = all <= two_rounds ? 1u : all >= 32 * two_rounds ? 32u : (uint32_t)((all + two_rounds - 1) / two_rounds);
  const unsigned long long warps = (p.n_tokens + p.per_warp - 1ull) / p.per_warp * 2 * p.H;
  const unsigned long long blocks = (warps + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (blocks > 0x7fffffffull) return DF_ERR_UNSUPPORTED;
  const int st = check_cuda(launch_kernel(p.D <= 64 ? k_cache_append<BF16, FORMAT, 8> : k_cache_append<BF16, FORMAT, 16>, dim3((unsigned)blocks), dim3(kAppendThreads), 0, s, p));
  note_launch();
  return st;
}

}  // namespace
}  // namespace df

using namespace df;

extern "C" int df_cache_append(const void *k, const void *v, const int32_t *slots, void *k_cache, void *v_cache, float *k_scale, float *v_scale,
                               uint32_t n_tokens, uint32_t n_kv_heads, uint32_t d_head, uint32_t page_size, uint32_t n_pages,
                               uint64_t k_row_stride, uint64_t v_row_stride, uint32_t kv_bf16, uint32_t format, void *stream) {
  DF_RANGE("df_cache_append");
  if (!cache_shape_valid(n_kv_heads, d_head, page_size, n_pages) || n_tokens >= (1u << 31)) return finish(DF_ERR_INVALID_ARG);
  if (format != DF_CACHE_INT8 && format != DF_CACHE_E4M3) return finish(DF_ERR_INVALID_ARG);
  const uint64_t width = (uint64_t)n_kv_heads * d_head;
  if (n_tokens > 1 && (k_row_stride < width || v_row_stride < width)) return finish(DF_ERR_INVALID_ARG);
  if (!cache_shape_supported(d_head, page_size)) return finish(DF_ERR_UNSUPPORTED);
  if (n_tokens == 0) return DF_OK;
  if (!k || !v || !slots || (n_pages && (!k_cache || !v_cache || !k_scale || !v_scale))) return finish(DF_ERR_INVALID_ARG);
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15u) != 0) return finish(DF_ERR_UNSUPPORTED);
  const uintptr_t elt = kv_bf16 ? 2 : 4;
  auto aligned = [&](const void *src, uint64_t stride) { return (reinterpret_cast<uintptr_t>(src) | (uintptr_t)(stride * elt)) % (4 * elt) == 0 ? 1u : 0u; };
  AppendParams p = {{k, v}, {static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache)}, {k_scale, v_scale}, slots, {k_row_stride, v_row_stride},
                    n_tokens, n_kv_heads, d_head, page_size, n_pages, 1, {aligned(k, k_row_stride), aligned(v, v_row_stride)}};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv_bf16) return finish(format == DF_CACHE_INT8 ? launch<true, DF_CACHE_INT8>(p, s) : launch<true, DF_CACHE_E4M3>(p, s));
  return finish(format == DF_CACHE_INT8 ? launch<false, DF_CACHE_INT8>(p, s) : launch<false, DF_CACHE_E4M3>(p, s));
}
