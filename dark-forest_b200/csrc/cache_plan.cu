// cache_plan.cu - block tables, slot maps and page accounting of a paged cache, for a whole step of requests in one launch (sm_100a).
//
// With len_r cached and new_r coming tokens, pages of P tokens, has_r = ceil(len_r / P) and need_r = ceil((len_r + new_r) / P) - has_r:
//   starts_r = sum_{i<r} new_i        first_r = sum_{i<r} need_i
//   page j of request r's need  = free_pages[*free_count - 1 - (first_r + j)]   -> block_table[r][has_r + j]
//   token j of request r        = position len_r + j, slot = page(position / P) * P + position % P
// The step moves a few hundred KB at most, so what it costs is a launch and the latency of its dependent loads. Two sums over the requests
// decide everything else: every block forms them itself (they come out of L2, 4 to 64 KB) rather than
// waiting for another block, and then writes its share of tokens and pages, whose request it finds by bisection in the
// sums, which lie in shared memory. No block reads what another writes: a table entry that a token needs is an old one, or is taken from
// the free pages again.
#include <initializer_list>
#include <mutex>

#include "df_common.cuh"
#include "sm100_ptx.cuh"

namespace df {
namespace {

constexpr uint32_t kMaxRequests = 16384;  // two sums of 4 bytes each in shared memory

struct PlanParams {
  const int32_t *lens, *new_tokens, *free_pages, *free_count;
  int32_t *block_table, *lens_out, *starts, *slots, *positions, *state;
  uint32_t n_requests, n_tokens, table_width, page_size, n_pages;
};

struct Sums {
  unsigned long long tokens, pages;
};

// Exclusive sums over the block's threads; *total gets the sums over all of them. One warp's lanes, then the warps.
template <int kThreads>
__device__ __forceinline__ Sums block_exclusive(Sums v, Sums *total) {
  __shared__ Sums warp_sum[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffu, in.tokens, o), p = __shfl_up_sync(0xffffffffu, in.pages, o);
    if (lane >= o) { in.tokens += t; in.pages += p; }
  }
  if (lane == 31) warp_sum[warp] = in;
  __syncthreads();
  Sums before = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) before = all;
    all.tokens += warp_sum[w].tokens;
    all.pages += warp_sum[w].pages;
  }
  *total = all;
  return {before.tokens + in.tokens - v.tokens, before.pages + in.pages - v.pages};
}

__device__ __forceinline__ uint32_t count_of(const int32_t *p) {  // negative lengths count as none
  const int32_t n = __ldg(p);
  return n > 0 ? (uint32_t)n : 0u;
}

// The last r < n with sum[r] <= at, where sum[0] = 0 <= at: the request that element `at` of the concatenation belongs to (empty ones are passed over).
__device__ __forceinline__ uint32_t owner_of(const uint32_t *sum, uint32_t n, uint32_t at) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (sum[mid] <= at) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) k_cache_plan(const PlanParams p) {
  ptx::pdl_wait();
  extern __shared__ uint32_t sums[];  // [n_requests] tokens, [n_requests] pages: exclusive
  __shared__ uint32_t first_bad;
  uint32_t *token_sum = sums, *page_sum = sums + p.n_requests;
  const uint32_t t = threadIdx.x, R = p.n_requests, P = p.page_size;
  if (t == 0) first_bad = ~0u;
  const uint32_t per = (R + kThreads - 1) / kThreads, r0 = min(R, t * per), r1 = min(R, r0 + per);
  const uint32_t free_count = min(count_of(p.free_count), p.n_pages);
  auto need_of = [&](uint32_t len, uint32_t n) {
    return (unsigned long long)(((unsigned long long)len + n + P - 1) / P) - (len + (unsigned long long)P - 1) / P;
  };
  Sums mine = {0, 0}, all;
  for (uint32_t r = r0; r < r1; ++r) {
    const uint32_t len = count_of(p.lens + r), n = count_of(p.new_tokens + r);
    mine.tokens += n;
    mine.pages += need_of(len, n);
  }
  Sums at = block_exclusive<kThreads>(mine, &all);
  for (uint32_t r = r0; r < r1; ++r) {
    const uint32_t len = count_of(p.lens + r), n = count_of(p.new_tokens + r);
    token_sum[r] = (uint32_t)min(at.tokens, (unsigned long long)p.n_tokens);
    page_sum[r] = (uint32_t)min(at.pages, 0xffffffffull);
    at.tokens += n;
    at.pages += need_of(len, n);
    if ((unsigned long long)len + n > (unsigned long long)p.table_width * P || at.tokens > p.n_tokens) atomicMin(&first_bad, r);
  }
  __syncthreads();
  const bool granted = first_bad == ~0u && all.pages <= free_count;
  const uint32_t me = blockIdx.x * kThreads + t, step = gridDim.x * kThreads;
  for (uint32_t r = me; r < R; r += step) {
    const uint32_t n = granted ? count_of(p.new_tokens + r) : 0u;
    p.lens_out[r] = (int32_t)(count_of(p.lens + r) + n);
    p.starts[r] = (int32_t)token_sum[r];
  }
  if (me == 0) {
    p.starts[R] = (int32_t)min(all.tokens, (unsigned long long)p.n_tokens);
    p.state[0] = (int32_t)(granted ? free_count - (uint32_t)all.pages : free_count);
    p.state[1] = granted ? 0 : first_bad != ~0u ? -1 - (int32_t)first_bad : (int32_t)min(all.pages - free_count, 0x7fffffffull);
  }
  const uint32_t tokens = granted ? (uint32_t)all.tokens : 0u, pages = granted ? (uint32_t)all.pages : 0u;
  for (uint32_t i = me; i < pages; i += step) {
    const uint32_t r = owner_of(page_sum, R, i), has = (count_of(p.lens + r) + P - 1) / P;
    p.block_table[(size_t)r * p.table_width + has + (i - page_sum[r])] = __ldg(p.free_pages + (free_count - 1 - i));
  }
  for (uint32_t i = me; i < p.n_tokens; i += step) {
    int32_t slot = -1, position = -1;
    if (i < tokens) {
      const uint32_t r = owner_of(token_sum, R, i), len = count_of(p.lens + r), has = (len + P - 1) / P;
      const uint32_t pos = len + (i - token_sum[r]), block = pos / P;
      // an entry of the table from before this step, or one of the pages that the loop above puts there
      const int32_t page = block < has ? p.block_table[(size_t)r * p.table_width + block] : __ldg(p.free_pages + (free_count - 1 - (page_sum[r] + (block - has))));
      slot = page * (int32_t)P + (int32_t)(pos - block * P);
      position = (int32_t)pos;
    }
    p.slots[i] = slot;
    p.positions[i] = position;
  }
}

// Pages of finished requests, in the order of the requests and of their tokens, go behind the free ones. One sum decides where.
template <int kThreads>
__global__ void __launch_bounds__(kThreads) k_cache_release(const int32_t *__restrict__ lens, const int32_t *__restrict__ finished,
                                                            const int32_t *__restrict__ block_table, int32_t *__restrict__ free_pages,
                                                            const int32_t *__restrict__ free_count, int32_t *__restrict__ lens_out,
                                                            int32_t *__restrict__ count_out, uint32_t R, uint32_t table_width, uint32_t P,
                                                            uint32_t n_pages) {
  ptx::pdl_wait();
  extern __shared__ uint32_t page_sum[];
  const uint32_t t = threadIdx.x;
  const uint32_t per = (R + kThreads - 1) / kThreads, r0 = min(R, t * per), r1 = min(R, r0 + per);
  const uint32_t count = min(count_of(free_count), n_pages);
  auto held = [&](uint32_t r) {
    const unsigned long long n = (count_of(lens + r) + (unsigned long long)P - 1) / P;
    return __ldg(finished + r) != 0 ? min(n, (unsigned long long)table_width) : 0ull;
  };
  Sums mine = {0, 0}, all;
  for (uint32_t r = r0; r < r1; ++r) mine.pages += held(r);
  Sums at = block_exclusive<kThreads>(mine, &all);
  for (uint32_t r = r0; r < r1; ++r) {
    page_sum[r] = (uint32_t)min(at.pages, 0xffffffffull);
    at.pages += held(r);
  }
  __syncthreads();
  // more pages than there are: lengths and tables that contradict each other; what does not fit is dropped
  const uint32_t pages = (uint32_t)min(all.pages, (unsigned long long)(n_pages - count));
  const uint32_t me = blockIdx.x * kThreads + t, step = gridDim.x * kThreads;
  for (uint32_t r = me; r < R; r += step) lens_out[r] = __ldg(finished + r) != 0 ? 0 : __ldg(lens + r);
  if (me == 0) *count_out = (int32_t)(count + pages);
  for (uint32_t i = me; i < pages; i += step) {
    const uint32_t r = owner_of(page_sum, R, i);
    free_pages[count + i] = __ldg(block_table + (size_t)r * table_width + (i - page_sum[r]));
  }
}

int finish(int st) {
  note_status(st);
  return st;
}

// Small blocks while a thread of 256 has four requests at most to sum over: they start sooner. A block for every two tokens a thread: all blocks form the
// sums, but at the same time, while tokens behind one another in a thread wait for each other's loads (17299 tokens of 512 requests:
// 9.2 us with 1024-thread blocks of 4096 tokens, 5.0 with 256-thread blocks of 512).
constexpr int kSmall = 256, kLarge = 1024;
constexpr uint32_t kSmallWork = 1024, kMaxBlocks = 296;
unsigned blocks_for(uint32_t work, uint32_t threads) {
  const uint32_t n = (work + 2 * threads - 1) / (2 * threads);
  return n < 1 ? 1 : n < kMaxBlocks ? n : kMaxBlocks;
}

// Shared memory for the most requests, asked for once per kernel and device: a launch may have 48 KB without, what the kernel holds itself included, and
// a limit that followed each call's size could be lowered by another thread's call.
template <auto K>
int prepare(size_t bytes) {
  static std::once_flag once[64];
  static bool ok[64];
  int dev = 0;
  if (check_cuda(cudaGetDevice(&dev)) != DF_OK || dev < 0 || dev >= 64) return DF_ERR_CUDA;
  std::call_once(once[dev], [&]() { ok[dev] = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess; });
  return ok[dev] ? DF_OK : DF_ERR_CUDA;
}

// Blocks read all inputs while others write: what a kernel writes may be nothing that it reads, and no two results the same.
struct Entries {
  const int32_t *at;
  uint64_t n;
};
bool apart(std::initializer_list<Entries> written, std::initializer_list<Entries> read) {
  auto meet = [](const Entries &a, const Entries &b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return a.n != 0 && b.n != 0 && x < y + 4 * b.n && y < x + 4 * a.n;
  };
  for (const Entries *a = written.begin(); a != written.end(); ++a) {
    for (const Entries *b = written.begin(); b != a; ++b)
      if (meet(*a, *b)) return false;
    for (const Entries &b : read)
      if (meet(*a, b)) return false;
  }
  return true;
}

bool page_layout_valid(uint32_t page_size, uint32_t n_pages) { return page_size != 0 && (uint64_t)page_size * n_pages < (1ull << 31); }

}  // namespace
}  // namespace df

using namespace df;

extern "C" {

int df_cache_plan(const int32_t *lens, const int32_t *new_tokens, int *block_table, const int32_t *free_pages, const int32_t *free_count,
                  int *lens_out, int *starts, int *slots, int *positions, int *state, uint32_t n_requests, uint32_t n_tokens,
                  uint32_t table_width, uint32_t page_size, uint32_t n_pages, void *stream) {
  DF_RANGE("df_cache_plan");
  if (!page_layout_valid(page_size, n_pages) || n_tokens >= (1u << 31)) return finish(DF_ERR_INVALID_ARG);
  if (n_requests > kMaxRequests) return finish(DF_ERR_UNSUPPORTED);
  if (!free_count || !starts || !state || (n_pages && !free_pages) || (n_tokens && (!slots || !positions))) return finish(DF_ERR_INVALID_ARG);
  if (n_requests && (!lens || !new_tokens || !lens_out || (table_width && !block_table))) return finish(DF_ERR_INVALID_ARG);
  const uint64_t R = n_requests;
  if (!apart({{lens_out, R}, {starts, R + 1}, {slots, n_tokens}, {positions, n_tokens}, {state, 2}, {block_table, R * table_width}},
             {{lens, R}, {new_tokens, R}, {free_pages, n_pages}, {free_count, 1}}))
    return finish(DF_ERR_INVALID_ARG);
  const PlanParams p = {lens, new_tokens, free_pages, free_count, block_table, lens_out, starts, slots, positions, state,
                        n_requests, n_tokens, table_width, page_size, n_pages};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t smem = 2 * sizeof(uint32_t) * (size_t)n_requests;
  int st;
  const uint32_t work = n_tokens > n_requests ? n_tokens : n_requests;
  if (n_requests <= kSmallWork) {
    st = check_cuda(launch_kernel(k_cache_plan<kSmall>, dim3(blocks_for(work, kSmall)), dim3(kSmall), smem, s, p));
  } else {
    st = prepare<k_cache_plan<kLarge>>(2 * sizeof(uint32_t) * kMaxRequests);
    if (st == DF_OK) st = check_cuda(launch_kernel(k_cache_plan<kLarge>, dim3(blocks_for(work, kLarge)), dim3(kLarge), smem, s, p));
  }
  note_launch();
  return finish(st);
}

int df_cache_release(const int32_t *lens, const int32_t *finished, const int32_t *block_table, int *free_pages, const int32_t *free_count,
                     int *lens_out, int *count_out, uint32_t n_requests, uint32_t table_width, uint32_t page_size, uint32_t n_pages,
                     void *stream) {
  DF_RANGE("df_cache_release");
  if (!page_layout_valid(page_size, n_pages)) return finish(DF_ERR_INVALID_ARG);
  if (n_requests > kMaxRequests) return finish(DF_ERR_UNSUPPORTED);
  if (!free_count || !count_out || (n_pages && !free_pages)) return finish(DF_ERR_INVALID_ARG);
  if (n_requests && (!lens || !finished || !lens_out || (table_width && !block_table))) return finish(DF_ERR_INVALID_ARG);
  const uint64_t R = n_requests;
  if (!apart({{lens_out, R}, {count_out, 1}, {free_pages, n_pages}}, {{lens, R}, {finished, R}, {block_table, R * table_width}, {free_count, 1}}))
    return finish(DF_ERR_INVALID_ARG);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t smem = sizeof(uint32_t) * (size_t)n_requests;
  int st;
  if (n_requests <= kSmallWork) {
    st = check_cuda(launch_kernel(k_cache_release<kSmall>, dim3(blocks_for(n_requests, kSmall)), dim3(kSmall), smem, s, lens, finished, block_table, free_pages, free_count,
                                  lens_out, count_out, n_requests, table_width, page_size, n_pages));
  } else {
    st = prepare<k_cache_release<kLarge>>(sizeof(uint32_t) * kMaxRequests);
    if (st == DF_OK)
      st = check_cuda(launch_kernel(k_cache_release<kLarge>, dim3(blocks_for(n_requests, kLarge)), dim3(kLarge), smem, s, lens, finished,
                                    block_table, free_pages, free_count, lens_out, count_out, n_requests, table_width, page_size, n_pages));
  }
  note_launch();
  return finish(st);
}

}  // extern "C"
