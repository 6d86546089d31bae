// A serving step's metadata from its requests' lengths (the host loops of prepare_prefill and
// prepare_decode, reference adallm/runtime/model_runner.py:234-300, on the device).
//
// Request b has c = cached_lens[b] tokens in its pages and n = new_lens[b] new ones (negative
// lengths count as 0).  With P rows a page it owns ceil(c / P) pages and takes
// ceil((c + n) / P) - ceil(c / P) from the free list, in request order from free_start on.  Its new
// tokens are t = cu_q[b] .. cu_q[b + 1] of the step: position c + t - cu_q[b], slot = page * P + row.
//
// A few words a request and 12 bytes a token: the time is one launch and the chain lengths ->
// prefix sums -> table -> slot.  Every CTA takes the prefix sums of all requests itself (they sit in
// L2 and take less than a second launch or a wait between CTAs would) and finds a token's request by
// bisection in shared memory; a new page's id comes from the free list and not from the table, which
// other CTAs write meanwhile.
#include "common.cuh"

namespace ada {
namespace meta {

constexpr int THREADS = 512;
constexpr int MAX_REQUESTS = 8192;
constexpr unsigned ERR_PAGES = 0x100, ERR_WIDTH = 0x200, ERR_TOKENS = 0x400;

struct Params {
  const int32_t *cached, *fresh;
  int requests;
  int32_t* tables;
  int64_t t_stride;
  int max_pages;
  const int32_t* free_pages;
  int64_t num_free;
  const int32_t* free_start;
  int page;
  int64_t tokens;
  int64_t* positions;
  int32_t *slots, *cu_q, *cu_k, *context, *free_next;
  unsigned* err;
};

// Sums of lengths stop at INT_MAX (addition that saturates is associative on values >= 0).
__device__ __forceinline__ int add_sat(int a, int b) {
  const unsigned s = (unsigned)a + (unsigned)b;
  return s > 0x7fffffffu ? 0x7fffffff : (int)s;
}
struct Sums {
  int q, k, p;
};
__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) {
  return {add_sat(a.q, b.q), add_sat(a.k, b.k), add_sat(a.p, b.p)};
}
__device__ __forceinline__ int pages_of(int tokens, int page) { return tokens / page + (tokens % page != 0); }

// Index of the segment of cu [n + 1] (ascending) that holds x < cu[n]: the first b with cu[b + 1] > x.
__device__ __forceinline__ int segment(const int* cu, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) step_metadata_kernel(Params P) {
  extern __shared__ int sm[];
  __shared__ Sums warp_sum[THREADS / 32];
  const int B = P.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* cu_q = sm;               // [B + 1]
  int* cu_p = sm + B + 1;       // [B + 1] pages taken before a request
  int* had = sm + 2 * (B + 1);  // [B] cached tokens
  pdl_wait();
  pdl_trigger();
  unsigned err = 0;

  // prefix sums: a thread's own requests in a row, then over the warp, then over the warps
  const int per = (B + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
  Sums sum{0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const int c = max(P.cached[b], 0), n = max(P.fresh[b], 0);
    const int all = add_sat(c, n);
    had[b] = c;
    sum = sum + Sums{n, all, pages_of(all, P.page) - pages_of(c, P.page)};
  }
  Sums inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums up{__shfl_up_sync(0xffffffffu, inc.q, o), __shfl_up_sync(0xffffffffu, inc.k, o),
                  __shfl_up_sync(0xffffffffu, inc.p, o)};
    if (lane >= o) inc = inc + up;
  }
  Sums run{__shfl_up_sync(0xffffffffu, inc.q, 1), __shfl_up_sync(0xffffffffu, inc.k, 1),
           __shfl_up_sync(0xffffffffu, inc.p, 1)};
  if (lane == 0) run = Sums{0, 0, 0};
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  for (int w = 0; w < warp; ++w) run = run + warp_sum[w];
  const bool first = blockIdx.x == 0;
  for (int b = b0; b < b1; ++b) {
    cu_q[b] = run.q;
    cu_p[b] = run.p;
    const int c = had[b], n = max(P.fresh[b], 0);
    const int all = add_sat(c, n);
    if (first) {
      P.cu_q[b] = run.q;
      P.cu_k[b] = run.k;
      P.context[b] = all;
    }
    run = run + Sums{n, all, pages_of(all, P.page) - pages_of(c, P.page)};
  }
  if (b0 < B && b1 == B) {  // the thread that holds the last request
    cu_q[B] = run.q;
    cu_p[B] = run.p;
    if (first) {
      P.cu_q[B] = run.q;
      P.cu_k[B] = run.k;
    }
  }
  if (B == 0 && tid == 0) {
    cu_q[0] = cu_p[0] = 0;
    if (first) P.cu_q[0] = P.cu_k[0] = 0;
  }
  __syncthreads();
  const int total = cu_q[B], taken = cu_p[B];
  const int64_t start = *P.free_start;
  if (first && tid == 0) {
    *P.free_next = (int)max(min(start + taken, P.num_free), min(start, P.num_free));
    if (total > P.tokens) err |= ERR_TOKENS;
  }

  const int64_t step = (int64_t)gridDim.x * THREADS, me = (int64_t)blockIdx.x * THREADS + tid;
  // the pages taken, into the tables
  for (int64_t i = me; i < taken; i += step) {
    const int b = segment(cu_p, B, (int)i);
    const int64_t at = start + i, col = pages_of(had[b], P.page) + (i - cu_p[b]);
    const bool listed = at >= 0 && at < P.num_free;
    if (!listed)
      err |= ERR_PAGES;
    else if (col >= P.max_pages)
      err |= ERR_WIDTH;
    // a page that is not there is none in the table either: what stood there may be a page of another request by now,
    // and the next step counts these columns as the request's own
    if (col < P.max_pages) P.tables[b * P.t_stride + col] = listed ? P.free_pages[at] : -1;
  }
  // the tokens
  for (int64_t t = me; t < P.tokens; t += step) {
    int64_t pos = 0, slot = -1;
    if (t < total) {
      const int b = segment(cu_q, B, (int)t);
      pos = (int64_t)had[b] + (t - cu_q[b]);
      const int64_t col = pos / P.page, owned = pages_of(had[b], P.page);
      int64_t id = -1;
      if (col < P.max_pages) {
        if (col < owned) {
          id = P.tables[b * P.t_stride + col];
        } else {
          const int64_t at = start + cu_p[b] + (col - owned);
          if (at >= 0 && at < P.num_free) id = P.free_pages[at];
        }
      } else {
        err |= ERR_WIDTH;
      }
      if (id >= 0) slot = id * P.page + (pos - col * P.page);
      if (slot > 0x7fffffff) {
        slot = -1;
        err |= ERR_TOKENS;
      }
    }
    P.positions[t] = pos;
    P.slots[t] = (int32_t)slot;
  }
  if (err && P.err) atomicOr(P.err, err);
}

}  // namespace meta
}  // namespace ada

using namespace ada;

extern "C" int ada_step_metadata(const int32_t* cached_lens, const int32_t* new_lens, int32_t requests,
                                 int32_t* block_tables, int64_t bt_stride, int32_t max_pages,
                                 const int32_t* free_pages, int64_t num_free, const int32_t* free_start,
                                 int32_t page_size, int64_t num_tokens, int64_t* positions, int32_t* slot_mapping,
                                 int32_t* cu_seqlens_q, int32_t* cu_seqlens_k, int32_t* context_lens,
                                 int32_t* free_next, unsigned int* err, void* stream) {
  if (requests < 0 || max_pages < 0 || num_free < 0 || page_size <= 0 || num_tokens < 0) return ADA_ERR_INVALID_ARG;
  if (!free_start || !free_next || !cu_seqlens_q || !cu_seqlens_k) return ADA_ERR_INVALID_ARG;
  if (requests > 0 && (!cached_lens || !new_lens || !context_lens)) return ADA_ERR_INVALID_ARG;
  if (requests > 0 && max_pages > 0 && (!block_tables || bt_stride < max_pages)) return ADA_ERR_INVALID_ARG;
  if (num_free > 0 && !free_pages) return ADA_ERR_INVALID_ARG;
  if (num_tokens > 0 && (!positions || !slot_mapping)) return ADA_ERR_INVALID_ARG;
  if (requests > meta::MAX_REQUESTS || num_tokens > 0x7fffffff) return ADA_ERR_UNSUPPORTED;
  const uintptr_t words = (uintptr_t)cached_lens | (uintptr_t)new_lens | (uintptr_t)block_tables |
                          (uintptr_t)free_pages | (uintptr_t)free_start | (uintptr_t)slot_mapping |
                          (uintptr_t)cu_seqlens_q | (uintptr_t)cu_seqlens_k | (uintptr_t)context_lens |
                          (uintptr_t)free_next | (uintptr_t)err;
  if ((words & 3) || ((uintptr_t)positions & 7)) return ADA_ERR_ALIGNMENT;
  // every CTA reads the inputs, the first one writes its results meanwhile: no output may lie in an input
  const struct { const void* p; int64_t n; } in[] = {{cached_lens, 4LL * requests}, {new_lens, 4LL * requests},
                                                     {free_pages, 4 * num_free}, {free_start, 4}},
      made[] = {{positions, 8 * num_tokens}, {slot_mapping, 4 * num_tokens}, {cu_seqlens_q, 4LL * (requests + 1)},
                {cu_seqlens_k, 4LL * (requests + 1)}, {context_lens, 4LL * requests}, {free_next, 4}};
  for (const auto& a : in)
    for (const auto& b : made)
      if (a.n > 0 && b.n > 0 && (uintptr_t)a.p < (uintptr_t)b.p + b.n && (uintptr_t)b.p < (uintptr_t)a.p + a.n)
        return ADA_ERR_INVALID_ARG;
  meta::Params P;
  P.cached = cached_lens;
  P.fresh = new_lens;
  P.requests = requests;
  P.tables = block_tables;
  P.t_stride = bt_stride;
  P.max_pages = max_pages;
  P.free_pages = free_pages;
  P.num_free = num_free;
  P.free_start = free_start;
  P.page = page_size;
  P.tokens = num_tokens;
  P.positions = positions;
  P.slots = slot_mapping;
  P.cu_q = cu_seqlens_q;
  P.cu_k = cu_seqlens_k;
  P.context = context_lens;
  P.free_next = free_next;
  P.err = err;
  const size_t smem = (size_t)(3 * requests + 2) * 4;
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ADA_ERR_CUDA;
  if (smem > 48 * 1024 && !ready[dev]) {
    if (cudaFuncSetAttribute(meta::step_metadata_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (3 * meta::MAX_REQUESTS + 2) * 4) != cudaSuccess)
      return ADA_ERR_CUDA;
    ready[dev] = true;
  }
  const int64_t grid = cdiv(num_tokens, meta::THREADS);
  (void)launch_k(meta::step_metadata_kernel, dim3((unsigned)(grid < 1 ? 1 : grid > 148 ? 148 : grid)),
                 dim3(meta::THREADS), smem, reinterpret_cast<cudaStream_t>(stream), P);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
