// Decode attention for batches that share prompt prefixes, on the FP8 paged cache (sm_100a).
//
// Sequences come in groups; the sequences of group g share the P_g keys of one list of prefix
// pages and each sequence b owns C_b further keys in pages of its own, the newest t_b of which
// belong to its query rows (one row for plain decode, 1 + drafted tokens when drafts are
// verified).  With key positions 0..P_g-1 for the prefix and P_g..P_g+C_b-1 for the sequence's
// own keys, query i of t_b stands at pos = P_g + C_b - t_b + i and
//   out = v_scale * sum_j p_j V_j,  p = softmax_j(scale * k_scale * q . K_j),
//   j <= pos and (window W > 0) j > pos - W, holes of the block tables left out;
// a row that sees no key is zeros.
#include "common.cuh"

namespace ada {
namespace sp {

constexpr int D = 128;
constexpr float LOG2E = 1.4426950408889634f;

struct Params {
  const void* q;
  int64_t q_st, q_sh;
  const uint8_t* k;
  const uint8_t* v;
  int64_t s_page, s_tok, s_head, num_pages;
  const int32_t* pt;  // [groups][max_prefix_pages]
  int64_t pt_stride;
  int32_t max_prefix_pages;
  const int32_t* prefix_lens;
  const int32_t* cu_groups;  // null: one group of every sequence
  int32_t num_groups;
  const int32_t* bt;  // [batch][max_pages]
  int64_t bt_stride;
  int32_t max_pages;
  const int32_t* ctx;
  const int32_t* cu_q;  // null: one row per sequence
  int32_t batch, total_q, num_heads, group, page, window;
  float scale_log2, v_scale;
  void* out;
  int64_t o_st, o_sh;
};

// Number of entries of the ascending list cu[0..n] that are <= x, minus one: the interval
// [cu[i], cu[i + 1]) that holds x (-1: before the first; n: past the last).
__device__ __forceinline__ int interval_of(const int32_t* cu, int n, int x) {
  int lo = 0, hi = n + 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= x) lo = mid + 1; else hi = mid;
  }
  return lo - 1;
}

// One warp per (row, query head): 32 keys at a time, lane = key for the scores, lane = four
// dimensions for the sum over V.
template <typename TQ, typename TO>
__global__ void __launch_bounds__(128) rows_kernel(Params P) {
  pdl_wait();
  pdl_trigger();
  __shared__ float qs[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + warp;
  if (item >= (int64_t)P.total_q * P.num_heads) return;
  const int n = (int)(item / P.num_heads), h = (int)(item % P.num_heads);
  const int kvh = h / P.group;
  const int b = P.cu_q ? interval_of(P.cu_q, P.batch, n) : n;
  const bool live = b >= 0 && b < P.batch;
  const int g = !live ? -1 : (P.cu_groups ? interval_of(P.cu_groups, P.num_groups, b) : 0);
  const int len_p =
      g >= 0 && g < P.num_groups ? max(0, min(__ldg(P.prefix_lens + g), P.max_prefix_pages * P.page)) : 0;
  const int len_c = live ? max(0, min(__ldg(P.ctx + b), P.max_pages * P.page)) : 0;
  const int pos = live ? len_p + len_c - (P.cu_q ? __ldg(P.cu_q + b + 1) - n : 1) : -1;
  const int lo = P.window > 0 ? max(0, pos - P.window + 1) : 0;

  const TQ* qp = reinterpret_cast<const TQ*>(P.q) + (int64_t)n * P.q_st + (int64_t)h * P.q_sh;
  for (int d = lane; d < D; d += 32) qs[warp][d] = to_f32(qp[d]) * P.scale_log2;
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = lo; j0 <= pos; j0 += 32) {
    const int j = j0 + lane;
    int64_t at = -1;  // byte offset of key j's row, -1: not visible
    if (j <= pos) {
      const bool pre = j < len_p;
      const int jj = pre ? j : j - len_p;
      const int32_t* tab = pre ? P.pt + (int64_t)g * P.pt_stride : P.bt + (int64_t)b * P.bt_stride;
      const int blk = __ldg(tab + jj / P.page);
      if (blk >= 0 && blk < P.num_pages) at = blk * P.s_page + (jj % P.page) * P.s_tok + kvh * P.s_head;
    }
    float s = -INFINITY;
    if (at >= 0) {
      s = 0.f;
      for (int c = 0; c < 8; ++c) {
        const uint4 e = *reinterpret_cast<const uint4*>(P.k + at + 16 * c);
        const uint32_t w[4] = {e.x, e.y, e.z, e.w};
        for (int i = 0; i < 8; ++i) {
          const uint32_t f = e4m3x2_to_f16x2((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
          const float2 kv = __half22float2(*reinterpret_cast<const __half2*>(&f));
          s = fmaf(qs[warp][16 * c + 2 * i], kv.x, s);
          s = fmaf(qs[warp][16 * c + 2 * i + 1], kv.y, s);
        }
      }
    }
    float mx = s;
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float mn = fmaxf(m, mx);
    if (mn == -INFINITY) continue;  // nothing visible so far
    const float al = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * al + p;
    for (int i = 0; i < 4; ++i) o[i] *= al;
    for (int t = 0; t < 32; ++t) {
      const int64_t a = __shfl_sync(0xffffffffu, at, t);
      const float pt = __shfl_sync(0xffffffffu, p, t);
      if (a < 0) continue;
      const uint32_t e = *reinterpret_cast<const uint32_t*>(P.v + a + 4 * lane);
      const uint32_t f0 = e4m3x2_to_f16x2((uint16_t)e), f1 = e4m3x2_to_f16x2((uint16_t)(e >> 16));
      const float2 v0 = __half22float2(*reinterpret_cast<const __half2*>(&f0));
      const float2 v1 = __half22float2(*reinterpret_cast<const __half2*>(&f1));
      o[0] = fmaf(pt, v0.x, o[0]);
      o[1] = fmaf(pt, v0.y, o[1]);
      o[2] = fmaf(pt, v1.x, o[2]);
      o[3] = fmaf(pt, v1.y, o[3]);
    }
  }
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  const float inv = l > 0.f ? P.v_scale / l : 0.f;
  TO* op = reinterpret_cast<TO*>(P.out) + (int64_t)n * P.o_st + (int64_t)h * P.o_sh;
  for (int i = 0; i < 4; ++i) op[4 * lane + i] = from_f32<TO>(o[i] * inv);
}

}  // namespace sp
}  // namespace ada

using namespace ada;

extern "C" size_t ada_fp8_shared_prefix_decode_workspace_size(int32_t total_q, int32_t num_groups, int32_t batch,
                                                              int32_t num_heads, int32_t num_kv_heads,
                                                              int32_t head_dim) {
  if (total_q <= 0 || num_groups < 0 || batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
  return 256;
}

extern "C" int ada_fp8_shared_prefix_decode(
    const void* q, int q_dtype, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* k_cache, const uint8_t* v_cache,
    int64_t kv_stride_page, int64_t kv_stride_tok, int64_t kv_stride_head, int64_t num_pages,
    const int32_t* prefix_tables, int64_t pt_stride, int32_t max_prefix_pages, const int32_t* prefix_lens,
    const int32_t* cu_groups, int32_t num_groups, const int32_t* block_tables, int64_t bt_stride, int32_t max_pages,
    const int32_t* context_lens, const int32_t* cu_seqlens_q, int32_t batch, int32_t total_q, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t page_size, float scale, float k_scale, float v_scale,
    int32_t window, void* out, int out_dtype, int64_t out_stride_t, int64_t out_stride_h, void* workspace,
    size_t workspace_bytes, unsigned int* err, void* stream) {
  if (batch < 0 || total_q < 0 || num_groups < 0 || num_heads <= 0 || num_kv_heads <= 0 || page_size <= 0 ||
      max_pages <= 0 || max_prefix_pages < 0)
    return ADA_ERR_INVALID_ARG;
  if (total_q == 0 || batch == 0) return ADA_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !out || !workspace) return ADA_ERR_INVALID_ARG;
  if (num_groups > 0 && (!prefix_lens || (max_prefix_pages > 0 && !prefix_tables))) return ADA_ERR_INVALID_ARG;
  if ((num_groups > 1 && !cu_groups) || (!cu_seqlens_q && total_q != batch)) return ADA_ERR_INVALID_ARG;
  if ((q_dtype != ADA_DT_BF16 && q_dtype != ADA_DT_F16) || (out_dtype != ADA_DT_BF16 && out_dtype != ADA_DT_F16))
    return ADA_ERR_INVALID_ARG;
  if (num_heads % num_kv_heads != 0) return ADA_ERR_INVALID_ARG;
  if (window < 0 || bt_stride < max_pages || pt_stride < max_prefix_pages || num_pages <= 0) return ADA_ERR_INVALID_ARG;
  if (!(scale * k_scale > 0.f)) return ADA_ERR_INVALID_ARG;  // row maxima are taken on unscaled scores
  if (head_dim != sp::D || page_size % 16 != 0 || num_heads / num_kv_heads > 128) return ADA_ERR_UNSUPPORTED;
  if (((int64_t)max_pages + max_prefix_pages) * page_size > (1LL << 30)) return ADA_ERR_UNSUPPORTED;
  if ((int64_t)total_q * num_heads > (1LL << 30)) return ADA_ERR_UNSUPPORTED;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return ADA_ERR_ALIGNMENT;
  if ((kv_stride_page | kv_stride_tok | kv_stride_head) & 15) return ADA_ERR_ALIGNMENT;
  if (((uintptr_t)q & 15) || (q_stride_t & 7) || (q_stride_h & 7)) return ADA_ERR_ALIGNMENT;
  if (((uintptr_t)out & 15) || (out_stride_t & 7) || (out_stride_h & 7)) return ADA_ERR_ALIGNMENT;
  if (((uintptr_t)workspace & 255) || ((uintptr_t)err & 3)) return ADA_ERR_ALIGNMENT;
  if (workspace_bytes < ada_fp8_shared_prefix_decode_workspace_size(total_q, num_groups, batch, num_heads,
                                                                    num_kv_heads, head_dim))
    return ADA_ERR_WORKSPACE;

  sp::Params P;
  P.q = q;
  P.q_st = q_stride_t;
  P.q_sh = q_stride_h;
  P.k = k_cache;
  P.v = v_cache;
  P.s_page = kv_stride_page;
  P.s_tok = kv_stride_tok;
  P.s_head = kv_stride_head;
  P.num_pages = num_pages;
  P.pt = prefix_tables;
  P.pt_stride = pt_stride;
  P.max_prefix_pages = max_prefix_pages;
  P.prefix_lens = prefix_lens;
  P.cu_groups = cu_groups;
  P.num_groups = num_groups;
  P.bt = block_tables;
  P.bt_stride = bt_stride;
  P.max_pages = max_pages;
  P.ctx = context_lens;
  P.cu_q = cu_seqlens_q;
  P.batch = batch;
  P.total_q = total_q;
  P.num_heads = num_heads;
  P.group = num_heads / num_kv_heads;
  P.page = page_size;
  P.window = window;
  P.scale_log2 = scale * k_scale * sp::LOG2E;
  P.v_scale = v_scale;
  P.out = out;
  P.o_st = out_stride_t;
  P.o_sh = out_stride_h;
  const dim3 grid((unsigned)cdiv((int64_t)total_q * num_heads, 4));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (q_dtype == ADA_DT_BF16) {
    if (out_dtype == ADA_DT_BF16)
      (void)ada::launch_k(sp::rows_kernel<__nv_bfloat16, __nv_bfloat16>, grid, dim3(128), 0, st, P);
    else
      (void)ada::launch_k(sp::rows_kernel<__nv_bfloat16, __half>, grid, dim3(128), 0, st, P);
  } else {
    if (out_dtype == ADA_DT_BF16)
      (void)ada::launch_k(sp::rows_kernel<__half, __nv_bfloat16>, grid, dim3(128), 0, st, P);
    else
      (void)ada::launch_k(sp::rows_kernel<__half, __half>, grid, dim3(128), 0, st, P);
  }
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
