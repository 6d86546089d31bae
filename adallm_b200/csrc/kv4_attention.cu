// Decode and prefill attention over the 4-bit paged KV cache (kv4.cuh), first form: one CTA a
// (query row, head), 128 keys a step -- a thread is a key for the scores and an element for the
// sums of values -- with the running maximum and sum of a softmax in fp32.
#include "kv4.cuh"

namespace ada {
namespace kv4 {

struct AttnParams {
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  const uint8_t *kc, *vc;
  int64_t s_page, s_head, num_pages;
  const int32_t* bt;
  int64_t bt_stride;
  int max_pages, page, group, window;
  const int32_t *lens;         // decode: context lengths
  const int32_t *cu_q, *cu_k;  // prefill
  int64_t rows;  // query rows of q and out
  float scale_log2, v_scale;
};

template <typename TQ, typename TO>
__global__ void __launch_bounds__(128) attn_kernel(AttnParams P) {
  __shared__ float qs[D], ps[128], red[4];
  __shared__ int64_t at[128];
  const int tid = threadIdx.x, head = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  int64_t row = b;
  int lo, hi;
  if (P.lens) {
    const int ctx = P.lens[b];
    hi = ctx;
    lo = P.window > 0 ? max(ctx - P.window, 0) : 0;
  } else {
    const int q0 = P.cu_q[b], len_q = P.cu_q[b + 1] - q0, len_k = P.cu_k[b + 1] - P.cu_k[b];
    const int t = blockIdx.x;
    if (t >= len_q) return;
    row = (int64_t)q0 + t;
    if (row < 0 || row >= P.rows) return;
    hi = min(len_k, t + len_k - len_q + 1);
    lo = P.window > 0 ? max(0, t + len_k - len_q - P.window) : 0;
  }
  hi = (int)min((int64_t)hi, (int64_t)P.max_pages * P.page);
  const TQ* q = reinterpret_cast<const TQ*>(P.q) + row * P.q_st + head * P.q_sh;
  float top = fabsf(to_f32(q[tid]));
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
  const int ex = query_exponent(max_nan(max_nan(red[0], red[1]), max_nan(red[2], red[3])));
  const float c = score_factor(P.scale_log2, ex);
  qs[tid] = to_f32(q[tid]) * pow2(ex);
  const int64_t hb = (int64_t)(head / P.group) * P.s_head;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int k0 = lo; k0 < hi; k0 += 128) {
    __syncthreads();
    const int key = k0 + tid;
    float s = -INFINITY;
    int64_t mine = -1;
    if (key < hi) {
      const int64_t id = P.bt[(int64_t)b * P.bt_stride + key / P.page];
      if (id >= 0 && id < P.num_pages) {
        const int r = key % P.page;
        const uint8_t* blk = P.kc + id * P.s_page + hb;
        mine = id * P.s_page + hb;
        s = 0.f;
        for (int j = 0; j < SROW; ++j) {
          const uint2 c = *reinterpret_cast<const uint2*>(blk + (int64_t)r * ROW + 8 * j);
          uint32_t h[8];
          e2m1x8_to_f16x8(c.x, h);
          e2m1x8_to_f16x8(c.y, h + 4);
          float a = 0.f;
          for (int i = 0; i < 8; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
            a = fmaf(f.x, qs[16 * j + 2 * i], fmaf(f.y, qs[16 * j + 2 * i + 1], a));
          }
          s = fmaf(a, scale_value(blk[(int64_t)P.page * ROW + r * SROW + j]), s);
        }
      }
    }
    at[tid] = mine;
    float mx = s;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
    const float base = mx == -INFINITY ? 0.f : mx;
    ps[tid] = exp2f((s - base) * c);
    const float alpha = exp2f((m - base) * c);
    m = mx;
    __syncthreads();
    l *= alpha;
    acc *= alpha;
    for (int j = 0; j < 128; ++j) {
      if (at[j] < 0) continue;
      const int r = (k0 + j) % P.page;
      const uint8_t* blk = P.vc + at[j];
      const uint32_t byte = blk[(int64_t)r * ROW + (tid >> 1)];
      uint32_t h[4];
      e2m1x8_to_f16x8(tid & 1 ? byte >> 4 : byte & 15u, h);
      const float v = __half2float(__ushort_as_half((unsigned short)(h[0] & 0xFFFFu))) *
                      scale_value(blk[(int64_t)P.page * ROW + r * SROW + (tid >> 4)]);
      l += ps[j];
      acc = fmaf(ps[j], v, acc);
    }
  }
  TO* out = reinterpret_cast<TO*>(P.out) + row * P.o_st + head * P.o_sh;
  out[tid] = from_f32<TO>(l != 0.f ? acc / l * P.v_scale : 0.f);
}

template <typename TQ, typename TO>
static void launch_attn(const AttnParams& P, dim3 grid, cudaStream_t st) {
  (void)launch_k(attn_kernel<TQ, TO>, grid, dim3(128), 0, st, P);
}
static void dispatch_attn(const AttnParams& P, dim3 grid, int qd, int od, cudaStream_t st) {
  if (qd == ADA_DT_BF16)
    od == ADA_DT_BF16 ? launch_attn<__nv_bfloat16, __nv_bfloat16>(P, grid, st)
                      : launch_attn<__nv_bfloat16, __half>(P, grid, st);
  else
    od == ADA_DT_BF16 ? launch_attn<__half, __nv_bfloat16>(P, grid, st) : launch_attn<__half, __half>(P, grid, st);
}

}  // namespace kv4
}  // namespace ada

using namespace ada;

extern "C" int ada_kv4_paged_prefill(const void* q, int q_dtype, int64_t q_stride_t, int64_t q_stride_h,
                                     const uint8_t* k_cache, const uint8_t* v_cache, int64_t kv_stride_page,
                                     int64_t kv_stride_head, int64_t num_pages, const int32_t* block_tables,
                                     int64_t bt_stride, int32_t max_pages, const int32_t* cu_seqlens_q,
                                     const int32_t* cu_seqlens_k, int32_t batch, int64_t total_q,
                                     int32_t max_seqlen_q, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                     float scale, float k_scale, float v_scale, int32_t window, void* out,
                                     int out_dtype, int64_t out_stride_t, int64_t out_stride_h, unsigned int* err,
                                     void* stream) {
  if (batch < 0 || max_seqlen_q < 0 || total_q < 0) return ADA_ERR_INVALID_ARG;
  if (batch == 0 || max_seqlen_q == 0 || total_q == 0) return ADA_OK;
  kv4::AttnParams P{q, q_stride_t, q_stride_h, out, out_stride_t, out_stride_h, k_cache, v_cache, kv_stride_page,
                    kv_stride_head, num_pages, block_tables, bt_stride, max_pages, page_size, 1, window, nullptr,
                    cu_seqlens_q, cu_seqlens_k, total_q, scale * k_scale * kv4::LOG2E, v_scale};
  if (!cu_seqlens_q || !cu_seqlens_k) return ADA_ERR_INVALID_ARG;
  if (const int e = kv4::attn_ok(q, q_dtype, q_stride_t, q_stride_h, out, out_dtype, out_stride_t, out_stride_h, k_cache,
                                 v_cache, kv_stride_page, kv_stride_head, num_pages, block_tables, bt_stride, max_pages,
                                 num_heads, num_kv_heads, head_dim, page_size, scale, k_scale, v_scale, window))
    return e;
  if ((reinterpret_cast<uintptr_t>(cu_seqlens_q) | reinterpret_cast<uintptr_t>(cu_seqlens_k)) & 3)
    return ADA_ERR_ALIGNMENT;
  if (batch > 65535 || num_heads > 65535) return ADA_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(err) & 3) return ADA_ERR_ALIGNMENT;
  P.group = num_heads / num_kv_heads;
  kv4::dispatch_attn(P, dim3((unsigned)max_seqlen_q, (unsigned)num_heads, (unsigned)batch), q_dtype, out_dtype,
                     reinterpret_cast<cudaStream_t>(stream));
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
