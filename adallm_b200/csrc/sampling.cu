// Sampling at a temperature and verification of drafted tokens (sm_100a).
//
// Both work on rows of logits x of one vocabulary with given random numbers.  With temperature T
// (T <= 1e-10: greedy, statistics at temperature 1) and z = x / T:
//   lse = max z + ln sum exp(z - max z),  p = exp(z - lse),
//   a draw from weights w is argmax_v w[v] / e[v], lowest index on ties, for given independent
//   exponentials e (read as max(e, 1e-10)): index v is the smallest of the times e / w with
//   probability w[v] / sum w.  The reference draws the same way (adallm/ops/sampler.py:10-15).
// A logit of -inf or NaN has probability 0, +inf is read as the largest float.  A row with no
// possible token has the token -1.
//
// Verification of the drafts x_1..x_d of a sequence against its target rows p_0..p_d and the
// draft distributions q_1..q_d (each the one that its draft was drawn from; without them every
// draft is taken as certain, q = 1 at x): draft i is accepted while u_i q_i(x_i) < p_{i-1}(x_i);
// at the first refusal the token is drawn from max(p_{i-1} - q_i, 0) (from p_{i-1} where that is
// zero everywhere), after d acceptances from p_d.  Tokens drawn this way are distributed as the
// target's own.  Greedy sequences accept a draft that is the target's first maximum and end with
// the first maximum.
#include <float.h>

#include "common.cuh"

namespace ada {
namespace smp {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;

template <typename T> __device__ __forceinline__ float load_logit(const T* p) {
  const float x = to_f32(*p);
  return x == x ? fminf(x, FLT_MAX) : -INFINITY;
}
template <> __device__ __forceinline__ float load_logit<float>(const float* p) {
  const float x = *p;
  return x == x ? fminf(x, FLT_MAX) : -INFINITY;
}

struct Best {
  float score;
  int index;
};
__device__ __forceinline__ void take(Best& a, float score, int index) {
  if (score > a.score || (score == a.score && index < a.index)) {
    a.score = score;
    a.index = index;
  }
}

__device__ float block_max(float v, float* red) {
  for (int x = 16; x > 0; x >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < WARPS; ++i) v = fmaxf(v, red[i]);
  return v;
}
__device__ float block_sum(float v, float* red) {
  for (int x = 16; x > 0; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < WARPS; ++i) v += red[i];
  return v;
}
__device__ Best block_best(Best b, float* red, int* redi) {
  for (int x = 16; x > 0; x >>= 1) {
    const float s = __shfl_xor_sync(0xffffffffu, b.score, x);
    const int i = __shfl_xor_sync(0xffffffffu, b.index, x);
    take(b, s, i);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = b.score;
    redi[threadIdx.x >> 5] = b.index;
  }
  __syncthreads();
  b.score = red[0];
  b.index = redi[0];
  for (int i = 1; i < WARPS; ++i) take(b, red[i], redi[i]);
  return b;
}

struct Row {
  float top, total;  // max z, sum exp(z - top); top = -inf: no possible token
};
__device__ __forceinline__ float scaled(float x, float t) { return fminf(x / t, FLT_MAX); }

template <typename T>
__device__ Row row_stats(const T* x, int64_t vocab, float t, float* red) {
  float m = -INFINITY;
  for (int64_t v = threadIdx.x; v < vocab; v += THREADS) m = fmaxf(m, scaled(load_logit(x + v), t));
  m = block_max(m, red);
  float s = 0.f;
  if (m != -INFINITY)
    for (int64_t v = threadIdx.x; v < vocab; v += THREADS) s += expf(scaled(load_logit(x + v), t) - m);
  return {m, block_sum(s, red)};
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
    sample_kernel(const T* __restrict__ logits, int64_t ld, int64_t vocab, const float* __restrict__ temps,
                  const float* __restrict__ noise, int64_t ld_noise, int64_t* tokens, float* logprobs, float* lse) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[WARPS];
  __shared__ int redi[WARPS];
  const int64_t r = blockIdx.x;
  const T* x = logits + r * ld;
  const float* e = noise + r * ld_noise;
  const float temp = temps[r];
  const bool greedy = !(temp > 1e-10f);
  const float t = greedy ? 1.f : temp;
  const Row st = row_stats(x, vocab, t, red);
  Best b{0.f, 0x7fffffff};
  if (st.top != -INFINITY)
    for (int64_t v = threadIdx.x; v < vocab; v += THREADS) {
      const float w = expf(scaled(load_logit(x + v), t) - st.top);
      const float s = greedy ? w : w / st.total / fmaxf(e[v], 1e-10f);
      if (s > 0.f) take(b, s, (int)v);
    }
  b = block_best(b, red, redi);
  if (threadIdx.x == 0) {
    const bool any = b.index != 0x7fffffff;
    const float l = any ? st.top + logf(st.total) : -INFINITY;
    tokens[r] = any ? b.index : -1;
    if (logprobs) logprobs[r] = any ? scaled(load_logit(x + b.index), t) - l : 0.f;
    if (lse) lse[r] = l;
  }
}

struct VerifyParams {
  const void* target;
  int64_t ld, vocab;
  const int64_t* ids;
  const int32_t* cu_q;
  int32_t total_q, max_drafts;
  const float* temps;
  const float* uniforms;
  int64_t ld_u;
  const float* noise;
  int64_t ld_noise;
  const void* draft;
  int64_t d_sb, d_sd;
  const float* draft_lse;
  int64_t l_sb, l_sd;
  int64_t* tokens;
  int32_t* accepted;
  float* logprobs;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) verify_kernel(VerifyParams P) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[WARPS];
  __shared__ int redi[WARPS];
  const int64_t b = blockIdx.x;
  const int first = max(0, __ldg(P.cu_q + b)), end = min(P.total_q, __ldg(P.cu_q + b + 1));
  const int drafts = min(end - first - 1, P.max_drafts);  // -1: an empty sequence
  const float temp = P.temps[b];
  const bool greedy = !(temp > 1e-10f);
  const float t = greedy ? 1.f : temp;
  int64_t* tokens = P.tokens + b * (P.max_drafts + 1);
  float* logprobs = P.logprobs + b * (P.max_drafts + 1);
  int count = 0, written = 0;
  for (int i = 0; i <= drafts; ++i) {
    const T* x = reinterpret_cast<const T*>(P.target) + (int64_t)(first + i) * P.ld;
    const Row st = row_stats(x, P.vocab, t, red);
    const T* dr = P.draft && i < drafts ? reinterpret_cast<const T*>(P.draft) + b * P.d_sb + i * P.d_sd : nullptr;
    const float dl = dr ? P.draft_lse[b * P.l_sb + i * P.l_sd] : 0.f;
    const int64_t id = i < drafts ? P.ids[first + i + 1] : -1;
    const bool inside = id >= 0 && id < P.vocab;
    auto p_of = [&](int64_t v) { return st.top != -INFINITY ? expf(scaled(load_logit(x + v), t) - st.top) / st.total : 0.f; };
    auto q_of = [&](int64_t v) { return dr ? expf(scaled(load_logit(dr + v), t) - dl) : (v == id ? 1.f : 0.f); };
    if (i < drafts && inside && !greedy && P.uniforms[b * P.ld_u + i] * q_of(id) < p_of(id)) {
      if (threadIdx.x == 0) {
        tokens[i] = id;
        logprobs[i] = scaled(load_logit(x + id), t) - (st.top + logf(st.total));
      }
      written = ++count;
      continue;
    }
    Best best{0.f, 0x7fffffff};
    if (!greedy && i < drafts)
      for (int64_t v = threadIdx.x; v < P.vocab; v += THREADS) {
        const float s = fmaxf(p_of(v) - q_of(v), 0.f) / fmaxf(P.noise[b * P.ld_noise + v], 1e-10f);
        if (s > 0.f) take(best, s, (int)v);
      }
    best = block_best(best, red, redi);
    if (best.index == 0x7fffffff) {
      for (int64_t v = threadIdx.x; v < P.vocab; v += THREADS) {
        const float s = greedy ? p_of(v) : p_of(v) / fmaxf(P.noise[b * P.ld_noise + v], 1e-10f);
        if (s > 0.f) take(best, s, (int)v);
      }
      best = block_best(best, red, redi);
    }
    const bool any = best.index != 0x7fffffff;
    if (threadIdx.x == 0) {
      tokens[i] = any ? best.index : -1;
      logprobs[i] = any ? scaled(load_logit(x + best.index), t) - (st.top + logf(st.total)) : 0.f;
    }
    written = i + 1;
    if (greedy && i < drafts && any && best.index == id) {
      ++count;
      continue;
    }
    break;
  }
  if (threadIdx.x == 0) {
    for (int i = written; i <= P.max_drafts; ++i) {
      tokens[i] = -1;
      logprobs[i] = 0.f;
    }
    P.accepted[b] = count;
  }
}

inline bool dtype_ok(int d) { return d == ADA_DT_BF16 || d == ADA_DT_F16 || d == ADA_DT_F32; }
inline bool misaligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == ADA_DT_F32 ? 3 : 1)) != 0; }

}  // namespace smp
}  // namespace ada

using namespace ada;

extern "C" size_t ada_sample_workspace_size(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  return 256;
}

extern "C" int ada_sample(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab,
                          const float* temperatures, const float* noise, int64_t ld_noise, int64_t* tokens,
                          float* logprobs, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || vocab <= 0 || ld < vocab || ld_noise < vocab || !smp::dtype_ok(dtype)) return ADA_ERR_INVALID_ARG;
  if (rows == 0) return ADA_OK;
  if (!logits || !temperatures || !noise || !tokens || !workspace) return ADA_ERR_INVALID_ARG;
  if (vocab > (1 << 30) || rows > (1 << 20)) return ADA_ERR_UNSUPPORTED;
  if (smp::misaligned(logits, dtype) || ((uintptr_t)noise & 3) || ((uintptr_t)temperatures & 3) ||
      ((uintptr_t)tokens & 7) || ((uintptr_t)logprobs & 3) || ((uintptr_t)lse & 3) || ((uintptr_t)workspace & 255))
    return ADA_ERR_ALIGNMENT;
  if (workspace_bytes < ada_sample_workspace_size(rows, vocab)) return ADA_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)rows), block(smp::THREADS);
  if (dtype == ADA_DT_BF16)
    (void)ada::launch_k(smp::sample_kernel<__nv_bfloat16>, grid, block, 0, st, (const __nv_bfloat16*)logits, ld, vocab,
                        temperatures, noise, ld_noise, tokens, logprobs, lse);
  else if (dtype == ADA_DT_F16)
    (void)ada::launch_k(smp::sample_kernel<__half>, grid, block, 0, st, (const __half*)logits, ld, vocab, temperatures,
                        noise, ld_noise, tokens, logprobs, lse);
  else
    (void)ada::launch_k(smp::sample_kernel<float>, grid, block, 0, st, (const float*)logits, ld, vocab, temperatures,
                        noise, ld_noise, tokens, logprobs, lse);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}

extern "C" size_t ada_verify_drafts_workspace_size(int32_t batch, int32_t max_drafts, int64_t vocab) {
  if (batch <= 0 || max_drafts < 0 || vocab <= 0) return 0;
  return 256;
}

extern "C" int ada_verify_drafts(const void* target, int dtype, int64_t ld, int32_t total_q, int64_t vocab,
                                 const int64_t* input_ids, const int32_t* cu_seqlens_q, int32_t batch,
                                 int32_t max_drafts, const float* temperatures, const float* uniforms, int64_t ld_u,
                                 const float* noise, int64_t ld_noise, const void* draft_logits,
                                 int64_t draft_stride_b, int64_t draft_stride_d, const float* draft_lse,
                                 int64_t lse_stride_b, int64_t lse_stride_d, int64_t* tokens, int32_t* accepted,
                                 float* logprobs, void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 0 || total_q < 0 || max_drafts < 0 || vocab <= 0 || ld < vocab || ld_noise < vocab ||
      ld_u < max_drafts || !smp::dtype_ok(dtype))
    return ADA_ERR_INVALID_ARG;
  if (batch == 0) return ADA_OK;
  if ((!target && total_q > 0) || (!input_ids && total_q > 0) || !cu_seqlens_q || !temperatures || !noise || !tokens ||
      !accepted || !logprobs || !workspace || (!uniforms && max_drafts > 0))
    return ADA_ERR_INVALID_ARG;
  if ((draft_logits == nullptr) != (draft_lse == nullptr)) return ADA_ERR_INVALID_ARG;
  if (draft_logits && (draft_stride_b < 0 || draft_stride_d < 0 || lse_stride_b < 0 || lse_stride_d < 0))
    return ADA_ERR_INVALID_ARG;
  if (vocab > (1 << 30) || batch > (1 << 20) || max_drafts > 1024) return ADA_ERR_UNSUPPORTED;
  if (smp::misaligned(target, dtype) || smp::misaligned(draft_logits, dtype) || ((uintptr_t)noise & 3) ||
      ((uintptr_t)temperatures & 3) || ((uintptr_t)uniforms & 3) || ((uintptr_t)draft_lse & 3) ||
      ((uintptr_t)input_ids & 7) || ((uintptr_t)cu_seqlens_q & 3) || ((uintptr_t)tokens & 7) ||
      ((uintptr_t)accepted & 3) || ((uintptr_t)logprobs & 3) || ((uintptr_t)workspace & 255))
    return ADA_ERR_ALIGNMENT;
  if (workspace_bytes < ada_verify_drafts_workspace_size(batch, max_drafts, vocab)) return ADA_ERR_WORKSPACE;
  smp::VerifyParams P;
  P.target = target;
  P.ld = ld;
  P.vocab = vocab;
  P.ids = input_ids;
  P.cu_q = cu_seqlens_q;
  P.total_q = total_q;
  P.max_drafts = max_drafts;
  P.temps = temperatures;
  P.uniforms = uniforms;
  P.ld_u = ld_u;
  P.noise = noise;
  P.ld_noise = ld_noise;
  P.draft = draft_logits;
  P.d_sb = draft_stride_b;
  P.d_sd = draft_stride_d;
  P.draft_lse = draft_lse;
  P.l_sb = lse_stride_b;
  P.l_sd = lse_stride_d;
  P.tokens = tokens;
  P.accepted = accepted;
  P.logprobs = logprobs;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)batch), block(smp::THREADS);
  if (dtype == ADA_DT_BF16)
    (void)ada::launch_k(smp::verify_kernel<__nv_bfloat16>, grid, block, 0, st, P);
  else if (dtype == ADA_DT_F16)
    (void)ada::launch_k(smp::verify_kernel<__half>, grid, block, 0, st, P);
  else
    (void)ada::launch_k(smp::verify_kernel<float>, grid, block, 0, st, P);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
