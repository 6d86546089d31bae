// Rotary positions in both layouts, and the 4-bit KV cache's store and read-back.
//
// Rotation (RotaryEmbedding.forward, reference adallm/ops/rotary_embedding.py:45-56, widened): of
// each head's D elements the first r = the table's width are turned, the others copied.  Pairs are
// (i, i + r/2) (half layout, the reference's) or (2i, 2i + 1) (interleaved):
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin,  in fp32, each operation rounded, then to T.
// The scaling for long contexts (linear, YaRN) lives in the fp32 table.
//
// Store: a row's rotated key, rounded to T as a model without the fusion has it, and its value are
// divided by the tensor's scale and packed as kv4.cuh describes.
#include "kv4.cuh"

namespace ada {
namespace kv4 {

struct RotaryParams {
  const int64_t* pos;
  const float* table;  // [max_pos][rot]: cos of rot/2 pairs, then sin
  int64_t max_pos;
  int rot, interleaved;
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // token, head strides (elements)
  void *q_out, *k_out;                         // contiguous [T, heads, D]; k_out may be null
  int hq, hk, hv, d;                           // heads of each (hv = 0: no values), head size
  int64_t tokens;
  // store (null cache: none)
  uint8_t *kc, *vc;
  int64_t s_page, s_head;
  const int32_t* slots;
  int64_t num_slots;
  int page;
  float k_scale, v_scale, k_inv, v_inv;
};

// Largest magnitude of 8 elements; NaN if one is.
template <typename T>
__device__ __forceinline__ float largest(const uint4& x) {
  return larger<T>(max_pairs<T>(0u, x));
}
// Codes of 8 elements over the tensor's scale `div` (inv near 1 / div) and the block's scale s; top: the block's largest
// quotient.
template <typename T>
__device__ __forceinline__ uint32_t pack_codes(const uint4& x, float div, float inv, float s, float top) {
  float y[8];
  unpack8<T>(x, y);
  if (div != 1.f) {
    if (top == INFINITY) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = any_quotient(y[i], div, inv);
    } else {
      quotients(y, div, inv);
    }
  }
  return codes8(y, s, top);
}

// A thread's unit is two chunks of 8 elements (16 bytes each) whose pairs lie within it: chunks i and
// i + r/16 of the turned part (half layout), or neighbours; it keeps U heads (blockIdx.y's share) and walks
// the tokens, so what belongs to a head is worked out once.  Rows and table entries of the next
// STAGES - 1 tokens are on their way by cp.async, each thread's rows into places of its own: with a token
// at a time, or one ahead in registers, an SM has 20-40 KB in flight where HBM wants 66 (95 us, with this
// 62.5, for 16,381 tokens of 40 heads: 83% of the copy rate).  The store's arithmetic (maxima, quotients,
// conversions) takes longer than its bytes: 54 us for 8,195 tokens of 32/16 heads, 34 by its bytes.
constexpr int U = 2, STAGES = 4;
// Bytes of a stage: the CTA's rows, then the table's row.
__host__ __device__ constexpr int stage_bytes(int threads, int heads, int rot) { return threads * heads * 32 + rot * 4; }

template <typename T, bool STORE>
__global__ void __launch_bounds__(256, STORE ? 2 : 3) rotary_store_kernel(const __grid_constant__ RotaryParams P) {
  extern __shared__ __align__(16) uint8_t sm[];
  pdl_wait();
  pdl_trigger();
  const int units = P.d >> 4;
  const int lanes = blockDim.x / units;  // heads side by side
  const int hl = (int)threadIdx.x / units, unit = (int)threadIdx.x - hl * units;
  const int half = P.rot >> 1;
  // Half layout: units of the first rc / 2 hold chunks (i, i + rc / 2), whose pairs lie across them.  The
  // others, and all of the interleaved layout, hold chunks half of what is left apart, so that
  // neighbouring lanes read and write neighbouring 16 bytes either time.
  const int rc = P.pos && !P.interleaved ? P.rot >> 3 : 0;
  const int rest = (2 * units - rc) >> 1;
  const bool apart = unit < (rc >> 1);
  const int c0 = apart ? unit : rc + unit - (rc >> 1), c1 = apart ? unit + (rc >> 1) : c0 + rest;
  const int step = 8 * (c1 - c0);
  // interleaved: which of the chunks are turned, and their 4 pairs' entries
  const bool turn0 = P.pos && P.interleaved && 8 * c0 < P.rot, turn1 = P.pos && P.interleaved && 8 * c1 < P.rot;
  // chunk c's neighbour in its block of 16 (c ^ 1): the lane that holds it, and as which of its two
  int lane0 = 0, lane1 = 0;
  bool one0 = false, one1 = false;
  if (STORE) {
    const int base = (int)(threadIdx.x & 31) - unit;  // (8 units a head: a head's lanes are in one warp)
    auto find = [&](int c, int& lane, bool& one) {
      const int first = c < rc ? 0 : rc, n = c < rc ? rc >> 1 : rest;
      one = c - first >= n;
      lane = base + (first >> 1) + (c - first) - (one ? n : 0);
    };
    find(c0 ^ 1, lane0, one0);
    find(c1 ^ 1, lane1, one1);
  }
  // the thread's heads
  const T* src[U];
  T* dst[U];
  int64_t src_st[U], dst_st[U];
  uint8_t* cache[U];
  bool turn[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = (int)blockIdx.y + (int)gridDim.y * (u * lanes + hl);  // (every share has queries, keys and values)
    src[u] = nullptr;
    dst[u] = nullptr;
    cache[u] = nullptr;
    src_st[u] = dst_st[u] = 0;
    turn[u] = false;
    if (h < P.hq) {
      src[u] = reinterpret_cast<const T*>(P.q) + h * P.q_sh + 8 * c0;
      dst[u] = reinterpret_cast<T*>(P.q_out) + (int64_t)h * P.d + 8 * c0;
      src_st[u] = P.q_st;
      dst_st[u] = (int64_t)P.hq * P.d;
      turn[u] = apart || turn0 || turn1;
    } else if (h < P.hq + P.hk) {
      const int n = h - P.hq;
      src[u] = reinterpret_cast<const T*>(P.k) + n * P.k_sh + 8 * c0;
      if (P.k_out) dst[u] = reinterpret_cast<T*>(P.k_out) + (int64_t)n * P.d + 8 * c0;
      src_st[u] = P.k_st;
      dst_st[u] = (int64_t)P.hk * P.d;
      turn[u] = apart || turn0 || turn1;
      if (STORE) cache[u] = P.kc + n * P.s_head;
    } else if (h < P.hq + P.hk + P.hv) {
      const int n = h - P.hq - P.hk;
      src[u] = reinterpret_cast<const T*>(P.v) + n * P.v_sh + 8 * c0;
      src_st[u] = P.v_st;
      if (STORE) cache[u] = P.vc + n * P.s_head;
    }
  }

  const unsigned tokens = (unsigned)P.tokens;
  const int stage = stage_bytes(blockDim.x, U, P.rot), rows = blockDim.x * U * 32;
  const int lines = P.pos ? P.rot >> 2 : 0;  // 16-byte pieces of a table row
  // the token whose rows are fetched next, and its position
  unsigned ft = blockIdx.x;
  auto place = [&](unsigned t) { return lines && t < tokens ? P.pos[t] : (int64_t)0; };
  int64_t fpos = place(ft);
  auto fetch = [&](int s) {
    if (ft < tokens) {
      const uint32_t at = smem_addr(sm) + s * stage + threadIdx.x * 16;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (src[u]) {
          const T* p = src[u] + ft * src_st[u];
          cp16(at + (2 * u) * blockDim.x * 16, p);
          cp16(at + (2 * u + 1) * blockDim.x * 16, p + step);
        }
      }
      const float* row = P.table + min(max(fpos, (int64_t)0), P.max_pos - 1) * P.rot;
      for (int i = threadIdx.x; i < lines; i += blockDim.x) cp16(smem_addr(sm) + s * stage + rows + 16 * i, row + 4 * i);
      ft += gridDim.x;
      fpos = place(ft);
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);
  int s = 0;
  int slot = -1;
  if (STORE && blockIdx.x < tokens) slot = P.slots[blockIdx.x];
  for (unsigned t = blockIdx.x; t < tokens; t += gridDim.x) {
    const bool store = STORE && slot >= 0 && slot < P.num_slots;
    const int page = store ? (int)((unsigned)slot / (unsigned)P.page) : 0;
    const int srow = store ? slot - page * P.page : 0;
    if (STORE && t + gridDim.x < tokens) slot = P.slots[t + gridDim.x];
    cp_wait<STAGES - 2>();
    __syncthreads();  // every thread's part of the table row is there, and the stage before is read
    fetch(s == 0 ? STAGES - 1 : s - 1);
    const uint8_t* mine = sm + s * stage + threadIdx.x * 16;
    float cs[8], sn[8];
    const float* row = reinterpret_cast<const float*>(sm + s * stage + rows);
    if (apart) {  // 8 pairs
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        *reinterpret_cast<float4*>(cs + i) = *reinterpret_cast<const float4*>(row + 8 * c0 + i);
        *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(row + half + 8 * c0 + i);
      }
    } else {
      if (turn0) {
        *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(row + 4 * c0);
        *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(row + half + 4 * c0);
      }
      if (turn1) {
        *reinterpret_cast<float4*>(cs + 4) = *reinterpret_cast<const float4*>(row + 4 * c1);
        *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(row + half + 4 * c1);
      }
    }
    s = s == STAGES - 1 ? 0 : s + 1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!src[u]) continue;
      uint4 o0 = *reinterpret_cast<const uint4*>(mine + (2 * u) * blockDim.x * 16);
      uint4 o1 = *reinterpret_cast<const uint4*>(mine + (2 * u + 1) * blockDim.x * 16);
      if (turn[u]) {
        float x[8], z[8], y[8], w[8];
        unpack8<T>(o0, x);
        unpack8<T>(o1, z);
        // single operations: joined to fused ones, or packed (which the compiler joins), they round differently
        if (!apart) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = __fsub_rn(__fmul_rn(x[2 * i], cs[i]), __fmul_rn(x[2 * i + 1], sn[i]));
            y[2 * i + 1] = __fadd_rn(__fmul_rn(x[2 * i + 1], cs[i]), __fmul_rn(x[2 * i], sn[i]));
            w[2 * i] = __fsub_rn(__fmul_rn(z[2 * i], cs[4 + i]), __fmul_rn(z[2 * i + 1], sn[4 + i]));
            w[2 * i + 1] = __fadd_rn(__fmul_rn(z[2 * i + 1], cs[4 + i]), __fmul_rn(z[2 * i], sn[4 + i]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] = __fsub_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(z[i], sn[i]));
            w[i] = __fadd_rn(__fmul_rn(z[i], cs[i]), __fmul_rn(x[i], sn[i]));
          }
        }
        if (apart || turn0) o0 = pack8<T>(y);
        if (apart || turn1) o1 = pack8<T>(w);
      }
      if (dst[u]) {
        T* p = dst[u] + t * dst_st[u];
        *reinterpret_cast<uint4*>(p) = o0;
        *reinterpret_cast<uint4*>(p + step) = o1;
      }
      if (!STORE || !store || cache[u] == nullptr) continue;  // (the same for a head's 8 lanes)
      const float top[2] = {largest<T>(o0), largest<T>(o1)};
      const uint32_t head_lanes = 0xFFu << (threadIdx.x & 24);
      const float a0 = __shfl_sync(head_lanes, top[0], lane0), a1 = __shfl_sync(head_lanes, top[1], lane0);
      const float b0 = __shfl_sync(head_lanes, top[0], lane1), b1 = __shfl_sync(head_lanes, top[1], lane1);
      const bool is_v = (int)blockIdx.y + (int)gridDim.y * (u * lanes + hl) >= P.hq + P.hk;
      const float div = is_v ? P.v_scale : P.k_scale, inv = is_v ? P.v_inv : P.k_inv;
      // (the largest quotient is the largest element's: rounding keeps the order)
      const float m0 = any_quotient(max_nan(top[0], one0 ? a1 : a0), div, inv);
      const float m1 = any_quotient(max_nan(top[1], one1 ? b1 : b0), div, inv);
      const uint32_t s0 = scale_code(m0), s1 = scale_code(m1);
      uint8_t* codes = cache[u] + page * P.s_page + srow * ROW;
      uint8_t* scales = cache[u] + page * P.s_page + P.page * ROW + srow * SROW;
      *reinterpret_cast<uint32_t*>(codes + 4 * c0) = pack_codes<T>(o0, div, inv, scale_value(s0), m0);
      *reinterpret_cast<uint32_t*>(codes + 4 * c1) = pack_codes<T>(o1, div, inv, scale_value(s1), m1);
      if (!(c0 & 1)) scales[c0 >> 1] = (uint8_t)s0;
      if (!(c1 & 1)) scales[c1 >> 1] = (uint8_t)s1;
    }
  }
}

struct ReadParams {
  const uint8_t *kc, *vc;
  int64_t s_page, s_head;
  const int32_t* slots;
  int64_t num_slots, tokens;
  int page, hk;
  float k_scale, v_scale;
  void *k, *v;  // contiguous [T, Hkv, D]
};

// A CTA reads READ_TOKENS tokens; a thread takes 8 elements (4 bytes of codes -> 16 of values) of one
// head of K or V of each of them, all loads before the first store.
constexpr int READ_TOKENS = 4;
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadParams P) {
  pdl_wait();
  pdl_trigger();
  const int64_t t0 = (int64_t)blockIdx.x * READ_TOKENS;
  int64_t page_at[READ_TOKENS];
  int row[READ_TOKENS];
  bool there[READ_TOKENS];
#pragma unroll
  for (int i = 0; i < READ_TOKENS; ++i) {
    const int slot = t0 + i < P.tokens ? P.slots[t0 + i] : -1;
    there[i] = slot >= 0 && slot < P.num_slots;
    const int page = there[i] ? (int)((unsigned)slot / (unsigned)P.page) : 0;
    page_at[i] = page * P.s_page;
    row[i] = there[i] ? slot - page * P.page : 0;
  }
  const int c = threadIdx.x & 15, e0 = 8 * c;
  for (int h = threadIdx.x >> 4; h < 2 * P.hk; h += 16) {
    const bool is_v = h >= P.hk;
    const int head = is_v ? h - P.hk : h;
    const uint8_t* src = (is_v ? P.vc : P.kc) + head * P.s_head;
    const float mul = is_v ? P.v_scale : P.k_scale;
    uint32_t codes[READ_TOKENS], sc[READ_TOKENS];
#pragma unroll
    for (int i = 0; i < READ_TOKENS; ++i) {
      codes[i] = sc[i] = 0;
      if (there[i]) {
        codes[i] = *reinterpret_cast<const uint32_t*>(src + page_at[i] + row[i] * ROW + 4 * c);
        sc[i] = src[page_at[i] + P.page * ROW + row[i] * SROW + (c >> 1)];
      }
    }
    T* out = reinterpret_cast<T*>(is_v ? P.v : P.k) + (t0 * P.hk + head) * D + e0;
#pragma unroll
    for (int i = 0; i < READ_TOKENS; ++i) {
      if (t0 + i >= P.tokens) break;
      uint32_t w[4];
      widen8(codes[i], w);
      const uint32_t s = scale_f16x2(sc[i]);
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = mul_f16x2(w[j], s);  // exact
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        f[2 * j] = mul == 1.f ? v.x : __fmul_rn(v.x, mul);
        f[2 * j + 1] = mul == 1.f ? v.y : __fmul_rn(v.y, mul);
      }
      *reinterpret_cast<uint4*>(out + (int64_t)i * P.hk * D) = pack8<T>(f);
    }
  }
}

template <typename T, bool STORE>
inline int launch_rotary_as(const RotaryParams& P, cudaStream_t st) {
  // heads side by side: as many as 256 threads hold, shared out evenly over the CTAs they take (by fours:
  // whole warps for the store's shuffles, 8 units a head there)
  const int units = P.d / 16, heads = P.hq + P.hk + P.hv, most = 256 / units;
  const int shares = (int)cdiv(heads, U * most);
  const int even = (int)cdiv(cdiv(heads, U * shares), 4) * 4, lanes = even <= most ? even : most;
  const int ys = (int)cdiv(heads, U * lanes), threads = lanes * units;
  const int smem = STAGES * stage_bytes(threads, U, P.pos ? P.rot : 0);
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ADA_ERR_CUDA;
  if (smem > 48 * 1024 && !ready[dev]) {
    if (cudaFuncSetAttribute(rotary_store_kernel<T, STORE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             STAGES * stage_bytes(256, U, 1024)) != cudaSuccess)
      return ADA_ERR_CUDA;
    ready[dev] = true;
  }
  // as many CTAs as the SMs hold (128 or 80 registers a thread, shared memory) stay and walk the tokens
  const int by_regs = 65536 / ((STORE ? 128 : 80) * threads), by_smem = 232448 / (smem + 1024);
  const int64_t walkers = cdiv(148 * (by_regs < by_smem ? by_regs : by_smem), ys);
  (void)launch_k(rotary_store_kernel<T, STORE>, dim3((unsigned)(P.tokens < walkers ? P.tokens : walkers), (unsigned)ys),
                 dim3((unsigned)threads), (size_t)smem, st, P);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
template <typename T>
inline int launch_rotary(const RotaryParams& P, cudaStream_t st) {
  return P.kc ? launch_rotary_as<T, true>(P, st) : launch_rotary_as<T, false>(P, st);
}

// Checks that ada_rotary and the store share.
static int rotary_ok(const RotaryParams& P, int64_t tokens, int dtype) {
  if (tokens < 0 || P.hq < 0 || P.hk < 0 || P.hv < 0 || P.d <= 0) return ADA_ERR_INVALID_ARG;
  if (dtype != ADA_DT_BF16 && dtype != ADA_DT_F16) return ADA_ERR_INVALID_ARG;
  if (P.pos) {
    if (!P.table || P.max_pos <= 0 || P.rot <= 0 || P.rot > P.d) return ADA_ERR_INVALID_ARG;
    if (P.rot % 16) return ADA_ERR_UNSUPPORTED;
    if (misaligned16(P.table)) return ADA_ERR_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(P.pos) & 7) return ADA_ERR_ALIGNMENT;
  }
  if (P.d % 16 || P.d > 1024 || tokens > 0x7fffffff) return ADA_ERR_UNSUPPORTED;
  if ((P.hq && (!P.q || !P.q_out)) || (P.hk && !P.k) || (P.hv && !P.v)) return ADA_ERR_INVALID_ARG;
  // a pair's halves belong to two threads: the outputs are not the inputs
  if ((P.hq && P.q_out == P.q) || (P.k_out && P.k_out == P.k)) return ADA_ERR_INVALID_ARG;
  if (misaligned16(P.q) || misaligned16(P.k) || misaligned16(P.v) || misaligned16(P.q_out) || misaligned16(P.k_out))
    return ADA_ERR_ALIGNMENT;
  if ((P.q_st | P.q_sh | P.k_st | P.k_sh | P.v_st | P.v_sh) & 7) return ADA_ERR_ALIGNMENT;
  return ADA_OK;
}

}  // namespace kv4
}  // namespace ada

using namespace ada;

extern "C" int ada_rotary(const int64_t* positions, const void* q, int64_t q_stride_t, int64_t q_stride_h,
                          const void* k, int64_t k_stride_t, int64_t k_stride_h, void* q_out, void* k_out,
                          int64_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                          const float* cos_sin, int64_t max_position, int32_t rotary_dim, int32_t interleaved,
                          int dtype, void* stream) {
  kv4::RotaryParams P{};
  P.pos = positions;
  P.table = cos_sin;
  P.max_pos = max_position;
  P.rot = rotary_dim;
  P.interleaved = interleaved != 0;
  P.q = q;
  P.k = k;
  P.q_st = q_stride_t;
  P.q_sh = q_stride_h;
  P.k_st = k_stride_t;
  P.k_sh = k_stride_h;
  P.q_out = q_out;
  P.k_out = k_out;
  P.hq = num_q_heads;
  P.hk = num_kv_heads;
  P.d = head_dim;
  P.tokens = num_tokens;
  if (num_tokens == 0) return ADA_OK;
  if (!positions || (num_kv_heads > 0 && !k_out)) return ADA_ERR_INVALID_ARG;
  if (const int e = kv4::rotary_ok(P, num_tokens, dtype)) return e;
  if (num_q_heads + num_kv_heads == 0) return ADA_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == ADA_DT_BF16 ? kv4::launch_rotary<__nv_bfloat16>(P, st) : kv4::launch_rotary<__half>(P, st);
}

extern "C" int ada_kv4_store(const int64_t* positions, const void* q, int64_t q_stride_t, int64_t q_stride_h,
                             const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                             int64_t v_stride_h, void* q_out, int64_t num_tokens, int32_t num_q_heads,
                             int32_t num_kv_heads, int32_t head_dim, const float* cos_sin, int64_t max_position,
                             int32_t rotary_dim, int32_t interleaved, const int32_t* slot_mapping, uint8_t* k_cache,
                             uint8_t* v_cache, int64_t kv_stride_page, int64_t kv_stride_head, int64_t num_pages,
                             int32_t page_size, float k_scale, float v_scale, int dtype, void* stream) {
  if (head_dim != kv4::D) return ADA_ERR_UNSUPPORTED;
  if (num_tokens < 0 || !kv4::scale_ok(k_scale) || !kv4::scale_ok(v_scale)) return ADA_ERR_INVALID_ARG;
  if (num_tokens == 0) return ADA_OK;
  if (!k || !v || !slot_mapping || (reinterpret_cast<uintptr_t>(slot_mapping) & 3)) return ADA_ERR_INVALID_ARG;
  if (const int e = kv4::cache_ok(k_cache, v_cache, kv_stride_page, kv_stride_head, num_pages, num_kv_heads, page_size))
    return e;
  kv4::RotaryParams P{};
  P.pos = positions;
  P.table = cos_sin;
  P.max_pos = max_position;
  P.rot = positions ? rotary_dim : 0;
  P.interleaved = interleaved != 0;
  P.q = q;
  P.k = k;
  P.v = v;
  P.q_st = q_stride_t;
  P.q_sh = q_stride_h;
  P.k_st = k_stride_t;
  P.k_sh = k_stride_h;
  P.v_st = v_stride_t;
  P.v_sh = v_stride_h;
  P.q_out = q_out;
  P.hq = num_q_heads;
  P.hk = P.hv = num_kv_heads;
  P.d = head_dim;
  P.tokens = num_tokens;
  P.kc = k_cache;
  P.vc = v_cache;
  P.s_page = kv_stride_page;
  P.s_head = kv_stride_head;
  P.slots = slot_mapping;
  P.num_slots = num_pages * page_size;
  P.page = page_size;
  P.k_scale = k_scale;
  P.v_scale = v_scale;
  P.k_inv = 1.f / k_scale;
  P.v_inv = 1.f / v_scale;
  if (const int e = kv4::rotary_ok(P, num_tokens, dtype)) return e;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == ADA_DT_BF16 ? kv4::launch_rotary<__nv_bfloat16>(P, st) : kv4::launch_rotary<__half>(P, st);
}

extern "C" int ada_kv4_read(const uint8_t* k_cache, const uint8_t* v_cache, int64_t kv_stride_page,
                            int64_t kv_stride_head, int64_t num_pages, int32_t page_size, int32_t num_kv_heads,
                            int32_t head_dim, const int32_t* slot_mapping, int64_t num_tokens, float k_scale,
                            float v_scale, void* k, void* v, int dtype, void* stream) {
  if (num_tokens < 0 || !kv4::scale_ok(k_scale) || !kv4::scale_ok(v_scale)) return ADA_ERR_INVALID_ARG;
  if (dtype != ADA_DT_BF16 && dtype != ADA_DT_F16) return ADA_ERR_INVALID_ARG;
  if (head_dim != kv4::D) return ADA_ERR_UNSUPPORTED;
  if (num_tokens == 0) return ADA_OK;
  if (const int e = kv4::cache_ok(k_cache, v_cache, kv_stride_page, kv_stride_head, num_pages, num_kv_heads, page_size))
    return e;
  if (!slot_mapping || !k || !v) return ADA_ERR_INVALID_ARG;
  if (kv4::misaligned16(k) || kv4::misaligned16(v) || (reinterpret_cast<uintptr_t>(slot_mapping) & 3))
    return ADA_ERR_ALIGNMENT;
  kv4::ReadParams P{};
  P.kc = k_cache;
  P.vc = v_cache;
  P.s_page = kv_stride_page;
  P.s_head = kv_stride_head;
  P.slots = slot_mapping;
  P.num_slots = num_pages * page_size;
  P.tokens = num_tokens;
  P.page = page_size;
  P.hk = num_kv_heads;
  P.k_scale = k_scale;
  P.v_scale = v_scale;
  P.k = k;
  P.v = v;
  const int64_t grid = cdiv(num_tokens, (int64_t)kv4::READ_TOKENS);
  if (grid > 0x7fffffff) return ADA_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == ADA_DT_BF16)
    (void)launch_k(kv4::read_kernel<__nv_bfloat16>, dim3((unsigned)grid), dim3(256), 0, st, P);
  else
    (void)launch_k(kv4::read_kernel<__half>, dim3((unsigned)grid), dim3(256), 0, st, P);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
