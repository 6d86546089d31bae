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
  // store (null cache: none)
  uint8_t *kc, *vc;
  int64_t s_page, s_head;
  const int32_t* slots;
  int64_t num_slots;
  int page;
  float k_scale, v_scale;
};

// One CTA per (token, y-th share of the heads).  A thread keeps one chunk of 8 elements (16 bytes)
// and walks the heads, so a token's cos and sin are read once per thread.
template <typename T>
__global__ void __launch_bounds__(256) rotary_store_kernel(RotaryParams P) {
  pdl_wait();
  pdl_trigger();
  const int chunks = P.d >> 3;
  const int lanes = blockDim.x / chunks;  // heads side by side
  const int c = threadIdx.x % chunks, e0 = 8 * c;
  const int64_t t = blockIdx.x;
  const int half = P.rot >> 1;
  const bool turned = P.pos != nullptr && e0 < P.rot;
  const bool second = !P.interleaved && e0 >= half;
  const int other = second ? e0 - half : e0 + half;  // the partners' chunk (half layout)
  float cs[8], sn[8];
  if (turned) {
    const int64_t p = min(max(__ldg(P.pos + t), (int64_t)0), P.max_pos - 1);
    const float* row = P.table + p * P.rot;
    if (P.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[i] = __ldg(row + e0 / 2 + i);
        sn[i] = __ldg(row + half + e0 / 2 + i);
      }
    } else {
      const int j = second ? other : e0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = __ldg(row + j + i);
        sn[i] = __ldg(row + half + j + i);
      }
    }
  }
  int64_t slot = -1;
  if (P.kc) slot = __ldg(P.slots + t);
  const bool store = slot >= 0 && slot < P.num_slots;
  const int64_t block = store ? slot / P.page : 0;
  const int srow = store ? (int)(slot - block * P.page) : 0;
  const int heads = P.hq + P.hk + P.hv;
  for (int h0 = blockIdx.y * lanes; h0 < heads; h0 += gridDim.y * lanes) {
    const int h = h0 + (int)threadIdx.x / chunks;
    const bool there = h < heads;
    const bool is_q = h < P.hq, is_v = h >= P.hq + P.hk;
    const int head = is_q ? h : is_v ? h - P.hq - P.hk : h - P.hq;
    float y[8];
    if (there) {
      const T* src = is_q   ? reinterpret_cast<const T*>(P.q) + t * P.q_st + head * P.q_sh
                     : is_v ? reinterpret_cast<const T*>(P.v) + t * P.v_st + head * P.v_sh
                            : reinterpret_cast<const T*>(P.k) + t * P.k_st + head * P.k_sh;
      uint4 own = *reinterpret_cast<const uint4*>(src + e0);
      if (turned && !is_v) {
        float x[8];
        unpack8<T>(own, x);
        if (P.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = __fsub_rn(__fmul_rn(x[2 * i], cs[i]), __fmul_rn(x[2 * i + 1], sn[i]));
            y[2 * i + 1] = __fadd_rn(__fmul_rn(x[2 * i + 1], cs[i]), __fmul_rn(x[2 * i], sn[i]));
          }
        } else {
          float z[8];
          unpack8<T>(*reinterpret_cast<const uint4*>(src + other), z);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            y[i] = second ? __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(z[i], sn[i]))
                          : __fsub_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(z[i], sn[i]));
        }
        own = pack8<T>(y);
      }
      if (is_q) {
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(P.q_out) + (t * P.hq + head) * P.d + e0) = own;
      } else if (!is_v && P.k_out) {
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(P.k_out) + (t * P.hk + head) * P.d + e0) = own;
      }
      unpack8<T>(own, y);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = 0.f;
    }
    if (!P.kc) continue;
    const float div = is_v ? P.v_scale : P.k_scale;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (div != 1.f) y[i] = __fdiv_rn(y[i], div);
      top = max_nan(top, fabsf(y[i]));
    }
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));  // a scale's 16 elements are two neighbouring lanes'
    if (!there || is_q || !store) continue;
    const uint32_t sc = scale_code(top);
    uint8_t* out = (is_v ? P.vc : P.kc) + block * P.s_page + head * P.s_head;
    *reinterpret_cast<uint32_t*>(out + (int64_t)srow * ROW + 4 * c) = codes8(y, scale_value(sc));
    if (!(c & 1)) out[(int64_t)P.page * ROW + srow * SROW + (c >> 1)] = (uint8_t)sc;
  }
}

struct ReadParams {
  const uint8_t *kc, *vc;
  int64_t s_page, s_head;
  const int32_t* slots;
  int64_t num_slots, items;
  int page, hk;
  float k_scale, v_scale;
  void *k, *v;  // contiguous [T, Hkv, D]
};

// One thread per (token, head, block of 16): its codes and scale of both caches.
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(ReadParams P) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= P.items) return;
  const int b = (int)(i % SROW);
  const int64_t th = i / SROW, t = th / P.hk;
  const int head = (int)(th - t * P.hk);
  const int64_t slot = __ldg(P.slots + t);
  const bool there = slot >= 0 && slot < P.num_slots;
  const int64_t blk = there ? slot / P.page : 0;
  const int64_t row = there ? slot - blk * P.page : 0;
  const int64_t at = blk * P.s_page + head * P.s_head;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint8_t* src = (w ? P.vc : P.kc) + at;
    const float mul = w ? P.v_scale : P.k_scale;
    uint2 codes = make_uint2(0, 0);
    uint32_t sc = 0;
    if (there) {
      codes = *reinterpret_cast<const uint2*>(src + row * ROW + 8 * b);
      sc = src[(int64_t)P.page * ROW + row * SROW + b];
    }
    const float s = scale_value(sc);
    T* out = reinterpret_cast<T*>(w ? P.v : P.k) + th * D + BLOCK * b;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t h[4];
      e2m1x8_to_f16x8(p ? codes.y : codes.x, h);
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        f[2 * j] = __fmul_rn(v.x * s, mul);  // code * scale is exact
        f[2 * j + 1] = __fmul_rn(v.y * s, mul);
      }
      *reinterpret_cast<uint4*>(out + 8 * p) = pack8<T>(f);
    }
  }
}

template <typename T>
inline void launch_rotary(const RotaryParams& P, int64_t tokens, cudaStream_t st) {
  const int chunks = P.d / 8;
  const int lanes = 256 / chunks;
  const int shares = (int)cdiv(P.hq + P.hk + P.hv, lanes);
  // few tokens: the heads' shares on CTAs of their own; many: one CTA walks a token's heads
  const int y = tokens * shares <= 1024 ? shares : 1;
  (void)launch_k(rotary_store_kernel<T>, dim3((unsigned)tokens, (unsigned)y), dim3((unsigned)(lanes * chunks)), 0, st, P);
}

// Checks that ada_rotary and the store share.
static int rotary_ok(const RotaryParams& P, int64_t tokens, int dtype) {
  if (tokens < 0 || P.hq < 0 || P.hk < 0 || P.hv < 0 || P.d <= 0) return ADA_ERR_INVALID_ARG;
  if (dtype != ADA_DT_BF16 && dtype != ADA_DT_F16) return ADA_ERR_INVALID_ARG;
  if (P.pos) {
    if (!P.table || P.max_pos <= 0 || P.rot <= 0 || P.rot > P.d) return ADA_ERR_INVALID_ARG;
    if (P.rot % 16) return ADA_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(P.table) & 3) return ADA_ERR_ALIGNMENT;
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
  if (num_tokens == 0) return ADA_OK;
  if (!positions || (num_kv_heads > 0 && !k_out)) return ADA_ERR_INVALID_ARG;
  if (const int e = kv4::rotary_ok(P, num_tokens, dtype)) return e;
  if (num_q_heads + num_kv_heads == 0) return ADA_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == ADA_DT_BF16)
    kv4::launch_rotary<__nv_bfloat16>(P, num_tokens, st);
  else
    kv4::launch_rotary<__half>(P, num_tokens, st);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}

extern "C" int ada_kv4_store(const int64_t* positions, const void* q, int64_t q_stride_t, int64_t q_stride_h,
                             const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                             int64_t v_stride_h, void* q_out, int64_t num_tokens, int32_t num_q_heads,
                             int32_t num_kv_heads, int32_t head_dim, const float* cos_sin, int64_t max_position,
                             int32_t rotary_dim, int32_t interleaved, const int32_t* slot_mapping, uint8_t* k_cache,
                             uint8_t* v_cache, int64_t kv_stride_page, int64_t kv_stride_head, int64_t num_pages,
                             int32_t page_size, float k_scale, float v_scale, int dtype, void* stream) {
  if (head_dim != kv4::D) return ADA_ERR_UNSUPPORTED;
  if (num_tokens < 0 || !(k_scale > 0.f) || !(v_scale > 0.f)) return ADA_ERR_INVALID_ARG;
  if (num_tokens == 0) return ADA_OK;
  if (!k || !v || !slot_mapping || (reinterpret_cast<uintptr_t>(slot_mapping) & 3)) return ADA_ERR_INVALID_ARG;
  if (const int e = kv4::cache_ok(k_cache, v_cache, kv_stride_page, kv_stride_head, num_pages, num_kv_heads, page_size))
    return e;
  kv4::RotaryParams P{};
  P.pos = positions;
  P.table = cos_sin;
  P.max_pos = max_position;
  P.rot = rotary_dim;
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
  P.kc = k_cache;
  P.vc = v_cache;
  P.s_page = kv_stride_page;
  P.s_head = kv_stride_head;
  P.slots = slot_mapping;
  P.num_slots = num_pages * page_size;
  P.page = page_size;
  P.k_scale = k_scale;
  P.v_scale = v_scale;
  if (const int e = kv4::rotary_ok(P, num_tokens, dtype)) return e;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == ADA_DT_BF16)
    kv4::launch_rotary<__nv_bfloat16>(P, num_tokens, st);
  else
    kv4::launch_rotary<__half>(P, num_tokens, st);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}

extern "C" int ada_kv4_read(const uint8_t* k_cache, const uint8_t* v_cache, int64_t kv_stride_page,
                            int64_t kv_stride_head, int64_t num_pages, int32_t page_size, int32_t num_kv_heads,
                            int32_t head_dim, const int32_t* slot_mapping, int64_t num_tokens, float k_scale,
                            float v_scale, void* k, void* v, int dtype, void* stream) {
  if (num_tokens < 0 || !(k_scale > 0.f) || !(v_scale > 0.f)) return ADA_ERR_INVALID_ARG;
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
  P.items = num_tokens * num_kv_heads * kv4::SROW;
  P.page = page_size;
  P.hk = num_kv_heads;
  P.k_scale = k_scale;
  P.v_scale = v_scale;
  P.k = k;
  P.v = v;
  const int64_t grid = cdiv(P.items, 256);
  if (grid > 0x7fffffff) return ADA_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == ADA_DT_BF16)
    (void)launch_k(kv4::read_kernel<__nv_bfloat16>, dim3((unsigned)grid), dim3(256), 0, st, P);
  else
    (void)launch_k(kv4::read_kernel<__half>, dim3((unsigned)grid), dim3(256), 0, st, P);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
