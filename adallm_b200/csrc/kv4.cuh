// The 4-bit paged KV cache: layout and conversions shared by its kernels.
//
// One block per (page, KV head), `page` rows of 128 elements (page a multiple of 16):
//   bytes [0, 64 * page)           the rows' e2m1 codes, 64 bytes a row, even element in the low nibble
//   bytes [64 * page, 72 * page)   the rows' e4m3 scales, 8 bytes a row, one for 16 elements
// value = code * scale * (the tensor's scale).  A block is contiguous, so a tile of 16 rows is two
// contiguous pieces (1,024 and 128 bytes) and a page of one head stays together in DRAM, where a
// row of 72 bytes among other heads' would leave no 16-byte alignment to load with.
// code * scale has at most 6 significant bits and lies in [2^-10, 2688]: exact in fp16 and in bf16.
//
// The kernels read lists, tables and queries by plain loads and not by those through the read-only path (ld.global.nc),
// whose data must not change while a kernel runs: theirs is written by the launch before, which
// overlaps their start (step_metadata.cu's CTAs read tables that others of it extend).
#pragma once

#include <type_traits>

#include "common.cuh"

namespace ada {
namespace kv4 {

constexpr int D = 128;
constexpr int BLOCK = 16;           // elements a scale
constexpr int ROW = D / 2;          // bytes of codes a row
constexpr int SROW = D / BLOCK;     // bytes of scales a row
constexpr int ROW_BYTES = ROW + SROW;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two floats in one register pair: the packed fp32 operations round each half like the single ones.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Largest magnitudes of the even and the odd elements of `acc` and 8 more, in a pair; NaN if one is.
template <typename T>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<T, __half>::value)
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t max_pairs(uint32_t acc, const uint4& x) {
  constexpr uint32_t MAGNITUDE = 0x7FFF7FFFu;
  return max2_nan<T>(max2_nan<T>(acc, max2_nan<T>(x.x & MAGNITUDE, x.y & MAGNITUDE)),
                     max2_nan<T>(x.z & MAGNITUDE, x.w & MAGNITUDE));
}
// The larger of a pair; NaN if one is.
template <typename T>
__device__ __forceinline__ float larger(const uint32_t& pair) {
  const T* h = reinterpret_cast<const T*>(&pair);
  return max_nan(to_f32(h[0]), to_f32(h[1]));
}

// x / d given r near 1 / d: one Newton step on the quotient's remainder (Markstein 1990).  Correctly rounded where x / d
// lies further than 2^-44 of itself from a midpoint of fp32 or on none: for divisors of few bits (6; the e4m3 scales)
// always (2^-27 and more), for others but for one quotient in 2^20, which is one step (2^-24) off then.  (x may be an
// infinity, or the quotient one.)
__device__ __forceinline__ float any_quotient(float x, float d, float r) {
  const float q = x * r;
  return fabsf(q) == INFINITY ? q : fmaf(fmaf(-q, d, x), r, q);
}

// The same of 8 finite elements, two an instruction.
__device__ __forceinline__ void quotients(float* x, float d, float r) {
  const uint64_t minus = pair(-d, -d), r2 = pair(r, r);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t a = pair(x[i], x[i + 1]), q = mul2(a, r2);
    unpair(fma2(fma2(q, minus, a), r2, q), x[i], x[i + 1]);
  }
}

// e4m3 byte of max|x| / 6, saturated to 448; NaN when the block holds one (the block then reads as NaN).
__device__ __forceinline__ uint32_t scale_code(float top) {
  return f32x2_to_e4m3x2(any_quotient(top, 6.f, 1.f / 6.f), 0.f) & 0xFFu;
}
__device__ __forceinline__ float scale_value(uint32_t code) {
  const uint32_t h = e4m3x2_to_f16x2((uint16_t)code);
  return __half2float(__ushort_as_half((unsigned short)(h & 0xFFFFu)));
}

// Eight elements -> eight codes: the nearest e2m1 to x / s, ties to even.  x * (1 / s) alone puts exact
// ties, which bf16 values often are, on either side; the quotient is the correctly rounded one.  A block
// whose scale is 0 (all below 2^-10 * 6) holds zeros.  top: the block's max |x|.
__device__ __forceinline__ uint32_t codes8(float* x, float s, float top) {
  if (!(s > 0.f)) return 0u;
  if (top == INFINITY) {  // infinities saturate like the largest floats (inf - inf would not)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -3.4028234663852886e38f), 3.4028234663852886e38f);
  }
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  quotients(x, s, r);
  return f32x8_to_e2m1x8(x);
}
// Eight codes -> their values, four f16x2 (low half = even element).
__device__ __forceinline__ void widen8(uint32_t w, uint32_t* h) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A scale's value in both halves.
__device__ __forceinline__ uint32_t scale_f16x2(uint32_t e4m3) {
  const uint32_t h = e4m3x2_to_f16x2((uint16_t)e4m3);
  return prmt(h, h, 0x1010);
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A query row enters the products multiplied by a power of two that brings its largest magnitude
// `top` into [2^14, 2^15), so that bf16 rows of any size keep their bits in fp16 (what falls under fp16's
// range is 2^-38 of the largest); the exponent is taken back in the factor of the scores, which stops
// at 2^90: |score| < 2^34 then keeps every product finite, and a row of such a factor is decided by its
// largest score alone.  (It is never 0: a masked score of -inf stays one.)  A row of zeros, or with an infinity or NaN, is left as it is.
__device__ __forceinline__ int query_exponent(float top) {
  if (!(top > 0.f) || !(top < INFINITY)) return 0;
  const int e = (int)(__float_as_uint(top) >> 23) - 127;  // (-127 for a subnormal)
  return 14 - max(e, -100);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -127 < e < 128
__device__ __forceinline__ float score_factor(float scale_log2, int exponent) {
  return fmaxf(fminf(scale_log2 * pow2(-exponent), 1.2379400392853803e27f), 1e-36f);
}

// Probabilities enter the products in fp16 as 2^6 times the weight against a row's reference, which a score passes by 8
// (log2) at most and, in the prefill kernel's rounding, 1 more: 2^15 then.  Their half step is 2^-11 of themselves from 2^-20
// of the reference's weight on, and 2^-31 of that below (without the factor 2^-25: thousands of keys of less, behind one
// that takes most, were all lost).  The sums, in fp32, carry the same factor.
constexpr float P_LOG2 = 6.f;

// A tensor's scale that both it and its reciprocal are good for as fp32 factors (no NaN, infinity or subnormal).
inline bool scale_ok(float s) { return s >= 1e-30f && s <= 1e30f; }
inline bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// Checks of a cache's layout that every entry shares.
inline int cache_ok(const void* kc, const void* vc, int64_t s_page, int64_t s_head, int64_t num_pages, int32_t heads,
                    int32_t page) {
  if (!kc || !vc || num_pages <= 0 || heads <= 0 || page <= 0) return ADA_ERR_INVALID_ARG;
  if (page % 16 || page > (1 << 24)) return ADA_ERR_UNSUPPORTED;  // (places in a block are counted in 32 bits)
  if (s_head < (int64_t)page * ROW_BYTES || s_page < (int64_t)page * ROW_BYTES) return ADA_ERR_INVALID_ARG;
  if (misaligned16(kc) || misaligned16(vc) || (s_page & 15) || (s_head & 15)) return ADA_ERR_ALIGNMENT;
  return ADA_OK;
}

// Checks that the attention entries share.
inline int attn_ok(const void* q, int qd, int64_t q_st, int64_t q_sh, const void* out, int od, int64_t o_st, int64_t o_sh,
                   const void* kc, const void* vc, int64_t s_page, int64_t s_head, int64_t num_pages, const int32_t* bt,
                   int64_t bt_stride, int32_t max_pages, int32_t hq, int32_t hkv, int32_t d, int32_t page, float scale,
                   float k_scale, float v_scale, int32_t window) {
  if (!q || !out || !bt || hq <= 0 || hkv <= 0 || max_pages <= 0) return ADA_ERR_INVALID_ARG;
  if ((qd != ADA_DT_BF16 && qd != ADA_DT_F16) || (od != ADA_DT_BF16 && od != ADA_DT_F16)) return ADA_ERR_INVALID_ARG;
  if (d != D) return ADA_ERR_UNSUPPORTED;
  if (const int e = cache_ok(kc, vc, s_page, s_head, num_pages, hkv, page)) return e;
  if (hq % hkv || window < 0 || bt_stride < max_pages) return ADA_ERR_INVALID_ARG;
  if (!(scale > 0.f) || !(scale <= 1e30f) || !scale_ok(k_scale) || !scale_ok(v_scale)) return ADA_ERR_INVALID_ARG;
  if ((int64_t)max_pages * page > (1LL << 30)) return ADA_ERR_UNSUPPORTED;
  if (misaligned16(q) || misaligned16(out) || ((q_st | q_sh | o_st | o_sh) & 7)) return ADA_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(bt) & 3) return ADA_ERR_ALIGNMENT;
  return ADA_OK;
}

// Prefill of a few new tokens a sequence, in kv4_decode.cu; workspace as sized there.
size_t rows_workspace_size(int32_t batch);
int rows_prefill(const void* q, int q_dtype, int64_t q_st, int64_t q_sh, const uint8_t* kc, const uint8_t* vc,
                 int64_t s_page, int64_t s_head, int64_t num_pages, const int32_t* bt, int64_t bt_stride,
                 int32_t max_pages, const int32_t* cu_q, const int32_t* cu_k, int32_t batch, int64_t rows, int32_t most,
                 int32_t hq, int32_t hkv, int32_t page, float scale_log2, float v_scale, int32_t window, void* out,
                 int out_dtype, int64_t o_st, int64_t o_sh, void* workspace, cudaStream_t st);

}  // namespace kv4
}  // namespace ada
