// Causal prefill attention over the 4-bit paged KV cache (kv4.cuh).
//
// Semantics as the e4m3 form (prefill_attention.cu): sequence b's len_q new rows see keys
// j <= i + len_k - len_q, with a window W > 0 also j >= i + len_k - len_q - W; a row without keys is
// zeros.  Rows are (token, head) pairs of a KV head's group, head fastest, so 256 / group tokens
// share every key block that a CTA widens.
//
// Floor of a block of 64 keys: 256 x 64 exponentials (16 a cycle and SM: 1,024 cycles), 2 x 256 x 64 x 128
// multiply-adds (4,096 a cycle: 1,024) and the operands' shared-memory reads (some 1,400).  It takes about 1,900: the
// softmax of the two tiles' rows on one scheduler runs in step (its exponentials 1,300 cycles side by side, 850 alone) and
// its loads, maxima and waits (600) come in between.  4 x 2,048 tokens behind 2,048, 32/8 heads: 413 us, 0.59 of
// the measured matrix rate (445 call after call, at the power cap).  Tried and left out: two threads a row (524: they have to agree on the reference),
// turns between the tiles (466), part of the exponentials as polynomials on the FMA pipe (426-454), 128 keys a block (564).
//
// One CTA a (256-row query block, KV head, sequence), or several that share its keys where there are few
// (merge_kernel joins them); 14 warps:
//   warp 0        TMEM owner, issues S_t = Q_t K^T for the two 128-row tiles t (M 128, N 64);
//   warp 1        issues O_t += P_t V with P_t as the A operand in TMEM;
//   warps 2-5     converters: a 16-key tile of each block each (in one page): its codes and scales by cp.async
//                 into a ring of the warp's own, codes x scales -> f16 K and V operand tiles (exact);
//   warps 6-9, 10-13   softmax of tile 0 and 1, thread = row: brings its query row into shared memory
//                 as f16 (times a power of two, kv4.cuh), then per block reads 64 scores from TMEM and
//                 writes 64 f16 probabilities there, where P V reads them: no shared memory and no
//                 proxy fence in between.  A row's reference moves when a score passes it by
//                 8 (log2); only then its O row is rescaled.
//
// A NaN scale of a value would reach every row through 0 * NaN, also those that do not see its key:
// the converters widen it as 0 and mark (key, scale block), and rows that see a marked key turn
// their 16 elements to NaN at the end.
//
// Barriers (block j, tile t): kv_empty[j % NKV] (commit after both P V); s_go[t][j % NKV]: S_j may run (4 converters;
// commit after P V of j - 2, whose probabilities lie in the same place); s_full[t][j & 1] (commit after S_j, an
// arrival of its issuer's own); p_full[t][j & 1] (4 warps); o_last[t] (commit after the last P V); q_ready (8
// warps); fin.  Few waits, as each takes 150-300 cycles also where it passes.
// A wait by parity needs the phase before to be known complete and the next one not begun.  Refills wait
// for the release of the use before, in every phase.  An arrival for the next phase of s_go[t][j % NKV] follows kv_empty of
// j or P V of j + 1; S_{j+2} and with it the next phases of s_full and p_full follow P V of j.  A softmax that
// rescales O waits for P V of j - 1 by kv_empty, whose phase before the converters of block j - 1 have seen.
// The end waits for o_last, which has one phase.
#include "kv4.cuh"
#include "tc_attention.cuh"

namespace ada {
namespace kv4 {
namespace pf4 {
using namespace tca;
using namespace sm100;

constexpr int NT = 2, BM = 128, BN = 64, TILE = 16;
constexpr int NSTG = 4, NKV = 3, NCONV = 4, NSOFT = 4;
constexpr int THREADS = (2 + NCONV + NT * NSOFT) * 32;
constexpr int Q_OFF = 0;                     // f16 Q, NT x [2 halves][128 rows][128 B]
constexpr int K_OFF = Q_OFF + NT * 32768;    // f16 K, NKV x [2 halves][64 keys][128 B]
constexpr int V_OFF = K_OFF + NKV * 16384;
constexpr int E_OFF = V_OFF + NKV * 16384;   // converter warps' rings: K codes, V codes, K scales, V scales of a tile
constexpr int E_BYTES = 2 * TILE * ROW_BYTES;
constexpr int EV = TILE * ROW, EKS = 2 * TILE * ROW, EVS = EKS + TILE * SROW;
constexpr int BAR_OFF = E_OFF + NCONV * NSTG * E_BYTES;
constexpr int NBAR = NKV + NT * (NKV + 5) + 2;
constexpr int FLAG_OFF = (BAR_OFF + NBAR * 8 + 15) & ~15;  // words a K/V slot: [4 tiles there][4 tiles' NaN flags][16 NaN masks]
constexpr int SLOT_WORDS = 24;
constexpr int SMEM = 1024 + FLAG_OFF + (NKV * SLOT_WORDS + 4) * 4;
static_assert(NCONV * TILE == BN, "a converter warp a tile");
constexpr uint32_t TMEM_COLS = 512, S_COL = 256;  // O of tile t at 128 t; S buffer b of tile t at 256 + 128 t + 64 b
constexpr float MOVE_LOG2 = 8.f;
// A partial (floats): O as [32 groups of 4 elements][256 rows][4], then (largest score, sum, factor, -) a row.
constexpr int ROWS = NT * BM, STATS = ROWS * D, PART = STATS + 4 * ROWS;
static_assert(SMEM <= 232448, "shared memory per CTA");
static_assert(E_BYTES % 16 == 0 && BAR_OFF % 16 == 0 && FLAG_OFF % 16 == 0 && SLOT_WORDS % 4 == 0, "alignment");
constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
// Up to this factor |score * factor| < 2^24, where the rounding of a row's reference is below 1 (log2).
constexpr float SAFE_FACTOR = 9.765625e-4f;  // 2^-10

struct Params {
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  const uint8_t *kc, *vc;
  int64_t s_page, s_head, num_pages;
  const int32_t* bt;
  int64_t bt_stride;
  int max_pages, page, window, group, qt, q_bf16, o_bf16;
  const int32_t *cu_q, *cu_k;
  int64_t rows;
  float scale_log2, v_scale;
  unsigned* err;
  int qblocks, splits;  // CTAs that share a query block's keys
  float* parts;         // workspace (splits > 1): a partial a CTA
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// High word of every shared-memory descriptor here: 1,024 bytes between 8-row groups, 128-byte swizzle.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | ((uint32_t)SWZ_128B << 29);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(DESC_HI), "r"(IDESC_S), "r"((int)accumulate)
      : "memory");
}
// A (f16, two a column) in TMEM.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(DESC_HI), "r"(IDESC_PV), "r"((int)accumulate)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// 64 columns of this thread's TMEM lane; load and wait are one statement, so no register of the load
// can be touched before the wait.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
}
// 16 codes times their scale as 16 f16 (two chunks).
__device__ __forceinline__ void widen16(uint2 codes, uint32_t scale2, uint4& lo, uint4& hi) {
  uint32_t h[8];
  widen8(codes.x, h);
  widen8(codes.y, h + 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = mul_f16x2(h[i], scale2);
  lo = make_uint4(h[0], h[1], h[2], h[3]);
  hi = make_uint4(h[4], h[5], h[6], h[7]);
}
// Keys [lo, hi) that new token t of a sequence sees.
__device__ __forceinline__ void key_range(const Params& P, int t, int off, int len_k, int& lo, int& hi) {
  hi = min(len_k, t + off + 1);
  lo = P.window > 0 ? max(0, t + off - P.window) : 0;
}

__global__ void __launch_bounds__(THREADS, 1) prefill_kernel(const __grid_constant__ Params P) {
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int kvh = blockIdx.x, b = blockIdx.y;
  int qblk = P.qblocks - 1 - blockIdx.z, split = 0;  // the longest causal rows of all heads and sequences first
  if (P.splits > 1) {
    qblk = P.qblocks - 1 - blockIdx.z / P.splits;
    split = blockIdx.z % P.splits;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *qs = base + Q_OFF, *kf = base + K_OFF, *vf = base + V_OFF, *es = base + E_OFF;
  uint64_t* kv_empty = reinterpret_cast<uint64_t*>(base + BAR_OFF);
  uint64_t* s_go = kv_empty + NKV;      // [NT][NKV]
  uint64_t* s_full = s_go + NT * NKV;   // [NT][2]
  uint64_t* p_full = s_full + 2 * NT;   // [NT][2]
  uint64_t* o_last = p_full + 2 * NT;   // [NT]
  uint64_t* q_ready = o_last + NT;
  uint64_t* fin = q_ready + 1;
  uint32_t* slots = reinterpret_cast<uint32_t*>(base + FLAG_OFF);
  uint32_t* tmem_slot = slots + NKV * SLOT_WORDS;
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NKV; ++i) mbar_init(&kv_empty[i], 1);
    for (int i = 0; i < NT * NKV; ++i) mbar_init(&s_go[i], NCONV + 1);
    for (int i = 0; i < 2 * NT; ++i) {
      mbar_init(&s_full[i], 2);
      mbar_init(&p_full[i], NSOFT);
    }
    for (int t = 0; t < NT; ++t) mbar_init(&o_last[t], 1);
    mbar_init(q_ready, NT * NSOFT);
    mbar_init(fin, 2);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  const int64_t q_begin = P.cu_q[b];
  const int len_q = (int)min(max((int64_t)P.cu_q[b + 1] - q_begin, (int64_t)0), (int64_t)1 << 30);
  const int len_k = (int)min(max((int64_t)P.cu_k[b + 1] - P.cu_k[b], (int64_t)0), (int64_t)1 << 30);
  const int t0 = qblk * P.qt;
  const bool active = t0 < len_q;
  const int off = len_k - len_q;
  int nblk = 0, kb0 = 0, k_end = 0;
  if (active) {
    const int t_last = min(t0 + P.qt, len_q) - 1;
    int k_lo, k_hi, dlo, dhi;
    key_range(P, t0, off, len_k, k_lo, dhi);
    key_range(P, t_last, off, len_k, dlo, k_hi);
    k_end = min(k_hi, P.max_pages * P.page);
    kb0 = (k_lo / BN) * BN;
    nblk = k_end > k_lo ? (k_end - kb0 + BN - 1) / BN : 0;
    if (P.splits > 1) {  // (2^24 blocks x 148: below 2^32)
      const unsigned n = nblk, first = n * split / P.splits;
      nblk = (int)(n * (split + 1) / P.splits - first);
      kb0 += (int)first * BN;
    }
  }

  if (warp < 2) {  // ---------------- MMA issuers: S, P V ----------------
    // The whole warp runs its loop, the values uniform, and one elected lane issues: the operands of the
    // tcgen05 instructions then stay in uniform registers (from a divergent lane an MMA takes about 100
    // cycles to issue, 24 of them a block: 629 us instead of 518 for 4 x 2,048 tokens behind 2,048, 32/8 heads).
    // S and P V have a warp each: a wait that passes takes 150-200 cycles, and five of them in turn left the
    // tensor pipe idle for half of a block.
    if (nblk > 0) {
      const bool leader = elect_one();
      const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
      // low words of the descriptors: address / 16, leading offset / 16 (V: 8 KB between the halves of d)
      const uint32_t q_lo = (smem_u32(qs) >> 4) | (1u << 16), k_lo = (smem_u32(kf) >> 4) | (1u << 16);
      const uint32_t v_lo = (smem_u32(vf) >> 4) | ((8192u >> 4) << 16);
      uint32_t slot = 0;
      bool ok = true;
      if (warp == 0) {
        ok = wait_b(q_ready, 0, abort_v, P.err);
        if (leader) {  // the first two places of each tile's scores are free
          for (int t = 0; t < NT; ++t) {
            mbar_arrive_plain(&s_go[NKV * t]);
            mbar_arrive_plain(&s_go[NKV * t + 1]);
          }
        }
        __syncwarp();
        for (int j = 0; j < nblk; ++j) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            ok = __all_sync(0xffffffffu, ok && wait_b(&s_go[NKV * t + slot], (j / NKV) & 1, abort_v, P.err));
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              const uint32_t d = tm + S_COL + 128u * (uint32_t)t + BN * (uint32_t)(j & 1);
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                mma_ss(d, q_lo + (uint32_t)t * 2048u + (uint32_t)(kk / 4) * 1024u + (uint32_t)(kk % 4) * 2u,
                       k_lo + slot * 1024u + (uint32_t)(kk / 4) * 512u + (uint32_t)(kk % 4) * 2u, kk > 0);
              tc_commit(&s_full[2 * t + (j & 1)]);
              mbar_arrive_plain(&s_full[2 * t + (j & 1)]);  // passes on what s_go ordered: flags, and V for P V
            }
            __syncwarp();
          }
          if (!ok) break;
          slot = slot + 1 == NKV ? 0 : slot + 1;
        }
      } else {
        for (int j = 0; ok && j < nblk; ++j) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            ok = __all_sync(0xffffffffu, ok && wait_b(&p_full[2 * t + (j & 1)], (j >> 1) & 1, abort_v, P.err));
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              const uint32_t p = tm + S_COL + 128u * (uint32_t)t + BN * (uint32_t)(j & 1);
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)
                mma_ts(tm + 128u * (uint32_t)t, p + 8u * (uint32_t)kk, v_lo + slot * 1024u + (uint32_t)kk * 128u,
                       j > 0 || kk > 0);
              tc_commit(j + 1 == nblk ? &o_last[t] : &s_go[NKV * t + (slot + 2) % NKV]);  // (S_{j+2} may come)
              if (t == NT - 1) tc_commit(&kv_empty[slot]);
            }
            __syncwarp();
          }
          slot = slot + 1 == NKV ? 0 : slot + 1;
        }
      }
      // every MMA issued above has completed before the teardown
      if (leader) tc_commit(fin);
      __syncwarp();
      uint32_t spins = 0;
      const uint64_t t_start = globaltimer();
      while (!mbar_try_wait(fin, 0)) {
        if ((++spins & 63u) == 0 && globaltimer() - t_start > 2000000000ull) {
          if (leader && P.err) atomicOr(P.err, ERR_TILE_WAIT);
          break;
        }
      }
    }
  } else if (warp < 2 + NCONV) {  // ---------------- converters ----------------
    // Warp w brings and converts tile w of every block.  Its ring holds the codes and scales of NSTG blocks, by
    // cp.async: a bulk copy takes a warp 60-100 cycles to issue, and a block has 16 contiguous pieces, so a warp that
    // did nothing else needed 1,400-1,700 cycles a block and was the bound.
    const int w = warp - 2, page_tiles = P.page / TILE;
    uint8_t* ring = es + w * (NSTG * E_BYTES);
    const uint8_t *kc = P.kc + (int64_t)kvh * P.s_head, *vc = P.vc + (int64_t)kvh * P.s_head;
    int64_t codes = -1;  // of the lane's block (32 of them from a multiple on): its tile's codes in the cache, -1: a hole
    int scales = 0;      // from there to its scales
    uint32_t there = 0;  // bit s: the tile in ring slot s
    int slot = 0;        // that the next block goes to
    auto fetch = [&](int j) {
      if (j < nblk) {
        if ((j & 31) == 0) {
          const int key0 = kb0 + BN * (j + lane) + TILE * w;
          codes = -1;
          if (j + lane < nblk && key0 < k_end) {
            const int tile = key0 / TILE, col = tile / page_tiles, at = tile - col * page_tiles;
            const int64_t id = P.bt[(int64_t)b * P.bt_stride + col];
            if (id >= 0 && id < P.num_pages) {
              codes = id * P.s_page + at * (TILE * ROW);
              scales = P.page * ROW - at * (TILE * (ROW - SROW));
            }
          }
        }
        const int64_t at = __shfl_sync(0xffffffffu, codes, j & 31);
        const int to = __shfl_sync(0xffffffffu, scales, j & 31);
        there = (there & ~(1u << slot)) | ((uint32_t)(at >= 0) << slot);
        if (at >= 0) {
          const uint32_t dst = smem_u32(ring + slot * E_BYTES) + 16 * lane;
          cp16(dst, kc + at + 16 * lane);
          cp16(dst + 512, kc + at + 512 + 16 * lane);
          cp16(dst + EV, vc + at + 16 * lane);
          cp16(dst + EV + 512, vc + at + 512 + 16 * lane);
          if (lane < 16) cp16(dst + EKS, (lane < 8 ? kc : vc - TILE * SROW) + at + to + 16 * lane);
        }
      }
      cp_commit();
      slot = slot + 1 == NSTG ? 0 : slot + 1;
    };
#pragma unroll
    for (int j = 0; j < NSTG - 1; ++j) fetch(j);
    int from = 0, kb = 0;
    for (int j = 0; j < nblk; ++j) {
      cp_wait<NSTG - 2>();
      __syncwarp();  // every lane's part has arrived, and the slot before has been read
      fetch(j + NSTG - 1);
      if (j >= NKV && !wait_w(&kv_empty[kb], ((j / NKV) - 1) & 1, abort_v, P.err)) break;
      const uint8_t* st = ring + from * E_BYTES;
      const bool ok = (there >> from) & 1u;
      uint32_t* flags = slots + kb * SLOT_WORDS;
      uint32_t nan_any = 0;
      // 16 keys x 8 blocks of 16 elements an operand: 4 units a lane, two read before the first is written (the compiler
      // cannot move a read over a write that may be to the same place; 1, 2, 4 at a time: 433, 423, 436 us)
#pragma unroll
      for (int u0 = 0; u0 < 4; u0 += 2) {
        uint2 k8[2], v8[2];
        uint32_t ks[2], vs[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int unit = lane + 32 * (u0 + i);
          k8[i] = *reinterpret_cast<const uint2*>(st + 8 * unit);
          v8[i] = *reinterpret_cast<const uint2*>(st + EV + 8 * unit);
          ks[i] = st[EKS + unit];
          vs[i] = st[EVS + unit];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int u = u0 + i, unit = lane + 32 * u, key = TILE * w + (unit >> 3), blk = unit & 7;
          if (!ok) ks[i] = 0;
          if (!ok || kb0 + j * BN + key >= len_k) vs[i] = 0;
          const bool nan = (vs[i] & 0x7Fu) == 0x7Fu;
          const uint32_t marked = __ballot_sync(0xffffffffu, nan);  // 4 keys x 8 blocks
          if (nan) vs[i] = 0;
          nan_any |= marked;
          if (lane == 0) flags[8 + 4 * w + u] = marked;
          uint4 lo, hi;
          // (blocks 4-7 lie 8 KB behind 0-3, in the same banks: they write their halves in the other order)
          const int c0 = ((blk & 3) * 2 + (blk >> 2)) ^ (key & 7), c1 = c0 ^ 1;
          if (blk & 4) k8[i] = make_uint2(k8[i].y, k8[i].x), v8[i] = make_uint2(v8[i].y, v8[i].x);
          const int at = kb * 16384 + (blk >> 2) * 8192 + key * 128;
          widen16(k8[i], scale_f16x2(ks[i]), lo, hi);
          *reinterpret_cast<uint4*>(kf + at + (c0 << 4)) = lo;
          *reinterpret_cast<uint4*>(kf + at + (c1 << 4)) = hi;
          widen16(v8[i], scale_f16x2(vs[i]), lo, hi);
          *reinterpret_cast<uint4*>(vf + at + (c0 << 4)) = lo;
          *reinterpret_cast<uint4*>(vf + at + (c1 << 4)) = hi;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        flags[w] = ok;
        flags[4 + w] = nan_any;
        mbar_arrive_plain(&s_go[kb]);
        mbar_arrive_plain(&s_go[NKV + kb]);
      }
      kb = kb + 1 == NKV ? 0 : kb + 1;
      from = from + 1 == NSTG ? 0 : from + 1;
    }
    cp_wait<0>();
  } else {  // ---------------- softmax: warpgroup t, thread = row r of tile t ----------------
    const int t = (warp - 2 - NCONV) / NSOFT;
    const int q4 = warp & 3;  // the TMEM lane quarter that this warp may access
    const int r = 32 * q4 + lane, R = t * BM + r;
    const uint32_t trow = tmem + ((uint32_t)(32 * q4) << 16);
    const uint32_t o_col = 128u * (uint32_t)t, s_col = S_COL + 128u * (uint32_t)t;
    const int tok = t0 + R / P.group;
    const int64_t row = q_begin + tok;
    const bool valid = active && R < P.qt * P.group && tok < len_q && row >= 0 && row < P.rows;
    const uint32_t there = __ballot_sync(0xffffffffu, valid);
    const int head = kvh * P.group + R % P.group;
    int lo = 0, hi = 0;
    if (valid) key_range(P, tok, off, len_k, lo, hi);
    float factor = 0.f;
    uint8_t* rows = qs + t * 32768 + 4096 * q4;  // the warp's 32 rows of the Q tile, [2 halves at 16 KB]
    const int c16 = lane & 15, r2 = lane >> 4;   // a half-warp a row
    auto chunk = [&](int rr, int c) {
      return reinterpret_cast<uint4*>(rows + rr * 128 + (c >> 3) * 16384 + (((c & 7) ^ (rr & 7)) << 4));
    };
    if (nblk > 0) {
      // The query rows -> f16, times a power of two, in place: elements come by cp.async to where their f16 form
      // will lie, so that a thread reads and writes its row without bank conflicts.  (By loads into registers the L1
      // beside this much shared memory, some 16 KB, holds a quarter of them at a time: 16,000 cycles a CTA, here 7,500.)
      const int64_t mine = row * P.q_st + head * P.q_sh;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int rr = 2 * i + r2;
        const int64_t at = __shfl_sync(0xffffffffu, mine, rr);
        if ((there >> rr) & 1u) cp16(smem_u32(chunk(rr, c16)), reinterpret_cast<const uint16_t*>(P.q) + at + 8 * c16);
      }
      cp_commit();
      cp_wait<0>();
      __syncwarp();
      int ex = 0;
      auto convert = [&](auto type) {
        using T = decltype(type);
        uint32_t top2 = 0;  // of pairs of magnitudes
#pragma unroll 4
        for (int c = 0; c < 16; ++c) top2 = max_pairs<T>(top2, *chunk(lane, c));
        ex = query_exponent(valid ? larger<T>(top2) : 0.f);
        const float mul = pow2(ex);
#pragma unroll 1
        for (int c = 0; c < 16; c += 4) {
          uint4 x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = valid ? *chunk(lane, c + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f[8];
            unpack8<T>(x[i], f);
            *chunk(lane, c + i) = make_uint4(pack_half2(f[0] * mul, f[1] * mul), pack_half2(f[2] * mul, f[3] * mul),
                                             pack_half2(f[4] * mul, f[5] * mul), pack_half2(f[6] * mul, f[7] * mul));
          }
        }
      };
      if (P.q_bf16) convert(__nv_bfloat16()); else convert(__half());
      factor = score_factor(P.scale_log2, ex);
      if (!valid) factor = fminf(factor, SAFE_FACTOR);  // (all its keys are masked)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_plain(q_ready);
    }
    const bool safe = __all_sync(0xffffffffu, factor <= SAFE_FACTOR);
    float m = -INFINITY;  // largest score that set the reference
    float shift = P_LOG2; // what the exponents get: P_LOG2, less the reference (log2) in safe rows
    uint64_t l2[2] = {0ull, 0ull};
    uint32_t nan_blocks = 0;
    bool failed = false;
    for (int j = 0; j < nblk; ++j) {
      // warp-uniform outcome: the TMEM accesses below are warp-collective
      if (!__all_sync(0xffffffffu, wait_b(&s_full[2 * t + (j & 1)], (j >> 1) & 1, abort_v, P.err))) {
        failed = true;
        break;
      }
      tc_fence_after();
      float x[64];
      uint32_t* sr = reinterpret_cast<uint32_t*>(x);
      tmem_ld64(trow + s_col + BN * (j & 1), sr);
      const uint32_t* flags = slots + (j % NKV) * SLOT_WORDS;
      const uint4 loaded = *reinterpret_cast<const uint4*>(flags);
      const uint32_t blk_ok = loaded.x | (loaded.y << 1) | (loaded.z << 2) | (loaded.w << 3);
      const uint4 marked = *reinterpret_cast<const uint4*>(flags + 4);
      const int key0 = kb0 + j * BN, a = lo - key0, e = hi - key0;  // visible columns [a, e) of loaded tiles
      if (!__all_sync(0xffffffffu, blk_ok == 15u && a <= 0 && e >= BN)) {
        if (__all_sync(0xffffffffu, a >= BN || e <= 0)) {  // none of the warp's rows sees the block
          uint32_t zero[16] = {};
          tmem_st16(trow + s_col + BN * (j & 1), zero);
          tmem_st16(trow + s_col + BN * (j & 1) + 16, zero);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_plain(&p_full[2 * t + (j & 1)]);
          continue;
        }
        const int a1 = max(a, 0);
        const unsigned n = (unsigned)max(min(e, BN) - a1, 0);
#pragma unroll
        for (int i = 0; i < 64; ++i) x[i] = (unsigned)(i - a1) < n ? x[i] : -INFINITY;
        if (blk_ok != 15u) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (!((blk_ok >> (i >> 4)) & 1u)) x[i] = -INFINITY;
        }
      }
      if (marked.x | marked.y | marked.z | marked.w) {
        for (int i = max(a, 0); i < min(e, BN); ++i) nan_blocks |= (flags[8 + (i >> 2)] >> (8 * (i & 3))) & 0xFFu;
      }
      float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < 60; i += 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], x[i + 2 * k], x[i + 2 * k + 1]);
      }
      const float top = max3(max3(mx[0], x[60], x[61]), max3(mx[1], x[62], x[63]), fmaxf(mx[2], mx[3]));
      float alpha = 1.f;
      if ((top - m) * factor > MOVE_LOG2) {
        const float to = safe ? fmaf(-top, factor, P_LOG2) : P_LOG2;
        alpha = m == -INFINITY ? 0.f : fast_exp2(safe ? to - shift : (m - top) * factor);
        m = top;
        shift = to;
      }
      if (!safe) {  // (warp-uniform) the difference first; the loop below then only takes the exponential
        const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < 64; ++i) x[i] = (x[i] - mm) * factor;
      }
      if (alpha != 1.f) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float s0, s1;
          unpair(l2[i], s0, s1);
          l2[i] = pair(s0 * alpha, s1 * alpha);
        }
      }
      const float c1 = safe ? factor : 1.f, r1 = shift;
      const uint64_t c2 = pair(c1, c1), r2 = pair(r1, r1);
      uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float p0, p1;
        unpair(fma2(pair(x[2 * i], x[2 * i + 1]), c2, r2), p0, p1);
        p0 = fast_exp2(p0);
        p1 = fast_exp2(p1);
        l2[i & 1] = add2(l2[i & 1], pair(p0, p1));  // fp32 probabilities feed the row's sum, fp16 ones P V
        pk[i] = pack_half2(p0, p1);
      }
      // the probabilities over the scores
#pragma unroll
      for (int i = 0; i < 2; ++i) tmem_st16(trow + s_col + BN * (j & 1) + 16 * i, pk + 16 * i);
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        // O is stable once P V of the block before has completed
        if (!__all_sync(0xffffffffu, wait_b(&kv_empty[(j - 1) % NKV], ((j - 1) / NKV) & 1, abort_v, P.err))) {
          failed = true;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16_async(trow + o_col + 16 * c, o);
          tmem_wait_ld16(o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st16(trow + o_col + 16 * c, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_plain(&p_full[2 * t + (j & 1)]);
    }
    // ---- epilogue: O row / l
    if (!failed && nblk > 0) {
      failed = !__all_sync(0xffffffffu, wait_b(&o_last[t], 0, abort_v, P.err));
      tc_fence_after();
    }
    failed = __any_sync(0xffffffffu, failed || *abort_v != 0);
    float s0, s1, s2, s3;
    unpair(l2[0], s0, s1);
    unpair(l2[1], s2, s3);
    float l = (s0 + s1) + (s2 + s3);
    const float nan = __uint_as_float(0x7FC00000u);
    const float inv = failed ? nan : l == 0.f ? 0.f : P.v_scale / l;
    if (P.splits > 1) {  // to the workspace, unnormalised: lanes' 16 bytes side by side
      if (failed) l = nan;
      float* part = P.parts + ((((int64_t)b * gridDim.x + kvh) * P.qblocks + qblk) * P.splits + split) * PART;
      reinterpret_cast<float4*>(part + STATS)[R] = make_float4(m, l, factor, 0.f);
      if (nblk > 0 && !failed) {
#pragma unroll 1
        for (int d0 = 0; d0 < D; d0 += 64) {
          float o[64];
          tmem_ld64(trow + o_col + d0, reinterpret_cast<uint32_t*>(o));
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float4 v = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
            if ((nan_blocks >> (d0 / 16 + c / 4)) & 1) v = make_float4(nan, nan, nan, nan);
            reinterpret_cast<float4*>(part)[(d0 / 4 + c) * ROWS + R] = v;
          }
        }
      }
    } else {
      // by way of the Q tile, which no MMA reads any more, so that a half-warp writes a row's 256 bytes at once
      __syncwarp();
#pragma unroll 1
      for (int d0 = 0; d0 < D; d0 += 64) {
        float o[64];
        if (nblk > 0 && !failed) {
          tmem_ld64(trow + o_col + d0, reinterpret_cast<uint32_t*>(o));
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float by = (nan_blocks >> (d0 / 16 + c)) & 1 ? nan : inv;
          float* f = o + 16 * c;
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] *= by;  // (without a key O is 0)
          *chunk(lane, d0 / 8 + 2 * c) = P.o_bf16 ? pack8<__nv_bfloat16>(f) : pack8<__half>(f);
          *chunk(lane, d0 / 8 + 2 * c + 1) = P.o_bf16 ? pack8<__nv_bfloat16>(f + 8) : pack8<__half>(f + 8);
        }
      }
      __syncwarp();
      const int64_t mine = row * P.o_st + head * P.o_sh;
#pragma unroll 8
      for (int i = 0; i < 16; ++i) {
        const int rr = 2 * i + r2;
        const int64_t at = __shfl_sync(0xffffffffu, mine, rr);
        const uint4 v = *chunk(rr, c16);
        if ((there >> rr) & 1u) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(P.out) + at + 8 * c16) = v;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, TMEM_COLS);
}

// Partials of the CTAs that share a query block: a CTA 32 rows (lane: row), a warp 16 elements of them.
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ Params P) {
  pdl_wait();
  pdl_trigger();
  const int kvh = blockIdx.x, b = blockIdx.y, qblk = blockIdx.z / (ROWS / 32);
  const int R = 32 * (blockIdx.z % (ROWS / 32)) + (threadIdx.x & 31), w = threadIdx.x >> 5;
  const int64_t q_begin = P.cu_q[b];
  const int len_q = (int)min(max((int64_t)P.cu_q[b + 1] - q_begin, (int64_t)0), (int64_t)1 << 30);
  const int tok = qblk * P.qt + R / P.group, head = kvh * P.group + R % P.group;
  const int64_t row = q_begin + tok;
  if (R >= P.qt * P.group || tok >= len_q || row < 0 || row >= P.rows) return;
  const float* part = P.parts + (((int64_t)b * gridDim.x + kvh) * P.qblocks + qblk) * P.splits * PART;
  float top = -INFINITY;
  for (int i = 0; i < P.splits; ++i) top = fmaxf(top, reinterpret_cast<const float4*>(part + i * PART + STATS)[R].x);
  float l = 0.f, o[16];
#pragma unroll
  for (int c = 0; c < 16; ++c) o[c] = 0.f;
  for (int i = 0; i < P.splits; ++i) {
    const float* p = part + i * PART;
    const float4 st = reinterpret_cast<const float4*>(p + STATS)[R];
    if (st.y == 0.f) continue;  // saw no key (a NaN sum stays)
    const float f = st.x == top ? 1.f : fast_exp2((st.x - top) * st.z);
    l = fmaf(f, st.y, l);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 v = reinterpret_cast<const float4*>(p)[(4 * w + c) * ROWS + R];
      o[4 * c] = fmaf(f, v.x, o[4 * c]);
      o[4 * c + 1] = fmaf(f, v.y, o[4 * c + 1]);
      o[4 * c + 2] = fmaf(f, v.z, o[4 * c + 2]);
      o[4 * c + 3] = fmaf(f, v.w, o[4 * c + 3]);
    }
  }
  const float inv = l == 0.f ? 0.f : P.v_scale / l;
#pragma unroll
  for (int c = 0; c < 16; ++c) o[c] = inv == 0.f ? 0.f : o[c] * inv;
  uint16_t* out = reinterpret_cast<uint16_t*>(P.out) + row * P.o_st + head * P.o_sh + 16 * w;
  reinterpret_cast<uint4*>(out)[0] = P.o_bf16 ? pack8<__nv_bfloat16>(o) : pack8<__half>(o);
  reinterpret_cast<uint4*>(out)[1] = P.o_bf16 ? pack8<__nv_bfloat16>(o + 8) : pack8<__half>(o + 8);
}

}  // namespace pf4
}  // namespace kv4
}  // namespace ada

using namespace ada;
namespace pf4 = ada::kv4::pf4;

constexpr int64_t FEW_ROWS = 32, FEW_KEYS = 256;

// A few rows a KV head behind tables of more than 256 keys go to the decode kernel's form, which shares the
// keys out over all SMs; this one has a CTA for 256 rows, which walks its keys alone.  Measured, 32/8 heads, 8
// sequences of 2 new tokens: 60 cached keys 12.9 us shared out and 8.6 here, 500: 16.7 and 17.0, 8,000: 32.6 and 149; 32
// sequences of 8: 60: 26 and 19.5, 500: 35.5 and 32, 8,000: 235 and 251; 16 tokens, 64 rows, behind 8,000: 455-470 and 258.
static bool prefill_few(int64_t batch, int64_t most, int32_t num_heads, int32_t num_kv_heads, int32_t max_pages,
                        int32_t page_size) {
  constexpr int64_t MOST = 1 << 30;  // steps of 32 keys, which that kernel counts in 32 bits
  const int64_t rows = most * (num_heads / num_kv_heads), items = batch * num_kv_heads * cdiv(rows, (int64_t)8);
  const int64_t keys = (int64_t)max_pages * page_size;
  return rows <= FEW_ROWS && keys > FEW_KEYS && keys <= MOST && batch <= 8192 && items <= MOST &&
         items * (cdiv(keys, (int64_t)32) + 1) <= MOST;
}

// CTAs that a query block's keys are shared by: as many as are resident at once, each with four blocks of 64 keys or more
// (a CTA costs 9 us around its blocks and the join 4-5; a row of new tokens sees half of them on average).  One
// sequence, 32/8 heads, alone and shared: 60 tokens behind 700 keys 23 and 19 us, 100 behind 1,500: 43 and 20, 128
// behind 8,000: 155 and 41, 512 behind 8,000: 161 and 95; 512 alone would take 20.3 instead of 18.0.  (Eight
// blocks at least: 25.0 for the first, 25.6 for the second.)
static int prefill_splits(int64_t batch, int64_t most, int32_t num_heads, int32_t num_kv_heads, int64_t reach,
                          int32_t window) {
  const int64_t group = num_heads / num_kv_heads, qt = group > 0 ? pf4::ROWS / group : 0;
  if (qt == 0 || reach > (1 << 30)) return 1;
  const int64_t ctas = batch * num_kv_heads * cdiv(most, qt);
  const int64_t seen = window > 0 && window + qt < reach ? window + qt : reach;
  const int64_t s = ctas > 0 && ctas <= 148 ? 148 / ctas : 1;
  const int64_t by_keys = (seen - (most < seen ? most : seen) / 2) / (4 * pf4::BN);
  return (int)(s < by_keys ? s : by_keys < 1 ? 1 : by_keys);
}

extern "C" size_t ada_kv4_paged_prefill_workspace_size(int32_t batch, int64_t total_q, int32_t max_seqlen_q,
                                                       int32_t num_heads, int32_t num_kv_heads, int32_t max_pages,
                                                       int32_t page_size) {
  if (batch <= 0 || total_q <= 0 || max_seqlen_q <= 0 || num_heads <= 0 || num_kv_heads <= 0 || max_pages <= 0 ||
      page_size <= 0)
    return 0;
  const int64_t most = max_seqlen_q < total_q ? max_seqlen_q : total_q;
  if (prefill_few(batch, most, num_heads, num_kv_heads, max_pages, page_size)) return kv4::rows_workspace_size(batch);
  const int splits = prefill_splits(batch, most, num_heads, num_kv_heads, (int64_t)max_pages * page_size, 0);
  if (splits == 1) return 0;
  return (size_t)(batch * num_kv_heads * cdiv(most, (int64_t)(pf4::ROWS / (num_heads / num_kv_heads))) * splits) * pf4::PART * 4;
}

extern "C" int ada_kv4_paged_prefill(const void* q, int q_dtype, int64_t q_stride_t, int64_t q_stride_h,
                                     const uint8_t* k_cache, const uint8_t* v_cache, int64_t kv_stride_page,
                                     int64_t kv_stride_head, int64_t num_pages, const int32_t* block_tables,
                                     int64_t bt_stride, int32_t max_pages, const int32_t* cu_seqlens_q,
                                     const int32_t* cu_seqlens_k, int32_t batch, int64_t total_q, int32_t max_seqlen_q,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                     float scale, float k_scale, float v_scale, int32_t window, void* out,
                                     int out_dtype, int64_t out_stride_t, int64_t out_stride_h, void* workspace,
                                     size_t workspace_bytes, unsigned int* err, void* stream) {
  if (batch < 0 || max_seqlen_q < 0 || total_q < 0) return ADA_ERR_INVALID_ARG;
  if (batch == 0 || max_seqlen_q == 0 || total_q == 0) return ADA_OK;
  if (!cu_seqlens_q || !cu_seqlens_k) return ADA_ERR_INVALID_ARG;
  if (const int e = kv4::attn_ok(q, q_dtype, q_stride_t, q_stride_h, out, out_dtype, out_stride_t, out_stride_h, k_cache,
                                 v_cache, kv_stride_page, kv_stride_head, num_pages, block_tables, bt_stride, max_pages,
                                 num_heads, num_kv_heads, head_dim, page_size, scale, k_scale, v_scale, window))
    return e;
  if ((reinterpret_cast<uintptr_t>(cu_seqlens_q) | reinterpret_cast<uintptr_t>(cu_seqlens_k) |
       reinterpret_cast<uintptr_t>(err)) & 3)
    return ADA_ERR_ALIGNMENT;
  const int group = num_heads / num_kv_heads;
  if (group > pf4::NT * pf4::BM || batch > 65535 || max_seqlen_q > (1 << 30)) return ADA_ERR_UNSUPPORTED;
  const int64_t most = max_seqlen_q < total_q ? (int64_t)max_seqlen_q : total_q;
  if (prefill_few(batch, most, num_heads, num_kv_heads, max_pages, page_size)) {
    if (!workspace || workspace_bytes < kv4::rows_workspace_size(batch)) return ADA_ERR_WORKSPACE;
    if (kv4::misaligned16(workspace)) return ADA_ERR_ALIGNMENT;
    return kv4::rows_prefill(q, q_dtype, q_stride_t, q_stride_h, k_cache, v_cache, kv_stride_page, kv_stride_head,
                             num_pages, block_tables, bt_stride, max_pages, cu_seqlens_q, cu_seqlens_k, batch, total_q,
                             (int32_t)most, num_heads, num_kv_heads, page_size, scale * k_scale * kv4::LOG2E, v_scale,
                             window, out, out_dtype, out_stride_t, out_stride_h, workspace,
                             reinterpret_cast<cudaStream_t>(stream));
  }
  pf4::Params P;
  P.q = q;
  P.q_st = q_stride_t;
  P.q_sh = q_stride_h;
  P.out = out;
  P.o_st = out_stride_t;
  P.o_sh = out_stride_h;
  P.kc = k_cache;
  P.vc = v_cache;
  P.s_page = kv_stride_page;
  P.s_head = kv_stride_head;
  P.num_pages = num_pages;
  P.bt = block_tables;
  P.bt_stride = bt_stride;
  P.max_pages = max_pages;
  P.page = page_size;
  P.window = window < (1 << 30) ? window : 1 << 30;  // (past every position: sums stay in 32 bits)
  P.group = group;
  P.qt = pf4::NT * pf4::BM / group;
  P.q_bf16 = q_dtype == ADA_DT_BF16;
  P.o_bf16 = out_dtype == ADA_DT_BF16;
  P.cu_q = cu_seqlens_q;
  P.cu_k = cu_seqlens_k;
  P.rows = total_q;
  P.scale_log2 = scale * k_scale * kv4::LOG2E;
  P.v_scale = v_scale;
  P.err = err;
  const int64_t qblocks = cdiv(most, P.qt);
  if (qblocks > 65535) return ADA_ERR_UNSUPPORTED;
  P.splits = prefill_splits(batch, most, num_heads, num_kv_heads, (int64_t)max_pages * page_size, window);
  P.qblocks = (int)qblocks;
  P.parts = static_cast<float*>(workspace);
  if (P.splits > 1) {
    if (!workspace || workspace_bytes < (size_t)(batch * num_kv_heads * qblocks * P.splits) * pf4::PART * 4)
      return ADA_ERR_WORKSPACE;
    if (kv4::misaligned16(workspace)) return ADA_ERR_ALIGNMENT;
  }
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ADA_ERR_CUDA;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(pf4::prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pf4::SMEM) != cudaSuccess)
      return ADA_ERR_CUDA;
    ready[dev] = true;
  }
  (void)launch_k(pf4::prefill_kernel, dim3((unsigned)num_kv_heads, (unsigned)batch, (unsigned)(qblocks * P.splits)),
                 dim3(pf4::THREADS), pf4::SMEM, reinterpret_cast<cudaStream_t>(stream), P);
  ADA_CHECK_LAUNCH();
  if (P.splits > 1) {
    (void)launch_k(pf4::merge_kernel, dim3((unsigned)num_kv_heads, (unsigned)batch, (unsigned)(qblocks * (pf4::ROWS / 32))),
                   dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), P);
    ADA_CHECK_LAUNCH();
  }
  return ADA_OK;
}
