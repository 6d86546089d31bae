// Decode attention over the 4-bit paged KV cache (kv4.cuh), one query token a sequence.
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q . k_t),   t over the visible keys.
//
// Bound by HBM: 144 bytes a key and KV head against 4 * 128 * group operations.  A warp takes a
// range of 32-key steps; the steps of all (sequence, KV head) items stand in one row and every warp
// gets the same number of them, whatever the lengths, so one wave ends together.  What an item's
// warps have found (maximum, sum, O) is joined in shared memory for the warps of a CTA and by a second
// small kernel for several CTAs; items inside one warp or CTA are finished there.
//
// Step: 32 keys, the K and V rows of two 16-key tiles (each in a page of its own when pages are
// short), brought by cp.async into the warp's own ring of two: half a warp copies a tile, so the
// places of both are one shuffle, and no barrier is needed but the warp's.  Products on m16n8k16 with
// fp16 operands and fp32 sums:
//   S^T = K Q^T    keys on M, heads on N.  The 128 elements are contracted in an order of our own:
//                  lane (g, c) multiplies elements [32c, 32c + 32) of keys g and g + 8, which are 16
//                  contiguous bytes of the row, with the same elements of Q (permuted once).
//   O^T += V^T P^T elements on M, heads on N: lane (g, c) needs keys 2c, 2c+1, 2c+8, 2c+9 of the 16
//                  elements of scale block g.  Row pairs' nibbles are joined in words of 8 before they are
//                  widened, so a byte becomes an operand register (key, key + 1) by one conversion.
// P^T comes from S^T by a transpose of 8x8 fragments (movmatrix).  A code times its scale is exact
// in fp16.  The running maximum moves when a score passes it by 8 (log2): a vote a step instead
// of a reduction; p (kv4.cuh, P_LOG2) is fp16 in the product, half a step 2^-11 of itself, and the sums are fp32.
//
// Instructions come next after HBM: widening takes 128 a lane and tile (a conversion, at half the rate, and a
// product for two elements), so everything else is kept per 32 keys.  32 sequences of 32,767 keys, 32/8 heads: 220 us,
// 0.84 of the copy rate; at the power cap (1.7 GHz) the instructions are the bound and it takes about 260.  (Past some 1,040
// sequences, 690 with few rows, the lists take more than half of an SM's shared memory beside the rings: one CTA an SM is
// resident then, and the equal shares of the grid are worked off in two waves.)
#include "kv4.cuh"

namespace ada {
namespace kv4 {
namespace dec {

constexpr int WARPS = 8;
constexpr int STAGES = 2;
constexpr int TILE = 16;                      // keys that lie in one page
constexpr int KEYS = 2 * TILE;                // keys a step
// a ring slot: of each tile K codes, V codes, then K scales, V scales
constexpr int V_OFF = TILE * ROW;
constexpr int KS_OFF = 2 * TILE * ROW;
constexpr int VS_OFF = KS_OFF + TILE * SROW;
constexpr int TILE_BYTES = 2 * TILE * ROW_BYTES;
constexpr int STEP_BYTES = 2 * TILE_BYTES;
constexpr int HEADS = 8;                         // heads side by side (N of the MMA)
constexpr int PART = HEADS * D + 2 * HEADS;      // floats of a partial: O, then (m, l) per head
constexpr int WARP_SMEM = STAGES * STEP_BYTES + PART * 4;
constexpr int MAX_BATCH = 8192;
constexpr int64_t MOST_STEPS = 1 << 30;
static_assert(STAGES * STEP_BYTES >= PART * 4, "a warp's last partial lies in its ring");

struct Params {
  const void* q;
  int64_t q_sb, q_sh;
  void* out;
  int64_t o_sb, o_sh;
  int q_bf16, o_bf16;
  const uint8_t *kc, *vc;
  int64_t s_page, s_head, num_pages;
  const int32_t* bt;
  int64_t bt_stride;
  int max_pages, page, batch;
  int span;              // keys that a row sees at most (0: all before it)
  int hkv, group, subs;  // subs: parts of 8 columns ((token, head) pairs of a KV head's group) a sequence has at most
  const int32_t* lens;          // decode: keys of each sequence
  const int32_t *cu_q, *cu_k;   // rows: prefix sums of new tokens and of keys
  int most;                     // rows: tokens of a sequence that are computed
  int64_t rows;                 // of q and out
  float scale_log2, v_scale;
  int* cum;      // workspace: [batch + 1] (steps x parts) before a sequence, then steps a CTA
  float* parts;  // workspace: [grid][2][PART]
};

// A sequence: its keys, its new tokens (1 for decode), and how many of them are computed.
struct Seq {
  int keys, fresh, tokens;
};
template <bool ROWS>
__device__ __forceinline__ Seq seq_of(const Params& P, int keys, int fresh) {
  constexpr int MOST = 1 << 30;
  if (!ROWS) return {min(max(keys, 0), MOST), 1, 1};
  const int n = min(max(fresh, 0), MOST);
  return {min(max(keys, 0), MOST), n, min(n, P.most)};
}
template <bool ROWS>
__device__ __forceinline__ Seq load_seq(const Params& P, int b) {
  if (!ROWS) return seq_of<ROWS>(P, P.lens[b], 1);
  // (differences of lists that do not ascend may wrap: any value is as good as another there)
  const unsigned k0 = (unsigned)P.cu_k[b], k1 = (unsigned)P.cu_k[b + 1];
  const unsigned q0 = (unsigned)P.cu_q[b], q1 = (unsigned)P.cu_q[b + 1];
  return seq_of<ROWS>(P, (int)(k1 - k0), (int)(q1 - q0));
}
// Keys [lo, hi) that token i of a sequence sees (0 <= i < tokens).
__device__ __forceinline__ int lo_of(const Params& P, const Seq& q, int i) {
  return P.span > 0 ? max(q.keys - q.fresh + i + 1 - P.span, 0) : 0;
}
__device__ __forceinline__ int hi_of(const Params& P, const Seq& q, int i) {
  return max(min(min(q.keys, P.max_pages * P.page), q.keys - q.fresh + i + 1), 0);
}
struct Range {
  int lo, hi, first;  // keys that any token sees, first step
};
__device__ __forceinline__ Range range_of(const Params& P, const Seq& q) {
  Range r;
  r.lo = lo_of(P, q, 0);
  r.hi = q.tokens > 0 ? hi_of(P, q, q.tokens - 1) : 0;
  r.first = r.lo / KEYS;
  return r;
}
__device__ __forceinline__ int steps_of(const Range& r) {
  return r.hi > r.lo ? (r.hi + KEYS - 1) / KEYS - r.first : 0;
}
template <bool ROWS>
__device__ __forceinline__ int parts_of(const Params& P, const Seq& q) {
  return ROWS ? (q.tokens * P.group + HEADS - 1) / HEADS : P.subs;
}

// One (sequence, KV head, part of its columns), and where its steps stand in the row of all.
struct Item {
  int b, kvh, part, base, end;
};
// The sequence of step t (cum: steps x parts before a sequence, for one KV head).
__device__ __forceinline__ int seq_at(const int* cum, int batch, int hkv, int t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid + 1] * hkv > t)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// Two rows lie in 128 bytes; a 16-byte chunk's place in them is moved by 2 * (line mod 4), so that
// both the 16-byte reads of 8 keys' quarter rows and the 8-byte reads of every other key's blocks
// fall on different banks.
__device__ __forceinline__ int chunk_at(int line, int chunk) { return line * 128 + ((chunk ^ (2 * (line & 3))) << 4); }

// A pair times one half of another (through the type, so that the instruction takes the half and no other makes a pair).
__device__ __forceinline__ uint32_t by_half(uint32_t a, uint32_t s, bool high) {
  const __half2 h = *reinterpret_cast<const __half2*>(&s);
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), high ? __high2half2(h) : __low2half2(h));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Row of one head to memory: 16 elements of lane's scale block.
__device__ __forceinline__ void write16(const Params& P, int64_t row, int head, int e0, const float* f) {
  if (P.o_bf16) {
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(P.out) + row * P.o_sb + head * P.o_sh + e0;
    *reinterpret_cast<uint4*>(o) = pack8<__nv_bfloat16>(f);
    *reinterpret_cast<uint4*>(o + 8) = pack8<__nv_bfloat16>(f + 8);
  } else {
    __half* o = reinterpret_cast<__half*>(P.out) + row * P.o_sb + head * P.o_sh + e0;
    *reinterpret_cast<uint4*>(o) = pack8<__half>(f);
    *reinterpret_cast<uint4*>(o + 8) = pack8<__half>(f + 8);
  }
}
__device__ __forceinline__ void write4(const Params& P, int64_t row, int head, int e0, float4 f) {
  if (P.o_bf16) {
    __nv_bfloat162 u[2] = {__floats2bfloat162_rn(f.x, f.y), __floats2bfloat162_rn(f.z, f.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(P.out) + row * P.o_sb + head * P.o_sh + e0) =
        *reinterpret_cast<uint2*>(u);
  } else {
    __half2 u[2] = {__floats2half2_rn(f.x, f.y), __floats2half2_rn(f.z, f.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(P.out) + row * P.o_sb + head * P.o_sh + e0) =
        *reinterpret_cast<uint2*>(u);
  }
}

// State of a warp's current piece of an item.
struct Acc {
  float o[8][4];  // M tile m: elements 16g + 2m (0, 1) and + 1 (2, 3), heads 2c (even) and 2c + 1
  float l[2];
};

// Column n of a part: its row of q and out and its head; false where there is none.
template <bool ROWS>
__device__ __forceinline__ bool column(const Params& P, const Item& it, const Seq& q, int64_t q0, int n, int64_t& row,
                                       int& head, int& token) {
  const int col = it.part * HEADS + n;
  token = ROWS ? col / P.group : 0;
  head = it.kvh * P.group + (ROWS ? col - token * P.group : col);
  row = ROWS ? q0 + token : it.b;
  return ROWS ? token < q.tokens && row >= 0 && row < P.rows : col < P.group;
}

// ALONE: one CTA an item, which it finishes; otherwise the steps of all items shared out equally.
// ROWS: a few new tokens a sequence, whose rows are columns beside each other as the heads are (the keys are
// read once for 8 of them), each with a last key of its own; otherwise one token, the newest.
template <bool ALONE, bool ROWS>
__global__ void __launch_bounds__(WARPS * 32, 2) split_kernel(const __grid_constant__ Params P) {
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int warp_sum[WARPS];
  __shared__ Item part_item[WARPS][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  uint8_t* ring = sm + warp * WARP_SMEM;
  float* slot0 = reinterpret_cast<float*>(ring + STAGES * STEP_BYTES);
  // steps before each sequence, and the lengths (a copy a warp for up to 32 sequences: no barrier)
  int* lists = reinterpret_cast<int*>(sm + WARPS * WARP_SMEM);
  const bool few = P.batch <= 32;
  int* cum = few ? lists + warp * 108 : lists;
  int* keys = few ? cum + 36 : lists + P.batch + 1;
  int* fresh = few ? keys + 36 : keys + P.batch;  // (ROWS)
  if (lane < 2) part_item[warp][lane].end = 0;  // no partial
  pdl_wait();
  pdl_trigger();

  int cta0, cta1, r0, r1;
  Item alone{0, 0, 0, 0, 0};
  Seq alone_seq{0, 0, 0};
  if (ALONE) {
    const int items = P.hkv * P.subs, h = blockIdx.x % items;
    alone.b = blockIdx.x / items;
    alone.kvh = h / P.subs;
    alone.part = h - alone.kvh * P.subs;
    alone_seq = load_seq<ROWS>(P, alone.b);
    alone.end = steps_of(range_of(P, alone_seq));
    const int per = (alone.end + WARPS - 1) / WARPS;
    cta0 = 0;
    cta1 = alone.end;
    r0 = min(warp * per, cta1);
    r1 = min(r0 + per, cta1);
  } else {
    auto cost = [&](const Seq& q) { return steps_of(range_of(P, q)) * parts_of<ROWS>(P, q); };
    if (few) {
      Seq q{0, 0, 0};
      if (lane < P.batch) q = load_seq<ROWS>(P, lane);
      int inc = lane < P.batch ? cost(q) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      cum[lane + 1] = inc;
      keys[lane] = q.keys;
      if (ROWS) fresh[lane] = q.fresh;
      if (lane == 0) cum[0] = 0;
      __syncwarp();
    } else {
      const int per = (P.batch + WARPS * 32 - 1) / (WARPS * 32);
      const int b0 = min(tid * per, P.batch), b1 = min(b0 + per, P.batch);
      int sum = 0;
      for (int b = b0; b < b1; ++b) {
        const Seq q = load_seq<ROWS>(P, b);
        keys[b] = q.keys;
        if (ROWS) fresh[b] = q.fresh;
        sum += cost(q);
      }
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (lane == 31) warp_sum[warp] = inc;
      __syncthreads();
      int run = inc - sum;
      for (int w = 0; w < warp; ++w) run += warp_sum[w];
      for (int b = b0; b < b1; ++b) {
        cum[b] = run;
        run += cost(seq_of<ROWS>(P, keys[b], ROWS ? fresh[b] : 1));
      }
      if (b0 < b1 && b1 == P.batch) cum[P.batch] = run;
      __syncthreads();
    }
    const int total = cum[P.batch] * P.hkv;
    const int workers = gridDim.x * WARPS;
    const int per = max((total + workers - 1) / workers, 1);
    if (blockIdx.x == 0) {  // for the merge (with few sequences every warp has the lists, and the first writes them)
      for (int b = few ? lane : tid; b <= P.batch; b += few ? 32 : WARPS * 32)
        if (!few || warp == 0) P.cum[b] = cum[b];
      if (tid == 0) P.cum[P.batch + 1] = per * WARPS;
    }
    const int64_t c0 = (int64_t)blockIdx.x * WARPS * per;  // this CTA's steps
    if (c0 >= total) return;
    cta0 = (int)c0;
    cta1 = (int)min(c0 + (int64_t)WARPS * per, (int64_t)total);
    r0 = min(cta0 + warp * per, total);
    r1 = min(r0 + per, total);
  }
  auto seq_in = [&](int b) { return ALONE ? alone_seq : seq_of<ROWS>(P, keys[b], ROWS ? fresh[b] : 1); };
  auto item_at = [&](int t) {  // (the step's item has steps, so there are parts)
    if (ALONE) return alone;
    Item it;
    it.b = seq_at(cum, P.batch, P.hkv, t);
    const Seq q = seq_in(it.b);
    const int n = steps_of(range_of(P, q)), parts = parts_of<ROWS>(P, q), h = (t - cum[it.b] * P.hkv) / n;
    it.kvh = h / parts;
    it.part = h - it.kvh * parts;
    it.base = cum[it.b] * P.hkv + h * n;
    it.end = it.base + n;
    return it;
  };
  auto range_at = [&](int b) { return range_of(P, seq_in(b)); };

  if (r0 < r1) {
    // ---- the loads' cursor: step `ld` of the row, its item, and 32 tiles (16 steps) from step `from` on in the
    // lanes: the page's id (-1: not there) and the tile's place in it
    Item li = item_at(r0);
    Range lr = range_at(li.b);
    int ld = r0, from = -64, id = -1, place = 0;
    const int page_tiles = P.page / TILE;
    const int half = lane >> 4, l16 = lane & 15;
    const int64_t head_off = (int64_t)li.kvh * P.s_head;
    const uint8_t *klane = P.kc + head_off + 16 * l16, *vlane = P.vc + head_off + 16 * l16;
    auto look = [&]() {
      from = ld;
      const int key = (lr.first + (ld - li.base)) * KEYS + lane * TILE;
      id = -1;
      place = 0;
      if (key < lr.hi) {
        const int tile = key / TILE, col = tile / page_tiles;
        place = tile - col * page_tiles;
        id = P.bt[(int64_t)li.b * P.bt_stride + col];
        if (id >= P.num_pages) id = -1;
      }
    };
    uint32_t there = 0;  // bits 2s, 2s + 1: the tiles in ring slot s are in the cache
    const uint32_t lane_dst = smem_addr(ring) + half * TILE_BYTES + (l16 >> 3) * 128;
    const uint32_t even = lane_dst + (((l16 & 7) ^ (2 * (l16 >> 3))) << 4);  // lines 0, 1 of each four, then 2, 3
    const uint32_t odd = lane_dst + (((l16 & 7) ^ (2 * (l16 >> 3)) ^ 4) << 4);
    const uint32_t scales = smem_addr(ring) + half * TILE_BYTES + KS_OFF + 16 * l16;
    auto load = [&](const int slot) {
      if (ld < r1) {
        if (ld == li.end) {
          li = item_at(ld);
          lr = range_at(li.b);
          from = -64;
          const int64_t off = (int64_t)li.kvh * P.s_head;
          klane = P.kc + off + 16 * l16;
          vlane = P.vc + off + 16 * l16;
        }
        if (ld >= from + 16) look();
        const int src = 2 * (ld - from) + half;
        const int my = __shfl_sync(0xffffffffu, id, src), at = __shfl_sync(0xffffffffu, place, src);
        const uint32_t ok = __ballot_sync(0xffffffffu, my >= 0);
        there = (there & ~(3u << (2 * slot))) | (((ok & 1u) | ((ok >> 15) & 2u)) << (2 * slot));
        if (my >= 0) {
          const int64_t page = (int64_t)my * P.s_page;
          const uint8_t *k = klane + page + at * (TILE * ROW), *v = vlane + page + at * (TILE * ROW);
          const uint32_t s = slot * STEP_BYTES;
          cp16(even + s, k);
          cp16(odd + s + 256, k + 256);
          cp16(even + s + 512, k + 512);
          cp16(odd + s + 768, k + 768);
          cp16(even + s + V_OFF, v);
          cp16(odd + s + V_OFF + 256, v + 256);
          cp16(even + s + V_OFF + 512, v + 512);
          cp16(odd + s + V_OFF + 768, v + 768);
          // 8 pieces of K's scales, 8 of V's
          cp16(scales + s, (l16 < 8 ? k : v - 128) + (P.page * ROW - at * (TILE * (ROW - SROW))));
        }
        ++ld;
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES; ++i) load(i);

    // ---- items of the range
    int t = r0, slot = 0;
    while (t < r1) {
      const Item it = item_at(t);
      const Range rg = range_at(it.b);
      const int stop = min(it.end, r1);
      const Seq sq = seq_in(it.b);
      const int64_t q0 = ROWS ? P.cu_q[it.b] : 0;
      int64_t row;
      int head, token;
      // ROWS: keys that this lane's columns 2c, 2c + 1 see, and where all columns of the part see the same
      int lo0 = 0, hi0 = 0, lo1 = 0, hi1 = 0, lo_all = rg.lo, hi_all = rg.hi;
      if (ROWS) {
        if (column<ROWS>(P, it, sq, q0, 2 * c, row, head, token)) lo0 = lo_of(P, sq, token), hi0 = hi_of(P, sq, token);
        if (column<ROWS>(P, it, sq, q0, 2 * c + 1, row, head, token))
          lo1 = lo_of(P, sq, token), hi1 = hi_of(P, sq, token);
        lo_all = lo_of(P, sq, min((it.part * HEADS + HEADS - 1) / P.group, sq.tokens - 1));
        hi_all = hi_of(P, sq, it.part * HEADS / P.group);
      }
      // queries: column g, elements [32c, 32c + 32)
      const bool mine = column<ROWS>(P, it, sq, q0, g, row, head, token);
      uint32_t qf[16];
      float fac[2];
      {
        float top = 0.f;
        float f[32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (mine) {
            const int64_t off = row * P.q_sb + head * P.q_sh + 32 * c + 8 * i;
            if (P.q_bf16)
              unpack8<__nv_bfloat16>(*reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(P.q) + off), f + 8 * i);
            else
              unpack8<__half>(*reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(P.q) + off), f + 8 * i);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[8 * i + j] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max_nan(top, fabsf(f[i]));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = query_exponent(top);
        const float mul = pow2(ex);
#pragma unroll
        for (int i = 0; i < 16; ++i) qf[i] = pack_half2(f[2 * i] * mul, f[2 * i + 1] * mul);
        const float mine = score_factor(P.scale_log2, ex);
        fac[0] = __shfl_sync(0xffffffffu, mine, 8 * c);
        fac[1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
      }
      Acc a;
#pragma unroll
      for (int m = 0; m < 8; ++m) a.o[m][0] = a.o[m][1] = a.o[m][2] = a.o[m][3] = 0.f;
      a.l[0] = a.l[1] = 0.f;
      float base0 = 0.f, base1 = 0.f;              // the running maxima
      // scores beyond these move them; -inf: there is none yet (rounded down: the next score above may be 16 further,
      // and its p an infinity in fp16)
      float pass0 = -INFINITY, pass1 = -INFINITY;

      // A step whose ring slot is a constant, and so its addresses (549 instead of 583 instructions, 224 -> 221 us for the
      // long case).  ROWS keeps the slot a variable: with its masks the step stands there once (36 bytes of spill stores
      // instead of 80: 32 x 8 tokens behind 500 keys 35.2 instead of 38.5 us, 8 x 2 behind 8,000 32.3 and 33.3, 32 x 8
      // behind 8,000 235 and 233).
      auto one = [&](auto at) {
        const int slot = at;
        cp_wait<STAGES - 1>();
        __syncwarp();
        const uint8_t* step = ring + slot * STEP_BYTES;
        const uint32_t ok = (there >> (2 * slot)) & 3u;
        const int key0 = (rg.first + (t - it.base)) * KEYS;
        const bool edge = key0 < lo_all || key0 + KEYS > hi_all || ok != 3u;
        // scores: tile i, keys g, g + 8 x heads 2c, 2c + 1
        float s[2][4];
        uint32_t vs[2][2];  // scales of block g, keys (2c, 2c + 1) and (2c + 8, 2c + 9)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint8_t* tile = step + i * TILE_BYTES;
          s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
          const uint4 k0 = *reinterpret_cast<const uint4*>(tile + chunk_at(g >> 1, (g & 1) * 4 + c));
          const uint4 k1 = *reinterpret_cast<const uint4*>(tile + chunk_at((g >> 1) + 4, (g & 1) * 4 + c));
          const uint32_t s0 = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(tile + KS_OFF + g * SROW + 2 * c));
          const uint32_t s1 = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(tile + KS_OFF + (g + 8) * SROW + 2 * c));
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t x[4], y[4];
            widen8(w0[w], x);
            widen8(w1[w], y);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t A[4] = {by_half(x[2 * j], s0, w >= 2), by_half(y[2 * j], s1, w >= 2),
                                     by_half(x[2 * j + 1], s0, w >= 2), by_half(y[2 * j + 1], s1, w >= 2)};
              mma_16816_f16(s[i], A, qf + 2 * (2 * w + j));
            }
          }
          const uint8_t* p = tile + VS_OFF + 2 * c * SROW + g;
          vs[i][0] = p[0] | ((uint32_t)p[SROW] << 8);
          vs[i][1] = p[8 * SROW] | ((uint32_t)p[9 * SROW] << 8);
        }
        if (edge) {  // what is not seen counts as 0, also where it would be NaN
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = key0 + i * TILE, hi = (ok >> i) & 1u ? rg.hi : 0;
            auto seen = [&](int key) { return key >= rg.lo && key < hi; };
            if (ROWS) {
              const int ha = min(hi0, hi), hb = min(hi1, hi);
              if (k + g < lo0 || k + g >= ha) s[i][0] = -INFINITY;
              if (k + g < lo1 || k + g >= hb) s[i][1] = -INFINITY;
              if (k + g + 8 < lo0 || k + g + 8 >= ha) s[i][2] = -INFINITY;
              if (k + g + 8 < lo1 || k + g + 8 >= hb) s[i][3] = -INFINITY;
            } else {
              if (!seen(k + g)) s[i][0] = s[i][1] = -INFINITY;
              if (!seen(k + g + 8)) s[i][2] = s[i][3] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (!seen(k + 2 * c + 8 * j)) vs[i][j] &= 0xFF00u;
              if (!seen(k + 2 * c + 8 * j + 1)) vs[i][j] &= 0x00FFu;
            }
          }
        }
        if (ROWS && edge) {
          // A value's NaN would reach columns that do not see its key, through 0 * NaN: it counts as 0, and the
          // columns that see it get their 16 elements' NaN here (rare: a vote says whether there is one).
          uint32_t bad = 0;  // bit 4i + 2j + x: key 16i + 8j + 2c + x
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const uint32_t v = vs[n >> 2][(n >> 1) & 1] >> (8 * (n & 1));
            if ((v & 0x7Fu) == 0x7Fu) bad |= 1u << n;
          }
          if (__any_sync(0xffffffffu, bad != 0)) {
            const float nan = __uint_as_float(0x7FC00000u);
            for (int o = 0; o < 4; ++o) {
              const uint32_t theirs = __shfl_sync(0xffffffffu, bad, (lane & ~3) + o);
              for (int n = 0; n < 8; ++n) {
                const int key = key0 + 16 * (n >> 2) + 8 * ((n >> 1) & 1) + 2 * o + (n & 1);
                if (!((theirs >> n) & 1u)) continue;
#pragma unroll
                for (int m = 0; m < 8; ++m) {
                  if (key >= lo0 && key < hi0) a.o[m][0] = a.o[m][2] = nan;
                  if (key >= lo1 && key < hi1) a.o[m][1] = a.o[m][3] = nan;
                }
              }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
              if ((bad >> n) & 1u) vs[n >> 2][(n >> 1) & 1] &= n & 1 ? 0x00FFu : 0xFF00u;
          }
        }
        const float x0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2]));
        const float x1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
        if (__any_sync(0xffffffffu, x0 > pass0 || x1 > pass1)) {
          float n0 = x0, n1 = x1;
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
          }
          float f0 = 1.f, f1 = 1.f;
          if (n0 > pass0) {
            f0 = pass0 == -INFINITY ? 0.f : fast_exp2((base0 - n0) * fac[0]);
            base0 = n0;
            pass0 = __fadd_rd(n0, 8.f / fac[0]);
          }
          if (n1 > pass1) {
            f1 = pass1 == -INFINITY ? 0.f : fast_exp2((base1 - n1) * fac[1]);
            base1 = n1;
            pass1 = __fadd_rd(n1, 8.f / fac[1]);
          }
          a.l[0] *= f0;
          a.l[1] *= f1;
#pragma unroll
          for (int m = 0; m < 8; ++m) {
            a.o[m][0] *= f0;
            a.o[m][1] *= f1;
            a.o[m][2] *= f0;
            a.o[m][3] *= f1;
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint8_t* tile = step + i * TILE_BYTES + V_OFF;
          const float p0 = fast_exp2(fmaf(s[i][0] - base0, fac[0], P_LOG2)), p1 = fast_exp2(fmaf(s[i][1] - base1, fac[1], P_LOG2));
          const float p2 = fast_exp2(fmaf(s[i][2] - base0, fac[0], P_LOG2)), p3 = fast_exp2(fmaf(s[i][3] - base1, fac[1], P_LOG2));
          a.l[0] += p0 + p2;
          a.l[1] += p1 + p3;
          const uint32_t pb[2] = {transpose8(pack_half2(p0, p1)), transpose8(pack_half2(p2, p3))};
          const uint32_t vs0 = e4m3x2_to_f16x2((uint16_t)vs[i][0]), vs1 = e4m3x2_to_f16x2((uint16_t)vs[i][1]);
          // values: keys 2c, 2c + 1, 2c + 8, 2c + 9, block g
          const int vch = g >> 1, vin = (g & 1) * 8;
          const uint2 va = *reinterpret_cast<const uint2*>(tile + chunk_at(c, vch) + vin);
          const uint2 vb = *reinterpret_cast<const uint2*>(tile + chunk_at(c, 4 + vch) + vin);
          const uint2 vc = *reinterpret_cast<const uint2*>(tile + chunk_at(c + 4, vch) + vin);
          const uint2 vd = *reinterpret_cast<const uint2*>(tile + chunk_at(c + 4, 4 + vch) + vin);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t a0 = w ? va.y : va.x, b0 = w ? vb.y : vb.x, c0_ = w ? vc.y : vc.x, d0 = w ? vd.y : vd.x;
            constexpr uint32_t LO = 0x0F0F0F0Fu;
            uint32_t e0[4], e1[4], f0[4], f1[4];  // (even, odd) elements of the first and second key pair
            widen8((a0 & LO) | ((b0 << 4) & ~LO), e0);
            widen8(((a0 >> 4) & LO) | (b0 & ~LO), e1);
            widen8((c0_ & LO) | ((d0 << 4) & ~LO), f0);
            widen8(((c0_ >> 4) & LO) | (d0 & ~LO), f1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t A[4] = {mul_f16x2(e0[j], vs0), mul_f16x2(e1[j], vs0), mul_f16x2(f0[j], vs1), mul_f16x2(f1[j], vs1)};
              mma_16816_f16(a.o[4 * w + j], A, pb);
            }
          }
        }
        __syncwarp();  // every lane has read the slot
        load(slot);
      };
      for (; t < stop; ++t) {
        if (ROWS)
          one(slot);
        else if (slot == 0)
          one(std::integral_constant<int, 0>());
        else
          one(std::integral_constant<int, 1>());
        slot ^= 1;
      }

      // ---- the piece's end
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        a.l[0] += __shfl_xor_sync(0xffffffffu, a.l[0], o);
        a.l[1] += __shfl_xor_sync(0xffffffffu, a.l[1], o);
      }
      const bool began = it.base >= r0, ended = it.end <= r1;
      if (began && ended) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!column<ROWS>(P, it, sq, q0, 2 * c + x, row, head, token)) continue;
          // (a NaN sum stays one)
          const float inv = a.l[x] == 0.f ? 0.f : P.v_scale / a.l[x];
          float f[16];
#pragma unroll
          for (int m = 0; m < 8; ++m) {
            f[2 * m] = a.o[m][x] * inv;
            f[2 * m + 1] = a.o[m][2 + x] * inv;
          }
          write16(P, row, head, 16 * g, f);
        }
      } else {
        // the last piece's partial may lie in the ring: its own copies have arrived
        const int which = began ? 1 : 0;
        float* dst = which ? reinterpret_cast<float*>(ring) : slot0;
        if (which) {
          cp_wait<0>();
          __syncwarp();
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float* o = dst + (2 * c + x) * D + 16 * g;
#pragma unroll
          for (int m = 0; m < 8; m += 2)
            *reinterpret_cast<float4*>(o + 2 * m) = make_float4(a.o[m][x], a.o[m][2 + x], a.o[m + 1][x], a.o[m + 1][2 + x]);
          if (g == 0) {
            const float top = x ? base1 : base0, pass = x ? pass1 : pass0;
            dst[HEADS * D + 2 * (2 * c + x)] = pass == -INFINITY ? -INFINITY : top * fac[x];
            dst[HEADS * D + 2 * (2 * c + x) + 1] = a.l[x];
          }
        }
        if (lane == 0) part_item[warp][which] = it;
      }
    }
  }
  __syncthreads();

  // ---- pieces of one item in several warps: joined here (thread: column, 4 elements)
  const int col = tid >> 5, e0 = 4 * lane;
  auto finish = [&](const Item& it, float4 o, float l) {
    const Seq q = seq_in(it.b);
    int64_t row;
    int head, token;
    if (!column<ROWS>(P, it, q, ROWS ? P.cu_q[it.b] : 0, col, row, head, token)) return;
    const float inv = l == 0.f ? 0.f : P.v_scale / l;
    write4(P, row, head, e0, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  };
  if (ALONE && cta1 == 0) {  // no key
    finish(alone, make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
    return;
  }
  int w = 0;
  while (w < 2 * WARPS) {
    const Item it = part_item[w >> 1][w & 1];
    if (it.end == 0) {
      ++w;
      continue;
    }
    int last = w;  // the item's last partial of this CTA: its others are the first slots of the next warps
    for (int n = ((w >> 1) + 1) * 2; n < 2 * WARPS; n += 2) {
      const Item x = part_item[n >> 1][0];
      if (x.end != it.end) break;
      last = n;
    }
    auto piece = [&](int n) {
      const uint8_t* r = sm + (n >> 1) * WARP_SMEM;
      return reinterpret_cast<const float*>(n & 1 ? r : r + STAGES * STEP_BYTES);
    };
    float m = -INFINITY;
    for (int n = w; n <= last; n = ((n >> 1) + 1) * 2) m = fmaxf(m, piece(n)[HEADS * D + 2 * col]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int n = w; n <= last; n = ((n >> 1) + 1) * 2) {
      const float* p = piece(n);
      const float pm = p[HEADS * D + 2 * col];
      const float f = m == -INFINITY ? 1.f : fast_exp2(pm - m);
      const float4 x = *reinterpret_cast<const float4*>(p + col * D + e0);
      l = fmaf(f, p[HEADS * D + 2 * col + 1], l);
      o.x = fmaf(f, x.x, o.x);
      o.y = fmaf(f, x.y, o.y);
      o.z = fmaf(f, x.z, o.z);
      o.w = fmaf(f, x.w, o.w);
    }
    if (it.base >= cta0 && it.end <= cta1) {
      finish(it, o, l);
    } else {
      float* dst = P.parts + ((int64_t)blockIdx.x * 2 + (it.base >= cta0 ? 1 : 0)) * PART;
      *reinterpret_cast<float4*>(dst + col * D + e0) = o;
      if (lane == 0) {
        dst[HEADS * D + 2 * col] = m;
        dst[HEADS * D + 2 * col + 1] = l;
      }
    }
    w = last + 1;
  }
}

// Items of several CTAs, and sequences without keys.  One CTA an item; thread: head, 4 elements.
constexpr int MAX_CTAS = 512, EARLY = 6;
template <bool ROWS>
__global__ void __launch_bounds__(HEADS * 32) merge_kernel(const __grid_constant__ Params P) {
  __shared__ float weight[HEADS][MAX_CTAS];
  pdl_wait();
  pdl_trigger();
  const int items = P.hkv * P.subs, b = blockIdx.x / items, h = blockIdx.x - b * items;
  const int head = threadIdx.x >> 5, lane = threadIdx.x & 31, e0 = 4 * lane;  // (head: the column)
  Item it{b, h / P.subs, h % P.subs, 0, 0};
  const int before = P.cum[b], all = P.cum[b + 1] - before, chunk = P.cum[P.batch + 1];
  const Seq q = load_seq<ROWS>(P, b);
  const int parts = parts_of<ROWS>(P, q);
  if (it.part >= parts) return;
  int64_t row;
  int row_head, token;
  const bool mine = column<ROWS>(P, it, q, ROWS ? P.cu_q[b] : 0, head, row, row_head, token);
  if (all == 0) {
    if (mine) write4(P, row, row_head, e0, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int n = all / parts;
  const int base = before * P.hkv + (it.kvh * parts + it.part) * n;
  const int first = base / chunk, pieces = (base + n - 1) / chunk - first + 1;
  if (pieces == 1) return;  // finished there
  // the first CTA's partial is its second (the item begins there), the others' their first
  auto at = [&](int i) { return P.parts + ((int64_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * PART; };
  float4 early[EARLY];  // the first partials, asked for along with the maxima
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
    early[i] = i < pieces ? *reinterpret_cast<const float4*>(at(i) + head * D + e0) : make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < pieces; i += 32) m = fmaxf(m, at(i)[HEADS * D + 2 * head]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  for (int i = lane; i < pieces; i += 32) {
    const float* p = at(i) + HEADS * D + 2 * head;
    const float f = m == -INFINITY ? 1.f : fast_exp2(p[0] - m);
    weight[head][i] = f;
    l = fmaf(f, p[1], l);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  __syncwarp();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < EARLY; ++i) {
    if (i >= pieces) break;
    const float f = weight[head][i];
    o.x = fmaf(f, early[i].x, o.x);
    o.y = fmaf(f, early[i].y, o.y);
    o.z = fmaf(f, early[i].z, o.z);
    o.w = fmaf(f, early[i].w, o.w);
  }
#pragma unroll 4
  for (int i = EARLY; i < pieces; ++i) {
    const float f = weight[head][i];
    const float4 x = *reinterpret_cast<const float4*>(at(i) + head * D + e0);
    o.x = fmaf(f, x.x, o.x);
    o.y = fmaf(f, x.y, o.y);
    o.z = fmaf(f, x.z, o.z);
    o.w = fmaf(f, x.w, o.w);
  }
  const float inv = l == 0.f ? 0.f : P.v_scale / l;
  if (mine) write4(P, row, row_head, e0, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

static int grid_size(int dev) {
  static std::atomic<int> sms[64];
  int n = sms[dev];
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 0;
    sms[dev] = n;
  }
  return n * 2 < MAX_CTAS ? n * 2 : MAX_CTAS;
}
// Shared memory limits of this device's kernels, once.
static int prepare() {
  static std::atomic<bool> ready[64];
  constexpr int lists = (3 * MAX_BATCH + 1) * 4;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ADA_ERR_CUDA;
  if (ready[dev]) return ADA_OK;
  if (cudaFuncSetAttribute(split_kernel<false, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           WARPS * WARP_SMEM + lists) != cudaSuccess ||
      cudaFuncSetAttribute(split_kernel<false, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           WARPS * WARP_SMEM + lists) != cudaSuccess ||
      cudaFuncSetAttribute(split_kernel<true, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, WARPS * WARP_SMEM) !=
          cudaSuccess)
    return ADA_ERR_CUDA;
  ready[dev] = true;
  return ADA_OK;
}
// Steps shared out equally, then the items of several CTAs joined.
template <bool ROWS>
static int launch_shared(const Params& P, cudaStream_t st) {
  if (const int e = prepare()) return e;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ADA_ERR_CUDA;
  const int grid = grid_size(dev);
  if (grid == 0) return ADA_ERR_CUDA;
  const size_t smem = WARPS * WARP_SMEM + (P.batch <= 32 ? WARPS * 108 * 4 : (size_t)((ROWS ? 3 : 2) * P.batch + 1) * 4);
  (void)launch_k(split_kernel<false, ROWS>, dim3((unsigned)grid), dim3(WARPS * 32), smem, st, P);
  ADA_CHECK_LAUNCH();
  (void)launch_k(merge_kernel<ROWS>, dim3((unsigned)(P.batch * P.hkv * P.subs)), dim3(HEADS * 32), 0, st, P);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}

}  // namespace dec
}  // namespace kv4
}  // namespace ada

using namespace ada;
namespace dec = ada::kv4::dec;

// The lists (cum and the steps a CTA), rounded up to 16 bytes, then two partials a CTA.
static size_t decode_lists(int32_t batch) { return ((size_t)(batch + 2) * 4 + 15) & ~(size_t)15; }

// One CTA an item, and one launch, where an item has at most 40 steps (five a warp) whatever its length and
// all items are resident at once; otherwise equal shares and a second launch that joins them.  (One sequence
// of 700 keys, 32/8 heads: 11.3 us shared out, 8.4 alone; 4 x 1,024 keys of a window, 32/16: 14.3 and 10.3.  With
// 16 warps a CTA 9.6 and 10.7: an SM issues the item's instructions no faster.)
static bool decode_alone(int64_t batch, int32_t num_heads, int32_t num_kv_heads, int32_t max_pages, int32_t page_size,
                         int32_t window) {
  const int64_t group = num_heads / num_kv_heads, items = num_kv_heads * cdiv(group, (int64_t)dec::HEADS);
  const int64_t all = (int64_t)max_pages * page_size;
  const int64_t reach = window > 0 && window < all ? (int64_t)window + dec::KEYS - 1 : all;
  return batch * items <= 2 * 148 && cdiv(reach, (int64_t)dec::KEYS) <= 5 * dec::WARPS;
}

extern "C" size_t ada_kv4_paged_decode_workspace_size(int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                                                      int32_t max_pages, int32_t page_size, int32_t window) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || max_pages <= 0 || page_size <= 0) return 0;
  if (decode_alone(batch, num_heads, num_kv_heads, max_pages, page_size, window)) return 0;
  return decode_lists(batch) + (size_t)dec::MAX_CTAS * 2 * dec::PART * 4;
}

extern "C" int ada_kv4_paged_decode(const void* q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h,
                                    const uint8_t* k_cache, const uint8_t* v_cache, int64_t kv_stride_page,
                                    int64_t kv_stride_head, int64_t num_pages, const int32_t* block_tables,
                                    int64_t bt_stride, int32_t max_pages, const int32_t* context_lens, int32_t batch,
                                    int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size,
                                    float scale, float k_scale, float v_scale, int32_t window, void* out,
                                    int out_dtype, int64_t out_stride_b, int64_t out_stride_h, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (batch < 0) return ADA_ERR_INVALID_ARG;
  if (batch == 0) return ADA_OK;
  if (!context_lens) return ADA_ERR_INVALID_ARG;
  if (const int e = kv4::attn_ok(q, q_dtype, q_stride_b, q_stride_h, out, out_dtype, out_stride_b, out_stride_h, k_cache,
                                 v_cache, kv_stride_page, kv_stride_head, num_pages, block_tables, bt_stride, max_pages,
                                 num_heads, num_kv_heads, head_dim, page_size, scale, k_scale, v_scale, window))
    return e;
  if (reinterpret_cast<uintptr_t>(context_lens) & 3) return ADA_ERR_ALIGNMENT;
  dec::Params P;
  P.hkv = num_kv_heads;
  P.group = num_heads / num_kv_heads;
  P.subs = (P.group + dec::HEADS - 1) / dec::HEADS;
  const int64_t items = (int64_t)num_kv_heads * P.subs;
  const int64_t steps = cdiv((int64_t)max_pages * page_size, dec::KEYS) + 1;
  // the row of all steps is counted in 32 bits
  if (batch > dec::MAX_BATCH || batch * items > dec::MOST_STEPS || batch * items * steps > dec::MOST_STEPS)
    return ADA_ERR_UNSUPPORTED;
  const bool alone = decode_alone(batch, num_heads, num_kv_heads, max_pages, page_size, window);
  if (!alone) {
    if (!workspace || workspace_bytes < ada_kv4_paged_decode_workspace_size(batch, num_heads, num_kv_heads, max_pages,
                                                                            page_size, window))
      return ADA_ERR_WORKSPACE;
    if (kv4::misaligned16(workspace)) return ADA_ERR_ALIGNMENT;
  }
  P.q = q;
  P.q_sb = q_stride_b;
  P.q_sh = q_stride_h;
  P.out = out;
  P.o_sb = out_stride_b;
  P.o_sh = out_stride_h;
  P.q_bf16 = q_dtype == ADA_DT_BF16;
  P.o_bf16 = out_dtype == ADA_DT_BF16;
  P.kc = k_cache;
  P.vc = v_cache;
  P.s_page = kv_stride_page;
  P.s_head = kv_stride_head;
  P.num_pages = num_pages;
  P.bt = block_tables;
  P.bt_stride = bt_stride;
  P.max_pages = max_pages;
  P.page = page_size;
  P.batch = batch;
  P.span = window;
  P.lens = context_lens;
  P.cu_q = P.cu_k = nullptr;
  P.most = 1;
  P.rows = batch;
  P.scale_log2 = scale * k_scale * kv4::LOG2E;
  P.v_scale = v_scale;
  P.cum = static_cast<int*>(workspace);
  P.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + decode_lists(batch));
  if (alone) {
    if (const int e = dec::prepare()) return e;
    (void)launch_k(dec::split_kernel<true, false>, dim3((unsigned)(batch * items)), dim3(dec::WARPS * 32),
                   dec::WARPS * dec::WARP_SMEM, reinterpret_cast<cudaStream_t>(stream), P);
    ADA_CHECK_LAUNCH();
    return ADA_OK;
  }
  return dec::launch_shared<false>(P, reinterpret_cast<cudaStream_t>(stream));
}

size_t ada::kv4::rows_workspace_size(int32_t batch) { return decode_lists(batch) + (size_t)dec::MAX_CTAS * 2 * dec::PART * 4; }

// The prefill entry's form for a few new tokens a sequence (its arguments are checked there).
int ada::kv4::rows_prefill(const void* q, int q_dtype, int64_t q_st, int64_t q_sh, const uint8_t* kc, const uint8_t* vc,
                           int64_t s_page, int64_t s_head, int64_t num_pages, const int32_t* bt, int64_t bt_stride,
                           int32_t max_pages, const int32_t* cu_q, const int32_t* cu_k, int32_t batch, int64_t rows,
                           int32_t most, int32_t hq, int32_t hkv, int32_t page, float scale_log2, float v_scale,
                           int32_t window, void* out, int out_dtype, int64_t o_st, int64_t o_sh, void* workspace,
                           cudaStream_t st) {
  dec::Params P;
  P.hkv = hkv;
  P.group = hq / hkv;
  P.subs = (most * P.group + dec::HEADS - 1) / dec::HEADS;
  P.q = q;
  P.q_sb = q_st;
  P.q_sh = q_sh;
  P.out = out;
  P.o_sb = o_st;
  P.o_sh = o_sh;
  P.q_bf16 = q_dtype == ADA_DT_BF16;
  P.o_bf16 = out_dtype == ADA_DT_BF16;
  P.kc = kc;
  P.vc = vc;
  P.s_page = s_page;
  P.s_head = s_head;
  P.num_pages = num_pages;
  P.bt = bt;
  P.bt_stride = bt_stride;
  P.max_pages = max_pages;
  P.page = page;
  P.batch = batch;
  P.span = window > 0 ? (window < (1 << 30) ? window + 1 : 0) : 0;  // (its own position and W before it)
  P.lens = nullptr;
  P.cu_q = cu_q;
  P.cu_k = cu_k;
  P.most = most;
  P.rows = rows;
  P.scale_log2 = scale_log2;
  P.v_scale = v_scale;
  P.cum = static_cast<int*>(workspace);
  P.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + decode_lists(batch));
  return dec::launch_shared<true>(P, st);
}
