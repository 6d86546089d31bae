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
//
// Work is cut into segments (a group's prefix, a sequence's own keys), a segment's (token, head of
// the GQA group) rows into blocks, its keys into splits, and each piece gives a partial softmax
// (maximum, sum, sum over V) in the workspace; a merge kernel joins a row's pieces.  What lies in a
// piece is worked out on the device from the lengths, so a call can be captured in a graph and
// follows the lengths it finds when it runs.
#include "common.cuh"
#include "sm100.cuh"

namespace ada {
namespace sp {

constexpr int D = 128;
constexpr int TILE = 16;              // keys of a tile: 16 rows of one page
constexpr int TILE_BYTES = TILE * D;  // 16 keys x 128 e4m3 bytes
constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned int ERR_TILE_WAIT = 0x90;

// Division of 0 <= n < 2^31 by a number fixed per launch: multiply and shift (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994): m = ceil(2^(31 + s) / d), s = ceil(log2 d).
struct Divisor {
  uint32_t m;
  int32_t shift, d;
  __host__ static Divisor of(int32_t d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s, d};
  }
  __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> shift); }
  __device__ __forceinline__ int divmod(int n, int& rest) const {
    const int q = div(n);
    rest = n - q * d;
    return q;
  }
};

// A token's partials.  Own keys: `own_splits` pieces, KV heads apart, from own_first + row block *
// own_splits * KV heads + KV head on, row own_row + head of the segment; prefix likewise, or with
// prefix_kernel the pieces of the `blocks` blocks from block `tc_from` + unit * blocks on (units: tc_units
// before the group).
struct RowPlan {
  int own_first, own_splits, own_row, pre_row;
  int pre_first, pre_splits, blocks, pad;
  int64_t tc_from, tc_units;
  int64_t tc_total, tc_ctas;
};

struct Params {
  const void* q;
  int64_t q_st, q_sh;
  const uint8_t* v;  // the V cache itself, for mark_nan, and its strides
  int64_t v_page, v_tok, v_head;
  int64_t num_pages;
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
  int32_t batch, total_q, num_heads, num_kv_heads, group, page, window;
  Divisor by_group, by_page, by_kv_heads, by_heads;
  float scale_log2, v_scale;
  void* out;
  int64_t o_st, o_sh;
  unsigned int* err;
  // workspace
  RowPlan* plan;       // [total_q]: where the merge finds a token's partials
  float* o_part;       // [piece][rows][D]
  float2* ml_part;     // [piece][rows]: maximum (log2 units), sum
  int32_t max_pieces;
  int32_t prefix_tc;   // prefixes are taken by tc::prefix_kernel, not by pieces_kernel
  int32_t tc_ctas;     // CTAs of prefix_kernel
  float* tc_o;         // [unit + CTA][256 rows][D]
  float2* tc_ml;       // [unit + CTA][256 rows]
  int64_t tc_rows;     // rows of the two
  unsigned int* tc_lost;  // [CTA of prefix_kernel]: a wait ran out, its partials are not valid
};

// ---- metadata (lengths are cut to what the tables reach, row ranges to the rows there are) ----
__device__ __forceinline__ int q_begin(const Params& P, int b) {
  return P.cu_q ? max(0, min(__ldg(P.cu_q + b), P.total_q)) : b;
}
__device__ __forceinline__ int own_len(const Params& P, int b) {
  return max(0, min(__ldg(P.ctx + b), P.max_pages * P.page));
}
__device__ __forceinline__ int prefix_len(const Params& P, int g) {
  return max(0, min(__ldg(P.prefix_lens + g), P.max_prefix_pages * P.page));
}
__device__ __forceinline__ int group_begin(const Params& P, int g) {  // first sequence
  return P.cu_groups ? max(0, min(__ldg(P.cu_groups + g), P.batch)) : g * P.batch;
}

// The interval [cu[i], cu[i + 1]) of the ascending list cu[0..n] that holds x (-1: before the first;
// n: past the last).
__device__ __forceinline__ int interval_of(const int32_t* cu, int n, int x) {
  int lo = 0, hi = n + 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= x) lo = mid + 1; else hi = mid;
  }
  return lo - 1;
}
__device__ __forceinline__ int sequence_of(const Params& P, int n) {  // row n's, or -1
  if (!P.cu_q) return n < P.batch ? n : -1;
  const int b = interval_of(P.cu_q, P.batch, n);
  return b < P.batch ? b : -1;
}

// A segment: rows [tok0, tok0 + tokens) x group heads over keys [k0, len) of a page list.
struct Segment {
  int tok0, tokens, k0, len;
  __device__ __forceinline__ int tiles() const { return len > k0 ? (len - k0 + TILE - 1) / TILE : 0; }
};
__device__ __forceinline__ Segment prefix_segment(const Params& P, int g) {
  Segment s;
  const int b0 = group_begin(P, g), b1 = max(b0, group_begin(P, g + 1));
  s.tok0 = q_begin(P, b0);
  s.tokens = max(0, q_begin(P, b1) - s.tok0);
  s.len = prefix_len(P, g);
  // with a window: no row of the group stands before len - tokens, so none sees keys before this
  s.k0 = P.window > 0 ? (max(0, s.len - s.tokens - P.window + 1) & ~(TILE - 1)) : 0;
  if (s.tokens == 0) s.len = s.k0 = 0;
  return s;
}
__device__ __forceinline__ Segment own_segment(const Params& P, int b) {
  Segment s;
  s.tok0 = q_begin(P, b);
  s.tokens = max(0, q_begin(P, b + 1) - s.tok0);
  s.len = own_len(P, b);
  s.k0 = P.window > 0 ? (max(0, s.len - s.tokens - P.window + 1) & ~(TILE - 1)) : 0;
  if (s.tokens == 0) s.len = s.k0 = 0;
  return s;
}

// Blocks of keys and units (blocks of 256 rows, KV heads) of a prefix in prefix_kernel.
constexpr int TC_KEYS = 128, TC_ROWS_LOG2 = 8;
__device__ __forceinline__ int tc_blocks(const Segment& x) {
  return x.len > x.k0 ? (x.len - x.k0 + TC_KEYS - 1) / TC_KEYS : 0;
}
__device__ __forceinline__ int64_t tc_units(const Segment& x, const Params& P) {
  return (((int64_t)x.tokens * P.group + (1 << TC_ROWS_LOG2) - 1) >> TC_ROWS_LOG2) * P.num_kv_heads;
}

// CTAs that share `total` blocks.  All SMs from three blocks an SM on; fewer blocks go to half of them, so that
// pieces_kernel, which cannot share an SM with prefix_kernel, runs beside it on the others: 192 rows x 8 heads
// behind 2,048 keys 35.2 -> 25.8 us, behind 4,096 38.4 -> 29.9; with 512 blocks (8,192 keys) there is nothing
// to win (32.7 on all SMs, 32.1 on 64).
__device__ __forceinline__ int64_t tc_ctas_of(int64_t total, int sms) {
  if (total > 2 * sms) return sms;
  const int half = max(1, sms / 2), each = max(1, ((int)total + half - 1) / half);
  return ((int)total + each - 1) / each;
}

// ---- NaN among the values ----------------------------------------------------------------------------
// A weight of 0 does not take a NaN out of P.V, so a NaN value would reach the rows that do not see its key
// (a later draft's token, a key that has left the window).  Where rows see different keys, NaN values are
// taken as 0 in shared memory, and the dimensions in which each row does see one are looked up in the cache
// and marked over the stored sums.  prefix_kernel looks for them in every block of such a piece (a warp of
// its own marks them); pieces_kernel, whose tiles are short, finds them in a piece's sums and runs the piece
// once more.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {  // e4m3 NaN: 0x80 in the byte
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t without_nan(uint32_t w) { return w & ~((nan_bytes(w) >> 7) * 0xFFu); }
// Thread `who` of `whos`: its share of the 16-byte chunks of a tile without NaN; whether there were any.
__device__ __forceinline__ bool clean(uint8_t* tile, int chunks, int who, int whos) {
  bool any = false;
#pragma unroll 1
  for (int i = who; i < chunks; i += whos) {
    const uint4 e = *reinterpret_cast<const uint4*>(tile + 16 * i);
    if (!(nan_bytes(e.x) | nan_bytes(e.y) | nan_bytes(e.z) | nan_bytes(e.w))) continue;
    any = true;
    *reinterpret_cast<uint4*>(tile + 16 * i) =
        make_uint4(without_nan(e.x), without_nan(e.y), without_nan(e.z), without_nan(e.w));
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the slot is loaded again
  }
  __syncwarp();
  return any;
}
// Warp-wide: NaN over the dimensions [d0, d0 + dims) of each lane's sums `o` in which one of the keys [lo, hi)
// that it sees has a NaN value; keys [from, to) of the page list are looked at.
__device__ __forceinline__ void mark_nan(const Params& P, const int32_t* table, int kvh, int from, int to, int lo, int hi,
                                         float* o, int d0, int dims) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int k0 = from; k0 < to; k0 += 32) {
    int blk = -1, row = 0;  // of this lane's key
    if (k0 + lane < to) {
      const int at = P.by_page.div(k0 + lane);
      row = k0 + lane - at * P.page;
      blk = __ldg(table + at);
    }
    const bool there = blk >= 0 && blk < P.num_pages;
    const uint32_t* x = reinterpret_cast<const uint32_t*>(
        P.v + (there ? blk * P.v_page + row * P.v_tok + kvh * P.v_head : 0));
    uint32_t any = 0;  // a first look, all of the key's loads in flight together: most keys have none
    if (there) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint4 e = reinterpret_cast<const uint4*>(x)[i];
        any |= nan_bytes(e.x) | nan_bytes(e.y) | nan_bytes(e.z) | nan_bytes(e.w);
      }
    }
    if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll 1
    for (int w = 0; w < D / 4; ++w) {
      const uint32_t bad = any ? nan_bytes(x[w]) : 0u;
#pragma unroll 1
      for (uint32_t who = __ballot_sync(0xffffffffu, bad != 0); who; who &= who - 1) {
        const int key = k0 + __ffs(who) - 1;
        const uint32_t b = __shfl_sync(0xffffffffu, bad, __ffs(who) - 1);
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
          if (((b >> (8 * i + 7)) & 1u) && key >= lo && key < hi && 4 * w + i >= d0 && 4 * w + i < d0 + dims)
            o[4 * w + i] = __int_as_float(0x7fc00000);
      }
    }
  }
}

// ---- pieces of few rows: one warp each, warp-level MMA --------------------------------------------
// Bound: HBM by its bytes, latency by measurement.  8 x 8 samples of prompts of 869 to 3,454 keys, 16 KV
// heads, window 1,024 (108 MB): 38 us, 2.8 TB/s = 0.43 of a measured copy; every further tile then costs its
// bytes at 0.96 of that rate, but about 5 us pass before the first load (lengths, plan, page look-up: some
// 1,500 instructions that run once, so fetching them is what takes the time) and 1 to 2 at either end of a
// piece.  A warp takes one piece (segment, block
// of 8 * NB rows, split, KV head) at a time, KV head fastest, so that neighbouring warps read the heads
// of the same pages together.  It streams the piece's 16-key tiles through its own ring of RING slots
// (TMA, 128-byte swizzle, one mbarrier a slot) and takes two tiles a step, so the steps' serial parts
// (waits, maxima, the way of P through shared memory) are paid once for 32 keys:
//   S^T = K . Q^T  mma.m16n8k16 (keys on M, rows on N), K widened to fp16 (exact) once for all rows, the
//     scaled queries as fp16: exact down to 2^-25 of the row's maximum (bf16; fp16 2^-22), to 2^-32 of it
//     below.  The head dimension is permuted so that lane (g, c) needs bytes [32c, 32c + 32) of keys g and
//     g + 8, Q likewise.  (The warp-level e4m3 product is no way round the widening: it runs as
//     conversions of both operands and two fp16 products, and queries need two or three e4m3 terms.)
//   O^T += V^T . P^T  mma.m16n8k16 with V widened to fp16 (exact) and P rounded to fp16, 2^-11 of a weight
//     (bf16 would leave 2^-8); the row sums add the unrounded weights in fp32.  The output dimension is
//     permuted so that the lane needs bytes [16g, 16g + 16) of keys 2c, 2c + 1, 2c + 8, 2c + 9.
// All shared-memory reads are 16 bytes a lane, conflict-free through the swizzle.  Statistics fp32; the
// sums are rescaled only when a row's maximum moved.
// A row of queries is scaled by a power of two to a maximum in [128, 256).  From the packed 16-bit maxima
// of |q| over its even and odd elements: the scale, and its inverse (NaN for a row with infinities or NaN).
template <typename TQ> __device__ __forceinline__ void term_scale(uint32_t top, float& up, float& down) {
  const uint16_t top16 = (uint16_t)max(top & 0xFFFFu, top >> 16);
  const uint32_t most = __float_as_uint(to_f32(*reinterpret_cast<const TQ*>(&top16)));
  const int sh = most ? min(134 - (int)(most >> 23), 126) : 0;  // tiny rows stop at 2^126
  up = __uint_as_float((uint32_t)(sh + 127) << 23);
  down = most < 0x7F800000u ? __uint_as_float((uint32_t)(127 - sh) << 23) : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ uint32_t top_of(uint32_t top, const uint4& u) {
  top = __vmaxu2(top, u.x & 0x7FFF7FFFu);
  top = __vmaxu2(top, u.y & 0x7FFF7FFFu);
  top = __vmaxu2(top, u.z & 0x7FFF7FFFu);
  return __vmaxu2(top, u.w & 0x7FFF7FFFu);
}
constexpr int RING = 4;
constexpr int WARPS = 4;
constexpr int MIN_TILES = 4;  // of a split: below, a piece's fixed cost outweighs its keys
constexpr int RING_BYTES = RING * 2 * TILE_BYTES;

__device__ __forceinline__ uint4 tile_ld16(const uint8_t* tile, int row, int chunk) {
  return *reinterpret_cast<const uint4*>(tile + row * 128 + ((chunk ^ (row & 7)) << 4));
}

// Tiles of a split: the fewest (>= MIN_TILES) with which the pieces do not exceed max_pieces, which is
// one piece for every warp of the grid, or twice the (segment, row block, head) units where those are
// more.  work[s] = (tiles, row blocks * heads).  Each lane tries a length, from the bound that the tiles
// alone give upwards; lengths past those (or of more segments than are worth trying) come from
// pieces <= tiles / length + units.  CTA-wide: each warp counts a share of the segments.
__device__ __forceinline__ int ceil_div_small(int a, float inverse) {  // a < 2^21: the half keeps it off the edges
  return (int)(((float)a - 0.5f) * inverse) + (a > 0);
}
__device__ __forceinline__ int split_tiles(const int2* work, int segs, int max_pieces, int (*counted)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float about = 0.f;  // the tiles of all pieces' rows: where the lengths tried begin
  int most = 0;
  for (int s = lane; s < segs; s += 32) {
    about += (float)work[s].x * (float)work[s].y;
    most = max(most, work[s].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) about += __shfl_xor_sync(0xffffffffu, about, o);
  most = __reduce_max_sync(0xffffffffu, most);
  const int least = (int)fminf(__fdividef(about, (float)max_pieces) + 1.f, (float)most);
  const int ct = max(MIN_TILES, least) + lane;
  bool fits = false;
  if (segs <= 256 && most < (1 << 21)) {  // the same in every warp
    const float inverse = 1.f / (float)ct;
    int n = 0;
#pragma unroll 4
    for (int s = warp; s < segs; s += WARPS) n += ceil_div_small(work[s].x, inverse) * work[s].y;
    counted[warp][lane] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) n += counted[w][lane];
    fits = n <= max_pieces && n >= 0;
  }
  const unsigned who = __ballot_sync(0xffffffffu, fits);
  if (who) return __shfl_sync(0xffffffffu, ct, __ffs(who) - 1);
  int64_t all = 0;
  int units = 0;
  for (int s = lane; s < segs; s += 32) {
    all += (int64_t)work[s].x * work[s].y;
    units += work[s].x ? work[s].y : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  units = __reduce_add_sync(0xffffffffu, units);
  return (int)min(max((int64_t)MIN_TILES, all / max(1, max_pieces - units) + 1), (int64_t)1 << 27);
}

// Pieces of a lane's segments.  Lists that overlap can name any number: the count stops at 2^26 - 1 (a
// workspace of as many pieces would be 256 GB), so that 32 lanes' sum stays in 32 bits and still ascends.
__device__ __forceinline__ int more_pieces(int before, int2 splits_units) {
  return (int)min(before + (int64_t)splits_units.x * splits_units.y, (int64_t)(1 << 26) - 1);
}

template <typename TQ, int NB>
__global__ void __launch_bounds__(WARPS * 32, NB == 1 ? 3 : 2)
    pieces_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, Params P) {
  using namespace sm100;
  constexpr int ROWS = 8 * NB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = base + warp * RING_BYTES;
  const int segs = P.num_groups + P.batch;
  Segment* seg = reinterpret_cast<Segment*>(base + WARPS * RING_BYTES);
  int2* work = reinterpret_cast<int2*>(seg + segs);  // tiles (0: not this kernel's), then splits; blocks * heads
  int* first = reinterpret_cast<int*>(work + segs);  // pieces before each segment, by heads
  int* begins = first + segs + 1;                    // first sequence of each group, and the end
  __shared__ uint64_t bars[WARPS][RING];
  __shared__ __align__(16) __half p_s[WARPS][NB][8][40];  // 32 keys a row; padded against bank conflicts
  __shared__ int abort_flag, s_cut, counted[WARPS][32];
  uint64_t* bar = bars[warp];
  if (threadIdx.x == 0) {
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
    abort_flag = 0;
    s_cut = P.window > 0;
  }
  if (lane < RING) mbar_init(&bar[lane], 1);
  fence_mbar_init();
  __syncthreads();
  // Behind prefix_kernel, which has waited for its predecessors before it let this kernel start, all
  // inputs are settled and nothing of prefix_kernel's is read: its end is waited for at the end.
  if (!P.prefix_tc) pdl_wait();
  pdl_trigger();

  // ---- the plan, the same in every CTA
  const int skip = P.prefix_tc ? P.num_groups : 0;  // segments that are not this kernel's
  for (int s = threadIdx.x; s < segs; s += WARPS * 32) {
    const Segment x = s < P.num_groups ? prefix_segment(P, s) : own_segment(P, s - P.num_groups);
    seg[s] = x;
    work[s] = make_int2(s >= skip ? x.tiles() : 0, (x.tokens * P.group + ROWS - 1) / ROWS * P.num_kv_heads);
    if (s >= P.num_groups && x.len < x.tokens) s_cut = 1;  // rows inside the prefix: it needs a mask too
  }
  for (int i = threadIdx.x; i <= P.num_groups; i += WARPS * 32) begins[i] = group_begin(P, i);
  __syncthreads();
  const int ct = split_tiles(work + skip, segs - skip, P.max_pieces, counted);
  __syncthreads();  // every warp has counted: splits take the tiles' place
  if (warp == 0) {  // each lane a run of segments: their splits in place of their tiles, the pieces before them
    const int run = (segs + 31) / 32, from = min(segs, lane * run), to = min(segs, from + run);
    const float inverse = 1.f / (float)ct;
    int mine = 0;
    for (int s = from; s < to; ++s) {
      const int tiles = work[s].x;
      work[s].x = tiles < (1 << 21) ? ceil_div_small(tiles, inverse) : (tiles + ct - 1) / ct;
      mine = more_pieces(mine, work[s]);
    }
    int acc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, acc, o);
      if (lane >= o) acc += up;
    }
    const int before = acc - mine;
    mine = 0;
    for (int s = from; s < to; ++s) {
      first[s] = before + mine;
      mine = more_pieces(mine, work[s]);
    }
    if (lane == 31) first[segs] = acc;
  }
  __syncthreads();
  const bool cut = s_cut != 0;
  // ---- for the merge: CTA i writes the tokens of sequences i, i + CTAs, ...
  for (int b = blockIdx.x; b < P.batch; b += gridDim.x) {
    const Segment x = seg[P.num_groups + b];
    if (x.tokens == 0) continue;
    int g = -1;  // the last group that begins at or before b, unless b is behind them all
    for (int i = 0; i <= P.num_groups; i += 32)
      g += __popc(__ballot_sync(0xffffffffu, i + lane <= P.num_groups && begins[i + lane] <= b));
    if (g == P.num_groups) g = -1;
    RowPlan r;
    r.own_first = first[P.num_groups + b];
    r.own_splits = work[P.num_groups + b].x;
    r.pre_first = r.pre_splits = r.blocks = r.pad = 0;
    r.tc_from = r.tc_units = r.tc_total = r.tc_ctas = 0;
    int tok0_g = 0;
    if (g >= 0) {
      tok0_g = seg[g].tok0;
      if (!P.prefix_tc) {
        r.pre_first = first[g];
        r.pre_splits = work[g].x;
      } else {  // prefix_kernel's units and blocks, as its Walk lays them out
        for (int i = 0; i < P.num_groups; ++i) {
          const int blocks = tc_blocks(seg[i]);
          const int64_t units = blocks ? tc_units(seg[i], P) : 0;
          if (i == g) {
            r.tc_from = r.tc_total;
            r.tc_units = r.tc_ctas;
            r.blocks = blocks;
          }
          r.tc_total += units * blocks;
          r.tc_ctas += units;
        }
        r.tc_ctas = tc_ctas_of(r.tc_total, P.tc_ctas);
      }
    }
    for (int i = threadIdx.x; i < x.tokens; i += WARPS * 32) {
      r.own_row = i * P.group;
      r.pre_row = (x.tok0 + i - tok0_g) * P.group;
      P.plan[x.tok0 + i] = r;
    }
  }
  if (blockIdx.x == gridDim.x - 1) {  // rows of no sequence
    const int from = q_begin(P, 0), to = P.cu_q ? q_begin(P, P.batch) : P.batch;
    const RowPlan none{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    for (int n = threadIdx.x; n < P.total_q; n += WARPS * 32)
      if (n < from || n >= to) P.plan[n] = none;
  }
  const int pieces = min(first[segs], P.max_pieces);  // (lists that overlap could name more than the workspace holds)
  uint32_t uses = 0;  // tiles through the ring (slot = uses % RING, parity = (uses / RING) & 1)
  bool careful = false;  // this piece's NaN values are to be taken as 0
  for (int piece = blockIdx.x * WARPS + warp; piece < pieces; piece += gridDim.x * WARPS) {
    int s = 0;  // the last segment with first[s] <= piece (it is not empty), 32 probes at a time
    for (int step = segs <= 32 ? 1 : (segs <= 1024 ? 32 : 1024);; step >>= 5) {
      const int at = s + lane * step;
      s += (__popc(__ballot_sync(0xffffffffu, at < segs && first[at] <= piece)) - 1) * step;
      if (step == 1) break;
    }
    const bool pre = s < P.num_groups;
    const Segment x = seg[s];
    const int splits = work[s].x, off = piece - first[s];
    int kvh;
    const int flat = P.by_kv_heads.divmod(off, kvh);
    const int rb = flat / splits, sp = flat - rb * splits;
    const int t_begin = x.k0 + sp * ct * TILE, t_end = min(x.len, t_begin + ct * TILE);
    const int nt = (t_end - t_begin + TILE - 1) / TILE;
    const int32_t* table = pre ? P.pt + (int64_t)s * P.pt_stride : P.bt + (int64_t)(s - P.num_groups) * P.bt_stride;

    int my_block = -1, my_row0 = 0;  // lane j: page of tile j (mod 32), refilled every 32 tiles
    auto look_up = [&](int from) {
      my_block = -1;
      if (from + lane < nt) {
        const int key = t_begin + TILE * (from + lane);
        const int at = P.by_page.div(key);
        my_row0 = key - at * P.page;
        my_block = __ldg(table + at);
        if (my_block >= P.num_pages) my_block = -1;
      }
    };
    auto issue = [&](int k, int blk, int row0) {
      if (lane == 0) {
        const uint32_t use = uses + k;
        const int slot = use % RING;
        if (blk >= 0) {
          mbar_arrive_expect_tx(&bar[slot], 2 * TILE_BYTES);
          tma_load_4d(ring + slot * 2 * TILE_BYTES, &tmk, &bar[slot], 0, kvh, row0, blk);
          tma_load_4d(ring + slot * 2 * TILE_BYTES + TILE_BYTES, &tmv, &bar[slot], 0, kvh, row0, blk);
        } else {
          mbar_arrive_plain(&bar[slot]);  // a hole: nothing to load
        }
      }
    };
    look_up(0);
    const int rows = x.tokens * P.group;
    uint4 raw[NB][4];  // queries of row g of each block of 8, d in [32c, 32c + 32)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = rb * ROWS + nb * 8 + g;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[nb][i] = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        int head;
        const int tok = P.by_group.divmod(r, head);
        const uint4* qp = reinterpret_cast<const uint4*>(
            reinterpret_cast<const TQ*>(P.q) + (int64_t)(x.tok0 + tok) * P.q_st +
            (int64_t)(kvh * P.group + head) * P.q_sh + 32 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[nb][i] = qp[i];
      }
    }
    uint32_t ok_mask = __ballot_sync(0xffffffffu, my_block >= 0);  // of the 32 tiles looked up last
    int looked = 0;
    for (int k = 0; k < RING && k < nt; ++k)
      issue(k, __shfl_sync(0xffffffffu, my_block, k), __shfl_sync(0xffffffffu, my_row0, k));

    // ---- the rows: queries as the B operand (lane: row g of each block of 8, d in [32c, 32c + 32)), and
    // for the rows 2c, 2c + 1 that this lane's scores belong to their scale and key range [lo, hi)
    uint32_t qf[NB][16];
    float cs[NB][2];
    int lo[NB][2], hi[NB][2], lo_max = 0, hi_min = 0x7fffffff;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = top_of(top, raw[nb][i]);
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float up, down;
      term_scale<TQ>(top, up, down);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[8];
        unpack8<TQ>(raw[nb][i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= up;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __half2 h = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
          qf[nb][4 * i + e] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      cs[nb][0] = P.scale_log2 * __shfl_sync(0xffffffffu, down, 8 * c);
      cs[nb][1] = P.scale_log2 * __shfl_sync(0xffffffffu, down, 8 * c + 4);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int re = rb * ROWS + nb * 8 + 2 * c + e;
        int from = 0, to = x.len;
        if (re < rows && (!pre || cut)) {
          const int n = x.tok0 + P.by_group.div(re);
          int pos;  // of the row, in this segment's key coordinates
          if (pre) {  // the last sequence that begins at or before row n (empty ones begin there too)
            int bl = 0, bh = P.batch;
            while (bh - bl > 1) {
              const int mid = (bl + bh) >> 1;
              if (seg[P.num_groups + mid].tok0 <= n) bl = mid; else bh = mid;
            }
            const Segment own = seg[P.num_groups + bl];
            pos = x.len + own.len - (own.tok0 + own.tokens - n);
          } else {
            pos = x.len - (x.tok0 + x.tokens - n);
          }
          to = min(to, pos + 1);
          if (P.window > 0) from = max(0, pos - P.window + 1);
        }
        lo[nb][e] = from;
        hi[nb][e] = to;
        lo_max = max(lo_max, from);
        hi_min = min(hi_min, to);
      }
    }
    lo_max = __reduce_max_sync(0xffffffffu, lo_max);
    hi_min = __reduce_min_sync(0xffffffffu, hi_min);

    float acc[NB][8][4], m[NB][2], l[NB][2];  // O^T fragments: d = 16g + 2mt (+1), rows 2c / 2c + 1
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[nb][i][0] = acc[nb][i][1] = acc[nb][i][2] = acc[nb][i][3] = 0.f;
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.f;
    }
    bool failed = false;
    int k = 0;
    for (; k < nt; k += 2) {
      const bool two = k + 1 < nt;
      bool came = true;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (u == 0 || two)
          came &= mbar_wait_bounded(&bar[(uses + k + u) % RING], ((uses + k + u) / RING) & 1, &abort_flag, P.err,
                                    ERR_TILE_WAIT);
      if (!__all_sync(0xffffffffu, came)) {
        failed = true;
        break;
      }
      if (__builtin_expect(careful, 0))
        for (int u = 0; u < (two ? 2 : 1); ++u)
          clean(ring + ((uses + k + u) % RING) * 2 * TILE_BYTES + TILE_BYTES, TILE_BYTES / 16, lane, 32);
      const int tt = t_begin + TILE * k;
      const uint32_t ok2 = (ok_mask >> (k & 31)) & (two ? 3u : 1u);  // which of the two tiles are there
      float sc[NB][2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sc[nb][u][0] = sc[nb][u][1] = sc[nb][u][2] = sc[nb][u][3] = 0.f;
        if (u == 1 && !two) break;
        const uint8_t* kt = ring + ((uses + k + u) % RING) * 2 * TILE_BYTES;
        uint4 kk[4];
        kk[0] = tile_ld16(kt, g, 2 * c);
        kk[1] = tile_ld16(kt, g, 2 * c + 1);
        kk[2] = tile_ld16(kt, g + 8, 2 * c);
        kk[3] = tile_ld16(kt, g + 8, 2 * c + 1);
        const uint32_t* kg = reinterpret_cast<const uint32_t*>(kk);
        const uint32_t* kg8 = reinterpret_cast<const uint32_t*>(kk + 2);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t a[4];
          a[0] = e4m3x2_to_f16x2((uint16_t)(kg[ks] & 0xFFFFu));
          a[1] = e4m3x2_to_f16x2((uint16_t)(kg8[ks] & 0xFFFFu));
          a[2] = e4m3x2_to_f16x2((uint16_t)(kg[ks] >> 16));
          a[3] = e4m3x2_to_f16x2((uint16_t)(kg8[ks] >> 16));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_16816_f16(sc[nb][u], a, qf[nb] + 2 * ks);
        }
      }
      const bool whole = ok2 == 3u && tt >= lo_max && tt + 2 * TILE <= hi_min;  // warp-uniform
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float v[2][4];  // [row 2c, 2c + 1][keys g, g + 8 of both tiles]
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          v[0][2 * u] = sc[nb][u][0] * cs[nb][0];
          v[1][2 * u] = sc[nb][u][1] * cs[nb][1];
          v[0][2 * u + 1] = sc[nb][u][2] * cs[nb][0];
          v[1][2 * u + 1] = sc[nb][u][3] * cs[nb][1];
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = tt + g + 8 * i;
            const bool there = (ok2 >> (i >> 1)) & 1u;
#pragma unroll
            for (int e = 0; e < 2; ++e) v[e][i] = there && key >= lo[nb][e] && key < hi[nb][e] ? v[e][i] : -INFINITY;
          }
        }
        float x0 = fmaxf(fmaxf(v[0][0], v[0][1]), fmaxf(v[0][2], v[0][3]));
        float x1 = fmaxf(fmaxf(v[1][0], v[1][1]), fmaxf(v[1][2], v[1][3]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
          x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
        }
        x0 = fmaxf(m[nb][0], x0);
        x1 = fmaxf(m[nb][1], x1);
        // nothing visible so far: against 0, so that no weight is NaN
        const float z0 = x0 == -INFINITY ? 0.f : x0, z1 = x1 == -INFINITY ? 0.f : x1;
        if (__any_sync(0xffffffffu, x0 != m[nb][0] || x1 != m[nb][1])) {
          const float al0 = fast_exp2(m[nb][0] - z0), al1 = fast_exp2(m[nb][1] - z1);
          m[nb][0] = x0;
          m[nb][1] = x1;
          l[nb][0] *= al0;
          l[nb][1] *= al1;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            acc[nb][mt][0] *= al0;
            acc[nb][mt][1] *= al1;
            acc[nb][mt][2] *= al0;
            acc[nb][mt][3] *= al1;
          }
        }
        __half(*ps)[40] = p_s[warp][nb];  // P through shared memory: the B operand wants (key pairs, row g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = fast_exp2(v[0][i] - z0), p1 = fast_exp2(v[1][i] - z1);
          l[nb][0] += p0;
          l[nb][1] += p1;
          ps[2 * c][g + 8 * i] = __float2half_rn(p0);
          ps[2 * c + 1][g + 8 * i] = __float2half_rn(p1);
        }
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (u == 1 && !two) break;
        const uint8_t* vt = ring + ((uses + k + u) % RING) * 2 * TILE_BYTES + TILE_BYTES;
        uint4 vv[4];
        const int keys[4] = {2 * c, 2 * c + 1, 2 * c + 8, 2 * c + 9};
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // rows of a hole or past the end may hold NaN: their weight is 0, V must be finite
          vv[i] = tile_ld16(vt, keys[i], g);
          if (!whole && !(((ok2 >> u) & 1u) && tt + TILE * u + keys[i] < x.len)) vv[i] = make_uint4(0, 0, 0, 0);
        }
        uint32_t bp[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          bp[nb][0] = *reinterpret_cast<const uint32_t*>(&p_s[warp][nb][g][TILE * u + 2 * c]);
          bp[nb][1] = *reinterpret_cast<const uint32_t*>(&p_s[warp][nb][g][TILE * u + 2 * c + 8]);
        }
        const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vv[0]);
        const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vv[1]);
        const uint32_t* v8 = reinterpret_cast<const uint32_t*>(&vv[2]);
        const uint32_t* v9 = reinterpret_cast<const uint32_t*>(&vv[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362u : 0x5140u;
            const uint32_t lo01 = prmt(v0[i], v1[i], sel);
            const uint32_t lo89 = prmt(v8[i], v9[i], sel);
            uint32_t a[4];
            a[0] = e4m3x2_to_f16x2((uint16_t)(lo01 & 0xFFFFu));
            a[1] = e4m3x2_to_f16x2((uint16_t)(lo01 >> 16));
            a[2] = e4m3x2_to_f16x2((uint16_t)(lo89 & 0xFFFFu));
            a[3] = e4m3x2_to_f16x2((uint16_t)(lo89 >> 16));
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma_16816_f16(acc[nb][2 * i + half], a, bp[nb]);
          }
        }
      }
      // every lane is done with the slots and with P: refill the slots with tiles k + RING, k + RING + 1
      __syncwarp();
      if (k + RING < nt) {
        const int nx = k + RING;
        if ((nx & 31) == 0) {
          look_up(nx);
          looked = nx;
        }
        if (lane == 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int blk = __shfl_sync(0xffffffffu, my_block, (nx + u) & 31);
          const int row0 = __shfl_sync(0xffffffffu, my_row0, (nx + u) & 31);
          if (nx + u < nt) issue(nx + u, blk, row0);
        }
      }
      // the mask of the next step's block of 32 (its look-up is RING tiles old by then)
      if (((k + 2) & 31) == 0 && looked == k + 2) ok_mask = __ballot_sync(0xffffffffu, my_block >= 0);
    }
    if (__builtin_expect((t_begin < lo_max || hi_min < t_end) && !careful && !failed, 0)) {
      float sum = 0.f;  // a key that some row does not see: a NaN may be another row's
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) sum += (acc[nb][mt][0] + acc[nb][mt][1]) + (acc[nb][mt][2] + acc[nb][mt][3]);
      if (__any_sync(0xffffffffu, sum != sum)) {  // the piece once more, without NaN values
        careful = true;
        uses += nt;
        piece -= gridDim.x * WARPS;
        continue;
      }
    }
    const float poison = failed ? __int_as_float(0x7fc00000) : 0.f;  // a tile never came: the result is not valid
    if (failed && lane == 0) {  // leave no copy in flight: wait (bounded) for the tiles asked for and not taken
      const uint64_t t0 = globaltimer();
      for (int i = k; i < nt && i < k + RING; ++i)
        while (!mbar_try_wait(&bar[(uses + i) % RING], ((uses + i) / RING) & 1) && globaltimer() - t0 < 1000000000ull) {
        }
    }
    uses += nt;

    float2* ml = P.ml_part + (int64_t)piece * ROWS;
    float* op = P.o_part + (int64_t)piece * ROWS * D;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float l0 = l[nb][0], l1 = l[nb][1];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, o);
        l1 += __shfl_xor_sync(0xffffffffu, l1, o);
      }
      const int r0 = nb * 8 + 2 * c;
      if (rb * ROWS + r0 < rows) {
        if (g == 0) ml[r0] = make_float2(m[nb][0] + poison, l0 + poison);
        if (m[nb][0] != -INFINITY)
#pragma unroll
          for (int mt = 0; mt < 8; ++mt)
            *reinterpret_cast<float2*>(op + r0 * D + 16 * g + 2 * mt) = make_float2(acc[nb][mt][0], acc[nb][mt][2]);
      }
      if (rb * ROWS + r0 + 1 < rows) {
        if (g == 0) ml[r0 + 1] = make_float2(m[nb][1] + poison, l1 + poison);
        if (m[nb][1] != -INFINITY)
#pragma unroll
          for (int mt = 0; mt < 8; ++mt)
            *reinterpret_cast<float2*>(op + (r0 + 1) * D + 16 * g + 2 * mt) =
                make_float2(acc[nb][mt][1], acc[nb][mt][3]);
      }
    }
    if (__builtin_expect(careful, 0)) {  // over the sums that this lane has just stored
#pragma unroll 1
      for (int r = 0; r < 2 * NB; ++r) {
        const int row = (r >> 1) * 8 + 2 * c + (r & 1);
        const int from = NB == 2 && r > 1 ? (r & 1 ? lo[NB - 1][1] : lo[NB - 1][0]) : (r & 1 ? lo[0][1] : lo[0][0]);
        const int to = NB == 2 && r > 1 ? (r & 1 ? hi[NB - 1][1] : hi[NB - 1][0]) : (r & 1 ? hi[0][1] : hi[0][0]);
        mark_nan(P, table, kvh, t_begin, t_end, from, rb * ROWS + row < rows ? to : 0, op + row * D, 16 * g, 16);
      }
      careful = false;
    }
    if (failed) {  // nor is anything that this warp has left to do
      for (piece += gridDim.x * WARPS; piece < pieces; piece += gridDim.x * WARPS)
        if (lane < ROWS) P.ml_part[(int64_t)piece * ROWS + lane] = make_float2(poison, poison);
      break;
    }
  }
  if (P.prefix_tc) pdl_wait();  // so that the merge, which waits for this kernel, finds both done
}

// ---- prefixes under many rows: tcgen05 ---------------------------------------------------------------
// Bound: the tensor cores, 4 * 128 flops for every (row, key).  1,024 rows x 8 KV heads x 32,768 keys (137 GFLOP):
// 142 us, 0.97 PFLOP/s = 0.59 of a measured bf16 product's rate; a block of 128 keys takes 3,550 cycles where its
// MMAs take 2,048 and its exponentials as many: a tile's scores, maxima, weights and products follow one another,
// and TMEM (O and S of both tiles fill it) has no room for a second S.  A unit is 256 rows (two 128-row
// tiles, the TMEM lanes) of one prefix and KV head over blocks of 128 keys; the blocks of all units are
// laid end to end and every CTA takes an equal range, so a range covers the end of one unit, whole
// ones and the start of another, each giving one partial (piece = unit + CTA index: one of the two
// moves on from each piece to the next).
//   S_t = Q_t . K^T  kind::f8f6f4 on the e4m3 bytes as they lie in the cache, the queries as sums of e4m3
//     terms (see Terms): K is never widened and the terms cost what the fp16 product would.
//   P  = 2^(S c - m) in fp16 (2^-11 of a weight; the sums add them unrounded), over S in TMEM, the A operand of
//   O_t += P_t . V  kind::f16; V is widened to fp16 (exact) by four warps, once for both tiles.
// Roles (16 warps): 0-3 widen V; 4-7 and 8-11 take tile 0's and tile 1's rows (thread = row: queries to
// terms, softmax, O to the workspace); 12 loads (TMA, eight 16-key tiles a block for K and V each);
// 13 issues the MMAs; 14 walks the CTA's range and hands out its pieces; 15 marks NaN values.  The row
// warps take 192 registers a thread (a row of S at once), the others 64.  P.V of a block and S of the next
// are issued together for a tile, so one tile's MMAs run under the other tile's softmax.  All tcgen05
// operations come from one thread in order, so s_full of block j + 1 also says that P.V of block j is
// complete: O may be rescaled.
// Barriers, phase = use: d_full/d_empty (pieces), k_full/k_empty (K slots), e_full/e_empty (e4m3 V
// slots), v_full/v_empty (fp16 V slots), s_full[t], p_full[t][half] (a block's S, P of tile t), q_full[t],
// o_full[t] (a piece's Q, O), stored (a cut piece's partial; the rows are at most two pieces ahead of the
// warp that waits for it).  A tile's next S and its next P.V wait for q_full and p_full, which its warps
// give after they have written the piece before.  Every wait is bounded and ends all roles through the
// abort flag.
namespace tc {
constexpr int BM = 128, BN = 128, TILES = 2, ROWS = TILES * BM;
static_assert(BN == TC_KEYS && ROWS == 1 << TC_ROWS_LOG2, "shape of a unit");
constexpr int THREADS = 16 * 32;
constexpr int NE = 2, NV = 2, ND = 2, NS = 4;
constexpr int REGS_LAUNCH = 128, REGS_ROWS = 192, REGS_REST = 64;  // a thread: 4 * 128 = 2 * 192 + 2 * 64
static_assert(2 * REGS_ROWS + 2 * REGS_REST <= 4 * REGS_LAUNCH, "registers of the block");
// Queries as sums of e4m3 terms.  Of a row scaled to a maximum in [128, 256) a
// term keeps 4 significant bits and what it leaves is exact, so two terms hold every bf16 value down to 2^-10
// of the row's maximum exactly (three hold fp16), smaller ones to 2^-18 of it.
template <typename TQ> struct Terms;
template <> struct Terms<__nv_bfloat16> { static constexpr int N = 2; };
template <> struct Terms<__half> { static constexpr int N = 3; };
// The next term of 4 values (packed), which are left with the rest.
__device__ __forceinline__ uint32_t next_term(float* f, bool last) {
  const uint32_t a = f32x2_to_e4m3x2(f[0], f[1]), b = f32x2_to_e4m3x2(f[2], f[3]);
  if (!last) {
    const uint32_t ha = e4m3x2_to_f16x2((uint16_t)a), hb = e4m3x2_to_f16x2((uint16_t)b);
    const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&ha));
    const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&hb));
    f[0] -= fa.x;
    f[1] -= fa.y;
    f[2] -= fb.x;
    f[3] -= fb.y;
  }
  return a | (b << 16);
}
// A piece: blocks [blk, blk + n) of a unit; n = 0: no more.
struct Piece {
  int tok0, tokens, k0, len;
  int g, rb, kvh, blk;
  int n, unit, cut;  // cut: some row may not see all of its prefix
};
template <int TERMS> struct Smem {
  static constexpr int NK = TERMS == 2 ? 3 : 2;
  static constexpr int Q = 0;                            // [tile][term][128 rows][128 B]
  static constexpr int K = Q + TILES * TERMS * 16384;    // e4m3 K slots [128 keys][128 B]
  static constexpr int E = K + NK * 16384;               // e4m3 V slots
  static constexpr int V = E + NE * 16384;               // fp16 V slots [2 halves of d][128 keys][128 B]
  static constexpr int BAR = V + NV * 32768;
  static constexpr int NBAR = 2 * ND + 2 * NK + 2 * NE + 2 * NV + 5 * TILES + 1 + NS;
  static constexpr int END = BAR + NBAR * 8 + ND * (int)sizeof(Piece) + NE * 4 + 12;
  static constexpr int BYTES = 1024 + END;
};
static_assert(Smem<2>::BYTES <= 232448 && Smem<3>::BYTES <= 232448, "shared memory per CTA");
constexpr uint32_t TMEM_COLS = 512;  // O of tile t at 128 t, S (then P) at 256 + 128 t
constexpr float RESCALE_LOG2 = 8.f;  // move a row's reference only when its maximum grew by more than this
constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);  // e4m3, f32 out
constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);

// Descriptors are passed by their low words (address and leading offset); the high words are the same
// for all operands here (1024 bytes between 8-row groups, 128-byte swizzle).
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | ((uint32_t)sm100::SWZ_128B << 29);
template <bool ACC> __device__ __forceinline__ void mma_f8(uint32_t d, uint32_t a_lo, uint32_t b_lo) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(DESC_HI), "r"(IDESC_S), "n"(ACC ? 1 : 0)
      : "memory");
}
template <bool ACC> __device__ __forceinline__ void mma_pv(uint32_t d, uint32_t a_tmem, uint32_t b_lo) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(DESC_HI), "r"(IDESC_PV), "n"(ACC ? 1 : 0)
      : "memory");
}
// 32 consecutive fp32 columns of this thread's TMEM lane; valid after ld_wait.
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Wait for this thread's loads, then pin the registers behind the wait.
__device__ __forceinline__ void ld_wait32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void store8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ bool wait_b(uint64_t* bar, uint32_t use, volatile int* abort_v, unsigned int* err) {
  const uint32_t parity = use & 1;
  if (sm100::mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = sm100::globaltimer();
  for (uint32_t n = 1;; ++n) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    if (n & 63u) continue;
    if (*abort_v) return false;
    if (sm100::globaltimer() - t0 > 2000000000ull) {
      *abort_v = 1;
      if (err) atomicOr(err, ERR_TILE_WAIT);
      return false;
    }
  }
}
// The same outcome in all lanes (the tcgen05 operations that follow are warp-collective).
__device__ __forceinline__ bool wait_w(uint64_t* bar, uint32_t use, volatile int* abort_v, unsigned int* err) {
  return __all_sync(0xffffffffu, wait_b(bar, use, abort_v, err));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ void copy16(void* smem_dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_u32(smem_dst)), "l"(src) : "memory");
}

// The blocks of one group: units (row block, KV head; head fastest) of `blocks` blocks each.
__device__ __forceinline__ void group_shape(const Params& P, int g, Segment& x, int64_t& units, int& blocks) {
  x = prefix_segment(P, g);
  blocks = tc_blocks(x);
  units = blocks ? tc_units(x, P) : 0;
}

__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {  // of non-negative numbers
  return (uint64_t)a < (1ull << 32) ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Walks a CTA's range of blocks piece by piece, warp-wide; 32 groups at a time are held in the lanes.
struct Walk {
  int64_t pos, end;        // blocks
  int g0;                  // first group in the lanes
  int64_t base, units0;    // blocks, units before it
  int64_t size, before;    // this lane's group: blocks, blocks before it
  int64_t units, ubefore;  // units, units before it
  int blocks, tok0, tokens, k0, len;

  __device__ __forceinline__ void fill(const Params& P) {
    const int lane = threadIdx.x & 31;
    Segment x{0, 0, 0, 0};
    units = 0;
    blocks = 0;
    if (g0 + lane < P.num_groups) group_shape(P, g0 + lane, x, units, blocks);
    tok0 = x.tok0;
    tokens = x.tokens;
    k0 = x.k0;
    len = x.len;
    size = units * blocks;
    before = size;
    ubefore = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, before, o), b = __shfl_up_sync(0xffffffffu, ubefore, o);
      if (lane >= o) {
        before += a;
        ubefore += b;
      }
    }
    before += base - size;
    ubefore += units0 - units;
  }
  __device__ __forceinline__ void begin(const Params& P) {
    g0 = 0;
    base = units0 = 0;
    fill(P);
  }
  __device__ __forceinline__ void forward(const Params& P) {  // the next 32 groups
    base = __shfl_sync(0xffffffffu, before + size, 31);
    units0 = __shfl_sync(0xffffffffu, ubefore + units, 31);
    g0 += 32;
    fill(P);
  }
  // The next piece of [pos, end).
  __device__ __forceinline__ Piece next(const Params& P) {
    Piece d{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    if (pos >= end) return d;
    while (pos >= __shfl_sync(0xffffffffu, before + size, 31)) {
      if (g0 >= P.num_groups) return d;
      forward(P);
    }
    const int at = __ffs(__ballot_sync(0xffffffffu, pos < before + size)) - 1;
    const int64_t off = pos - __shfl_sync(0xffffffffu, before, at);
    const int nb = __shfl_sync(0xffffffffu, blocks, at);
    const int u = (int)divide(off, nb);
    d.g = g0 + at;
    d.blk = (int)(off - (int64_t)u * nb);
    d.n = (int)min((int64_t)(nb - d.blk), end - pos);
    d.rb = u / P.num_kv_heads;
    d.kvh = u - d.rb * P.num_kv_heads;
    d.unit = (int)__shfl_sync(0xffffffffu, ubefore, at) + u;
    d.tok0 = __shfl_sync(0xffffffffu, tok0, at);
    d.tokens = __shfl_sync(0xffffffffu, tokens, at);
    d.k0 = __shfl_sync(0xffffffffu, k0, at);
    d.len = __shfl_sync(0xffffffffu, len, at);
    pos += d.n;
    return d;
  }
};
// CTA c of `ctas` takes blocks [c * total / ctas, (c + 1) * total / ctas).
__device__ __forceinline__ int64_t range_begin(int64_t total, int64_t ctas, int64_t c) { return divide(c * total, ctas); }
__device__ __forceinline__ int64_t cta_of(int64_t total, int64_t ctas, int64_t block) {
  return divide((block + 1) * ctas - 1, total);
}

template <int N> __device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <typename TQ, int TERMS>
__global__ void __launch_bounds__(THREADS, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, Params P) {
  using namespace sm100;
  using L = Smem<TERMS>;
  constexpr int NK = L::NK;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* d_full = reinterpret_cast<uint64_t*>(base + L::BAR);
  uint64_t* d_empty = d_full + ND;
  uint64_t* k_full = d_empty + ND;
  uint64_t* k_empty = k_full + NK;
  uint64_t* e_full = k_empty + NK;
  uint64_t* e_empty = e_full + NE;
  uint64_t* v_full = e_empty + NE;
  uint64_t* v_empty = v_full + NV;
  uint64_t* s_full = v_empty + NV;
  uint64_t* p_full = s_full + TILES;
  uint64_t* q_full = p_full + 2 * TILES;
  uint64_t* o_full = q_full + TILES;
  uint64_t* fin = o_full + TILES;
  uint64_t* stored = fin + 1;
  Piece* pieces = reinterpret_cast<Piece*>(stored + NS);
  int* e_ok = reinterpret_cast<int*>(pieces + ND);  // which of a V slot's page tiles are there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(e_ok + NE);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abort_v = abort_flag;
  volatile int* nan_v = abort_flag + 1;  // a NaN value was taken as 0
  if (threadIdx.x == 0) {
    for (int i = 0; i < ND; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 15);
    }
    for (int i = 0; i < NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < NE; ++i) {
      mbar_init(&e_full[i], 1);
      mbar_init(&e_empty[i], 4);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 1);
    }
    for (int t = 0; t < TILES; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], 4);
      mbar_init(&p_full[2 * t + 1], 4);
      mbar_init(&q_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(fin, 1);
    for (int i = 0; i < NS; ++i) mbar_init(&stored[i], 8);
    *abort_flag = 0;
    *nan_v = 0;
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
    fence_mbar_init();
  }
  if (warp == 13) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  // The next piece (number `d`) for a role's warp; n = 0 at the end or after an abort.
  auto take = [&](uint32_t d) {
    Piece x;
    x.n = 0;
    if (!wait_w(&d_full[d % ND], d / ND, abort_v, P.err)) return x;
    x = pieces[d % ND];
    __syncwarp();
    if (lane == 0) mbar_arrive_plain(&d_empty[d % ND]);
    return x;
  };

  // The keys [lo, hi) of a piece's prefix that row `row` of its group sees.
  auto seen_keys = [&](int row, const Piece& x, int& lo, int& hi) {
    const int n = x.tok0 + P.by_group.div(row), b = max(0, sequence_of(P, n));  // (-1: only from lists that do not ascend)
    const int pos = x.len + own_len(P, b) - (q_begin(P, b + 1) - n);
    hi = min(x.len, pos + 1);
    lo = P.window > 0 ? max(0, pos - P.window + 1) : 0;
  };

  if (warp < 4) {  // ---------------- V: e4m3 -> fp16 ----------------
    regs_down<REGS_REST>();
    const int ct = threadIdx.x;
    uint32_t j = 0;
    bool ok = true;
    for (uint32_t d = 0; ok; ++d) {
      const Piece x = take(d);
      if (!x.n) break;
      for (int i = 0; i < x.n; ++i, ++j) {
        const int se = j % NE, sv = j % NV;
        if (!wait_w(&e_full[se], j / NE, abort_v, P.err) ||
            (j >= NV && !wait_w(&v_empty[sv], j / NV - 1, abort_v, P.err))) {
          ok = false;
          break;
        }
        const int key0 = x.k0 + (x.blk + i) * BN, there = e_ok[se];
        uint8_t* src = base + L::E + se * 16384;
        uint8_t* dst = base + L::V + sv * 32768;
        // (what this warp widens below; published by the arrive there, the product and its commit)
        if (x.cut && clean(src, min(BN, x.len - key0) * 8, ct, 128)) *nan_v = 1;
#pragma unroll 4
        for (int u = 0; u < 8; ++u) {
          const int id = ct + 128 * u, key = id >> 3, ch = id & 7;
          uint4 e = *reinterpret_cast<const uint4*>(src + key * 128 + ((ch ^ (key & 7)) << 4));
          // a hole or a row past the end may hold NaN: its weight is 0, V must be finite
          if (!((there >> (key >> 4)) & 1) || key0 + key >= x.len) e = make_uint4(0, 0, 0, 0);
          uint4 lo, hi;
          lo.x = e4m3x2_to_f16x2((uint16_t)(e.x & 0xFFFFu));
          lo.y = e4m3x2_to_f16x2((uint16_t)(e.x >> 16));
          lo.z = e4m3x2_to_f16x2((uint16_t)(e.y & 0xFFFFu));
          lo.w = e4m3x2_to_f16x2((uint16_t)(e.y >> 16));
          hi.x = e4m3x2_to_f16x2((uint16_t)(e.z & 0xFFFFu));
          hi.y = e4m3x2_to_f16x2((uint16_t)(e.z >> 16));
          hi.z = e4m3x2_to_f16x2((uint16_t)(e.w & 0xFFFFu));
          hi.w = e4m3x2_to_f16x2((uint16_t)(e.w >> 16));
          uint8_t* dd = dst + (ch >> 2) * 16384 + key * 128;
          const int c0 = (ch & 3) * 2;
          *reinterpret_cast<uint4*>(dd + ((c0 ^ (key & 7)) << 4)) = lo;
          *reinterpret_cast<uint4*>(dd + (((c0 + 1) ^ (key & 7)) << 4)) = hi;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_plain(&v_full[sv]);
          mbar_arrive_plain(&e_empty[se]);
        }
      }
    }
  } else if (warp < 12) {  // ---------------- rows: Q terms, softmax, O ----------------
    regs_up<REGS_ROWS>();
    const int t = (warp - 4) >> 2;
    const int r = 32 * (warp & 3) + lane;  // row of the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tmem + lane_off + 256u + 128u * t, o_addr = tmem + lane_off + 128u * t;
    uint32_t j = 0, done = 0;
    bool ok = true;
    for (uint32_t d = 0; ok; ++d) {
      const Piece x = take(d);
      if (!x.n) break;
      const int row = x.rb * ROWS + t * BM + r, rows = x.tokens * P.group;
      if (x.rb * ROWS + t * BM >= rows) {  // the unit has no rows in this tile
        if (x.cut && lane == 0) mbar_arrive_plain(&stored[d % NS]);
        continue;
      }
      const bool valid = row < rows;
      // ---- the warp's 32 rows of queries as e4m3 terms, eight lanes a row.  The rows are copied into the
      // place of their first two terms and converted there; the loop is kept short, since this runs once
      // a piece and fetching unrolled code took longer than running it.
      float c = P.scale_log2;
      {
        uint8_t* qt = base + L::Q + t * TERMS * 16384;
#pragma unroll 1
        for (int k = 0; k < 8; ++k) {
          const int rl = 32 * (warp & 3) + 4 * k + (lane >> 3), rr = x.rb * ROWS + t * BM + rl;
          uint8_t* to = qt + rl * 128 + 16 * (lane & 7);
          if (rr < rows) {
            int head;
            const int tok = P.by_group.divmod(rr, head);
            const TQ* qp = reinterpret_cast<const TQ*>(P.q) + (int64_t)(x.tok0 + tok) * P.q_st +
                           (int64_t)(x.kvh * P.group + head) * P.q_sh + 16 * (lane & 7);
            copy16(to, qp);
            copy16(to + 16384, qp + 8);
          } else {
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(to + 16384) = make_uint4(0, 0, 0, 0);
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
#pragma unroll 1
        for (int k = 0; k < 8; ++k) {
          const int rl = 32 * (warp & 3) + 4 * k + (lane >> 3);
          uint8_t* row_at = qt + rl * 128;
          const uint4 raw[2] = {*reinterpret_cast<const uint4*>(row_at + 16 * (lane & 7)),
                                *reinterpret_cast<const uint4*>(row_at + 16384 + 16 * (lane & 7))};
          uint32_t top = top_of(top_of(0, raw[0]), raw[1]);
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
          float up, down;
          term_scale<TQ>(top, up, down);
          const float mine = __shfl_sync(0xffffffffu, down, 8 * (lane & 3));
          if (lane >> 2 == k) c *= mine;  // lane = row 4 k + (lane & 3)
          __syncwarp();                   // the row has been read
          float f[16];
          unpack8<TQ>(raw[0], f);
          unpack8<TQ>(raw[1], f + 8);
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] *= up;
#pragma unroll
          for (int term = 0; term < TERMS; ++term) {
            uint32_t out[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = next_term(f + 4 * e, term + 1 == TERMS);
            *reinterpret_cast<uint4*>(row_at + term * 16384 + (((lane & 7) ^ (rl & 7)) << 4)) =
                make_uint4(out[0], out[1], out[2], out[3]);
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_plain(&q_full[t]);
      // ---- the keys that the row sees
      int lo = 0, hi = 0;
      if (valid) hi = x.len;
      if (valid && x.cut) seen_keys(row, x, lo, hi);
      const int32_t* table = P.pt + (int64_t)x.g * P.pt_stride;
      const int tile0 = x.blk * (BN / TILE);  // of the piece's first block, from k0
      auto entry = [&](int tile) {            // is the page of this lane's key tile there?
        const int key = x.k0 + (tile0 + tile) * TILE;
        if (tile >= x.n * (BN / TILE) || key >= x.len) return 0;
        const int blk = __ldg(table + P.by_page.div(key));
        return blk >= 0 && blk < P.num_pages ? 1 : 0;
      };
      int coming = entry(lane);
      uint32_t there = 0;
      float m = -INFINITY, m_raw = 0.f, l = 0.f;  // reference, scaled and as a raw score; sum
      for (int i = 0; i < x.n; ++i, ++j) {
        if ((i & 3) == 0) {  // 32 key tiles = 4 blocks
          there = __ballot_sync(0xffffffffu, coming != 0);
          coming = entry(32 * (i / 4 + 1) + lane);
        }
        const uint32_t okb = (there >> (8 * (i & 3))) & 0xFFu;
        const int key0 = x.k0 + (x.blk + i) * BN;
        const int a = lo - key0, e = hi - key0;  // the row sees columns [a, e) of pages that are there
        const bool whole = __all_sync(0xffffffffu, !valid || (okb == 0xFFu && a <= 0 && e >= BN));
        if (!wait_w(&s_full[t], j, abort_v, P.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sr[128];
#pragma unroll
        for (int q = 0; q < 4; ++q) ld32(s_addr + 32 * q, sr + 32 * q);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int k = 0; k < 128; ++k) asm volatile("" : "+r"(sr[k]));
        if (!whole) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // bit k: column 32 q + k is visible
            const int from = min(max(a - 32 * q, 0), 32), to = min(max(e - 32 * q, 0), 32);
            uint32_t vis = (to >= 32 ? 0xFFFFFFFFu : (1u << to) - 1u) & (from >= 32 ? 0u : 0xFFFFFFFFu << from);
            vis &= ((okb >> (2 * q)) & 1u ? 0xFFFFu : 0u) | ((okb >> (2 * q + 1)) & 1u ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int k = 0; k < 32; ++k) sr[32 * q + k] = (vis >> k) & 1u ? sr[32 * q + k] : 0xFF800000u;
          }
        }
        float mq[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          mq[q] = __uint_as_float(sr[q]);
#pragma unroll
          for (int k = 8; k < 120; k += 16)
            mq[q] = fmaxf(fmaxf(mq[q], __uint_as_float(sr[k + q])), __uint_as_float(sr[k + 8 + q]));
          mq[q] = fmaxf(mq[q], __uint_as_float(sr[120 + q]));
        }
        const float raw = fmaxf(fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])),
                                fmaxf(fmaxf(mq[4], mq[5]), fmaxf(mq[6], mq[7])));
        const float mx = raw * c;
        // The reference of a row's O and l follows its maximum only when that grew by more than
        // 2^RESCALE_LOG2: weights stay <= 2^8, exact enough in fp16, and O / l does not change.  (By the difference,
        // which is exact: near 2^27 m + 8 may round up to the next score, 16 above m.)
        float alpha = 1.f;
        if (mx - m > RESCALE_LOG2 || (m == -INFINITY && mx != -INFINITY)) {
          alpha = fast_exp2(m - mx);
          m = mx;
          m_raw = raw;
        }
        // Weights are 2^(s c - m) by one fma, m carrying a rounding of 2^-24 |m|; where that could be seen,
        // the maximum is taken off s first.
        const bool huge = fabsf(m) > 16384.f && m != -INFINITY;
        if (__any_sync(0xffffffffu, huge)) {
#pragma unroll
          for (int k = 0; k < 128; ++k)
            if (huge) sr[k] = __float_as_uint(__uint_as_float(sr[k]) - m_raw);
        }
        const float ref = m != -INFINITY && !huge ? m : 0.f;
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {  // P.V of the block before is complete: see s_full
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            uint32_t o[32];
            ld32(o_addr + 32 * q, o);
            ld_wait32(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            st16(o_addr + 32 * q, o);
            st16(o_addr + 32 * q + 16, o + 16);
          }
        }
        const float2 c2 = make_float2(c, c), off = make_float2(-ref, -ref);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float2 y =
                fma2(make_float2(__uint_as_float(sr[32 * q + k]), __uint_as_float(sr[32 * q + k + 1])), c2, off);
            const float2 p = make_float2(fast_exp2(y.x), fast_exp2(y.y));
            sum = add2(sum, p);
            pk[k >> 1] = pack_half2(p.x, p.y);
          }
          st16(s_addr + 16 * q, pk);  // over S, which is in registers
          if (q & 1) {                // half of the block's keys: their P.V may begin
            st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_plain(&p_full[2 * t + (q >> 1)]);
          }
        }
        l = l * alpha + (sum.x + sum.y);
      }
      // ---- the piece's partial
      if (ok) ok = wait_w(&o_full[t], done, abort_v, P.err);
      if (!ok) break;  // (see tc_lost)
      ++done;
      tc_fence_after();
      const int64_t at = ((int64_t)x.unit + blockIdx.x) * ROWS + t * BM + r;
      if ((uint64_t)at < (uint64_t)P.tc_rows) {
        if (valid) P.tc_ml[at] = make_float2(m, l);
        float* op = P.tc_o + at * D;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t o[32];
          ld32(o_addr + 32 * q, o);
          ld_wait32(o);
          if (valid)
#pragma unroll
            for (int k = 0; k < 32; k += 8) store8(op + 32 * q + k, reinterpret_cast<const float*>(o + k));
        }
      }
      tc_fence_before();
      if (x.cut) {
        __syncwarp();
        if (lane == 0) mbar_arrive_plain(&stored[d % NS]);
      }
    }
  } else {
    regs_down<REGS_REST>();
    if (warp == 12) {  // ---------------- loads ----------------
      uint32_t j = 0, keys = 0;  // blocks asked for: V, K
      bool ok = true;
      for (uint32_t d = 0; ok; ++d) {
        const Piece x = take(d);
        if (!x.n) break;
        const int32_t* table = P.pt + (int64_t)x.g * P.pt_stride;
        const int tile0 = x.blk * (BN / TILE), tiles = x.n * (BN / TILE);
        int blk = -1, row0 = 0, blk_n = -1, row_n = 0;  // lane: key tile of the current and the next 4 blocks
        auto entry = [&](int tile, int& b, int& rr) {
          const int key = x.k0 + (tile0 + tile) * TILE;
          b = -1;
          rr = 0;
          if (tile >= tiles || key >= x.len) return;
          const int at = P.by_page.div(key);
          rr = key - at * P.page;
          b = __ldg(table + at);
          if (b >= P.num_pages) b = -1;
        };
        entry(lane, blk_n, row_n);
        for (int i = 0; i < x.n; ++i, ++j) {
          if ((i & 3) == 0) {
            blk = blk_n;
            row0 = row_n;
            entry(32 * (i / 4 + 1) + lane, blk_n, row_n);
          }
          const uint32_t there = (__ballot_sync(0xffffffffu, blk >= 0) >> (8 * (i & 3))) & 0xFFu;
          const int sk = j % NK, se = j % NE, tile = lane - 8 * (i & 3);
          const bool mine = tile >= 0 && tile < 8 && blk >= 0;
          ok = j < NK || wait_w(&k_empty[sk], j / NK - 1, abort_v, P.err);
          if (!ok) break;
          if (lane == 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive_expect_tx(&k_full[sk], __popc(there) * TILE_BYTES);
          }
          __syncwarp();
          if (mine) tma_load_4d(base + L::K + sk * 16384 + tile * TILE_BYTES, &tmk, &k_full[sk], 0, x.kvh, row0, blk);
          keys = j + 1;
          ok = j < NE || wait_w(&e_empty[se], j / NE - 1, abort_v, P.err);
          if (!ok) break;
          if (lane == 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            e_ok[se] = (int)there;  // published by the arrive below
            mbar_arrive_expect_tx(&e_full[se], __popc(there) * TILE_BYTES);
          }
          __syncwarp();
          if (mine) tma_load_4d(base + L::E + se * 16384 + tile * TILE_BYTES, &tmv, &e_full[se], 0, x.kvh, row0, blk);
        }
      }
      if (lane == 0) {  // leave no copy in flight: wait (bounded) for the last use of every slot
        const uint64_t t0 = globaltimer();
        for (int i = 0; i < NK + NE; ++i) {
          uint64_t* bar = i < NK ? &k_full[i] : &e_full[i - NK];
          const uint32_t ns = i < NK ? NK : NE, slot = i < NK ? i : i - NK, asked = i < NK ? keys : j;
          if (asked <= slot) continue;
          const uint32_t use = (asked - 1 - slot) / ns;
          while (!mbar_try_wait(bar, use & 1) && globaltimer() - t0 < 1000000000ull) {
          }
        }
      }
    } else if (warp == 13) {  // ---------------- MMA ----------------
      // low descriptor words: address >> 4, and the leading offset >> 4 (K-major: unused, 1; V: 16 KB
      // between its halves of d)
      const uint32_t q_lo = (smem_u32(base + L::Q) >> 4) | (1u << 16), k_lo = (smem_u32(base + L::K) >> 4) | (1u << 16);
      const uint32_t v_lo = (smem_u32(base + L::V) >> 4) | ((16384u >> 4) << 16);
      // The whole warp runs this loop, its values uniform, and one elected lane issues: the operands of
      // the tcgen05 instructions then stay in uniform registers (issued from a divergent lane, an MMA
      // took about 100 cycles to issue, longer than the 64 it runs).
      const bool leader = elect_one();
      const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
      uint32_t j = 0, sk = 0, sv = 0, s0 = 0, s1 = 0, p0 = 0, p1 = 0;  // blocks, slots, P and pieces by tile
      bool ok = true;
      auto issue_s = [&](int t, uint32_t slot) {
        const uint32_t dd = tm + 256u + 128u * t, q = q_lo + t * (TERMS * 1024u), k = k_lo + slot * 1024u;
        if (leader) {
          mma_f8<false>(dd, q, k);
#pragma unroll
          for (int kk = 1; kk < 4 * TERMS; ++kk)
            mma_f8<true>(dd, q + (kk / 4) * 1024u + (kk % 4) * 2u, k + (kk % 4) * 2u);
          tc_commit(&s_full[t]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int half, uint32_t v, bool first) {  // 64 keys
        const uint32_t o = tm + 128u * t, pt = tm + 256u + 128u * t + 32u * half;
        v += half * 512u;
        if (leader) {
          if (first)
            mma_pv<false>(o, pt, v);
          else
            mma_pv<true>(o, pt, v);
#pragma unroll
          for (int kk = 1; kk < 4; ++kk) mma_pv<true>(o, pt + 8u * kk, v + kk * 128u);  // 16 keys each
        }
        __syncwarp();
      };
      for (uint32_t d = 0; ok; ++d) {
        const Piece x = take(d);
        const int n = __reduce_max_sync(0xffffffffu, x.n);
        if (!n) break;
        const bool two = __any_sync(0xffffffffu, x.rb * ROWS + BM < x.tokens * P.group);
        // V of a block and K of the next are waited for under the MMAs of the block before
        auto operands = [&](bool more) {
          const uint32_t next = sk + 1 == NK ? 0 : sk + 1;
          return (!more || wait_w(&k_full[next], (j + 1) / NK, abort_v, P.err)) &&
                 wait_w(&v_full[sv], j / NV, abort_v, P.err);
        };
        ok = wait_w(&k_full[sk], j / NK, abort_v, P.err) && wait_w(&q_full[0], p0++, abort_v, P.err) &&
             (!two || wait_w(&q_full[1], p1++, abort_v, P.err));
        if (!ok) break;
        tc_fence_after();
        issue_s(0, sk);
        if (two) issue_s(1, sk);
        if (leader) tc_commit(&k_empty[sk]);
        __syncwarp();
        ok = operands(n > 1);
        for (int i = 0; ok && i < n; ++i) {
          const bool more = i + 1 < n;
          const uint32_t v = v_lo + sv * 2048u, next = sk + 1 == NK ? 0 : sk + 1;
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            if (t == 1 && !two) break;
            uint32_t& use = t ? s1 : s0;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && wait_w(&p_full[2 * t + half], use, abort_v, P.err);
              if (!ok) break;
              tc_fence_after();
              issue_pv(t, half, v, i == 0 && half == 0);
            }
            if (!ok) break;
            ++use;
            if (more)
              issue_s(t, next);
            else if (leader)
              tc_commit(&o_full[t]);
            __syncwarp();
          }
          if (!ok) break;
          if (leader) {
            tc_commit(&v_empty[sv]);
            if (more) tc_commit(&k_empty[next]);
          }
          __syncwarp();
          ++j;
          sk = next;
          sv = sv + 1 == NV ? 0 : sv + 1;
          if (more) ok = operands(i + 2 < n);
        }
      }
      if (leader) {  // everything issued has completed before the teardown
        tc_commit(fin);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(fin, 0) && globaltimer() - t0 < 2000000000ull) {
        }
      }
      __syncwarp();
    } else if (warp == 14) {  // ---------------- pieces ----------------
      int cut = P.window > 0;  // a window, or a sequence with fewer own keys than rows: its rows stand in the prefix
      for (int b = lane; b < P.batch; b += 32) cut |= own_len(P, b) < q_begin(P, b + 1) - q_begin(P, b);
      Walk w;
      w.begin(P);
      cut = __any_sync(0xffffffffu, cut);
      while (w.g0 + 32 < P.num_groups) w.forward(P);
      const int64_t total = __shfl_sync(0xffffffffu, w.before + w.size, 31);
      const int64_t ctas = tc_ctas_of(total, (int)gridDim.x);
      if (w.g0 > 0) w.begin(P);
      const bool work = (int64_t)blockIdx.x < ctas;
      w.pos = work ? range_begin(total, ctas, blockIdx.x) : 0;
      w.end = work ? range_begin(total, ctas, blockIdx.x + 1) : 0;
      for (uint32_t d = 0;; ++d) {
        Piece x = w.next(P);
        x.cut = cut;
        if (d >= ND && !wait_w(&d_empty[d % ND], d / ND - 1, abort_v, P.err)) break;
        if (lane == 0) {
          pieces[d % ND] = x;
          mbar_arrive_plain(&d_full[d % ND]);
        }
        if (!x.n) break;
      }
    } else {  // ---------------- NaN values (cut is the same for all pieces) ----------------
      for (uint32_t d = 0;; ++d) {
        const Piece x = take(d);
        if (!x.n) break;
        if (!x.cut) continue;
        if (!wait_w(&stored[d % NS], d / NS, abort_v, P.err)) break;
        if (!*nan_v) continue;
        const int rows = min(ROWS, x.tokens * P.group - x.rb * ROWS);
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 32) {
          int lo = 0, hi = 0;
          const int64_t at = ((int64_t)x.unit + blockIdx.x) * ROWS + r0 + lane;
          if (r0 + lane < rows && (uint64_t)at < (uint64_t)P.tc_rows) seen_keys(x.rb * ROWS + r0 + lane, x, lo, hi);
          mark_nan(P, P.pt + x.g * P.pt_stride, x.kvh, x.k0 + x.blk * BN, min(x.len, x.k0 + (x.blk + x.n) * BN), lo, hi,
                   P.tc_o + at * D, 0, D);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 13) tmem_dealloc(tmem, TMEM_COLS);
  if (threadIdx.x == 0) P.tc_lost[blockIdx.x] = (unsigned)*abort_v;
}

// The row warps wait for registers that the others give back: only what the block was launched with is
// there, so the compiled kernel has to come with REGS_LAUNCH a thread.
template <auto Kernel>
inline bool registers_ready() {
  static std::atomic<int> ok{-1};
  int v = ok;
  if (v < 0) {
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, Kernel) != cudaSuccess) return false;
    ok = v = a.numRegs >= REGS_LAUNCH ? 1 : 0;
  }
  return v == 1;
}
}  // namespace tc

// ---- merge: one warp per (row, head), four dimensions a lane --------------------------------------
// out = v_scale * sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over the row's pieces i, M = max m_i, in the
// order of the pieces.  Bound: the partials' bytes, latency for few rows: 256 rows x 32 heads (48 MB of partials)
// 21.0 us from a cold L2, 2.3 TB/s; 64 rows x 32 heads 10.8 us, a chain of three loads (plan, maxima, sums).
template <typename TO>
__global__ void __launch_bounds__(128) merge_kernel(Params P, int piece_rows) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x * 4 + warp;
  if (item >= P.total_q * P.num_heads) return;
  int h, hg;
  const int n = P.by_heads.divmod(item, h), kvh = P.by_group.divmod(h, hg);
  const RowPlan plan = P.plan[n];
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  // `count` partials of this row, `step` rows apart from row0 on, in order
  auto gather = [&](int count, int64_t row0, int64_t step, const float2* mls, const float* os, int64_t limit) {
    for (int s0 = 0; s0 < count; s0 += 32) {
      float2 ml = make_float2(-INFINITY, 0.f);
      const int64_t mine = row0 + (s0 + lane) * step;
      if (s0 + lane < count && (uint64_t)mine < (uint64_t)limit) ml = mls[mine];
      float most = ml.x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float to = fmaxf(M, most);
      if (to == -INFINITY && !__any_sync(0xffffffffu, ml.x != ml.x || ml.y != ml.y)) continue;
      const float by = M == -INFINITY ? 0.f : fast_exp2(M - to);
      M = to;
      L *= by;
      O.x *= by, O.y *= by, O.z *= by, O.w *= by;
      const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - to);
      float add = ml.y * w;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
      L += add;
      const int here = min(32, count - s0);
#pragma unroll 4
      for (int j = 0; j < here; ++j) {
        const float wj = __shfl_sync(0xffffffffu, w, j);
        if (wj != 0.f) {  // (0 for a piece without a visible key, which holds no sum)
          const float4 v = *reinterpret_cast<const float4*>(os + (row0 + (s0 + j) * step) * D + 4 * lane);
          O.x = fmaf(v.x, wj, O.x);
          O.y = fmaf(v.y, wj, O.y);
          O.z = fmaf(v.z, wj, O.z);
          O.w = fmaf(v.w, wj, O.w);
        }
      }
    }
  };
  unsigned int lost = 0;
  if (plan.blocks > 0) {
    const int r = plan.pre_row + hg;
    const int64_t unit = (int64_t)(r / tc::ROWS) * P.num_kv_heads + kvh, from = plan.tc_from + unit * plan.blocks;
    const int64_t c0 = tc::cta_of(plan.tc_total, plan.tc_ctas, from);
    const int64_t c1 = tc::cta_of(plan.tc_total, plan.tc_ctas, from + plan.blocks - 1);
    for (int64_t c = max(c0, (int64_t)0) + lane; c <= c1 && c < P.tc_ctas; c += 32) lost |= P.tc_lost[c];
    gather((int)(c1 - c0 + 1), (plan.tc_units + unit + c0) * tc::ROWS + r % tc::ROWS, tc::ROWS, P.tc_ml, P.tc_o,
           P.tc_rows);
  }
  // the pieces of a segment that hold row r, in order of their splits
  auto join = [&](int first, int splits, int r) {
    const int64_t piece0 = first + (int64_t)(r / piece_rows) * splits * P.num_kv_heads + kvh;
    gather(splits, piece0 * piece_rows + r % piece_rows, (int64_t)P.num_kv_heads * piece_rows, P.ml_part, P.o_part,
           (int64_t)P.max_pieces * piece_rows);
  };
  join(plan.pre_first, plan.pre_splits, plan.pre_row + hg);
  join(plan.own_first, plan.own_splits, plan.own_row + hg);
  if (__any_sync(0xffffffffu, lost != 0)) L = __int_as_float(0x7fc00000);
  const float inv = L > 0.f ? P.v_scale / L : (L != L ? L : 0.f);  // a poisoned piece stays visible
  TO* op = reinterpret_cast<TO*>(P.out) + (int64_t)n * P.o_st + (int64_t)h * P.o_sh + 4 * lane;
  TO v[4] = {from_f32<TO>(O.x * inv), from_f32<TO>(O.y * inv), from_f32<TO>(O.z * inv), from_f32<TO>(O.w * inv)};
  *reinterpret_cast<uint2*>(op) = *reinterpret_cast<const uint2*>(v);
}

// ---- launch -----------------------------------------------------------------------------------------
inline int sm_count() {
  static std::atomic<int> sms[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = sms[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 0;
    sms[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <auto Kernel>
inline bool smem_ready(int bytes) {
  static std::atomic<int> done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (done[dev] == bytes) return true;
  if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
      cudaFuncSetAttribute(Kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared) !=
          cudaSuccess)
    return false;
  done[dev] = bytes;
  return true;
}

// Blocks of 8 rows that a warp takes together: two where the sequences have more than 8 rows on average, one
// otherwise (then 16 cost more than a prefix's K and V read half as often give back: 42 against 56 us for
// 8 x 8 samples of 2 rows, 23 against 31 for 16 sequences of 4).
inline int row_blocks(int64_t rows) { return rows <= 8 ? 1 : 2; }

// pieces_kernel keeps the segments in shared memory behind its rings; its limit is set once, for the most
// there may be, so that calls of different batches on different threads cannot lower it under one another.
constexpr int MAX_SEGMENTS = 4096;
constexpr int pieces_smem(int groups, int batch) {
  return 1024 + WARPS * RING_BYTES + (groups + batch) * ((int)sizeof(Segment) + 12) + groups * 4 + 8;
}
static_assert(pieces_smem(MAX_SEGMENTS, 0) + 8 * 1024 <= 227 * 1024, "the segments have to fit beside the rings");
constexpr int PIECES_PER_SM = 3 * WARPS;

// prefix_kernel takes the prefixes from 33 rows a prefix and KV head on (with fewer, its 128-row tiles stay
// emptier than the pieces' blocks of 8), where (rows) x (keys that the prefix tables reach) x (KV heads)
// is at least 3 * 2^19, where its start-up and partials (about 15 us) are made up for.  The host knows the
// tables' width, not the lengths: behind tables padded to a long reach (and under a window, which is not
// counted either) a short prefix takes it too, and pays those 15 us.  By pieces and with it, tables cut to
// the prefix, in us: 64 rows x 8 heads behind 2,048 keys 22.6, 21.8, behind 8,192 38.1, 32.7; 192 rows behind 1,024 32.0,
// 24.1; 256 rows behind 512 27.3, 31.2.
constexpr int64_t TC_ROWS = 33, TC_WORK = 3 << 19;

struct Layout {
  int nb;
  bool tc;  // enough rows for prefix_kernel
  int64_t pieces, tc_pieces;
  size_t plan, ml, o, tc_lost, tc_ml, tc_o, bytes;  // offsets of the workspace's parts, its size
};
inline Layout layout(int64_t total_q, int64_t groups, int64_t batch, int64_t heads, int64_t kv_heads) {
  Layout y;
  const int64_t group = heads / kv_heads;
  y.tc = groups > 0 && total_q * group >= TC_ROWS * groups;
  y.nb = row_blocks(cdiv(total_q * group, batch));
  const int64_t rows = 8 * y.nb;
  // every row lies in at most two segments (its prefix and its own keys)
  const int64_t units = (2 * cdiv(total_q * group, rows) + groups + batch) * kv_heads;
  y.pieces = units * 2 > 148 * PIECES_PER_SM ? units * 2 : 148 * PIECES_PER_SM;
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  y.tc_pieces = y.tc ? (cdiv(total_q * group, tc::ROWS) + groups) * kv_heads + 148 : 0;
  y.plan = 0;
  y.ml = up((size_t)total_q * sizeof(RowPlan));
  y.o = up(y.ml + (size_t)y.pieces * rows * sizeof(float2));
  y.tc_lost = up(y.o + (size_t)y.pieces * rows * D * sizeof(float));
  y.tc_ml = up(y.tc_lost + (y.tc ? 148 * sizeof(unsigned int) : 0));
  y.tc_o = up(y.tc_ml + (size_t)y.tc_pieces * tc::ROWS * sizeof(float2));
  y.bytes = y.tc_o + (size_t)y.tc_pieces * tc::ROWS * D * sizeof(float);
  return y;
}

}  // namespace sp
}  // namespace ada

using namespace ada;

extern "C" size_t ada_fp8_shared_prefix_decode_workspace_size(int32_t total_q, int32_t num_groups, int32_t batch,
                                                              int32_t num_heads, int32_t num_kv_heads,
                                                              int32_t head_dim) {
  if (total_q <= 0 || num_groups < 0 || batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      num_heads % num_kv_heads != 0)
    return 0;
  return sp::layout(total_q, num_groups, batch, num_heads, num_kv_heads).bytes;
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
  if ((int64_t)num_groups + batch > sp::MAX_SEGMENTS) return ADA_ERR_UNSUPPORTED;
  if (((int64_t)max_pages + max_prefix_pages) * page_size > (1LL << 30)) return ADA_ERR_UNSUPPORTED;
  if ((int64_t)total_q * num_heads > (1LL << 30)) return ADA_ERR_UNSUPPORTED;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return ADA_ERR_ALIGNMENT;
  if ((kv_stride_page | kv_stride_tok | kv_stride_head) & 15) return ADA_ERR_ALIGNMENT;
  if (((uintptr_t)q & 15) || (q_stride_t & 7) || (q_stride_h & 7)) return ADA_ERR_ALIGNMENT;
  if (((uintptr_t)out & 15) || (out_stride_t & 7) || (out_stride_h & 7)) return ADA_ERR_ALIGNMENT;
  if (((uintptr_t)workspace & 255) || ((uintptr_t)err & 3)) return ADA_ERR_ALIGNMENT;
  const sp::Layout y = sp::layout(total_q, num_groups, batch, num_heads, num_kv_heads);
  if (workspace_bytes < y.bytes) return ADA_ERR_WORKSPACE;

  sp::Params P;
  P.q = q;
  P.q_st = q_stride_t;
  P.q_sh = q_stride_h;
  P.v = v_cache;
  P.v_page = kv_stride_page;
  P.v_tok = kv_stride_tok;
  P.v_head = kv_stride_head;
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
  P.num_kv_heads = num_kv_heads;
  P.group = num_heads / num_kv_heads;
  P.page = page_size;
  P.by_group = sp::Divisor::of(P.group);
  P.by_page = sp::Divisor::of(page_size);
  P.by_kv_heads = sp::Divisor::of(num_kv_heads);
  P.by_heads = sp::Divisor::of(num_heads);
  // a window as wide as all positions cuts nothing off; any other leaves the differences below in 32 bits
  P.window = window < ((int64_t)max_pages + max_prefix_pages) * page_size ? window : 0;
  P.scale_log2 = scale * k_scale * sp::LOG2E;
  P.v_scale = v_scale;
  P.out = out;
  P.o_st = out_stride_t;
  P.o_sh = out_stride_h;
  P.err = err;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  P.plan = reinterpret_cast<sp::RowPlan*>(ws + y.plan);
  P.ml_part = reinterpret_cast<float2*>(ws + y.ml);
  P.o_part = reinterpret_cast<float*>(ws + y.o);
  P.max_pieces = (int32_t)(y.pieces < (1 << 26) ? y.pieces : (1 << 26) - 1);
  const int64_t reach = (int64_t)max_prefix_pages * page_size;
  P.prefix_tc = y.tc && total_q * (int64_t)P.group * num_kv_heads * reach >= sp::TC_WORK ? 1 : 0;
  P.tc_lost = reinterpret_cast<unsigned int*>(ws + y.tc_lost);
  P.tc_ml = reinterpret_cast<float2*>(ws + y.tc_ml);
  P.tc_o = reinterpret_cast<float*>(ws + y.tc_o);
  P.tc_rows = y.tc_pieces * sp::tc::ROWS;

  // K / V caches as 4-D byte tensors [num_pages][page][Hkv][D] -> TMA box of 16 rows x 128 B
  CUtensorMap tmk, tmv;
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)num_kv_heads, (cuuint64_t)page_size,
                              (cuuint64_t)num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)kv_stride_head, (cuuint64_t)kv_stride_tok, (cuuint64_t)kv_stride_page};
  const cuuint32_t box[4] = {(cuuint32_t)head_dim, 1, (cuuint32_t)sp::TILE, 1};
  if (!sm100::encode_bytes(&tmk, k_cache, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !sm100::encode_bytes(&tmv, v_cache, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
    return ADA_ERR_CUDA;
  const int sms = sp::sm_count();
  if (!sms) return ADA_ERR_CUDA;
  P.tc_ctas = sms < 148 ? sms : 148;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (P.prefix_tc) {
    const dim3 grid((unsigned)P.tc_ctas), block(sp::tc::THREADS);
    if (q_dtype == ADA_DT_BF16) {
      constexpr int bytes = sp::tc::Smem<2>::BYTES;
      if (!sp::tc::registers_ready<sp::tc::prefix_kernel<__nv_bfloat16, 2>>()) return ADA_ERR_UNSUPPORTED;
      if (!sp::smem_ready<sp::tc::prefix_kernel<__nv_bfloat16, 2>>(bytes)) return ADA_ERR_CUDA;
      (void)ada::launch_k(sp::tc::prefix_kernel<__nv_bfloat16, 2>, grid, block, bytes, st, tmk, tmv, P);
    } else {
      constexpr int bytes = sp::tc::Smem<3>::BYTES;
      if (!sp::tc::registers_ready<sp::tc::prefix_kernel<__half, 3>>()) return ADA_ERR_UNSUPPORTED;
      if (!sp::smem_ready<sp::tc::prefix_kernel<__half, 3>>(bytes)) return ADA_ERR_CUDA;
      (void)ada::launch_k(sp::tc::prefix_kernel<__half, 3>, grid, block, bytes, st, tmk, tmv, P);
    }
    ADA_CHECK_LAUNCH();
  }
  const int smem = sp::pieces_smem(num_groups, batch);
#define ADA_SP(TQ, NB)                                                                                              \
  do {                                                                                                              \
    if (!sp::smem_ready<sp::pieces_kernel<TQ, NB>>(sp::pieces_smem(sp::MAX_SEGMENTS, 0))) return ADA_ERR_CUDA;         \
    (void)ada::launch_k(sp::pieces_kernel<TQ, NB>, dim3((unsigned)(sms * (NB == 1 ? 3 : 2))), dim3(sp::WARPS * 32), \
                        smem, st, tmk, tmv, P);                                                                     \
  } while (0)
  if (q_dtype == ADA_DT_BF16) {
    if (y.nb == 1) ADA_SP(__nv_bfloat16, 1); else ADA_SP(__nv_bfloat16, 2);
  } else {
    if (y.nb == 1) ADA_SP(__half, 1); else ADA_SP(__half, 2);
  }
#undef ADA_SP
  ADA_CHECK_LAUNCH();
  const dim3 grid((unsigned)cdiv((int64_t)total_q * num_heads, 4));
  if (out_dtype == ADA_DT_BF16)
    (void)ada::launch_k(sp::merge_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, P, 8 * y.nb);
  else
    (void)ada::launch_k(sp::merge_kernel<__half>, grid, dim3(128), 0, st, P, 8 * y.nb);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}
