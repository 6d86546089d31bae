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
//
// Bound: HBM (a logit costs 2 or 4 bytes and about ten instructions).  One thread-block cluster
// takes one row (or one sequence's rows), each CTA a contiguous share of the vocabulary, so a call is
// one launch without a workspace: the CTAs exchange their partial results through distributed
// shared memory.  A thread keeps a running maximum m of its raw logits and its sum of
// 2^((x - m) c), c = log2(e) / T; x - m is exact or nearly so where the weight matters, so the
// statistics do not pay for the size of x.
#include <float.h>

#include <type_traits>

#include "cluster.cuh"

namespace ada {
namespace smp {

constexpr int MAX_CLUSTER = 16;  // non-portable size: few rows on many SMs
constexpr int NONE = 0x7fffffff;
constexpr float LN2 = 0.6931471805599453f;

// ---- reading a row in packets of 16 bytes a thread -------------------------------------------
// VEC: packet k is the N elements from k * N, one 16-byte load (rows start on 16 bytes).  Otherwise
// the 32 packets of a warp share 32 * N elements in turn (coalesced scalar loads, any alignment).
template <typename T> constexpr int pack_n() { return 16 / (int)sizeof(T); }
template <typename T, bool VEC> __device__ __forceinline__ int pack_index(int k, int i) {
  constexpr int N = pack_n<T>();
  return VEC ? k * N + i : (k & ~31) * N + (k & 31) + 32 * i;
}
__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return to_f32(v); }
__device__ __forceinline__ float as_f32(__half v) { return to_f32(v); }
template <typename T> __device__ __forceinline__ T minus_inf();
template <> __device__ __forceinline__ float minus_inf<float>() { return -INFINITY; }
template <> __device__ __forceinline__ __nv_bfloat16 minus_inf<__nv_bfloat16>() { return __ushort_as_bfloat16(0xFF80); }
template <> __device__ __forceinline__ __half minus_inf<__half>() { return __ushort_as_half(0xFC00); }

template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_pack(const T* __restrict__ x, int k, int n) {
  constexpr int N = pack_n<T>();
  if (VEC && (k + 1) * N <= n) return ldg_stream16(x + k * N);
  uint4 u;
  T* h = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = pack_index<T, VEC>(k, i);
    h[i] = at < n ? x[at] : minus_inf<T>();
  }
  return u;
}
template <typename T> __device__ __forceinline__ void unpack(const uint4& u, float* f) {
  const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < pack_n<T>(); ++i) f[i] = as_f32(h[i]);
}
// The noise beside packet k of a T row.
template <typename T, bool VEC>
__device__ __forceinline__ void load_noise(const float* __restrict__ e, int k, int n, float* f) {
  constexpr int N = pack_n<T>();
  if (VEC && (k + 1) * N <= n) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 u = ldg_stream16(e + k * N + i);
      f[i] = __uint_as_float(u.x);
      f[i + 1] = __uint_as_float(u.y);
      f[i + 2] = __uint_as_float(u.z);
      f[i + 3] = __uint_as_float(u.w);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = pack_index<T, VEC>(k, i);
    f[i] = at < n ? e[at] : 1.f;
  }
}

// ---- weights ---------------------------------------------------------------------------------
struct Scale {
  float c, c_lo;  // log2(e) / T in two floats
  float least;    // differences below this have weight 0 (2^-200)
  bool greedy;
  float t;
  __device__ __forceinline__ explicit Scale(float temp) {
    greedy = !(temp > 1e-10f);
    t = greedy ? 1.f : temp;
    const double cd = 1.4426950408889634 / (double)t;
    c = (float)cd;
    c_lo = (float)(cd - (double)c);
    least = -200.f / c;
  }
  // x - m, at most 0: -inf and NaN give `least` (weight 0), +inf gives 0.
  __device__ __forceinline__ float diff(float x, float m) const { return fminf(fmaxf(x - m, least), 0.f); }
  // 2^(d c) to about 2^-21 relative: enough for sums
  __device__ __forceinline__ float weight(float d) const { return fast_exp2(d * c); }
  // to about 2^-22 whatever d: the product's rounding is carried into the result
  __device__ __forceinline__ float weight_exact(float d) const {
    const float y = d * c;
    const float low = fmaf(d, c, -y) + d * c_lo;
    const float w = fast_exp2(y);
    return fmaf(w, low * LN2, w);
  }
};

// Maximum and sum of the logits a thread (warp, CTA, cluster) has seen: s = sum 2^((x - m) c).
struct Stats {
  float m, s;
  int at;  // a thread's packet that first held the maximum, then the index of the first maximum
  __device__ __forceinline__ void init() {
    m = -FLT_MAX;
    s = 0.f;
    at = NONE;
  }
  __device__ __forceinline__ void merge(float m2, float s2, int at2, const Scale& sc) {
    const float top = fmaxf(m, m2);
    at = m == m2 ? min(at, at2) : (m > m2 ? at : at2);
    s = s * sc.weight(fmaxf(m - top, sc.least)) + s2 * sc.weight(fmaxf(m2 - top, sc.least));
    m = top;
  }
  __device__ __forceinline__ void merge_warp(const Scale& sc) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
      merge(m2, s2, at2, sc);
    }
  }
  __device__ __forceinline__ bool any() const { return s > 0.f; }
};
// Fold packet k (values v) in; returns whether the maximum moved.
template <int N>
__device__ __forceinline__ bool fold(Stats& st, const float* v, int k, const Scale& sc) {
  float top = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
  const bool moved = top > st.m || (st.at == NONE && top == -FLT_MAX);
  if (moved) {
    top = fminf(top, FLT_MAX);
    st.s *= sc.weight(fmaxf(st.m - top, sc.least));
    st.m = top;
    st.at = k;
  }
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    s0 += sc.weight(sc.diff(v[i], st.m));
    s1 += sc.weight(sc.diff(v[i + 1], st.m));
  }
  st.s += s0 + s1;
  return moved;
}
// A thread's packet of the first maximum -> the index of that maximum.
template <typename T, bool VEC>
__device__ __forceinline__ int first_maximum(const T* x, const Stats& st, int n) {
  if (st.at == NONE) return NONE;
  float v[pack_n<T>()];
  unpack<T>(load_pack<T, VEC>(x, st.at, n), v);
  int at = NONE;
#pragma unroll
  for (int i = pack_n<T>() - 1; i >= 0; --i)
    if (v[i] >= st.m) at = pack_index<T, VEC>(st.at, i);
  return at;
}

// The winner of a race: the largest w / e, lowest index on ties.  Compared crosswise, so no
// division: w1 / e1 > w2 / e2 as w1 e2 > w2 e1.
struct Best {
  float w, e;
  int at;
  __device__ __forceinline__ void init() {
    w = 0.f;
    e = 1.f;
    at = NONE;
  }
  __device__ __forceinline__ void merge(float w2, float e2, int at2) {
    const float a = w2 * e, b = w * e2;
    if (a > b || (a == b && at2 < at)) {
      w = w2;
      e = e2;
      at = at2;
    }
  }
  __device__ __forceinline__ void merge_warp() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float w2 = __shfl_xor_sync(0xffffffffu, w, o), e2 = __shfl_xor_sync(0xffffffffu, e, o);
      const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
      merge(w2, e2, at2);
    }
  }
};
__device__ __forceinline__ float exponential(float e) { return fmaxf(e, 1e-10f); }

// This CTA's packets [k0, k1) of a row of n elements, in shares of whole warps.
template <typename T> __device__ __forceinline__ void share(int n, int rank, int ranks, int& k0, int& k1) {
  constexpr int N = pack_n<T>();
  const int packs = ((n + 32 * N - 1) / (32 * N)) * 32;
  const int per = ((packs / 32 + ranks - 1) / ranks) * 32;
  k0 = min(rank * per, packs);
  k1 = min(k0 + per, packs);
}

// ---- sampling: one cluster per row -------------------------------------------------------------
struct SampleWord {
  float m, s, x, e;  // x, e: the candidate's logit and noise
  int at, first;     // its index; the index of the first maximum
  int pad[2];
};

template <typename T, bool VEC, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT)
    sample_kernel(const T* __restrict__ logits, int64_t ld, int n, const float* __restrict__ temps,
                  const float* __restrict__ noise, int64_t ld_noise, int64_t* tokens, float* logprobs, float* lse) {
  constexpr int N = pack_n<T>(), WARPS = NT / 32, U = 2;
  __shared__ float wm[WARPS], wsum[WARPS], we[WARPS], wx[WARPS];
  __shared__ int wat[WARPS], wfirst[WARPS];
  __shared__ SampleWord words[MAX_CLUSTER];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cl::ctarank(), ranks = (int)cl::nctarank();
  cl::cluster_arrive_relaxed();
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x / ranks;
  const T* x = logits + r * ld;
  const float* e = noise + r * ld_noise;
  const Scale sc(temps[r]);
  int k0, k1;
  share<T>(n, rank, ranks, k0, k1);

  Stats st;
  st.init();
  float bx = -INFINITY, be = 1.f, bw = 0.f;  // the thread's candidate: logit, noise, weight against st.m
  int bat = NONE;
  for (int base = k0 + warp * 32; base < k1; base += NT * U) {  // warp-uniform
    uint4 raw[U];
    float ns[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = base + u * NT + lane;
      if (base + u * NT < k1) {
        raw[u] = load_pack<T, VEC>(x, k, n);
        if (!sc.greedy) load_noise<T, VEC>(e, k, n, ns[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * NT >= k1) break;
      const int k = base + u * NT + lane;
      float v[N];
      unpack<T>(raw[u], v);
      if (sc.greedy) {
        fold<N>(st, v, k, sc);
        continue;
      }
      float top = v[0];
#pragma unroll
      for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
      if (top > st.m || (st.at == NONE && top == -FLT_MAX)) {
        top = fminf(top, FLT_MAX);
        st.s *= sc.weight(fmaxf(st.m - top, sc.least));
        st.m = top;
        st.at = k;
        bw = sc.weight_exact(sc.diff(bx, top));
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float w = sc.weight_exact(sc.diff(v[i], st.m)), ei = exponential(ns[u][i]);
        st.s += w;
        if (w * be > bw * ei) {
          bw = w;
          bx = v[i];
          be = ei;
          bat = pack_index<T, VEC>(k, i);
        }
      }
    }
  }
  int first = sc.greedy ? first_maximum<T, VEC>(x, st, n) : NONE;
  // the CTA's maximum, then everything against it
  st.at = first;
  st.merge_warp(sc);
  Best b;
  b.w = bat != NONE ? sc.weight_exact(sc.diff(bx, st.m)) : 0.f;
  b.e = be;
  b.at = bat;
  b.merge_warp();
  // the winning lane's logit travels with it
  const unsigned who = __ballot_sync(0xffffffffu, bat == b.at);
  const float x_best = __shfl_sync(0xffffffffu, bx, __ffs(who) - 1);
  if (lane == 0) {
    wm[warp] = st.m;
    wsum[warp] = st.s;
    wfirst[warp] = st.at;
    wx[warp] = x_best;
    we[warp] = b.e;
    wat[warp] = b.at;
  }
  __syncthreads();
  cl::cluster_wait();  // every CTA of the cluster runs
  auto reduce = [&](int count, auto get) {  // lanes hold entries; result in every lane
    SampleWord w = get(lane < count ? lane : 0);
    if (lane >= count) {
      w.s = 0.f;
      w.m = -FLT_MAX;
      w.at = w.first = NONE;
    }
    Stats a{w.m, w.s, w.first};
    a.merge_warp(sc);
    Best c{w.at != NONE ? sc.weight_exact(sc.diff(w.x, a.m)) : 0.f, w.e, w.at};
    c.merge_warp();
    const unsigned hit = __ballot_sync(0xffffffffu, w.at == c.at);
    w.x = __shfl_sync(0xffffffffu, w.x, __ffs(hit) - 1);
    w.m = a.m;
    w.s = a.s;
    w.first = a.at;
    w.e = c.e;
    w.at = c.at;
    return w;
  };
  if (warp == 0) {
    const SampleWord w = reduce(WARPS, [&](int i) { return SampleWord{wm[i], wsum[i], wx[i], we[i], wat[i], wfirst[i], {0, 0}}; });
    if (lane == 0) {
      const uint32_t to = cl::mapa(&words[rank], 0);
      cl::st_cluster_v4(to, w.m, w.s, w.x, w.e);
      cl::st_cluster_v4(to + 16, __int_as_float(w.at), __int_as_float(w.first), 0.f, 0.f);
    }
  }
  cl::cluster_sync();
  if (rank != 0 || warp != 0) return;
  const SampleWord w = reduce(ranks, [&](int i) { return words[i]; });
  if (lane != 0) return;
  const bool any = w.s > 0.f && (sc.greedy || w.at != NONE);
  const float ln_s = logf(w.s);
  const float xt = sc.greedy ? w.m : w.x;
  const int at = sc.greedy ? w.first : w.at;
  tokens[r] = any ? at : -1;
  if (logprobs) logprobs[r] = any ? sc.diff(xt, w.m) / sc.t - ln_s : 0.f;
  if (lse) lse[r] = any ? w.m / sc.t + ln_s : -INFINITY;
}

// ---- verification: one cluster per sequence -----------------------------------------------------
struct VerifyParams {
  const void* target;
  int64_t ld;
  int n;  // vocabulary
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

constexpr int TILE_ROWS = 16;  // rows whose statistics are taken before their drafts are judged

template <typename T, bool VEC, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) verify_kernel(VerifyParams P) {
  constexpr int N = pack_n<T>(), WARPS = NT / 32, U = 4;
  __shared__ float wm[WARPS][TILE_ROWS], wsum[WARPS][TILE_ROWS];
  __shared__ int wfirst[WARPS][TILE_ROWS];
  __shared__ float cm[TILE_ROWS][MAX_CLUSTER], cs[TILE_ROWS][MAX_CLUSTER];
  __shared__ int cfirst[TILE_ROWS][MAX_CLUSTER];
  __shared__ float rm[TILE_ROWS], rs[TILE_ROWS];  // the rows' statistics over the whole vocabulary
  __shared__ int rfirst[TILE_ROWS];
  __shared__ float id_x[TILE_ROWS], id_q[TILE_ROWS];  // target logit and draft probability of each draft
  __shared__ int id_at[TILE_ROWS];
  __shared__ float bw[WARPS], be[WARPS];
  __shared__ int bat[WARPS];
  __shared__ float cw[2][MAX_CLUSTER], ce[2][MAX_CLUSTER];
  __shared__ int cat[2][MAX_CLUSTER];
  __shared__ int s_count, s_winner;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cl::ctarank(), ranks = (int)cl::nctarank();
  cl::cluster_arrive_relaxed();
  pdl_wait();
  pdl_trigger();
  const int64_t b = blockIdx.x / ranks;
  const int begin = max(0, __ldg(P.cu_q + b)), end = min(P.total_q, __ldg(P.cu_q + b + 1));
  const int drafts = min(end - begin - 1, P.max_drafts);  // -1: an empty sequence
  const Scale sc(P.temps[b]);
  const int n = P.n;
  int k0, k1;
  share<T>(n, rank, ranks, k0, k1);
  int64_t* tokens = P.tokens + b * (P.max_drafts + 1);
  float* logprobs = P.logprobs + b * (P.max_drafts + 1);
  cl::cluster_wait();  // every CTA of the cluster runs

  int count = 0;  // accepted drafts; cluster-uniform from here on
  for (int i0 = 0; i0 <= drafts; i0 += TILE_ROWS) {
    const int rows = min(TILE_ROWS, drafts + 1 - i0);
    const T* x0 = reinterpret_cast<const T*>(P.target) + (int64_t)(begin + i0) * P.ld;
    // what the judgement needs of each draft, asked for before the statistics are taken
    if (tid < rows) {
      const int i = i0 + tid;
      int at = -1;
      float xv = -INFINITY, q = 1.f;
      if (i < drafts) {
        const int64_t id = P.ids[begin + i + 1];
        if (id >= 0 && id < n) {
          at = (int)id;
          xv = as_f32(x0[(int64_t)tid * P.ld + at]);
          if (P.draft) {
            const float xd = as_f32(reinterpret_cast<const T*>(P.draft)[b * P.d_sb + i * P.d_sd + at]);
            const float d = fminf(xd, FLT_MAX) / sc.t - P.draft_lse[b * P.l_sb + i * P.l_sd];
            q = xd == xd ? expf(d) : 0.f;
          }
        }
      }
      id_at[tid] = at;
      id_x[tid] = xv;
      id_q[tid] = q;
    }
    // ---- statistics of the tile's rows over this CTA's share, U packets in flight a thread
    const int np = k0 + warp * 32 < k1 ? (k1 - (k0 + warp * 32) + NT - 1) / NT : 0;  // warp-uniform
    const int total = rows * np;
    Stats st;
    st.init();
    int row = 0, p = 0, lrow = 0, lp = 0;
    auto flush = [&]() {
      if (sc.greedy) st.at = first_maximum<T, VEC>(x0 + (int64_t)row * P.ld, st, n);
      st.merge_warp(sc);
      if (lane == 0) {
        wm[warp][row] = st.m;
        wsum[warp][row] = st.s;
        wfirst[warp][row] = st.at;
      }
      st.init();
      ++row;
      p = 0;
    };
    for (int t = 0; t < total; t += U) {
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t + u < total) {
          raw[u] = load_pack<T, VEC>(x0 + (int64_t)lrow * P.ld, k0 + warp * 32 + lane + lp * NT, n);
          if (++lp == np) {
            lp = 0;
            ++lrow;
          }
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t + u < total) {
          float v[N];
          unpack<T>(raw[u], v);
          fold<N>(st, v, k0 + warp * 32 + lane + p * NT, sc);
          if (++p == np) flush();
        }
    }
    while (row < rows) flush();  // warps without packets
    __syncthreads();
    // warp w merges rows w, w + WARPS, ... over the CTA's warps and tells every CTA
    for (int i = warp; i < rows; i += WARPS) {
      Stats a;
      a.init();
      if (lane < WARPS) a = Stats{wm[lane][i], wsum[lane][i], wfirst[lane][i]};
      a.merge_warp(sc);
      if (lane < ranks) {
        cl::st_cluster_f32(cl::mapa(&cm[i][rank], lane), a.m);
        cl::st_cluster_f32(cl::mapa(&cs[i][rank], lane), a.s);
        cl::st_cluster_f32(cl::mapa(&cfirst[i][rank], lane), __int_as_float(a.at));
      }
    }
    cl::cluster_sync();
    for (int i = warp; i < rows; i += WARPS) {
      Stats a;
      a.init();
      if (lane < ranks) a = Stats{cm[i][lane], cs[i][lane], cfirst[i][lane]};
      a.merge_warp(sc);
      if (lane == 0) {
        rm[i] = a.m;
        rs[i] = a.s;
        rfirst[i] = a.at;
      }
    }
    __syncthreads();
    // ---- judge the tile's drafts: lane = draft; the first refusal ends the run of acceptances
    if (warp == 0) {
      bool ok = false;
      float lp_id = 0.f;
      if (lane < rows && i0 + lane < drafts) {
        const int at = id_at[lane];
        const bool any = rs[lane] > 0.f;
        const float d = sc.diff(id_x[lane], rm[lane]);
        if (sc.greedy)
          ok = any && at == rfirst[lane];
        else
          ok = any && at >= 0 &&
               P.uniforms[b * P.ld_u + i0 + lane] * id_q[lane] < sc.weight_exact(d) / rs[lane];
        lp_id = d / sc.t - logf(rs[lane]);
      }
      const unsigned good = __ballot_sync(0xffffffffu, ok);
      const int run = __ffs(~good) - 1;  // rows <= 16 < 32: a zero bit exists
      if (rank == 0 && lane < run) {
        tokens[i0 + lane] = id_at[lane];
        logprobs[i0 + lane] = lp_id;
      }
      if (lane == 0) s_count = run;
    }
    __syncthreads();
    const int run = s_count;
    count += run;
    if (run == TILE_ROWS && i0 + TILE_ROWS <= drafts) {
      cl::cluster_sync();  // the exchange words are read before the next tile overwrites them
      continue;
    }
    // ---- the token after the accepted drafts, from row `run` of the tile
    const int i = i0 + run;
    const T* x = x0 + (int64_t)run * P.ld;
    const float m = rm[run], s = rs[run];
    int winner = NONE;
    if (sc.greedy) {
      winner = s > 0.f ? rfirst[run] : NONE;
    } else if (s > 0.f) {
      const T* dr = P.draft && i < drafts ? reinterpret_cast<const T*>(P.draft) + b * P.d_sb + i * P.d_sd : nullptr;
      const float dl = dr ? P.draft_lse[b * P.l_sb + i * P.l_sd] : 0.f;
      const float* e = P.noise + b * P.ld_noise;
      const int struck = !P.draft && i < drafts ? id_at[run] : -1;  // a certain draft: q = 1 there
      const float inv = 1.f / s;
      for (int attempt = 0; attempt < 2; ++attempt) {  // the second draws from p: nothing was left
        Best best;
        best.init();
        for (int k = k0 + tid; k < k1; k += NT) {
          float v[N], ns[N];
          const uint4 raw = load_pack<T, VEC>(x, k, n);
          uint4 rawd;
          if (dr) rawd = load_pack<T, VEC>(dr, k, n);
          load_noise<T, VEC>(e, k, n, ns);
          unpack<T>(raw, v);
          float w[N];
#pragma unroll
          for (int c = 0; c < N; ++c) w[c] = sc.weight_exact(sc.diff(v[c], m)) * inv;
          if (attempt == 0 && dr) {
            float d[N];
            unpack<T>(rawd, d);
#pragma unroll
            for (int c = 0; c < N; ++c) {
              const float q = d[c] == d[c] ? expf(fminf(d[c], FLT_MAX) / sc.t - dl) : 0.f;
              w[c] = fmaxf(w[c] - q, 0.f);
            }
          }
#pragma unroll
          for (int c = 0; c < N; ++c) {
            const int at = pack_index<T, VEC>(k, c);
            if (attempt == 0 && at == struck) w[c] = fmaxf(w[c] - 1.f, 0.f);
            const float ei = exponential(ns[c]);
            if (w[c] * best.e > best.w * ei) best = Best{w[c], ei, at};
          }
        }
        best.merge_warp();
        if (lane == 0) {
          bw[warp] = best.w;
          be[warp] = best.e;
          bat[warp] = best.at;
        }
        __syncthreads();
        if (warp == 0) {
          best.init();
          if (lane < WARPS) best = Best{bw[lane], be[lane], bat[lane]};
          best.merge_warp();
          if (lane < ranks) {
            cl::st_cluster_f32(cl::mapa(&cw[attempt][rank], lane), best.w);
            cl::st_cluster_f32(cl::mapa(&ce[attempt][rank], lane), best.e);
            cl::st_cluster_f32(cl::mapa(&cat[attempt][rank], lane), __int_as_float(best.at));
          }
        }
        cl::cluster_sync();
        if (warp == 0) {
          best.init();
          if (lane < ranks) best = Best{cw[attempt][lane], ce[attempt][lane], cat[attempt][lane]};
          best.merge_warp();
          if (lane == 0) s_winner = best.at;
        }
        __syncthreads();
        winner = s_winner;
        if (winner != NONE) break;
      }
    }
    if (rank == 0 && tid == 0) {
      tokens[i] = winner != NONE ? winner : -1;
      logprobs[i] = winner != NONE ? sc.diff(as_f32(x[winner]), m) / sc.t - logf(s) : 0.f;
    }
    break;
  }
  if (rank == 0) {
    const int written = drafts < 0 ? 0 : count + 1;
    for (int i = written + tid; i <= P.max_drafts; i += NT) {
      tokens[i] = -1;
      logprobs[i] = 0.f;
    }
    if (tid == 0) P.accepted[b] = count;
  }
}

// ---- launch ------------------------------------------------------------------------------------
// CTAs per row: as many as fill the SMs' 2,048 resident threads once (592 CTAs of 256), so that few
// rows still pull from all of HBM, but no less than 2,048 logits a CTA (below that the exchange
// costs more than the reading saves).  Up to 148 CTAs in all take 1,024 threads each.
struct Split {
  int ctas;
  bool wide;
};
inline Split split_for(int64_t rows, int64_t vocab) {
  int c = 1;
  while (c < MAX_CLUSTER && rows * (2 * c) <= (c < 8 ? 592 : 148) && vocab >= 2048 * 2 * c) c *= 2;
  return {c, rows * c <= 148};
}

template <auto Kernel, typename... Args>
inline int launch(int64_t rows, const Split& sp, cudaStream_t st, Args... args) {
  if (sp.ctas > 8) {  // set once per device
    static std::atomic<bool> done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ADA_ERR_CUDA;
    if (!done[dev]) {
      if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return ADA_ERR_CUDA;
      done[dev] = true;
    }
  }
  (void)ada::launch_kc(Kernel, dim3((unsigned)(rows * sp.ctas)), dim3(sp.wide ? 1024 : 256), 0, st, sp.ctas, args...);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}

inline bool on16(const void* p, int64_t stride_bytes) { return (((uintptr_t)p | (uintptr_t)stride_bytes) & 15) == 0; }
inline bool dtype_ok(int d) { return d == ADA_DT_BF16 || d == ADA_DT_F16 || d == ADA_DT_F32; }
inline int dtype_size(int d) { return d == ADA_DT_F32 ? 4 : 2; }
inline bool misaligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype_size(dtype) - 1)) != 0; }

template <typename T, bool VEC, typename... Args>
int sample_typed(int64_t rows, int64_t vocab, cudaStream_t st, const void* logits, Args... args) {
  const Split sp = split_for(rows, vocab);
  return sp.wide ? launch<sample_kernel<T, VEC, 1024>>(rows, sp, st, (const T*)logits, args...)
                 : launch<sample_kernel<T, VEC, 256>>(rows, sp, st, (const T*)logits, args...);
}
template <typename T, bool VEC>
int verify_typed(int64_t batch, const VerifyParams& P, cudaStream_t st) {
  const Split sp = split_for(batch, P.n);
  return sp.wide ? launch<verify_kernel<T, VEC, 1024>>(batch, sp, st, P)
                 : launch<verify_kernel<T, VEC, 256>>(batch, sp, st, P);
}

}  // namespace smp
}  // namespace ada

using namespace ada;

extern "C" int ada_sample(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab,
                          const float* temperatures, const float* noise, int64_t ld_noise, int64_t* tokens,
                          float* logprobs, float* lse, void* stream) {
  if (rows < 0 || vocab <= 0 || ld < vocab || ld_noise < vocab || !smp::dtype_ok(dtype)) return ADA_ERR_INVALID_ARG;
  if (rows == 0) return ADA_OK;
  if (!logits || !temperatures || !noise || !tokens) return ADA_ERR_INVALID_ARG;
  if (vocab > (1 << 30) || rows > (1 << 20)) return ADA_ERR_UNSUPPORTED;
  if (smp::misaligned(logits, dtype) || ((uintptr_t)noise & 3) || ((uintptr_t)temperatures & 3) ||
      ((uintptr_t)tokens & 7) || ((uintptr_t)logprobs & 3) || ((uintptr_t)lse & 3))
    return ADA_ERR_ALIGNMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = smp::on16(logits, ld * smp::dtype_size(dtype)) && smp::on16(noise, ld_noise * 4);
#define ADA_SAMPLE(T)                                                                                             \
  return vec ? smp::sample_typed<T, true>(rows, vocab, st, logits, ld, (int)vocab, temperatures, noise, ld_noise, \
                                          tokens, logprobs, lse)                                                  \
             : smp::sample_typed<T, false>(rows, vocab, st, logits, ld, (int)vocab, temperatures, noise, ld_noise, \
                                           tokens, logprobs, lse)
  if (dtype == ADA_DT_BF16) ADA_SAMPLE(__nv_bfloat16);
  if (dtype == ADA_DT_F16) ADA_SAMPLE(__half);
  ADA_SAMPLE(float);
#undef ADA_SAMPLE
}

extern "C" int ada_verify_drafts(const void* target, int dtype, int64_t ld, int32_t total_q, int64_t vocab,
                                 const int64_t* input_ids, const int32_t* cu_seqlens_q, int32_t batch,
                                 int32_t max_drafts, const float* temperatures, const float* uniforms, int64_t ld_u,
                                 const float* noise, int64_t ld_noise, const void* draft_logits,
                                 int64_t draft_stride_b, int64_t draft_stride_d, const float* draft_lse,
                                 int64_t lse_stride_b, int64_t lse_stride_d, int64_t* tokens, int32_t* accepted,
                                 float* logprobs, void* stream) {
  if (batch < 0 || total_q < 0 || max_drafts < 0 || vocab <= 0 || ld < vocab || ld_noise < vocab ||
      ld_u < max_drafts || !smp::dtype_ok(dtype))
    return ADA_ERR_INVALID_ARG;
  if (batch == 0) return ADA_OK;
  if ((!target && total_q > 0) || (!input_ids && total_q > 0) || !cu_seqlens_q || !temperatures || !noise || !tokens ||
      !accepted || !logprobs || (!uniforms && max_drafts > 0))
    return ADA_ERR_INVALID_ARG;
  if ((draft_logits == nullptr) != (draft_lse == nullptr)) return ADA_ERR_INVALID_ARG;
  if (draft_logits && (draft_stride_b < 0 || draft_stride_d < 0 || lse_stride_b < 0 || lse_stride_d < 0))
    return ADA_ERR_INVALID_ARG;
  if (vocab > (1 << 30) || batch > (1 << 20) || max_drafts > 1024) return ADA_ERR_UNSUPPORTED;
  if (smp::misaligned(target, dtype) || smp::misaligned(draft_logits, dtype) || ((uintptr_t)noise & 3) ||
      ((uintptr_t)temperatures & 3) || ((uintptr_t)uniforms & 3) || ((uintptr_t)draft_lse & 3) ||
      ((uintptr_t)input_ids & 7) || ((uintptr_t)cu_seqlens_q & 3) || ((uintptr_t)tokens & 7) ||
      ((uintptr_t)accepted & 3) || ((uintptr_t)logprobs & 3))
    return ADA_ERR_ALIGNMENT;
  smp::VerifyParams P;
  P.target = target;
  P.ld = ld;
  P.n = (int)vocab;
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
  const int size = smp::dtype_size(dtype);
  const bool vec = smp::on16(target, ld * size) && smp::on16(noise, ld_noise * 4) &&
                   (!draft_logits || smp::on16(draft_logits, (draft_stride_b | draft_stride_d) * size));
  if (dtype == ADA_DT_BF16)
    return vec ? smp::verify_typed<__nv_bfloat16, true>(batch, P, st)
               : smp::verify_typed<__nv_bfloat16, false>(batch, P, st);
  if (dtype == ADA_DT_F16)
    return vec ? smp::verify_typed<__half, true>(batch, P, st) : smp::verify_typed<__half, false>(batch, P, st);
  return vec ? smp::verify_typed<float, true>(batch, P, st) : smp::verify_typed<float, false>(batch, P, st);
}
