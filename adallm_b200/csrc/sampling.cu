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
// Bound: HBM (a logit costs 2 or 4 bytes and about ten instructions).  A row is read once: a warp
// keeps a running maximum m of its raw logits and each lane its sum of 2^((x - m) c),
// c = log2(e) / T; x - m is exact or nearly so where the weight matters, so the statistics do not pay
// for the size of x.  Sampling takes one thread-block cluster per row, each CTA a share of the
// vocabulary; the CTAs meet in distributed shared memory, so a call is one launch without a
// workspace.
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
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
// A packet's values with NaN replaced by -inf (a maximum takes the operand that is a number), and
// their maximum.
template <typename H2> __device__ __forceinline__ float unpack_halves(const uint4& u, H2 low, float* f) {
  H2 h[4];
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmax2(*reinterpret_cast<const H2*>(&w[i]), low);
  const H2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = as_f32(h[i].x);
    f[2 * i + 1] = as_f32(h[i].y);
  }
  return fmaxf(as_f32(m.x), as_f32(m.y));
}
template <typename T> __device__ __forceinline__ float unpack(const uint4& u, float* f) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return unpack_halves(u, __halves2bfloat162(minus_inf<T>(), minus_inf<T>()), f);
  } else if constexpr (std::is_same<T, __half>::value) {
    return unpack_halves(u, __halves2half2(minus_inf<T>(), minus_inf<T>()), f);
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = fmaxf(__uint_as_float(w[i]), -INFINITY);
    return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
  }
}
// Raw element i of a packet.
template <typename T> __device__ __forceinline__ float element(const uint4& u, int i) {
  return as_f32(reinterpret_cast<const T*>(&u)[i]);
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
    constexpr float L = 1.4426950408889634f, L_LO = (float)(1.4426950408889634 - (double)1.4426950408889634f);
    greedy = !(temp > 1e-10f);
    t = greedy ? 1.f : temp;
    c = L / t;
    c_lo = (fmaf(-c, t, L) + L_LO) / t;
    least = -138.62944f * t;  // -200 ln 2 T
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

// Maximum and sum of a set of logits: s = sum 2^((x - m) c); at = the index of the first maximum
// (greedy rows).
struct Stats {
  float m, s;
  int at;
  __device__ __forceinline__ void merge(float m2, float s2, int at2, const Scale& sc) {
    const float top = fmaxf(m, m2);
    at = m == m2 ? min(at, at2) : (m > m2 ? at : at2);
    s = s * sc.weight(sc.diff(m, top)) + s2 * sc.weight(sc.diff(m2, top));
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
};
__device__ __forceinline__ Stats no_stats() { return Stats{-FLT_MAX, 0.f, NONE}; }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// A warp's statistics while it reads a row.  The maximum is the warp's (it moves a handful of times
// a row, found by one vote a packet), so a logit costs half a cleaning and half a maximum (packed
// 16-bit), its widening, half a difference and half a product (f32x2), an ex2 and half an add.
struct Fold {
  float m;       // the warp's maximum
  float2 s;      // this lane's sum against it, in two parts
  float top;     // this lane's own maximum and the packet that first held it (greedy rows)
  int top_pack;
  __device__ __forceinline__ void init() {
    m = -FLT_MAX;
    s = make_float2(0.f, 0.f);
    top = -INFINITY;
    top_pack = NONE;
  }
  // Fold packet k with values v and maximum `most` in; every lane of the warp calls.  w: the
  // packet's weights against m.  Returns whether m moved.
  template <int N>
  __device__ __forceinline__ bool add(float* v, float most, int k, const Scale& sc, float* w) {
    const float reach = fminf(most, FLT_MAX);  // +inf is the largest float: no later maximum than one of that
    if (reach > top) {
      top = reach;
      top_pack = k;
    }
    const bool moved = __any_sync(0xffffffffu, most > m);
    if (moved) {
      float to = warp_max(most);
      if (to > FLT_MAX) {  // +inf among them: read as the largest float (such a packet always gets here)
        to = FLT_MAX;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = fminf(v[i], FLT_MAX);
      }
      const float by = sc.weight(sc.diff(m, to));
      s = mul2(s, make_float2(by, by));
      m = to;
    }
    const float2 off = make_float2(-m, -m), c2 = make_float2(sc.c, sc.c);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 y = mul2(add2(make_float2(v[i], v[i + 1]), off), c2);  // -inf stays -inf: weight 0
      w[i] = fast_exp2(y.x);
      w[i + 1] = fast_exp2(y.y);
      s = add2(s, make_float2(w[i], w[i + 1]));
    }
    return moved;
  }
  // The warp's statistics, in every lane.
  template <typename T, bool VEC>
  __device__ __forceinline__ Stats finish(const T* x, int n, const Scale& sc) const {
    Stats st{m, s.x + s.y, NONE};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
    if (sc.greedy) {
      if (top_pack != NONE && top >= m) {
        float v[pack_n<T>()];
        unpack<T>(load_pack<T, VEC>(x, top_pack, n), v);
#pragma unroll
        for (int i = pack_n<T>() - 1; i >= 0; --i)
          if (v[i] >= m) st.at = pack_index<T, VEC>(top_pack, i);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) st.at = min(st.at, __shfl_xor_sync(0xffffffffu, st.at, o));
    }
    return st;
  }
};

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
// How far a score that filters candidates is lowered: above the roundings of the weights it is made of.
constexpr float SLACK = 1.f - 1.f / 16384.f;
__device__ __forceinline__ unsigned long long pack2(float a, float b) {
  return ((unsigned long long)__float_as_uint(b) << 32) | __float_as_uint(a);
}
__device__ __forceinline__ float2 unpack2(unsigned long long v) {
  return make_float2(__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32)));
}
__device__ __forceinline__ float exponential(float e) { return fmaxf(e, 1e-10f); }

// Probability of a draft's logit given its row's log-normaliser (-inf and NaN: 0, +inf: the largest float).
// Below temperature 1 the largest floats' quotients, of either sign, and with them the normaliser, stop at the
// largest float.
__device__ __forceinline__ float divided(float x, float t) { return fminf(fmaxf(x / t, -FLT_MAX), FLT_MAX); }
__device__ __forceinline__ float draft_prob(float x, const Scale& sc, float lse) {
  return x >= -FLT_MAX ? expf(divided(x, sc.t) - (lse > FLT_MAX ? FLT_MAX : lse)) : 0.f;
}

// This CTA's packets [k0, k1) of a row of n elements, in shares of whole warps.
template <typename T> __device__ __forceinline__ void share(int n, int rank, int ranks, int& k0, int& k1) {
  constexpr int N = pack_n<T>();
  const int packs = ((n + 32 * N - 1) / (32 * N)) * 32;
  const int per = ((packs / 32 + ranks - 1) / ranks) * 32;
  k0 = min(rank * per, packs);
  k1 = min(k0 + per, packs);
}

// ---- sampling: one cluster per row -------------------------------------------------------------
// 64 rows of 151,936 bf16 logits (58 MB with the noise): 14.9 us, 3.9 TB/s = 0.60 of a measured copy, bound by
// the instructions of a logit and the start and end of a 15 us kernel; one row 7.0 us, a chain of latencies
// (launch, one read, the cluster's exchange).  The statistics and the race share one read of the row, which
// is why the race filters by a score shared as raw numbers: the row's maximum is not known yet.
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
  __shared__ SampleWord mine[WARPS], words[MAX_CLUSTER];
  __shared__ unsigned long long bound;  // (maximum, score): see below
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cl::ctarank(), ranks = (int)cl::nctarank();
  cl::cluster_arrive_relaxed();
  if (threadIdx.x == 0) bound = pack2(-FLT_MAX, 0.f);
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x / ranks;
  const T* x = logits + r * ld;
  const float* e = noise + r * ld_noise;
  const Scale sc(temps[r]);
  int k0, k1;
  share<T>(n, rank, ranks, k0, k1);

  // The race.  A lane keeps its best (logit, noise), with its weight against the warp's maximum;
  // the CTA shares a score that some lane has reached, with the maximum that it is against, so only
  // a few packets a row hold anything that could still win and are looked at element by element.
  Fold f;
  f.init();
  float bx = -INFINITY, be = 1.f, bw = 0.f;
  int bat = NONE;
  // U packets a lane are in flight: each is asked for again as soon as it has been used
  uint4 raw[U];
  float ns[U][N];
  auto load = [&](int u, int base) {
    if (base >= k1) return;
    raw[u] = load_pack<T, VEC>(x, base + lane, n);
    if (!sc.greedy) load_noise<T, VEC>(e, base + lane, n, ns[u]);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, k0 + warp * 32 + u * NT);
  for (int base = k0 + warp * 32; base < k1; base += NT * U) {  // warp-uniform
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * NT >= k1) break;
      const int k = base + u * NT + lane;
      float v[N], w[N];
      const float most = unpack<T>(raw[u], v);
      const bool moved = f.add<N>(v, most, k, sc, w);
      if (!sc.greedy) {
        if (moved) bw = sc.weight(sc.diff(bx, f.m));
        const float2 known = unpack2(*const_cast<volatile unsigned long long*>(&bound));
        const float score = known.y * sc.weight(known.x - f.m);  // against f.m
        const float least = score * SLACK;
        bool hit = false;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float2 t = mul2(make_float2(ns[u][i], ns[u][i + 1]), make_float2(least, least));
          hit |= !(w[i] <= t.x) | !(w[i + 1] <= t.y);
        }
        if (__any_sync(0xffffffffu, hit)) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float ei = exponential(ns[u][i]);
            if (w[i] * be > bw * ei) {
              bw = w[i];
              bx = v[i];
              be = ei;
              bat = pack_index<T, VEC>(k, i);
            }
          }
          const float reached = warp_max(bw / be);
          if (lane == 0 && reached > score) *const_cast<volatile unsigned long long*>(&bound) = pack2(f.m, reached);
        }
      }
      load(u, base + (u + U) * NT);
    }
  }
  // entries (statistics, candidate) of a warp's lanes -> their merge, in every lane
  auto reduce = [&](SampleWord w) {
    Stats a{w.m, w.s, w.first};
    a.merge_warp(sc);
    Best c{w.at != NONE ? sc.weight(sc.diff(w.x, a.m)) : 0.f, w.e, w.at};
    c.merge_warp();
    const unsigned hit = __ballot_sync(0xffffffffu, w.at == c.at);
    return SampleWord{a.m, a.s, __shfl_sync(0xffffffffu, w.x, __ffs(hit) - 1), c.e, c.at, a.at, {0, 0}};
  };
  {
    const Stats st = f.finish<T, VEC>(x, n, sc);
    SampleWord w{st.m, lane == 0 ? st.s : 0.f, bx, be, bat, st.at, {0, 0}};
    w = reduce(w);
    if (lane == 0) mine[warp] = w;
  }
  __syncthreads();
  cl::cluster_wait();  // every CTA of the cluster runs
  const SampleWord nothing{-FLT_MAX, 0.f, -INFINITY, 1.f, NONE, NONE, {0, 0}};
  if (warp == 0) {
    const SampleWord w = reduce(lane < WARPS ? mine[lane] : nothing);
    if (lane == 0) {
      const uint32_t to = cl::mapa(&words[rank], 0);
      cl::st_cluster_v4(to, w.m, w.s, w.x, w.e);
      cl::st_cluster_v4(to + 16, __int_as_float(w.at), __int_as_float(w.first), 0.f, 0.f);
    }
  }
  cl::cluster_sync();
  if (rank != 0 || warp != 0) return;
  const SampleWord w = reduce(lane < ranks ? words[lane] : nothing);
  if (lane != 0) return;
  const int at = sc.greedy ? w.first : w.at;
  const bool any = w.s > 0.f;
  const float ln_s = logf(w.s);
  tokens[r] = any && at != NONE ? at : -1;
  if (logprobs) logprobs[r] = any ? sc.diff(sc.greedy ? w.m : w.x, w.m) / sc.t - ln_s : 0.f;
  if (lse) lse[r] = any ? divided(w.m, sc.t) + ln_s : -INFINITY;
}

// ---- verification ---------------------------------------------------------------------------------
// Two kernels: the statistics of every target row, then the draw from one row of every sequence
// (by then in L2).  In both any CTA takes any share of any row, so ragged numbers of drafts cost no
// balance; in the second each CTA judges its sequence's drafts for itself (a few words) and the
// shares meet in one 64-bit atomic maximum of (score, lowest index), whose order does not matter.
// 230 rows of 151,936 bf16 logits for 64 sequences (128 MB): 38.8 us.  The statistics take 21 us, 3.3 TB/s = 0.51 of
// a measured copy, issue slots 0.66 busy (12 instructions a logit, fixed costs of a warp's share included);
// the draw about 20, of which the judging, a chain of dependent reads, is 6 to 8 before its first load.
struct VerifyParams {
  const void* target;
  int64_t ld;
  int n;  // vocabulary
  const int64_t* ids;
  const int32_t* cu_q;
  int32_t batch, total_q, max_drafts;
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
  float4* part;  // [total_q][chunks]: maximum, sum, first maximum
  int32_t chunks, chunk_packs;
  unsigned long long* best;  // [batch]: score bits << 32 | ~index; 0: no candidate yet
  unsigned int* done;        // [batch]: shares drawn
  int32_t draw_chunks, draw_packs;
};
constexpr int STAT_THREADS = 256;

// Warp-wide: how many entries of the ascending list cu[0..count) are <= x, 32 probes at a time.
__device__ __forceinline__ int count_up_to(const int32_t* cu, int count, int x) {
  const int lane = threadIdx.x & 31;
  int lo = 0, end = count;
  while (lo < end) {
    const int step = (end - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool below = at < end && __ldg(cu + min(at + step, end) - 1) <= x;
    const int blocks = __popc(__ballot_sync(0xffffffffu, below));
    lo = min(lo + blocks * step, end);
    if (step == 1) break;
    end = min(lo + step, end);
  }
  return lo;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(STAT_THREADS, 4) row_stats_kernel(VerifyParams P) {
  constexpr int N = pack_n<T>(), WARPS = STAT_THREADS / 32, U = 4;
  __shared__ Stats mine[WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x == 0)  // the draw's words, for the kernel after this one
    for (int i = threadIdx.x; i < P.batch; i += STAT_THREADS) {
      P.best[i] = 0;
      P.done[i] = 0;
    }
  const int row = blockIdx.x / P.chunks, chunk = blockIdx.x % P.chunks;
  if (row >= P.total_q) return;  // a call without rows
  const T* x = reinterpret_cast<const T*>(P.target) + (int64_t)row * P.ld;
  const int k0 = chunk * P.chunk_packs, k1 = k0 + P.chunk_packs;  // packets past the row's end are -inf
  uint4 raw[U];
  auto load = [&](int u, int base) {
    if (base < k1) raw[u] = load_pack<T, VEC>(x, base + lane, P.n);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, k0 + warp * 32 + u * STAT_THREADS);
  const int seq = count_up_to(P.cu_q, P.batch + 1, row) - 1;
  if (seq < 0 || seq >= P.batch || row - __ldg(P.cu_q + seq) > P.max_drafts) return;  // no one asks for this row
  const Scale sc(P.temps[seq]);
  Fold f;
  f.init();
  for (int base = k0 + warp * 32; base < k1; base += STAT_THREADS * U) {  // warp-uniform
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * STAT_THREADS >= k1) break;
      float v[N], w[N];
      const float most = unpack<T>(raw[u], v);
      f.add<N>(v, most, base + u * STAT_THREADS + lane, sc, w);
      load(u, base + (u + U) * STAT_THREADS);
    }
  }
  const Stats st = f.finish<T, VEC>(x, P.n, sc);
  if (lane == 0) mine[warp] = st;
  __syncthreads();
  if (warp == 0) {
    Stats a = lane < WARPS ? mine[lane] : no_stats();
    a.merge_warp(sc);
    if (lane == 0) P.part[blockIdx.x] = make_float4(a.m, a.s, __int_as_float(a.at), 0.f);
  }
}

// A share of the race for one token: the candidates of packets [k0, k1) of a row, weights
// max(p - q, 0), returned as (score bits << 32 | ~index) in every lane of the warp; 0: none.  `known`
// is a score that some share has reached.  p bounds what is left of it, so elements whose p / e does not
// reach that score are done with; the others (about 1 / (1 - a) of a row's tokens, where a is the chance
// that the draft was accepted) take q into account.  Every thread of the CTA calls.
template <typename T, bool VEC, int NT>
__device__ __forceinline__ unsigned long long draw_share(const T* x, const T* dr, const float* e, int n, int k0, int k1,
                                                         const Scale& sc, float m, float s, float dl, int struck,
                                                         volatile int* known) {
  constexpr int N = pack_n<T>(), U = 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float inv = 1.f / s;
  Best best;
  best.init();
  uint4 raw[U], rawd[U];
  float ns[U][N];
  auto load = [&](int u, int base) {
    if (base >= k1) return;
    raw[u] = load_pack<T, VEC>(x, base + lane, n);
    if (dr) rawd[u] = load_pack<T, VEC>(dr, base + lane, n);
    load_noise<T, VEC>(e, base + lane, n, ns[u]);
  };
  auto consider = [&](float v, float d, float noise, int at) {
    float w = sc.weight_exact(sc.diff(v, m)) * inv;
    if (dr) w = fmaxf(w - draft_prob(d, sc, dl), 0.f);
    if (at == struck) w = fmaxf(w - 1.f, 0.f);
    const float ei = exponential(noise);
    if (w * best.e > best.w * ei) best = Best{w, ei, at};
  };
  auto publish = [&](float score) {
    const float reached = warp_max(best.w / best.e);
    if (lane == 0 && reached > score) atomicMax(const_cast<int*>(known), __float_as_int(reached));
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, k0 + warp * 32 + u * NT);
  // A first bound: of each lane's first packet the element with the largest p / e.
  if (k0 + warp * 32 < k1) {
    float v[N], most = -1.f, mv = 0.f, md = 0.f, me = 1.f;
    int mi = 0;
    unpack<T>(raw[0], v);
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const float r = __fdividef(sc.weight(sc.diff(v[c], m)), exponential(ns[0][c]));
      if (r > most) {
        most = r;
        mv = v[c];
        md = dr ? element<T>(rawd[0], c) : 0.f;
        me = ns[0][c];
        mi = c;
      }
    }
    consider(mv, md, me, pack_index<T, VEC>(k0 + warp * 32 + lane, mi));
    publish(0.f);
  }
  __syncthreads();
  for (int base = k0 + warp * 32; base < k1; base += NT * U) {  // warp-uniform
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * NT >= k1) break;
      const int k = base + u * NT + lane;
      const float score = __int_as_float(*known);
      const float least = score * SLACK * s;  // against s p
      float v[N];
      unpack<T>(raw[u], v);
      unsigned hits = 0;
#pragma unroll
      for (int c = 0; c < N; c += 2) {
        const float2 t = mul2(make_float2(ns[u][c], ns[u][c + 1]), make_float2(least, least));
        hits |= !(sc.weight(sc.diff(v[c], m)) <= t.x) ? 1u << c : 0u;
        hits |= !(sc.weight(sc.diff(v[c + 1], m)) <= t.y) ? 2u << c : 0u;
      }
      const unsigned any = __reduce_or_sync(0xffffffffu, hits);
      if (any) {
#pragma unroll
        for (int c = 0; c < N; ++c)
          if ((any >> c) & 1u)  // warp-uniform: the few places where some lane has a candidate
            consider(v[c], dr ? element<T>(rawd[u], c) : 0.f, ns[u][c], pack_index<T, VEC>(k, c));
        publish(score);
      }
      load(u, base + (u + U) * NT);
    }
  }
  unsigned long long word =
      best.at == NONE ? 0ull : ((unsigned long long)__float_as_uint(best.w / best.e) << 32) | (unsigned)~best.at;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, word, o);
    word = other > word ? other : word;
  }
  return word;
}

constexpr int TILE_ROWS = 16;  // rows judged at a time
constexpr int DRAW_THREADS = 256;

template <typename T, bool VEC>
__global__ void __launch_bounds__(DRAW_THREADS, 3) draw_kernel(VerifyParams P) {
  constexpr int WARPS = DRAW_THREADS / 32;
  __shared__ Stats rows_s[TILE_ROWS];  // over the whole vocabulary
  __shared__ float id_x[TILE_ROWS], id_q[TILE_ROWS], id_u[TILE_ROWS];  // of each draft: target logit, q, uniform
  __shared__ int id_at[TILE_ROWS];
  __shared__ unsigned long long words[WARPS];
  __shared__ int s_count, s_last;
  __shared__ int s_known;  // bits of a score that the race has reached (scores are >= 0)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // The kernel before this one (the row statistics) has waited for its predecessors before it let
  // this one start: all inputs are settled, only its own results are waited for below.
  const int64_t b = blockIdx.x / P.draw_chunks;
  const int chunk = blockIdx.x % P.draw_chunks;
  const int begin = min(max(0, __ldg(P.cu_q + b)), P.total_q), end = min(max(0, __ldg(P.cu_q + b + 1)), P.total_q);
  const int drafts = min(end - begin - 1, P.max_drafts);  // -1: an empty sequence
  const Scale sc(P.temps[b]);
  int64_t* tokens = P.tokens + b * (P.max_drafts + 1);
  float* logprobs = P.logprobs + b * (P.max_drafts + 1);
  bool waited = false;

  int count = 0;  // accepted drafts
  int run = 0;
  for (int i0 = 0; i0 <= drafts; i0 += TILE_ROWS) {
    const int rows = min(TILE_ROWS, drafts + 1 - i0);
    const T* x0 = reinterpret_cast<const T*>(P.target) + (int64_t)(begin + i0) * P.ld;
    if (tid < rows) {
      const int i = i0 + tid;
      int at = -1;
      float xv = -INFINITY, q = 1.f, un = 0.f;
      if (i < drafts) {
        const int64_t id = P.ids[begin + i + 1];
        un = P.uniforms[b * P.ld_u + i];
        if (id >= 0 && id < P.n) {
          at = (int)id;
          xv = as_f32(x0[(int64_t)tid * P.ld + at]);
          if (P.draft)
            q = draft_prob(as_f32(reinterpret_cast<const T*>(P.draft)[b * P.d_sb + i * P.d_sd + at]), sc,
                           P.draft_lse[b * P.l_sb + i * P.l_sd]);
        }
      }
      id_at[tid] = at;
      id_x[tid] = xv;
      id_q[tid] = q;
      id_u[tid] = un;
    }
    if (!waited) {
      pdl_wait();
      pdl_trigger();
      waited = true;
      if (tid == 0) s_known = (int)(*const_cast<volatile unsigned long long*>(P.best + b) >> 32);
    }
    for (int i = warp; i < rows; i += WARPS) {
      Stats a = no_stats();
      const float4* part = P.part + (int64_t)(begin + i0 + i) * P.chunks;
      for (int c = lane; c < P.chunks; c += 32) {
        const float4 w = part[c];
        a.merge(w.x, w.y, __float_as_int(w.z), sc);
      }
      a.merge_warp(sc);
      if (lane == 0) rows_s[i] = a;
    }
    __syncthreads();
    // ---- judge the tile's drafts: lane = draft; the first refusal ends the run of acceptances
    if (warp == 0) {
      bool ok = false;
      float lp = 0.f;
      if (lane < rows && i0 + lane < drafts) {
        const int at = id_at[lane];
        const Stats st = rows_s[lane];
        const float d = sc.diff(id_x[lane], st.m);
        ok = st.s > 0.f && at >= 0 &&
             (sc.greedy ? at == st.at : id_u[lane] * id_q[lane] < sc.weight_exact(d) / st.s);
        lp = d / sc.t - logf(st.s);
      }
      const unsigned good = __ballot_sync(0xffffffffu, ok);
      const int ran = __ffs(~good) - 1;  // rows <= 16 < 32: a zero bit exists
      if (chunk == 0 && lane < ran) {
        tokens[i0 + lane] = id_at[lane];
        logprobs[i0 + lane] = lp;
      }
      if (lane == 0) s_count = ran;
    }
    __syncthreads();
    run = s_count;
    count += run;
    if (run < TILE_ROWS) break;
    __syncthreads();  // every row's draft was accepted: the next tile (it exists)
  }
  if (!waited) {
    pdl_wait();
    pdl_trigger();
  }
  if (chunk == 0) {
    for (int i = (drafts < 0 ? 0 : count + 1) + tid; i <= P.max_drafts; i += DRAW_THREADS) {
      tokens[i] = -1;
      logprobs[i] = 0.f;
    }
    if (tid == 0) P.accepted[b] = count;
  }
  if (drafts < 0) return;
  // ---- the token after the accepted drafts: row `count`, row `run` of the last tile
  const T* x = reinterpret_cast<const T*>(P.target) + (int64_t)(begin + count) * P.ld;
  const Stats st = rows_s[run];
  auto finish = [&](int winner) {  // (a list that does not ascend leaves rows without statistics, and any winner)
    const bool any = winner >= 0 && winner < P.n;
    tokens[count] = any ? winner : -1;
    logprobs[count] = any ? sc.diff(as_f32(x[winner]), st.m) / sc.t - logf(st.s) : 0.f;
  };
  if (sc.greedy || !(st.s > 0.f)) {
    if (chunk == 0 && tid == 0) finish(st.s > 0.f ? st.at : NONE);
    return;
  }
  const bool refused = count < drafts;
  const T* dr = P.draft && refused ? reinterpret_cast<const T*>(P.draft) + b * P.d_sb + count * P.d_sd : nullptr;
  const float dl = dr ? P.draft_lse[b * P.l_sb + count * P.l_sd] : 0.f;
  const float* e = P.noise + b * P.ld_noise;
  const int struck = !P.draft && refused ? id_at[run] : -1;  // a certain draft: q = 1 there
  const int k0 = chunk * P.draw_packs;
  unsigned long long word =
      draw_share<T, VEC, DRAW_THREADS>(x, dr, e, P.n, k0, k0 + P.draw_packs, sc, st.m, st.s, dl, struck, &s_known);
  if (lane == 0) words[warp] = word;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < WARPS; ++i) word = words[i] > word ? words[i] : word;
    if (word) atomicMax(P.best + b, word);
    __threadfence();
    s_last = atomicAdd(P.done + b, 1u) == (unsigned)P.draw_chunks - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  word = *const_cast<volatile unsigned long long*>(P.best + b);
  if (!word && refused) {  // nothing was left anywhere: the token is drawn from p
    if (tid == 0) s_known = 0;
    __syncthreads();
    word = draw_share<T, VEC, DRAW_THREADS>(x, nullptr, e, P.n, 0, (int)cdiv(P.n, 32 * pack_n<T>()) * 32, sc, st.m, st.s,
                                            0.f, -1, &s_known);
    if (lane == 0) words[warp] = word;
    __syncthreads();
    for (int i = 0; i < WARPS; ++i) word = words[i] > word ? words[i] : word;
  }
  if (tid == 0) finish(word ? (int)~(unsigned)word : NONE);
}

// ---- launch ------------------------------------------------------------------------------------
// CTAs per row of the sampling kernel: as many as fill the SMs' threads once (592 CTAs of 256; 512 in
// clusters of 16, which have to fit a GPC), so that few rows still pull from all of HBM, but no less
// than 2,048 logits a CTA (below that the exchange costs more than the reading saves).  Up to 148
// CTAs in all take 1,024 threads each.
struct Split {
  int ctas;
  bool wide;
};
inline Split split_for(int64_t rows, int64_t vocab) {
  int c = 1;
  while (c < MAX_CLUSTER && rows * (2 * c) <= (c < 8 ? 592 : 512) && vocab >= 2048 * 2 * c) c *= 2;
  return {c, rows * c <= 148};
}

// Shares of a row in the verification kernels (256 threads, `resident` CTAs on the card at once): what
// takes least if a wave of CTAs takes `fixed` + the packets a thread of one of its shares reads, up to four
// waves, at least one packet a thread.  Nothing fixed for the row statistics; for the draw the judging of
// the drafts, about 8 us or 12 packets: 100 sequences of 3 rows of 151936 in one wave 49 us, in four full
// ones 62.
inline void row_shares(int64_t rows, int64_t vocab, int pack, int64_t resident, int64_t fixed, int* chunks,
                       int* packs) {
  const int64_t units = cdiv(vocab, 256 * pack);  // packets a thread of a lone CTA
  int64_t best = units, least = INT64_MAX;        // packets a thread of a share, its cost
  for (int w = 1; w <= 4; ++w) {
    int64_t c = rows > 0 ? w * resident / rows : 1;
    c = c < 1 ? 1 : (c > units ? units : c);
    const int64_t per = cdiv(units, c), cost = cdiv(rows * cdiv(units, per), resident) * (per + fixed);
    if (cost < least) {
      least = cost;
      best = per;
    }
  }
  *packs = (int)best * 256;
  *chunks = (int)cdiv(units, best);
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
int verify_typed(VerifyParams P, cudaStream_t st) {
  const unsigned stat_ctas = (unsigned)P.total_q * P.chunks;
  (void)ada::launch_k(row_stats_kernel<T, VEC>, dim3(stat_ctas ? stat_ctas : 1), dim3(STAT_THREADS), 0, st, P);
  ADA_CHECK_LAUNCH();
  (void)ada::launch_k(draw_kernel<T, VEC>, dim3((unsigned)P.batch * P.draw_chunks), dim3(DRAW_THREADS), 0, st, P);
  ADA_CHECK_LAUNCH();
  return ADA_OK;
}

// Workspace: the row statistics, then the draw's words.
inline size_t verify_layout(VerifyParams& P, int64_t total_q, int64_t batch, int64_t vocab, int dtype, void* ws) {
  const int pack = 16 / dtype_size(dtype);
  row_shares(total_q, vocab, pack, 4 * 148, 0, &P.chunks, &P.chunk_packs);
  row_shares(batch, vocab, pack, 3 * 148, 12, &P.draw_chunks, &P.draw_packs);
  const size_t part = (size_t)total_q * P.chunks * sizeof(float4);
  P.part = reinterpret_cast<float4*>(ws);
  P.best = reinterpret_cast<unsigned long long*>(reinterpret_cast<char*>(ws) + part);
  P.done = reinterpret_cast<unsigned int*>(P.best + batch);
  return part + (size_t)batch * 12;
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

extern "C" size_t ada_verify_drafts_workspace_size(int32_t total_q, int32_t batch, int64_t vocab, int dtype) {
  if (total_q < 0 || batch <= 0 || vocab <= 0 || !smp::dtype_ok(dtype)) return 0;
  smp::VerifyParams P;
  return smp::verify_layout(P, total_q, batch, vocab, dtype, nullptr);
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
      !accepted || !logprobs || (!uniforms && max_drafts > 0) || !workspace)
    return ADA_ERR_INVALID_ARG;
  if ((draft_logits == nullptr) != (draft_lse == nullptr)) return ADA_ERR_INVALID_ARG;
  if (draft_logits && (draft_stride_b < 0 || draft_stride_d < 0 || lse_stride_b < 0 || lse_stride_d < 0))
    return ADA_ERR_INVALID_ARG;
  if (vocab > (1 << 30) || batch > (1 << 20) || max_drafts > 1024) return ADA_ERR_UNSUPPORTED;
  if (smp::misaligned(target, dtype) || smp::misaligned(draft_logits, dtype) || ((uintptr_t)noise & 3) ||
      ((uintptr_t)temperatures & 3) || ((uintptr_t)uniforms & 3) || ((uintptr_t)draft_lse & 3) ||
      ((uintptr_t)input_ids & 7) || ((uintptr_t)cu_seqlens_q & 3) || ((uintptr_t)tokens & 7) ||
      ((uintptr_t)accepted & 3) || ((uintptr_t)logprobs & 3) || ((uintptr_t)workspace & 15))
    return ADA_ERR_ALIGNMENT;
  smp::VerifyParams P;
  if (workspace_bytes < smp::verify_layout(P, total_q, batch, vocab, dtype, workspace)) return ADA_ERR_WORKSPACE;
  if ((int64_t)total_q * P.chunks > 0x7fffffff || (int64_t)batch * P.draw_chunks > 0x7fffffff)
    return ADA_ERR_UNSUPPORTED;
  P.target = target;
  P.ld = ld;
  P.n = (int)vocab;
  P.ids = input_ids;
  P.cu_q = cu_seqlens_q;
  P.batch = batch;
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
    return vec ? smp::verify_typed<__nv_bfloat16, true>(P, st)
               : smp::verify_typed<__nv_bfloat16, false>(P, st);
  if (dtype == ADA_DT_F16)
    return vec ? smp::verify_typed<__half, true>(P, st) : smp::verify_typed<__half, false>(P, st);
  return vec ? smp::verify_typed<float, true>(P, st) : smp::verify_typed<float, false>(P, st);
}
