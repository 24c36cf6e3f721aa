// Log probabilities of given tokens from rows of logits, with each row's entropy, the
// token's rank and the most likely alternatives, in one read of the logits.
#include <math.h>
#include "common.cuh"

namespace tpp {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kU = 4;          // 16-byte vectors a thread has in flight
constexpr int kCap = 2048;     // candidates for the alternatives; see below
constexpr int kMaxTop = 32;
constexpr int kMaxCtas = 8;    // CTAs (one cluster) a row

struct LogprobArgs {
  const void* logits;
  int64_t ld, V;
  const int64_t* tokens;
  float c;      // log2(e) / temperature
  float inv_t;  // 1 / temperature
  int top;
  float* logprob;
  float* entropy;
  int64_t* rank;
  float* top_logprob;
  int64_t* top_token;
};

// Weights of a set of logits: S = sum 2^(c (x - m)), E = sum 2^(c (x - m)) (x - m).
struct Stat {
  float m, S, E;
};
__device__ __forceinline__ Stat merge(Stat a, Stat b, float c) {
  const float M = fmaxf(a.m, b.m);
  Stat r{M, 0.f, 0.f};
  // (a set without weight adds nothing whatever its m, and one that vanishes beside the
  // other no E, whose sum may be infinite; NaN sums stay NaN)
  if (!(a.S == 0.f)) {
    const float d = a.m - M, f = exp2f(c * d);
    r.S += a.S * f;
    r.E += f == 0.f ? 0.f : (a.E + a.S * d) * f;
  }
  if (!(b.S == 0.f)) {
    const float d = b.m - M, f = exp2f(c * d);
    r.S += b.S * f;
    r.E += f == 0.f ? 0.f : (b.E + b.S * d) * f;
  }
  return r;
}

// Order of logits as unsigned numbers: NaN above all, -0 equal to 0; never 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (isnan(x)) return 0xfffffffeu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k == 0xfffffffeu ? 0x7fffffffu : k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// Larger logit first, then the lower index.
__device__ __forceinline__ uint64_t item_of(float x, int64_t i) {
  return (uint64_t)key_of(x) << 32 | (uint32_t)~(uint32_t)i;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
               "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <typename V>
__device__ __forceinline__ V peer_load(const V* p, uint32_t rank) {
  static_assert(sizeof(V) == 4 || sizeof(V) == 8, "");
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  V v;
  if constexpr (sizeof(V) == 4) {
    uint32_t w;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
    memcpy(&v, &w, 4);
  } else {
    uint64_t w;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(w) : "r"(at) : "memory");
    memcpy(&v, &w, 8);
  }
  return v;
}

// The elements of a 16-byte vector, their largest (NaN aside), how many exceed t.
template <typename T> struct Lane {
  static constexpr int E = 8;
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2,
                                       __nv_bfloat162>::type;
  static __device__ __forceinline__ T2 as(uint32_t w) { return *reinterpret_cast<T2*>(&w); }
  static __device__ __forceinline__ void get(const uint4& u, float* f) { unpack8<T>(u, f); }
  static __device__ __forceinline__ float most(const uint4& u) {
    const T2 m = __hmax2(__hmax2(as(u.x), as(u.y)), __hmax2(as(u.z), as(u.w)));
    return fmaxf(to_f32(m.x), to_f32(m.y));
  }
};
template <> struct Lane<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void get(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float most(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                 fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
};

// One row a cluster of gridDim.y CTAs, each a slice of 16-byte vectors (of the row
// and the unaligned elements at its ends).
//
// Weights: exponents are taken against a reference that the first chunk's largest logit
// sets and that only a logit 2^8 times as likely moves (exact: the final quotients
// use the same reference), so an element costs a difference, a product, an exponential
// and two sums.  The differences are taken before the scale: masks of the type's lowest
// value stay finite, and a row of nothing else is uniform.
//
// Alternatives: every warp's ceil(top / 8)-th largest of its threads' maxima over the
// first chunk; the least of these eight is a lower bound of the slice's top-th largest
// logit (at least `top` elements are no smaller).  What is no smaller there, and larger
// later (a later equal one loses by its index), is kept: some 20 to 400 candidates, ranked at the
// end by counting.  More than kCap (long runs of equal logits, ascending rows), or a NaN, and the
// slice is searched `top` times over instead.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 3) token_logprobs_kernel(LogprobArgs p) {
  constexpr int E = Lane<T>::E;
  __shared__ uint64_t cand[TOP ? kCap : 1];
  __shared__ uint64_t list[TOP ? kMaxTop : 1];
  __shared__ uint64_t wbest[kWarps];
  __shared__ uint32_t wkey[2][kWarps];
  __shared__ Stat wstat[kWarps], slice;
  __shared__ int wcount[kWarps];
  __shared__ int count, above;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = gridDim.y, cr = C > 1 ? (int)cluster_rank() : 0;
  if (tid == 0) count = 0;
  pdl_wait();
  pdl_trigger();

  const int64_t row_i = blockIdx.x;
  const T* row = static_cast<const T*>(p.logits) + row_i * p.ld;
  const int64_t V = p.V;
  const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const T* base = row - shift;  // vector v holds elements v E - shift ...
  const int64_t tok = p.tokens[row_i];
  const bool has = tok >= 0 && tok < V;
  const float xt = has ? to_f32(row[tok]) : INFINITY;
  // whole vectors [va, vb); the ends' elements go one by one
  const int64_t nv = (shift + V + E - 1) / E;
  const int64_t fa = shift > 0 ? 1 : 0, fb = (shift + V) / E;
  const int64_t per = (nv + C - 1) / C;
  const int64_t s0 = per * cr < nv ? per * cr : nv, s1 = s0 + per < nv ? s0 + per : nv;
  const int64_t va = s0 > fa ? s0 : fa, vb = s1 < fb ? s1 : fb;
  // the slice's elements [e0, e1)
  const int64_t e0 = s0 * E - shift > 0 ? s0 * E - shift : 0;
  const int64_t e1 = s1 * E - shift < V ? (s1 * E - shift > 0 ? s1 * E - shift : 0) : V;
  // those outside its whole vectors: [e0, ea) and [eb, e1)
  const int64_t ea = va < vb ? va * E - shift : e1, eb = va < vb ? vb * E - shift : e1;

  const float c = p.c;
  float ref = -INFINITY, S = 0.f, En = 0.f;
  int greater = 0;
  float T0 = INFINITY;  // what a candidate has to exceed, from the second chunk on

  auto push = [&](float x, int64_t i) {
    const int at = atomicAdd(&count, 1);
    if (at < kCap) cand[at] = item_of(x, i);
  };
  // chunk by chunk: kU vectors a thread, the next chunk's loads in flight
  uint4 nxt[kU];
  const int64_t step = (int64_t)kThreads * kU;
  auto fetch = [&](int64_t v0) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int64_t v = v0 + u * kThreads + tid;
      nxt[u] = v < vb ? ldg_nc_v4(base + v * E) : make_uint4(0, 0, 0, 0);
    }
  };
  fetch(va);
  bool start = true;
  for (int64_t v0 = va; start || v0 < vb; v0 += step) {
    uint4 cur[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) cur[u] = nxt[u];
    if (v0 + step < vb) fetch(v0 + step);
    float cm = -INFINITY;  // of this thread's elements
    const bool any = v0 + tid < vb;
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (v0 + u * kThreads + tid < vb) cm = fmaxf(cm, Lane<T>::most(cur[u]));
    if (start) {
      // the ends' elements (fewer than 2 E a row) belong to the first chunk, but not to
      // the bound: one at the row's end loses to equal ones before it
      float edge = 0.f;
      int64_t ei = -1;
      if (tid < ea - e0) ei = e0 + tid;
      else if (tid - (ea - e0) < e1 - eb) ei = eb + tid - (ea - e0);
      uint32_t key = any ? key_of(cm) : 0u, last = 0;
      if (ei >= 0) {
        edge = to_f32(row[ei]);
        cm = fmaxf(cm, edge);
      }
      const uint32_t first = __reduce_max_sync(0xffffffffu, key_of(cm));
      const int rounds = TOP ? (p.top + kWarps - 1) / kWarps : 0;
      for (int r = 0; r < rounds; ++r) {
        last = __reduce_max_sync(0xffffffffu, key);
        const uint32_t who = __ballot_sync(0xffffffffu, key == last);
        if (lane == __ffs(who) - 1) key = 0;
      }
      if (lane == 0) {
        wkey[0][warp] = first;
        wkey[1][warp] = last;
      }
      __syncthreads();
      uint32_t big = 0, least = 0xffffffffu;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        big = max(big, wkey[0][w]);
        least = min(least, wkey[1][w]);
      }
      ref = value_of(big);
      T0 = least == 0 ? -INFINITY : value_of(least);
      if (ei >= 0) {
        if (TOP && !(edge < T0)) push(edge, ei);
        if (edge > xt) ++greater;
        if (edge != -INFINITY) {
          const float q = edge - ref, w = ex2_ftz(q * c);
          S += w;
          En += w * q;
        }
      }
    }
    if ((cm - ref) * c > 8.f) {  // (rare)
      const float d = ref - cm, f = S == 0.f ? 0.f : exp2f(c * d);
      En = f == 0.f ? 0.f : (En + S * d) * f;
      S *= f;
      ref = cm;
    }
    if (TOP && any && (start ? cm >= T0 : cm > T0)) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t v = v0 + u * kThreads + tid;
        if (v >= vb) break;
        const float vm = Lane<T>::most(cur[u]);
        if (!(start ? vm >= T0 : vm > T0)) continue;
        float f[E];
        Lane<T>::get(cur[u], f);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (start ? f[j] >= T0 : f[j] > T0) push(f[j], v * E - shift + j);
      }
    }
    if (cm > xt) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (v0 + u * kThreads + tid >= vb) break;
        float f[E];
        Lane<T>::get(cur[u], f);
#pragma unroll
        for (int j = 0; j < E; ++j) greater += f[j] > xt;
      }
    }
    if (ref != -INFINITY) {
      const uint64_t c2 = f2_pack(c, c), r2 = f2_pack(-ref, -ref);
      uint64_t s2[2] = {0ull, 0ull}, e2[2] = {0ull, 0ull};
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (v0 + u * kThreads + tid >= vb) break;
        float f[E];
        Lane<T>::get(cur[u], f);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
          const uint64_t q2 = f2_add(f2_pack(f[j], f[j + 1]), r2);
          float d0, d1;
          f2_unpack(f2_mul(q2, c2), d0, d1);
          const uint64_t w2 = f2_pack(ex2_ftz(d0), ex2_ftz(d1));
          s2[(j >> 1) & 1] = f2_add(s2[(j >> 1) & 1], w2);
          e2[(j >> 1) & 1] = f2_fma(w2, q2, e2[(j >> 1) & 1]);
        }
      }
      float a0, a1;
      f2_unpack(f2_add(s2[0], s2[1]), a0, a1);
      S += a0 + a1;
      f2_unpack(f2_add(e2[0], e2[1]), a0, a1);
      En += a0 + a1;
    } else {
      // nothing but -inf so far, which weighs nothing, or NaN
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (v0 + u * kThreads + tid >= vb) break;
        float f[E];
        Lane<T>::get(cur[u], f);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (isnan(f[j])) S = f[j];
      }
    }
    start = false;
  }

  // ---- the slice's weights and rank
  auto reduce = [&](Stat st) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Stat ot;
      ot.m = __shfl_xor_sync(0xffffffffu, st.m, o);
      ot.S = __shfl_xor_sync(0xffffffffu, st.S, o);
      ot.E = __shfl_xor_sync(0xffffffffu, st.E, o);
      // (both lanes of a pair add in the same order)
      st = lane & o ? merge(ot, st, c) : merge(st, ot, c);
    }
    __syncthreads();
    if (lane == 0) wstat[warp] = st;
    __syncthreads();
    st = wstat[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) st = merge(st, wstat[w], c);
    return st;
  };
  auto total = [&](int n) {
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (lane == 0) wcount[warp] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) n += wcount[w];
    return n;
  };
  Stat st = reduce(Stat{ref, S, En});
  if (!isnan(st.S) && isnan(st.E)) {
    // -inf among the logits made 0 * -inf: once more, without those
    const float m = st.m;
    S = En = 0.f;
    for (int64_t i = e0 + tid; i < e1; i += kThreads) {
      const float x = to_f32(row[i]);
      const float q = x - m, w = ex2_ftz(q * c);
      if (w == 0.f) continue;
      S += w;
      En += w * q;
    }
    st = reduce(Stat{m, S, En});
  }
  const bool odd = isnan(st.S);  // NaN or +inf: order by keys
  if (odd) {
    greater = 0;
    const uint32_t kt = key_of(xt);
    for (int64_t i = e0 + tid; i < e1; i += kThreads) greater += key_of(to_f32(row[i])) > kt;
  }
  greater = total(greater);  // (its barriers also order the candidates)

  // ---- the slice's alternatives, in order
  if constexpr (TOP) {
    const int K = p.top, n = count;
    if (odd || n > kCap) {
      uint64_t prev = ~0ull;
      for (int k = 0; k < K; ++k) {
        uint64_t best = 0;
        for (int64_t i = e0 + tid; i < e1; i += kThreads) {
          const uint64_t it = item_of(to_f32(row[i]), i);
          if (it < prev && it > best) best = it;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        __syncthreads();
        if (lane == 0) wbest[warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) best = max(best, wbest[w]);
        if (tid == 0) list[k] = best;
        prev = best;  // (0, none left, stays 0)
      }
    } else {
      if (tid < K) list[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t me = cand[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += cand[j] > me;
        if (r < K) list[r] = me;
      }
    }
    __syncthreads();
  }

  // ---- the row's, by the first CTA
  if (C > 1) {
    if (tid == 0) {
      slice = st;
      above = greater;
    }
    cluster_sync();
    if (cr != 0) {
      cluster_sync();  // its shared memory lives until the first CTA has read it
      return;
    }
    for (int r = 1; r < C; ++r) {
      st = merge(st, Stat{peer_load(&slice.m, r), peer_load(&slice.S, r), peer_load(&slice.E, r)}, c);
      greater += peer_load(&above, r);
    }
    if constexpr (TOP) {
      const int K = p.top, n = C * K;
      if (tid < n) cand[tid] = peer_load(&list[tid % K], tid / K);
      __syncthreads();
      uint64_t me = tid < n ? cand[tid] : 0;
      int r = 0;
      if (me != 0)
        for (int j = 0; j < n; ++j) r += cand[j] > me;
      cluster_sync();
      if (me != 0 && r < K) list[r] = me;
      __syncthreads();
    } else {
      cluster_sync();
    }
  }
  constexpr float kLn2 = 0.69314718055994531f;
  const float lz = log2f(st.S);
  // no weight at all (every logit -inf): no token has any probability
  auto logp = [&](float x) {
    if (isnan(st.S)) return NAN;
    if (st.S == 0.f || x == -INFINITY) return -INFINITY;
    return (x - st.m) * p.inv_t - lz * kLn2;  // (finite for every finite logit)
  };
  if (tid == 0) {
    p.logprob[row_i] = has ? logp(xt) : 0.f;
    p.entropy[row_i] = isnan(st.S) ? NAN : st.S == 0.f ? 0.f : lz * kLn2 - st.E / st.S * p.inv_t;
    p.rank[row_i] = has ? greater + 1 : 0;
  }
  if constexpr (TOP) {
    if (tid < p.top) {
      const uint64_t it = list[tid];
      p.top_logprob[row_i * p.top + tid] = logp(value_of((uint32_t)(it >> 32)));
      p.top_token[row_i * p.top + tid] = (int64_t)(uint32_t)~(uint32_t)it;
    }
  }
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int tpp_token_logprobs(const void* logits, int64_t ld, int64_t N, int64_t V,
                                  const int64_t* tokens, double temperature, int64_t top,
                                  float* logprobs, float* entropy, int64_t* ranks,
                                  float* top_logprobs, int64_t* top_tokens, int dtype,
                                  void* stream) {
  if (N == 0) return TPP_OK;
  TPP_REQUIRE(logits && tokens && logprobs && entropy && ranks, TPP_ERR_SHAPE, "null pointer");
  TPP_REQUIRE(N > 0 && N < (1ll << 31) && V > 0 && V < (1ll << 31) && ld >= V, TPP_ERR_SHAPE,
              "bad sizes");
  TPP_REQUIRE(temperature > 0 && isfinite(temperature) && temperature >= 1e-6, TPP_ERR_SHAPE,
              "temperature must be positive");
  TPP_REQUIRE(top >= 0 && top <= kMaxTop && top <= V, TPP_ERR_SHAPE,
              "top must be at most 32 and at most V");
  TPP_REQUIRE(top == 0 || (top_logprobs && top_tokens), TPP_ERR_SHAPE, "null pointer");
  const LogprobArgs a{logits, ld, V, tokens, (float)(1.4426950408889634 / temperature),
                      (float)(1 / temperature), (int)top,
                      logprobs, entropy, ranks, top_logprobs, top_tokens};
  // CTAs a row: enough rows for three on every SM want one each
  int C = 1;
  while (C < kMaxCtas && N * C < 3 * (int64_t)num_sms()) C *= 2;
  auto go = [&](auto tag) -> int {
    using T = decltype(tag);
    TPP_REQUIRE(reinterpret_cast<uintptr_t>(logits) % sizeof(T) == 0, TPP_ERR_ALIGN,
                "logits must be aligned to their type");
    return launch("token_logprobs_kernel",
                  top > 0 ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>,
                  dim3((unsigned)N, (unsigned)C), dim3(kThreads), 0, as_stream(stream),
                  C > 1 ? (unsigned)C : 0u, a);
  };
  if (dtype == TPP_F16) return go(__half());
  if (dtype == TPP_BF16) return go(__nv_bfloat16());
  if (dtype == TPP_F32) return go(float());
  set_error("tpp_token_logprobs: dtype must be f16, bf16 or f32");
  return TPP_ERR_DTYPE;
}
