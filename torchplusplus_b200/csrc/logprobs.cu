// Log probabilities of given tokens from rows of logits, with each row's entropy, the
// token's rank and the most likely alternatives, in one read of the logits.
#include <math.h>
#include "common.cuh"

namespace tpp {
namespace {

constexpr int kU = 4;          // 16-byte vectors a thread has in flight
constexpr int kCap = 1024;     // candidates for the alternatives; see below
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
  // how many of a chunk's elements exceed t: ones summed in the type (at most 16 a lane, exact)
  struct Count {
    T2 n{}, t;
    __device__ __forceinline__ explicit Count(float v) {
      const T e = from_f32<T>(v);
      t.x = t.y = e;
      n.x = n.y = from_f32<T>(0.f);
    }
    __device__ __forceinline__ void add(const uint4& u) {
      n = __hadd2(__hadd2(n, __hadd2(__hgt2(as(u.x), t), __hgt2(as(u.y), t))),
                  __hadd2(__hgt2(as(u.z), t), __hgt2(as(u.w), t)));
    }
    __device__ __forceinline__ int get() const { return (int)(to_f32(n.x) + to_f32(n.y)); }
  };
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
  struct Count {
    int n = 0;
    float t;
    __device__ __forceinline__ explicit Count(float v) : t(v) {}
    __device__ __forceinline__ void add(const uint4& u) {
      n += (__uint_as_float(u.x) > t) + (__uint_as_float(u.y) > t) + (__uint_as_float(u.z) > t) +
           (__uint_as_float(u.w) > t);
    }
    __device__ __forceinline__ int get() const { return n; }
  };
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
// Alternatives: of each warp with a full first chunk, the r-th largest of its lanes'
// maxima, r = ceil(top / such warps); the least of these is a lower bound of the slice's
// top-th largest logit (at least `top` elements are no smaller).  What is no smaller there,
// and larger later (a later equal one loses by its index), is a candidate.  After chunks
// 1, 2, 4, 8 .. the candidates are ranked by counting and all but `top` dropped, which
// raises the bound: some `top` new ones come in between.  More than kCap, or kHits chunks of a thread (long runs of
// equal logits, ascending rows), or a NaN, and the slice is searched `top` times over instead.
//
// Measured, bf16: 4096 x 151936 224 us without alternatives (5.55 TB/s, 85 % of a copy's rate), 288
// with 20; 4096 x 32003 62 and 100; a single row of 151936 over 8 CTAs 10.6, with 5 14.6.
// Bound by HBM without alternatives (issue slots 69 % busy), by issue slots and barriers with
// them, a single row by latency.  Narrowing after chunks 1, 3, 9 .. takes as long, 1, 8, 64: 313.
// A row with -inf is read once more, an element a thread at a time, and one whose first chunk's
// bound is -inf `top` times more: 10 % of the 4096 x 151936 at -inf 2290 us, 2380 with 20
// alternatives; all but 100 of each row 2290, and 45 ms (8 such rows: 139 us, of others 17).
template <typename T, bool TOP, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT)
    token_logprobs_kernel(LogprobArgs p) {
  constexpr int E = Lane<T>::E, kWarps = NT / 32;
  __shared__ __align__(16) uint64_t cand[TOP ? kCap : 1];
  __shared__ uint64_t list[TOP ? kMaxTop : 1];
  __shared__ uint64_t wbest[kWarps];
  __shared__ uint32_t wkey[2][kWarps];
  __shared__ Stat wstat[kWarps], slice;
  __shared__ int wcount[kWarps];
  __shared__ int count, above;
  // With whole rows a CTA (128 threads) a chunk's hit costs its warp as little as possible:
  // the thread's vectors are noted and looked at when the candidates are narrowed.  (Where a
  // row has several CTAs, latency counts, and they are looked at on the spot.)
  constexpr bool LATER = TOP && NT == 128;
  constexpr int kHits = 512;
  __shared__ int hit[LATER ? kHits : 1], hits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = gridDim.y, cr = C > 1 ? (int)cluster_rank() : 0;
  if (tid == 0) count = hits = 0;
  pdl_wait();
  pdl_trigger();

  const int64_t row_i = blockIdx.x;
  const T* row = static_cast<const T*>(p.logits) + row_i * p.ld;
  const int V = (int)p.V;
  const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const T* base = row - shift;  // vector v holds elements v E - shift ...
  // whole vectors [va, vb); the ends' elements go one by one
  const int nv = (int)(((int64_t)shift + V + E - 1) / E);
  const int fa = shift > 0 ? 1 : 0, fb = (int)(((int64_t)shift + V) / E);
  const int per = (nv + C - 1) / C;
  const int s0 = min(per * cr, nv), s1 = min(s0 + per, nv);
  const int va = max(s0, fa), vb = min(s1, fb);
  // the slice's elements [e0, e1)
  const int e0 = max(s0 * E - shift, 0), e1 = (int)min((int64_t)s1 * E - shift, (int64_t)V);
  // those outside its whole vectors: [e0, ea) and [eb, e1)
  const int ea = va < vb ? va * E - shift : e1, eb = va < vb ? vb * E - shift : e1;

  // chunk by chunk: kU vectors a thread, the next chunk's loads in flight
  constexpr int step = NT * kU;
  uint4 nxt[kU];
  auto fetch = [&](int v0) {
    if (v0 + step <= vb) {
#pragma unroll
      for (int u = 0; u < kU; ++u) nxt[u] = ldg_nc_v4(base + (int64_t)(v0 + u * NT + tid) * E);
    } else {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int v = v0 + u * NT + tid;
        nxt[u] = v < vb ? ldg_nc_v4(base + (int64_t)v * E) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  fetch(va);

  const int64_t tok = p.tokens[row_i];
  const bool has = tok >= 0 && tok < V;
  const float xt = has ? to_f32(row[tok]) : INFINITY;
  const float c = p.c;
  const uint64_t c2 = f2_pack(c, c);
  float ref = -INFINITY, S = 0.f, En = 0.f;
  int greater = 0;
  float T0 = INFINITY;   // what a candidate has to exceed
  float edge = 0.f;      // this thread's element of the ends, number ei
  int ei = -1;
  // the first chunk's bound as a key; at or below that of -inf everything is a candidate
  // (below 0 comes -0, which equals it, and then the largest negative number)
  constexpr uint32_t kLeastKey = 0x007fffffu, kZeroKey = 0x80000000u;
  uint32_t first_key = 0;
  bool everything = false;

  auto push = [&](float x, int i) {
    const int at = atomicAdd(&count, 1);
    if (at < kCap) cand[at] = item_of(x, i);
  };
  // how many of the first n candidates come before `me`
  auto place = [&](uint64_t me, int n) {
    int r = 0, j = 0;
#pragma unroll 4
    for (; j + 2 <= n; j += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(cand + j);
      r += (o.x > me) + (o.y > me);
    }
    if (j < n) r += cand[j] > me;
    return r;
  };
  // the candidates in order, all but the first `top` dropped; returns how many are left
  // (more than kCap: too many, and none dropped)
  auto narrow = [&]() {
    __syncthreads();
    if (LATER) {
      const int noted = hits;
      if (noted > kHits) return kCap + 1;
#pragma unroll 1
      for (int e = tid; e < noted * kU; e += NT) {
        const int v = hit[e / kU] + e % kU * NT;
        if (v >= vb) continue;
        float f[E];
        Lane<T>::get(ldg_nc_v4(base + (int64_t)v * E), f);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (f[j] > T0 || (everything && v < va + step)) push(f[j], v * E - shift + j);
      }
      __syncthreads();
      if (tid == 0) hits = 0;
    }
    const int n = count;
    if (n > kCap) return n;
#pragma unroll 1
    for (int i = tid; i < n; i += NT) {
      const uint64_t me = cand[i];
      const int r = place(me, n);
      if (r < p.top) list[r] = me;
    }
    __syncthreads();
    const int left = min(n, p.top);
#pragma unroll 1
    for (int i = tid; i < left; i += NT) cand[i] = list[i];
    if (tid == 0) count = left;
    __syncthreads();
    return left;
  };
  // One chunk; FULL: every thread has kU vectors.
  auto chunk = [&](int v0, auto full) {
    constexpr bool FULL = decltype(full)::value;
    uint4 cur[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) cur[u] = nxt[u];
    if (v0 + step < vb) fetch(v0 + step);
    const int mine = FULL ? kU : max(0, min(kU, (vb - v0 - tid + NT - 1) / NT));
    float cm = -INFINITY;  // this thread's largest
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (FULL || u < mine) cm = fmaxf(cm, Lane<T>::most(cur[u]));
    if (v0 == va) {
      // the ends' elements (fewer than 2 E a row) belong to the first chunk, but not to
      // the bound, and those of the row's end are candidates last: one loses to equal ones
      // before it
      if (tid < ea - e0) ei = e0 + tid;
      else if (tid - max(ea - e0, 0) < e1 - eb) ei = eb + tid - max(ea - e0, 0);
      uint32_t key = key_of(cm), last = 0;
      if (ei >= 0) {
        edge = to_f32(row[ei]);
        cm = fmaxf(cm, edge);
      }
      const uint32_t first = __reduce_max_sync(0xffffffffu, key_of(cm));
      const int whole = min(kWarps, (vb - va) / 32);  // warps with data in every lane
      if (TOP && warp < whole) {
        const int rounds = min(32, (p.top + whole - 1) / whole);
#pragma unroll 1
        for (int r = 0; r < rounds; ++r) {
          last = __reduce_max_sync(0xffffffffu, key);
          const uint32_t who = __ballot_sync(0xffffffffu, key == last);
          if (lane == __ffs(who) - 1) key = 0;
        }
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
        if (w < whole) least = min(least, wkey[1][w]);
      }
      ref = value_of(big);
      // (reached, not exceeded, is enough in this chunk: the next value below)
      first_key = whole * 32 < p.top ? 0u : least;
      everything = first_key <= kLeastKey;
      T0 = everything ? -INFINITY : value_of(first_key - (first_key == kZeroKey ? 2 : 1));
      if (ei >= 0) {
        if (TOP && ei < eb && (everything || edge > T0)) push(edge, ei);
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
    const bool all = everything && v0 == va;
    if (LATER && (cm > T0 || all)) {
      const int at = atomicAdd(&hits, 1);
      if (at < kHits) hit[at] = v0 + tid;
    }
    if (TOP && !LATER && (cm > T0 || all)) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (!FULL && u >= mine) break;
        if (!(Lane<T>::most(cur[u]) > T0 || all)) continue;
        float f[E];
        Lane<T>::get(cur[u], f);
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) hits |= (uint32_t)(f[j] > T0 || all) << j;
        const int i0 = (v0 + u * NT + tid) * E - shift;
        while (hits != 0) {
          const int j = __ffs(hits) - 1;
          hits &= hits - 1;
          float x = f[0];
#pragma unroll
          for (int k = 1; k < E; ++k) x = j == k ? f[k] : x;
          push(x, i0 + j);
        }
      }
    }
    if (cm > xt) {
      typename Lane<T>::Count above_t(xt);
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (FULL || u < mine) above_t.add(cur[u]);
      greater += above_t.get();
    }
    if (ref != -INFINITY) {
      const uint64_t r2 = f2_pack(-ref, -ref);
      uint64_t s2[2] = {0ull, 0ull}, e2[2] = {0ull, 0ull};
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (!FULL && u >= mine) break;
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
        if (!FULL && u >= mine) break;
        float f[E];
        Lane<T>::get(cur[u], f);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (isnan(f[j])) S = f[j];
      }
    }
  };
  int done = 0, next = 1;
#pragma unroll 1
  for (int v0 = va; v0 < vb || v0 == va; v0 += step) {
    if (TOP && done > 0 && done == next) {
      next *= 2;
      const int left = narrow();
      if (left == p.top) T0 = value_of((uint32_t)(cand[left - 1] >> 32));
    }
    ++done;
    if (v0 + step <= vb) chunk(v0, std::true_type{});
    else chunk(v0, std::false_type{});
  }
  if (TOP && ei >= eb && !(edge < T0)) push(edge, ei);

  // ---- the slice's weights and rank
  auto reduce = [&](Stat st) {
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) {
      Stat ot;
      ot.m = __shfl_xor_sync(0xffffffffu, st.m, o);
      ot.S = __shfl_xor_sync(0xffffffffu, st.S, o);
      ot.E = __shfl_xor_sync(0xffffffffu, st.E, o);
      // (both lanes of a pair add in the same order)
      const bool up = lane & o;
      st = merge(up ? ot : st, up ? st : ot, c);
    }
    __syncthreads();
    if (lane == 0) wstat[warp] = st;
    __syncthreads();
    st = wstat[0];
#pragma unroll 1
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
#pragma unroll 1
    for (int i = e0 + tid; i < e1; i += NT) {
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
#pragma unroll 1
    for (int i = e0 + tid; i < e1; i += NT) greater += key_of(to_f32(row[i])) > kt;
  }
  greater = total(greater);  // (its barriers also order the candidates)

  // ---- the slice's alternatives, in order
  if constexpr (TOP) {
    const int K = p.top, n = odd ? kCap + 1 : narrow();
    if (n > kCap) {
      uint64_t prev = ~0ull;
#pragma unroll 1
      for (int k = 0; k < K; ++k) {
        uint64_t best = 0;
#pragma unroll 1
        for (int i = e0 + tid; i < e1; i += NT) {
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
    } else if (tid >= n && tid < K) {
      list[tid] = 0;
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
#pragma unroll 1
    for (int r = 1; r < C; ++r) {
      st = merge(st, Stat{peer_load(&slice.m, r), peer_load(&slice.S, r), peer_load(&slice.E, r)}, c);
      greater += peer_load(&above, r);
    }
    if constexpr (TOP) {
      const int K = p.top, n = C * K;
#pragma unroll 1
      for (int i = tid; i < n; i += NT) cand[i] = peer_load(&list[i % K], i / K);
      cluster_sync();  // (its barrier is the CTA's too)
#pragma unroll 1
      for (int i = tid; i < n; i += NT) {
        const uint64_t me = cand[i];
        const int r = place(me, n);
        if (me != 0 && r < K) list[r] = me;
      }
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
  TPP_REQUIRE(N > 0 && N < (1ll << 31) && V > 0 && V < (1ll << 31) - 4096 && ld >= V,
              TPP_ERR_SHAPE, "bad sizes");
  TPP_REQUIRE(temperature > 0 && isfinite(temperature) && temperature >= 1e-6, TPP_ERR_SHAPE,
              "temperature must be positive");
  TPP_REQUIRE(top >= 0 && top <= kMaxTop && top <= V, TPP_ERR_SHAPE,
              "top must be at most 32 and at most V");
  TPP_REQUIRE(top == 0 || (top_logprobs && top_tokens), TPP_ERR_SHAPE, "null pointer");
  const LogprobArgs a{logits, ld, V, tokens, (float)(1.4426950408889634 / temperature),
                      (float)(1 / temperature), (int)top,
                      logprobs, entropy, ranks, top_logprobs, top_tokens};
  // CTAs a row: enough rows for three on every SM want one each.  Measured (bf16, top 20, us with
  // 1, 2, 4, 8 CTAs): one of 151936 39.5, 27.6, 21.2, 16.7; 130 46, 33, 28, 46 (takes 4); 300 51, 52,
  // 53, 98 (2); 1200 113, 116, 147, 349 (1).  Not the best between, and for small rows: 110 of
  // 151936 46, 33, 28, 44 (8); 600 84, 72, 85, 182 (1), without alternatives 64, 44, 47, 93; one of
  // 32003 15.9, 13.2, 11.3, 17.0 (8).
  int C = 1;
  while (C < kMaxCtas && N * C < 3 * (int64_t)num_sms()) C *= 2;
  auto go = [&](auto tag, auto threads) -> int {
    using T = decltype(tag);
    constexpr int NT = decltype(threads)::value;
    TPP_REQUIRE(reinterpret_cast<uintptr_t>(logits) % sizeof(T) == 0, TPP_ERR_ALIGN,
                "logits must be aligned to their type");
    return launch("token_logprobs_kernel",
                  top > 0 ? token_logprobs_kernel<T, true, NT> : token_logprobs_kernel<T, false, NT>,
                  dim3((unsigned)N, (unsigned)C), dim3(NT), 0, as_stream(stream),
                  C > 1 ? (unsigned)C : 0u, a);
  };
  auto size = [&](auto tag) -> int {
    // a thread's chunk is 64 bytes: small slices want few threads, a row over several CTAs
    // the latency of many, and eight CTAs on an SM hide each other's barriers
    if (V * (int64_t)sizeof(tag) / C < 128 * 64) return go(tag, std::integral_constant<int, 64>{});
    if (C < 8) return go(tag, std::integral_constant<int, 128>{});
    return go(tag, std::integral_constant<int, 256>{});
  };
  if (dtype == TPP_F16) return size(__half());
  if (dtype == TPP_BF16) return size(__nv_bfloat16());
  if (dtype == TPP_F32) return size(float());
  set_error("tpp_token_logprobs: dtype must be f16, bf16 or f32");
  return TPP_ERR_DTYPE;
}
