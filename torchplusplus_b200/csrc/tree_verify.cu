// Verification of a drafted tree against the target's logits (tpp_verify_tree).
//
// One cluster walks one sequence's tree from the root.  At a node it needs the
// softmax of one row of logits (and of the draft's row, where the children were
// drawn from one).  Every CTA of the cluster holds its part of the row; every
// thread makes the same decisions from the exchanged sums.
//
// Weights are exp((l - max) / temperature) in fp32; sums and cumulative sums of
// weights run over 64-bit integers, round(w * 2^40), so they are exact and a
// result does not depend on the order or the split of a row (fp32 cumulative
// sums over 150k tokens move the boundaries of a draw by about 1e-6).
//
// What a walk costs is its chain of passes and exchanges, and the exact weights
// are 23 instructions an element.  So a node's tests go by its maximum and an fp32
// sum, taken in one pass of 7 instructions an element and one exchange; the exact
// sums follow only where a test comes within the fp32 sum's error of a tie, and
// at the last node, for the draw.  For chains with a draft verify_stats_kernel takes
// these of all rows ahead of the walk, on all SMs.  An exchange is one remote store a
// warp and CTA (st.async, counted by the receiver's mbarrier) and no barrier of the
// CTA or the cluster, 1.0 us.
//
// Bound by latency: one chain of 5 nodes over 151936 tokens with its draft takes
// 26.6 us (first form 123), of which statistics 5, set-up 3, tests 3, exact sums 6,
// residual 7, draw 3; 32 trees of 32 nodes 31 us (49), greedily 48 (longer paths).
// Code fetched once a walk counts: unrolling the second passes' loops over a lane's
// groups cost 8 us.  With 64 registers a thread, for 1024 threads an SM, the walk
// spills some 200 bytes.
#include <limits.h>
#include <math.h>
#include <cooperative_groups.h>
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace tpp {
namespace {

constexpr int kMaxNodes = 256;
constexpr int kMaxDraftVocab = 400000;  // with a draft: 196 KB of cache a CTA
constexpr int kSlice = 1024;         // groups of a row for a CTA of the statistics
constexpr double kFix = 1099511627776.0;  // 2^40
using ull = unsigned long long;

struct VerifyArgs {
  const void* logits; int64_t l_sb, l_st;
  const void* draft; int64_t d_sb, d_st;   // null: no draft distribution
  const int64_t* tokens; int64_t tok_sb;
  const int32_t* parents; int64_t par_sb;
  const float* u; int64_t u_sb;
  float inv_t;                             // 1 / temperature
  int greedy;
  int32_t* path; int32_t* count; int64_t* next;
  int B, T; int V;
  float2* stats;                           // [row][slices] of (max, sum), or null
  int slices;
  float sum_error;                         // relative error of the fp32 sums, at most
  int* err;
};

// A row in groups of 16 bytes: group k holds elements [k*VE - mis, k*VE - mis
// + VE), where mis makes the groups 16-byte aligned whatever the row's start.
template <typename T>
struct Row {
  static constexpr int VE = 16 / sizeof(T);
  const T* p;
  int mis, groups;
  __device__ __forceinline__ Row(const T* row, int V) : p(row) {
    mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    groups = (V + mis + VE - 1) / VE;
  }
};

template <typename T>
__device__ __forceinline__ void unpack_group(const uint4& w, float* f) { unpack8<T>(w, f); }
template <>
__device__ __forceinline__ void unpack_group<float>(const uint4& w, float* f) {
  f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y);
  f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
}

// Elements [e0, e0 + VE) of a row of V as they are stored, -inf outside it, one by
// one: a row's ends, and a draft row whose start is aligned otherwise than the
// target's.  (All loads first: one after the other they held up the CTAs at a row's
// ends by some 3 us a pass.)
template <typename T>
__device__ __noinline__ uint4 load_edge(const T* row, int e0, int V) {
  constexpr int VE = 16 / sizeof(T);
  T x[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j)
    x[j] = e0 + j >= 0 && e0 + j < V ? row[e0 + j] : from_f32<T>(-INFINITY);
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 4) {
      w[q] = __float_as_uint(x[q]);
    } else {
      w[q] = (uint32_t)*reinterpret_cast<const unsigned short*>(&x[2 * q]) |
             (uint32_t)*reinterpret_cast<const unsigned short*>(&x[2 * q + 1]) << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ uint4 load_group(const T* row, int e0, int V) {
  const T* a = row + e0;
  if (e0 >= 0 && e0 + (int)(16 / sizeof(T)) <= V && (reinterpret_cast<uintptr_t>(a) & 15) == 0)
    return __ldg(reinterpret_cast<const uint4*>(a));
  return load_edge<T>(row, e0, V);
}

// exp((l - m) / temperature), 0 where that is NaN (NaN logits; no finite max).
__device__ __forceinline__ float weight(float l, float m, float inv_t) {
  const float w = expf((l - m) * inv_t);
  return w == w ? w : 0.f;
}
// round(w * 2^40) for w in [0, 2), to even, in two parts of 20 bits by adding
// constants at whose size an ulp is 2^-20 and 2^-40: full-rate instructions, where
// a conversion to 64 bits has a sixteenth of that rate.
__device__ __forceinline__ void fixed_parts(float w, uint32_t& hi, int& lo) {
  const float a = __fadd_rn(w, 12.f);
  hi = __float_as_uint(a) - 0x41400000u;
  const float r = __fsub_rn(w, __fsub_rn(a, 12.f));     // exact, at most 2^-21
  lo = (int)(__float_as_uint(__fadd_rn(r, 1.1444091796875e-05f)) - 0x37400000u);
}
__device__ __forceinline__ ull fixed_sum(ull hi, long long lo) { return (hi << 20) + lo; }
__device__ __forceinline__ ull fixed(float w) {
  uint32_t hi;
  int lo;
  fixed_parts(w, hi, lo);
  return fixed_sum(hi, lo);
}
__device__ __forceinline__ float unfixed(ull s) { return (float)((double)s / kFix); }
__device__ __forceinline__ float share(float w, float z) { return z > 0.f ? __fdiv_rn(w, z) : 0.f; }

__device__ __forceinline__ ull warp_sum_u64(ull v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A thread's sum of integer weights: some 2^22 / 2048 of them at most (8 CTAs of 256
// threads, to whole groups) of up to 1, so that either half's sum (of 2^20 and of
// 2^19) fits 32 bits.
struct Sum {
  uint32_t hi = 0;
  int lo = 0;
  template <int N> __device__ __forceinline__ void add(const float* w) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      uint32_t h;
      int l;
      fixed_parts(w[j], h, l);
      hi += h;
      lo += l;
    }
  }
  __device__ __forceinline__ ull warp() const { return warp_sum_u64(fixed_sum(hi, lo)); }
};

// ---- every row's maximum and sum ---------------------------------------------
// Row r < B*T: the target's at (r / T, r % T); after those, the draft's.
template <typename T>
__global__ void __launch_bounds__(256) verify_stats_kernel(VerifyArgs p) {
  constexpr int VE = 16 / sizeof(T), U = kSlice / 256;
  __shared__ float sm[8], ss[8];
  pdl_wait();
  pdl_trigger();
  const int nt = p.B * p.T, r = blockIdx.y, tid = threadIdx.x;
  const int nd = p.T - 1;  // nodes that can have children
  const T* src = r < nt
      ? static_cast<const T*>(p.logits) + (r / p.T) * p.l_sb + (r % p.T) * p.l_st
      : static_cast<const T*>(p.draft) + ((r - nt) / nd) * p.d_sb + ((r - nt) % nd) * p.d_st;
  const Row<T> row(src, p.V);
  const uint4* at = reinterpret_cast<const uint4*>(row.p - row.mis);
  const int whole = (p.V + row.mis) / VE;  // groups 1 .. whole - 1 lie within the row
  uint4 raw[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int k = blockIdx.x * kSlice + i * 256 + tid;
    raw[i] = k > 0 && k < whole ? __ldg(at + k)
                                : load_edge<T>(row.p, k < row.groups ? k * VE - row.mis : p.V, p.V);
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float f[VE];
    unpack_group<T>(raw[i], f);
#pragma unroll
    for (int j = 0; j < VE; j += 2) m = fmax3(m, f[j], f[j + 1]);
  }
  m = warp_max(m);
  if ((tid & 31) == 0) sm[tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < 8; ++w) m = fmaxf(m, sm[w]);
  // pairs on the two-lane fp32 pipe; a NaN argument is clamped to a weight of 0
  const float c = p.inv_t * 1.4426950408889634f;
  const uint64_t m2 = f2_pack(-m, -m), c2 = f2_pack(c, c), zero = f2_pack(0.f, 0.f);
  uint64_t s2 = zero;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float f[VE];
    unpack_group<T>(raw[i], f);
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
      float x, y;
      f2_unpack(f2_fma(f2_add(f2_pack(f[j], f[j + 1]), m2), c2, zero), x, y);
      s2 = f2_add(s2, f2_pack(ex2_ftz(fmaxf(x, -200.f)), ex2_ftz(fmaxf(y, -200.f))));
    }
  }
  float s, s_hi;
  f2_unpack(s2, s, s_hi);
  s += s_hi;
  s = warp_sum(s);
  if ((tid & 31) == 0) ss[tid >> 5] = s;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 8; ++w) s += ss[w];
    p.stats[(int64_t)r * p.slices + blockIdx.x] = make_float2(m, s);
  }
}

// ---- the walk ----------------------------------------------------------------
struct __align__(16) Part { ull a, b; };  // a warp's part of an exchange

template <int PARTS>
struct Shared {
  Part in[2][PARTS];       // every warp's part, by the exchange's parity
  ull bar[2];
  float stage[kMaxNodes];  // sums of the residual after each rejection
  int out[kMaxNodes];      // rejected tokens
  int par[kMaxNodes];
  int tok[kMaxNodes];      // -1: not a token
  float u[kMaxNodes];
  float lt[kMaxNodes], qt[kMaxNodes];  // a node's own logit in its parent's rows
  float m[kMaxNodes], z[kMaxNodes], mq[kMaxNodes], zq[kMaxNodes];  // from the statistics
  float pt[kMaxNodes], uq[kMaxNodes];  // and from those, a node's own test
};

// How the cluster's warps share a row: `gc` groups a CTA, of which this warp owns
// [g0, g1) (counted from the row's first, whatever its alignment).
struct Share { int first, g0, g1; };

// f(group, values) over the warp's groups of a row.  The first pass over a row has
// U loads in flight (5: with 8 CTAs of 512, all of a lane's part of 160k 16-bit
// logits); the later ones find it in L1 or L2 and keep two, since their code, run
// once or twice a walk, costs more to fetch than to run when it is unrolled (half
// of the stalls of a single sequence's walk were instruction fetches).  The row's
// first and last groups go apart, so that the loop holds plain loads and arithmetic.
template <typename T, int U, typename F>
__device__ __forceinline__ void each(const Share& sh, const T* src, int mis, int V, F f) {
  constexpr int VE = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const bool plain = (reinterpret_cast<uintptr_t>(src - mis) & 15) == 0;
  // whole groups: those from 1 on that end within the row
  const int lo = plain ? min(max(sh.g0, 1), sh.g1) : sh.g0;
  const int hi = plain ? max(min(sh.g1, (V + mis) / VE), lo) : sh.g0;
  const uint4* at = reinterpret_cast<const uint4*>(src - mis);
  if constexpr (U > 1) {
    for (int k0 = lo + lane; k0 < hi; k0 += 32 * U) {
      uint4 raw[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + 32 * i < hi) raw[i] = __ldg(at + k0 + 32 * i);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (k0 + 32 * i < hi) {
          float v[VE];
          unpack_group<T>(raw[i], v);
          f(k0 + 32 * i, v);
        }
    }
  }
  // with U = 1 all groups take this loop, the plain ones with a load ahead
  const int n = U > 1 ? lo - sh.g0 + sh.g1 - hi : sh.g1 - sh.g0;
  auto group = [&](int j) { return U > 1 && j >= lo - sh.g0 ? hi + j - (lo - sh.g0) : sh.g0 + j; };
  auto load = [&](int k) {
    return k >= lo && k < hi ? __ldg(at + k) : load_edge<T>(src, k * VE - mis, V);
  };
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (lane < n) raw = load(group(lane));
#pragma unroll 1
  for (int j = lane; j < n; j += 32) {
    uint4 next = raw;
    if (j + 32 < n) next = load(group(j + 32));
    float v[VE];
    unpack_group<T>(raw, v);
    f(group(j), v);
    raw = next;
  }
}
// f(group, values, other row's values) over the warp's groups of two rows, one
// group's loads ahead.
template <typename T, typename F>
__device__ __forceinline__ void each2(const Share& sh, const T* src, const T* other, int mis, int V,
                                      F f) {
  constexpr int VE = 16 / sizeof(T);
  const bool plain = (reinterpret_cast<uintptr_t>(src - mis) & 15) == 0;
  const bool plain2 = (reinterpret_cast<uintptr_t>(other - mis) & 15) == 0;
  const int whole = (V + mis) / VE;  // groups 1 .. whole - 1 lie within the row
  auto load = [&](const T* s, bool pl, int k) {
    return pl && k > 0 && k < whole ? __ldg(reinterpret_cast<const uint4*>(s - mis) + k)
                                    : load_edge<T>(s, k * VE - mis, V);
  };
  int k = sh.g0 + (threadIdx.x & 31);
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (k < sh.g1) {
    a = load(src, plain, k);
    b = load(other, plain2, k);
  }
#pragma unroll 1
  for (; k < sh.g1; k += 32) {
    uint4 a1 = a, b1 = b;
    if (k + 32 < sh.g1) {
      a1 = load(src, plain, k + 32);
      b1 = load(other, plain2, k + 32);
    }
    float v[VE], w[VE];
    unpack_group<T>(a, v);
    unpack_group<T>(b, w);
    f(k, v, w);
    a = a1;
    b = b1;
  }
}
__device__ __forceinline__ ull pack_f2(float x, float y) {
  return (ull)__float_as_uint(y) << 32 | __float_as_uint(x);
}
// The maximum of the warp's part of a row and the fp32 sum of its weights over
// that maximum.  (A NaN argument, of a NaN logit or of inf - inf, is clamped to a
// weight of 0.)
template <typename T>
__device__ __noinline__ ull approx_of(Share sh, const T* src, int mis, int V, float inv_t) {
  constexpr int VE = 16 / sizeof(T);
  const float c = inv_t * 1.4426950408889634f;
  float m = -INFINITY, s = 0.f;
  each<T, 5>(sh, src, mis, V, [&](int, const float* v) {
    float top = m;
#pragma unroll
    for (int j = 0; j < VE; ++j) top = fmaxf(top, v[j]);
    if (top > m) {
      s *= ex2_ftz((m - top) * c);
      m = top;
    }
    // (subtracted first: a product with logits near the type's lowest value
    // would overflow)
#pragma unroll
    for (int j = 0; j < VE; ++j) s += ex2_ftz(fmaxf((v[j] - m) * c, -200.f));
  });
  const float top = warp_max(m);
  s = warp_sum(s * ex2_ftz(fmaxf((m - top) * c, -200.f)));
  return pack_f2(top, s);
}
// The maximum of the warp's part of a row and the lowest index that has it.
template <typename T>
__device__ __noinline__ ull max_of(Share sh, const T* src, int mis, int V) {
  constexpr int VE = 16 / sizeof(T);
  float m = -INFINITY;
  int ix = INT_MAX;
  each<T, 5>(sh, src, mis, V, [&](int k, const float* v) {
    float top = v[0];
#pragma unroll
    for (int j = 1; j < VE; ++j) top = fmaxf(top, v[j]);
    const int e0 = k * VE - mis;
    if (top > m || (top == m && e0 < ix)) {  // (the row's first group comes late)
      m = top;
#pragma unroll
      for (int j = VE - 1; j >= 0; --j)
        if (v[j] == top) ix = e0 + j;
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const int oi = __shfl_xor_sync(0xffffffffu, ix, o);
    if (om > m || (om == m && oi < ix)) { m = om; ix = oi; }
  }
  return (ull)(uint32_t)ix << 32 | __float_as_uint(m);
}
// The sums of the integer weights of the warp's parts of a row and, if there is
// one, of the draft's.
template <typename T>
__device__ __noinline__ Part sum_weights(Share sh, const T* src, const T* other, int mis, int V,
                                         float top, float top2, float inv_t) {
  constexpr int VE = 16 / sizeof(T);
  Sum s, s2;
  if (other) {
    each2<T>(sh, src, other, mis, V, [&](int, const float* v, const float* w) {
      float x[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = weight(v[j], top, inv_t);
      s.add<VE>(x);
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = weight(w[j], top2, inv_t);
      s2.add<VE>(x);
    });
  } else {
    each<T, 1>(sh, src, mis, V, [&](int, const float* v) {
      float x[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = weight(v[j], top, inv_t);
      s.add<VE>(x);
    });
  }
  return {s.warp(), s2.warp()};
}
// With a draft, what is left of p is kept in `cache`, this CTA's part of the row:
// shares() puts the warp's part of p = w / z there, reject() takes p = max(p / s - q,
// 0) (s 0: p as it is; s < 0: p = w / z is taken from the row), and both return the
// sum of the integer weights; scale() that of p / s without changing it.
//
// Many quotients by one divisor: with r = 1 / b rounded to nearest, q = a r and one
// correction by the exact remainder a - q b give a / b rounded to nearest
// (Markstein, Computation of elementary functions on the IBM RISC System/6000,
// 1990), three instructions.  Numerators below 2^-80, 40 powers of two under what
// an integer weight can show, are set to 0: their remainders could be denormal.
struct Divisor {
  float b, r;
  __device__ __forceinline__ explicit Divisor(float by) {
    b = by;
    r = by > 0.f ? __fdiv_rn(1.f, by) : 0.f;
  }
  __device__ __forceinline__ float of(float a) const {
    const float q = __fmul_rn(a, r);
    const float x = __fmaf_rn(__fmaf_rn(-q, b, a), r, q);
    return a >= 8.271806e-25f ? x : 0.f;
  }
};
template <typename T>
__device__ __noinline__ ull shares(Share sh, const T* src, int mis, int V, float top, float z,
                                   float inv_t, float* cache) {
  constexpr int VE = 16 / sizeof(T);
  Sum s;
  const Divisor by(z);
  each<T, 1>(sh, src, mis, V, [&](int k, const float* v) {
    float* c = cache + (k - sh.first) * VE;
    float x[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) x[j] = by.of(weight(v[j], top, inv_t));
    s.add<VE>(x);
#pragma unroll
    for (int j = 0; j < VE; j += 4)
      *reinterpret_cast<float4*>(c + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
  });
  return s.warp();
}
template <typename T>
__device__ __noinline__ ull reject(Share sh, const T* src, const T* other, int mis, int V,
                                   float top, float z, float top2, float zq, float inv_t, float s,
                                   float* cache) {
  constexpr int VE = 16 / sizeof(T);
  Sum sum;
  const bool first = s < 0.f;
  const Divisor by(zq), over(first ? z : s > 0.f ? s : 1.f);
  each2<T>(sh, src, other, mis, V, [&](int k, const float* v, const float* w) {
    float* c = cache + (k - sh.first) * VE;
    float x[VE];
    if (first) {
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = weight(v[j], top, inv_t);
    } else {
#pragma unroll
      for (int j = 0; j < VE; j += 4) {
        const float4 y = *reinterpret_cast<const float4*>(c + j);
        x[j] = y.x; x[j + 1] = y.y; x[j + 2] = y.z; x[j + 3] = y.w;
      }
    }
#pragma unroll
    for (int j = 0; j < VE; ++j)
      x[j] = fmaxf(over.of(x[j]) - by.of(weight(w[j], top2, inv_t)), 0.f);
    sum.add<VE>(x);
#pragma unroll
    for (int j = 0; j < VE; j += 4)
      *reinterpret_cast<float4*>(c + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
  });
  return sum.warp();
}
template <int VE>
__device__ __noinline__ ull scale(Share sh, float s, const float* cache) {
  Sum sum;
  const Divisor over(s > 0.f ? s : 1.f);
#pragma unroll 1
  for (int k = sh.g0 + (threadIdx.x & 31); k < sh.g1; k += 32) {
    const float* c = cache + (k - sh.first) * VE;
    float x[VE];
#pragma unroll
    for (int j = 0; j < VE; j += 4) {
      const float4 y = *reinterpret_cast<const float4*>(c + j);
      x[j] = over.of(y.x); x[j + 1] = over.of(y.y);
      x[j + 2] = over.of(y.z); x[j + 3] = over.of(y.w);
    }
    sum.add<VE>(x);
  }
  return sum.warp();
}
// The element of the warp's part at which the cumulative weight, `before` ahead
// of the part, passes `at`: in one lane, -1 in the others.  `weights` gives a
// group's.
template <int VE, typename F>
__device__ __forceinline__ long long find_at(const Share& sh, int mis, ull before, ull at,
                                             F weights) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int k0 = sh.g0; k0 < sh.g1; k0 += 32) {
    const int k = k0 + lane;
    ull w[VE], sum = 0;
#pragma unroll
    for (int j = 0; j < VE; ++j) w[j] = 0;
    if (k < sh.g1) weights(k, w);
#pragma unroll
    for (int j = 0; j < VE; ++j) sum += w[j];
    ull incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const ull up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const ull mine = before + incl - sum;
    const bool hit = at >= mine && at < mine + sum;
    if (__any_sync(0xffffffffu, hit)) {
      if (!hit) return -1;
      ull c = mine;
      int j = 0;  // elements whose cumulative weight does not pass `at`
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        c += w[e];
        j += c <= at;
      }
      return (long long)k * VE - mis + j;
    }
    before = __shfl_sync(0xffffffffu, before + incl, 31);
  }
  return -1;
}

// A token's share of a row's weights.
__device__ __noinline__ float share_of(float l, float m, float z, float inv_t) {
  return share(weight(l, m, inv_t), z);
}
// p of a token after the rejections so far, from its p and q before them.
__device__ __noinline__ float left_of(float pv, float qv, int nst, const float* stage) {
  for (int k = 0; k < nst; ++k)
    if (stage[k] > 0.f) pv = __fdiv_rn(fmaxf(pv - qv, 0.f), stage[k]);
  return pv;
}
// The first child of `cur` after node `after`, n if there is none.
__device__ __noinline__ int next_child(const int* par, int n, int cur, int after) {
  for (int base = (after + 1) & ~31; base < n; base += 32) {
    const int j = base + (threadIdx.x & 31);
    const unsigned hit = __ballot_sync(0xffffffffu, j > after && j < n && par[j] == cur);
    if (hit) return base + __ffs(hit) - 1;
  }
  return n;
}
// Whether an earlier child had node i's token (and so took its weight).
__device__ __noinline__ bool seen_before(const int* par, const int* tok, int cur, int i) {
  bool s = false;
  for (int j = cur + 1 + (threadIdx.x & 31); j < i; j += 32) s |= par[j] == cur && tok[j] == tok[i];
  return __any_sync(0xffffffffu, s) != 0;
}
// Sums of all parts' a and b.
template <int PARTS>
__device__ __noinline__ Part total(const Part* in) {
  Part r = {0, 0};
#pragma unroll 4
  for (int i = 0; i < PARTS / 32; ++i) {
    r.a += in[(threadIdx.x & 31) + 32 * i].a;
    r.b += in[(threadIdx.x & 31) + 32 * i].b;
  }
  r.a = warp_sum_u64(r.a);
  r.b = warp_sum_u64(r.b);
  return r;
}

// Gives this warp's part (in every lane) to all CTAs of the cluster and waits for
// all parts of the same turn.  A buffer is written again two turns later, when
// every warp has given its part of the turn between, and so has read this one's.
template <int C, int PARTS>
__device__ __noinline__ const Part* exchange(Shared<PARTS>& sm, int turn, int rank, ull a, ull b,
                                             int* err) {
  constexpr int W = PARTS / C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Part* in = sm.in[turn & 1];
  uint64_t* bar = reinterpret_cast<uint64_t*>(&sm.bar[turn & 1]);
  if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, sizeof(Part) * PARTS);
  if (lane < C) {
    uint32_t to, tb;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(in + rank * W + warp)), "r"(lane));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(tb) : "r"(smem_u32(bar)), "r"(lane));
    asm volatile(
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
        "r"((uint32_t)a), "r"((uint32_t)(a >> 32)), "r"((uint32_t)b), "r"((uint32_t)(b >> 32)), "r"(tb)
        : "memory");
  }
  const uint32_t parity = (turn >> 1) & 1;
  bool ok = false;
  for (uint32_t i = 0; i < kWaitLimit && !ok; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    ok = done != 0;
  }
  if (!ok && err) atomicExch(err, 71);
  __syncwarp();
  return in;
}

// C CTAs of TH threads a sequence; rank = blockIdx.y.
template <typename T, int C, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) verify_tree_kernel(VerifyArgs p) {
  constexpr int VE = 16 / sizeof(T), W = TH / 32, PARTS = C * W;
  __shared__ Shared<PARTS> sm;
  extern __shared__ __align__(16) float cache[];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.y, b = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool with_q = p.draft != nullptr && !p.greedy;
  if (tid == 0) {
    mbar_init(reinterpret_cast<uint64_t*>(&sm.bar[0]), 1);
    mbar_init(reinterpret_cast<uint64_t*>(&sm.bar[1]), 1);
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  const T* lb = static_cast<const T*>(p.logits) + b * p.l_sb;
  const T* db = with_q ? static_cast<const T*>(p.draft) + b * p.d_sb : nullptr;
  for (int i = tid; i < p.T; i += TH) {
    const int par = p.parents[b * p.par_sb + i];
    const int64_t t = p.tokens[b * p.tok_sb + i];
    const bool known = i > 0 && par >= 0 && par < i && t >= 0 && t < p.V;
    sm.par[i] = known ? par : -1;  // (a node without a token is nobody's child)
    sm.tok[i] = known ? (int)t : -1;
    const float u = p.greedy ? 0.f : p.u[b * p.u_sb + i];
    // outside [0, 1) its ends: a test would accept a token without weight, or reject
    // the only one left (the draw, with node 0's, sees to that itself)
    sm.u[i] = i == 0 ? u : u < 0.f ? 0.f : u >= 1.f ? 0x1.fffffep-1f : u;
    sm.lt[i] = known ? to_f32(lb[par * p.l_st + t]) : -INFINITY;
    sm.qt[i] = known && with_q ? to_f32(db[par * p.d_st + t]) : -INFINITY;
  }
  if (p.stats) {
    // a warp a row: its slices' maxima and sums
    const int rows = 2 * p.T - 1;  // (they are taken with a draft only)
    for (int i = warp; i < rows; i += W) {
      const int r = i < p.T ? b * p.T + i : p.B * p.T + b * (p.T - 1) + i - p.T;
      const float2* st = p.stats + (int64_t)r * p.slices;
      float m = -INFINITY, s = 0.f;
      for (int k = lane; k < p.slices; k += 32) m = fmaxf(m, st[k].x);
      m = warp_max(m);
      for (int k = lane; k < p.slices; k += 32) {
        const float f = ex2_ftz((st[k].x - m) * p.inv_t * 1.4426950408889634f);
        s += f == f ? st[k].y * f : 0.f;
      }
      s = warp_sum(s);
      if (lane == 0) {
        if (i < p.T) { sm.m[i] = m; sm.z[i] = s; }
        else { sm.mq[i - p.T] = m; sm.zq[i - p.T] = s; }
      }
    }
  }
  if (p.stats) {
    __syncthreads();
    for (int i = tid; i < p.T; i += TH) {
      const int par = max(sm.par[i], 0);
      const float w = weight(sm.lt[i], sm.m[par], p.inv_t);
      sm.pt[i] = share(w, sm.z[par]);
      if (i > 0)
        sm.uq[i] = __fmul_rn(sm.u[i], share(weight(sm.qt[i], sm.mq[par], p.inv_t), sm.zq[par]));
    }
  }
  cluster.sync();  // all CTAs run: their shared memory can be written

  const int gc = ((p.V + 2 * VE - 2) / VE + C - 1) / C;
  const int gw = (gc + W - 1) / W;
  Share sh;
  sh.first = rank * gc;
  sh.g0 = min(sh.first + warp * gw, sh.first + gc);
  sh.g1 = min(sh.g0 + gw, sh.first + gc);
  int turn = 0;  // exchanges so far
  auto sum1 = [&](ull mine) {
    const Part* in = exchange<C>(sm, turn++, rank, mine, 0, p.err);
    return total<PARTS>(in).a;
  };

  int32_t* path = p.path + (int64_t)b * p.T;
  int cur = 0, last = 0, n = 1, best = -1;
  for (;;) {
    const T* row = lb + cur * p.l_st;
    const T* qrow = with_q && cur < p.T - 1 ? db + cur * p.d_st : nullptr;
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    float m, mq = -INFINITY, z = 0.f, zq = 0.f;
    ull left = 0;         // integer weights left at the node (no draft)
    bool summed = false;  // z, zq and left are exact, not the statistics'
    int nst = 0;          // rejections with a draft: stages of the residual
    float over = 0.f;     // the cache holds p times this (0: p itself)
    auto sums = [&]() {   // the exact sums of the node's weights
      const Part s = sum_weights<T>(sh, row, qrow, mis, p.V, m, mq, p.inv_t);
      const Part* in = exchange<C>(sm, turn++, rank, s.a, s.b, p.err);
      const Part r = total<PARTS>(in);
      left = r.a;
      z = unfixed(r.a);
      zq = unfixed(r.b);
      summed = true;
    };
    if (p.stats) {
      m = sm.m[cur];
      z = sm.z[cur];
      if (qrow) { mq = sm.mq[cur]; zq = sm.zq[cur]; }
      left = (ull)((double)z * kFix);
    } else if (p.greedy) {
      const Part* in = exchange<C>(sm, turn, rank, max_of<T>(sh, row, mis, p.V), 0, p.err);
      ++turn;
      m = -INFINITY;
      int ix = INT_MAX;
#pragma unroll 4
      for (int i = 0; i < PARTS / 32; ++i) {  // (ascending indexes)
        const ull o = in[lane * (PARTS / 32) + i].a;
        const float x = __uint_as_float((uint32_t)o);
        if (x > m) { m = x; ix = (int)(o >> 32); }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oi = __shfl_xor_sync(0xffffffffu, ix, o);
        if (om > m || (om == m && oi < ix)) { m = om; ix = oi; }
      }
      best = m > -INFINITY ? ix : -1;
    } else {
      const ull a = approx_of<T>(sh, row, mis, p.V, p.inv_t);
      const ull c = qrow ? approx_of<T>(sh, qrow, mis, p.V, p.inv_t) : pack_f2(-INFINITY, 0.f);
      const Part* in = exchange<C>(sm, turn, rank, a, c, p.err);
      ++turn;
      const float sc = p.inv_t * 1.4426950408889634f;
      m = -INFINITY;
#pragma unroll 4
      for (int i = 0; i < PARTS / 32; ++i) {
        m = fmaxf(m, __uint_as_float((uint32_t)in[lane + 32 * i].a));
        mq = fmaxf(mq, __uint_as_float((uint32_t)in[lane + 32 * i].b));
      }
      m = warp_max(m);
      mq = warp_max(mq);
#pragma unroll 4
      for (int i = 0; i < PARTS / 32; ++i) {
        const Part o = in[lane + 32 * i];
        z += __uint_as_float((uint32_t)(o.a >> 32)) *
             ex2_ftz(fmaxf((__uint_as_float((uint32_t)o.a) - m) * sc, -200.f));
        zq += __uint_as_float((uint32_t)(o.b >> 32)) *
              ex2_ftz(fmaxf((__uint_as_float((uint32_t)o.b) - mq) * sc, -200.f));
      }
      z = warp_sum(z);
      zq = warp_sum(zq);
      left = (ull)((double)z * kFix);
    }
    // ---- the children, in index order ----
    bool down = false;
    for (int i = next_child(sm.par, p.T, cur, last); i < p.T;) {
      const int t = sm.tok[i];
      bool ok = false, again = false;  // again: with the exact sums
      if (p.greedy) {
        ok = t == best && best >= 0;
      } else if (with_q) {
        float uq, pt;
        if (p.stats && !summed) {
          uq = sm.uq[i];
          pt = sm.pt[i];
        } else {
          const float qv = share_of(sm.qt[i], mq, zq, p.inv_t);
          uq = __fmul_rn(sm.u[i], qv);
          pt = left_of(share_of(sm.lt[i], m, z, p.inv_t), qv, nst, sm.stage);
        }
        again = !summed && fabsf(uq - pt) <= 3.f * p.sum_error * fmaxf(uq, pt);
        ok = uq < pt;
        again |= !summed && !ok;  // the residual needs them
        if (!again && !ok) {
          const ull r = sum1(reject<T>(sh, row, qrow, mis, p.V, m, z, mq, zq, p.inv_t,
                                       nst == 0 ? -1.f : over, cache));
          sm.stage[nst] = unfixed(r);  // (all threads write the same)
          if (r > 0) {
            over = unfixed(r);
          } else {
            // nothing left: p stays as it was, rebuilt stage by stage
            shares<T>(sh, row, mis, p.V, m, z, p.inv_t, cache);
            float s = 0.f;
#pragma unroll 1
            for (int k = 0; k < nst; ++k)
              if (sm.stage[k] > 0.f) {
                reject<T>(sh, row, qrow, mis, p.V, m, z, mq, zq, p.inv_t, s, cache);
                s = sm.stage[k];
              }
          }
          ++nst;
        }
      } else {
        const ull w = seen_before(sm.par, sm.tok, cur, i)
                          ? 0 : fixed(weight(sm.lt[i], m, p.inv_t));
        const double u = (double)sm.u[i];
        ok = u * (double)left < (double)w;
        again = !summed && fabs(u * (double)left - (double)w) <= u * p.sum_error * kFix * (double)z;
        if (!again && !ok) left -= min(left, w);
      }
      if (again) {
        sums();
        if (!with_q)  // less what the earlier children took
          for (int j = next_child(sm.par, p.T, cur, cur); j < i; j = next_child(sm.par, p.T, cur, j))
            if (!seen_before(sm.par, sm.tok, cur, j))
              left -= fixed(weight(sm.lt[j], m, p.inv_t));
        continue;  // the same child
      }
      last = i;
      if (ok) {
        if (rank == 0 && tid == 0) path[n] = i;
        ++n;
        cur = i;
        down = true;
        break;
      }
      i = next_child(sm.par, p.T, cur, last);
    }
    if (down) continue;

    // ---- the draw from what is left at the last node ----
    long long next = -1;
    bool owner = rank == 0 && tid == 0;
    if (p.greedy) {
      next = best;
    } else {
      if (!summed) sums();
      int nout = 0;
      if (with_q) {
        sum1(nst == 0 ? shares<T>(sh, row, mis, p.V, m, z, p.inv_t, cache)
                      : scale<VE>(sh, over, cache));
      } else {
        for (int j = next_child(sm.par, p.T, cur, cur); j < p.T; j = next_child(sm.par, p.T, cur, j))
          if (!seen_before(sm.par, sm.tok, cur, j)) sm.out[nout++] = j;  // (all threads write the same)
      }
      // the parts of the last exchange, less the rejected tokens
      const Part* in = sm.in[(turn - 1) & 1];
      const int me = rank * W + warp;
      ull all = 0, before = 0, mine = in[me].a;
#pragma unroll
      for (int i = 0; i < PARTS / 32; ++i) {
        const int e = lane + 32 * i;
        all += in[e].a;
        if (e < me) before += in[e].a;
      }
      all = warp_sum_u64(all);
      before = warp_sum_u64(before);
      for (int j = 0; j < nout; ++j) {
        const int i = sm.out[j], k = (sm.tok[i] + mis) / VE;
        const ull w = fixed(weight(sm.lt[i], m, p.inv_t));
        const int e = k / gc * W + k % gc / gw;
        all -= w;
        if (e < me) before -= w;
        if (e == me) mine -= w;
      }
      if (all > 0) {
        ull at = (ull)(fmax((double)sm.u[0], 0.0) * (double)all);  // (u outside [0, 1): its ends)
        if (at >= all) at = all - 1;
        owner = false;
        if (at >= before && at < before + mine) {  // in this warp's part
          if (with_q) {
            const Divisor by(over > 0.f ? over : 1.f);
            next = find_at<VE>(sh, mis, before, at, [&](int k, ull* w) {
              const float* c = cache + (k - sh.first) * VE;
#pragma unroll
              for (int j = 0; j < VE; ++j) w[j] = fixed(by.of(c[j]));
            });
          } else {
            next = find_at<VE>(sh, mis, before, at, [&](int k, ull* w) {
              const int e0 = k * VE - mis;
              float f[VE];
              unpack_group<T>(load_group<T>(row, e0, p.V), f);
              for (int j = 0; j < nout; ++j) {
                const int d = sm.tok[sm.out[j]] - e0;
#pragma unroll
                for (int q = 0; q < VE; ++q)
                  if (d == q) f[q] = -INFINITY;
              }
#pragma unroll
              for (int j = 0; j < VE; ++j) w[j] = fixed(weight(f[j], m, p.inv_t));
            });
          }
          owner = next >= 0;
        }
      }
    }
    if (owner) p.next[b] = next;
    break;
  }
  if (rank == 0) {
    if (tid == 0) { path[0] = 0; p.count[b] = n; }
    for (int i = n + tid; i < p.T; i += TH) path[i] = -1;
  }
  cluster.sync();  // a CTA's shared memory outlives its writers
}

int stats_slices(int64_t V, int64_t item) {
  return (int)((V * item / 16 + 1 + kSlice) / kSlice);  // whatever the rows' alignment
}
// Statistics ahead of the walk, or as it goes: ahead where a node takes two rows
// (a draft's too) and the rows off the path are few.  Measured (us, ahead / going):
// 1 chain of 5 nodes over 151936 tokens with its draft 28.0 / 44.9, 64 of 9 over
// 32003 51.8 / 79.3, 32 of 16 over 151936 126.7 / 168.3; 8 trees of 32 with a draft
// 94.5 / 74.0; without a draft 1 tree of 32 19.5 / 16.6, 32 of them 106 / 32.
bool use_stats(int64_t B, int64_t T, int with_q) {
  return with_q && T > 1 && T <= 16 && B * (2 * T - 1) <= 65535;
}

// 8 CTAs a sequence, of 512 threads for few sequences, of 256 for more, so that all
// of them fit the SMs at once: 64 chains of 9 nodes over 32003 tokens 69.8 us with 512,
// 52.6 with 256; 1 chain of 5 over 151936 28.2 and 33.8.  (16 CTAs of 1024: 31.4.)
int walk_threads(int64_t B) {
  return 16 * B <= 2 * num_sms() ? 512 : 256;
}

// Bytes of the cache of what is left of p: a CTA's part of a row, in fp32.
template <typename T, int C>
constexpr size_t cache_bytes(int V) {
  constexpr int VE = 16 / sizeof(T);
  return (size_t)((V + 2 * VE - 2) / VE + C - 1) / C * VE * sizeof(float);
}
template <typename T, int C, int TH>
int walk_launch(const VerifyArgs& a, int64_t B, cudaStream_t st) {
  static std::atomic<bool> reserved[64];
  auto kern = verify_tree_kernel<T, C, TH>;
  const size_t cache = a.draft && !a.greedy ? cache_bytes<T, C>(a.V) : 0;
  if (cache > 16 * 1024)
    if (const int e = reserve_smem(reinterpret_cast<const void*>(kern), reserved,
                                   cache_bytes<T, C>(kMaxDraftVocab), "verify_tree_kernel"))
      return e;
  return launch("verify_tree_kernel", kern, dim3((unsigned)B, C), dim3(TH), cache, st, C, a);
}
template <typename T>
int walk_as(const VerifyArgs& a, int64_t B, cudaStream_t st) {
  return walk_threads(B) == 512 ? walk_launch<T, 8, 512>(a, B, st) : walk_launch<T, 8, 256>(a, B, st);
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int64_t tpp_verify_tree_workspace(int64_t B, int64_t T, int64_t V, int with_draft,
                                             double temperature, int dtype) {
  const int64_t item = dtype == TPP_F32 ? 4 : 2;
  if (B <= 0 || T <= 0 || V <= 0 || temperature <= 0.0) return 0;
  if (!use_stats(B, T, with_draft)) return 0;
  return B * (2 * T - 1) * stats_slices(V, item) * (int64_t)sizeof(float2);
}

extern "C" int tpp_verify_tree(const void* logits, int64_t l_sb, int64_t l_st,
                               const void* draft_logits, int64_t d_sb, int64_t d_st,
                               const int64_t* tokens, int64_t tok_sb, const int32_t* parents,
                               int64_t par_sb, const float* u, int64_t u_sb, double temperature,
                               int32_t* path, int32_t* count, int64_t* next_token, int64_t B,
                               int64_t T, int64_t V, void* workspace, int64_t workspace_bytes,
                               int dtype, void* stream) {
  if (B == 0) return TPP_OK;
  TPP_REQUIRE(logits && tokens && parents && path && count && next_token, TPP_ERR_SHAPE,
              "null pointer");
  TPP_REQUIRE(temperature >= 0.0 && temperature <= 1e30, TPP_ERR_SHAPE,
              "temperature must be finite and not negative");
  TPP_REQUIRE(temperature == 0.0 || (u != nullptr && temperature >= 1e-30), TPP_ERR_SHAPE,
              "temperature > 0 needs the uniform numbers");
  TPP_REQUIRE(B > 0 && B <= 65535 && T > 0 && T <= kMaxNodes && V > 0 && V <= (1 << 22),
              TPP_ERR_SHAPE, "need 1..65535 sequences, 1..256 nodes and 1..2^22 tokens");
  TPP_REQUIRE(dtype == TPP_F16 || dtype == TPP_BF16 || dtype == TPP_F32, TPP_ERR_DTYPE,
              "dtype must be f16, bf16 or f32");
  const int64_t need =
      tpp_verify_tree_workspace(B, T, V, draft_logits != nullptr, temperature, dtype);
  TPP_REQUIRE(need == 0 || (workspace && workspace_bytes >= need &&
                            (reinterpret_cast<uintptr_t>(workspace) & 7) == 0),
              TPP_ERR_WORKSPACE, "workspace missing, too small or not 8-byte aligned");
  VerifyArgs a;
  a.logits = logits; a.l_sb = l_sb; a.l_st = l_st;
  a.draft = draft_logits; a.d_sb = d_sb; a.d_st = d_st;
  a.tokens = tokens; a.tok_sb = tok_sb; a.parents = parents; a.par_sb = par_sb;
  a.u = u; a.u_sb = u_sb;
  a.greedy = temperature == 0.0;
  a.inv_t = a.greedy ? 1.f : (float)(1.0 / temperature);
  a.path = path; a.count = count; a.next = next_token;
  a.B = (int)B; a.T = (int)T; a.V = (int)V;
  a.stats = need ? static_cast<float2*>(workspace) : nullptr;
  a.slices = stats_slices(V, dtype == TPP_F32 ? 4 : 2);
  // A lane adds V / 2048 terms (8 CTAs of 256) one by one, then some dozens of
  // partial sums; an exponential's argument is rounded thrice at |x| <= 46 (smaller
  // weights do not count), itself twice.
  a.sum_error = 8e-6f + (float)(V / 2048 + 64) * 5.9604645e-8f;
  a.err = device_error_flag();
  TPP_REQUIRE(!draft_logits || a.greedy || V <= kMaxDraftVocab, TPP_ERR_UNSUPPORTED,
              "draft logits need a vocabulary of at most 400000 tokens");
  if (need) {
    const dim3 grid((unsigned)a.slices, (unsigned)(B * (2 * T - 1)));
    auto stats = [&](auto kern) {
      return launch("verify_stats_kernel", kern, grid, dim3(256), 0, as_stream(stream), 0u, a);
    };
    const int rc = dtype == TPP_F16 ? stats(verify_stats_kernel<__half>)
                 : dtype == TPP_BF16 ? stats(verify_stats_kernel<__nv_bfloat16>)
                                     : stats(verify_stats_kernel<float>);
    if (rc != TPP_OK) return rc;
  }
  if (dtype == TPP_F16) return walk_as<__half>(a, B, as_stream(stream));
  if (dtype == TPP_BF16) return walk_as<__nv_bfloat16>(a, B, as_stream(stream));
  return walk_as<float>(a, B, as_stream(stream));
}
