// Verification of a drafted tree against the target's logits (tpp_verify_tree).
//
// One cluster of 8 CTAs walks one sequence's tree from the root.  At a node it
// needs the softmax of one row of logits (and of the draft's row, where the
// children were drawn from one).  Every CTA of the cluster holds an eighth of the
// row; every thread makes the same decisions from the exchanged sums.
//
// Weights are exp((l - max) / temperature) in fp32; sums and cumulative sums of
// weights run over 64-bit integers, round(w * 2^40), so they are exact and a
// result does not depend on the order or the split of a row (fp32 cumulative
// sums over 150k tokens move the boundaries of a draw by about 1e-6).
//
// What a walk costs is its chain of passes and exchanges, two a node (the maximum,
// the sum).  An exchange is one remote store a warp and CTA (st.async, counted by
// the receiver's mbarrier) and no barrier of the CTA or the cluster.  For small
// batches verify_stats_kernel first takes every row's maximum and an fp32 sum on
// all SMs; the walk decides from those, and goes through the exact sums only where
// a test comes within the fp32 sum's error of a tie, and for the draw.  For larger
// ones reading the rows off the path costs more than the exchanges: rows are then
// read as the walk reaches them.
#include <limits.h>
#include <math.h>
#include <cstdlib>
#include <cooperative_groups.h>
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace tpp {
namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxNodes = 256;
constexpr int kUnroll = 5;           // groups a lane has in flight: all of its
                                     // share of 160k tokens of 16 bits
constexpr int kSlice = 1024;         // groups of a row for a CTA of the statistics
constexpr double kFix = 1099511627776.0;  // 2^40
// Relative error of the statistics' sums: fp32 sums of at most 32 + 13 + 512 / 32
// terms in a row and an exponential within 2^-21 of exact (its argument rounded at
// |x| < 32; weights below e^-32 do not count).
constexpr float kSumError = 1e-5f;
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
  int* err;
  int slices;
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

// Elements [e0, e0 + VE) of a row of V as they are stored, -inf outside it.  The
// slow way is for a row's ends, and for a draft row whose start is aligned
// otherwise than the target's.
template <typename T>
__device__ __forceinline__ uint4 load_group(const T* row, int e0, int V) {
  constexpr int VE = 16 / sizeof(T);
  const T* a = row + e0;
  if (e0 >= 0 && e0 + VE <= V && (reinterpret_cast<uintptr_t>(a) & 15) == 0)
    return __ldg(reinterpret_cast<const uint4*>(a));
  ull w[2] = {0, 0};
#pragma unroll 1
  for (int j = 0; j < VE; ++j) {
    const T x = e0 + j >= 0 && e0 + j < V ? a[j] : from_f32<T>(-INFINITY);
    ull bits;
    if constexpr (sizeof(T) == 4) bits = __float_as_uint(x);
    else bits = *reinterpret_cast<const unsigned short*>(&x);
    bits <<= (j * sizeof(T) * 8) & 63;
    if (j < VE / 2) w[0] |= bits;
    else w[1] |= bits;
  }
  return make_uint4((uint32_t)w[0], (uint32_t)(w[0] >> 32), (uint32_t)w[1],
                    (uint32_t)(w[1] >> 32));
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
  uint4 raw[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int k = blockIdx.x * kSlice + i * 256 + tid;
    raw[i] = load_group<T>(row.p, k < row.groups ? k * VE - row.mis : p.V, p.V);
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float f[VE];
    unpack_group<T>(raw[i], f);
#pragma unroll
    for (int j = 0; j < VE; ++j) m = fmaxf(m, f[j]);
  }
  m = warp_max(m);
  if ((tid & 31) == 0) sm[tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < 8; ++w) m = fmaxf(m, sm[w]);
  float s = 0.f;
  const float c = p.inv_t * 1.4426950408889634f;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float f[VE];
    unpack_group<T>(raw[i], f);
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float w = ex2_ftz((f[j] - m) * c);
      s += w == w ? w : 0.f;
    }
  }
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

struct Shared {
  Part in[2][kCluster * kWarps];  // every warp's part, by the exchange's parity
  ull bar[2];
  float stage[kMaxNodes];  // sums of the residual after each rejection
  int out[kMaxNodes];      // rejected tokens
  int par[kMaxNodes];
  int tok[kMaxNodes];      // -1: not a token
  float u[kMaxNodes];
  float lt[kMaxNodes], qt[kMaxNodes];  // a node's own logit in its parent's rows
  float m[kMaxNodes], z[kMaxNodes], mq[kMaxNodes], zq[kMaxNodes];  // from the statistics
};

// How the cluster's warps share a row: `gc` groups a CTA, of which this warp owns
// [g0, g1) (counted from the row's first, whatever its alignment).
struct Share { int first, g0, g1; };

// f(group, values) over the warp's groups of a row, kUnroll loads at a time; the
// second pass over a row finds it in L1.
template <typename T, typename F>
__device__ __forceinline__ void each(const Share& sh, const T* src, int mis, int V, F f) {
  constexpr int VE = 16 / sizeof(T);
  for (int k0 = sh.g0 + (threadIdx.x & 31); k0 < sh.g1; k0 += 32 * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (k0 + 32 * i < sh.g1) raw[i] = load_group<T>(src, (k0 + 32 * i) * VE - mis, V);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (k0 + 32 * i < sh.g1) {
        float v[VE];
        unpack_group<T>(raw[i], v);
        f(k0 + 32 * i, v);
      }
  }
}
// The maximum of the warp's part of a row and the lowest index that has it.
template <typename T>
__device__ __noinline__ ull max_of(Share sh, const T* src, int mis, int V) {
  constexpr int VE = 16 / sizeof(T);
  float m = -INFINITY;
  int ix = INT_MAX;
  each<T>(sh, src, mis, V, [&](int k, const float* v) {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (v[j] > m) { m = v[j]; ix = k * VE - mis + j; }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const int oi = __shfl_xor_sync(0xffffffffu, ix, o);
    if (om > m || (om == m && oi < ix)) { m = om; ix = oi; }
  }
  return (ull)(uint32_t)ix << 32 | __float_as_uint(m);
}
// The sum of the integer weights of the warp's part of a row.
template <typename T>
__device__ __noinline__ ull sum_weights(Share sh, const T* src, int mis, int V, float top,
                                        float inv_t) {
  constexpr int VE = 16 / sizeof(T);
  ull hi = 0;
  long long lo = 0;
  each<T>(sh, src, mis, V, [&](int, const float* v) {
    uint32_t h = 0;
    int l = 0;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      uint32_t hj;
      int lj;
      fixed_parts(weight(v[j], top, inv_t), hj, lj);
      h += hj;
      l += lj;
    }
    hi += h;
    lo += l;
  });
  return warp_sum_u64(fixed_sum(hi, lo));
}
// With a draft, what is left of p is kept in `cache`, this CTA's part of the row:
// shares() puts the warp's part of p = w / z there, reject() takes p = max(p / s - q,
// 0) (s 0: p as it is), and both return the sum of the integer weights; scale()
// that of p / s without changing it.
template <typename T>
__device__ __noinline__ ull shares(Share sh, const T* src, int mis, int V, float top, float z,
                                   float inv_t, float* cache) {
  constexpr int VE = 16 / sizeof(T);
  ull s = 0;
  each<T>(sh, src, mis, V, [&](int k, const float* v) {
    float* c = cache + (k - sh.first) * VE;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      c[j] = share(weight(v[j], top, inv_t), z);
      s += fixed(c[j]);
    }
  });
  return warp_sum_u64(s);
}
__device__ __forceinline__ float scaled(float p, float s) { return s > 0.f ? __fdiv_rn(p, s) : p; }
template <typename T>
__device__ __noinline__ ull reject(Share sh, const T* src, int mis, int V, float top, float zq,
                                   float inv_t, float s, float* cache) {
  constexpr int VE = 16 / sizeof(T);
  ull sum = 0;
  each<T>(sh, src, mis, V, [&](int k, const float* v) {
    float* c = cache + (k - sh.first) * VE;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      c[j] = fmaxf(scaled(c[j], s) - share(weight(v[j], top, inv_t), zq), 0.f);
      sum += fixed(c[j]);
    }
  });
  return warp_sum_u64(sum);
}
template <int VE>
__device__ __noinline__ ull scale(Share sh, float s, const float* cache) {
  ull sum = 0;
  for (int k = sh.g0 + (threadIdx.x & 31); k < sh.g1; k += 32) {
    const float* c = cache + (k - sh.first) * VE;
#pragma unroll
    for (int j = 0; j < VE; ++j) sum += fixed(scaled(c[j], s));
  }
  return warp_sum_u64(sum);
}
// The element of the warp's part at which the cumulative weight, `before` ahead
// of the part, passes `at`: in one lane, -1 in the others.  `weights` gives a
// group's.
template <int VE, typename F>
__device__ __forceinline__ long long find_at(const Share& sh, int mis, ull before, ull at,
                                             F weights) {
  const int lane = threadIdx.x & 31;
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

// Gives this warp's part (in every lane) to all CTAs of the cluster and waits for
// all parts of the same turn.  A buffer is written again two turns later, when
// every warp has given its part of the turn between, and so has read this one's.
__device__ __noinline__ const Part* exchange(Shared& sm, int turn, int rank, ull a, ull b, int* err) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Part* in = sm.in[turn & 1];
  uint64_t* bar = reinterpret_cast<uint64_t*>(&sm.bar[turn & 1]);
  if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, sizeof(Part) * kCluster * kWarps);
  if (lane < kCluster) {
    uint32_t to, tb;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(in + rank * kWarps + warp)), "r"(lane));
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) __cluster_dims__(kCluster, 1, 1)
    verify_tree_kernel(VerifyArgs p) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ Shared sm;
  extern __shared__ __align__(16) float cache[];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x, b = blockIdx.y;
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
  for (int i = tid; i < p.T; i += kThreads) {
    const int par = p.parents[b * p.par_sb + i];
    const int64_t t = p.tokens[b * p.tok_sb + i];
    const bool known = i > 0 && par >= 0 && par < i && t >= 0 && t < p.V;
    sm.par[i] = i > 0 && par < i ? par : -1;
    sm.tok[i] = known ? (int)t : -1;
    sm.u[i] = p.greedy ? 0.f : p.u[b * p.u_sb + i];
    sm.lt[i] = known ? to_f32(lb[par * p.l_st + t]) : -INFINITY;
    sm.qt[i] = known && with_q ? to_f32(db[par * p.d_st + t]) : -INFINITY;
  }
  if (p.stats) {
    // a warp a row: its slices' maxima and sums
    const int rows = p.T + (with_q ? p.T - 1 : 0);
    for (int i = warp; i < rows; i += kWarps) {
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
  cluster.sync();  // all CTAs run: their shared memory can be written

  const int gc = ((p.V + 2 * VE - 2) / VE + kCluster - 1) / kCluster;
  const int gw = (gc + kWarps - 1) / kWarps;
  Share sh;
  sh.first = rank * gc;
  sh.g0 = min(sh.first + warp * gw, sh.first + gc);
  sh.g1 = min(sh.g0 + gw, sh.first + gc);
  int turn = 0;  // exchanges so far
  // sums of a and b over all parts
  auto total = [&](const Part* in, ull& a, ull& c) {
    a = c = 0;
#pragma unroll
    for (int i = 0; i < kCluster * kWarps / 32; ++i) {
      a += in[lane + 32 * i].a;
      c += in[lane + 32 * i].b;
    }
    a = warp_sum_u64(a);
    c = warp_sum_u64(c);
  };
  auto sum1 = [&](ull mine) {
    ull a, c;
    total(exchange(sm, turn, rank, mine, 0, p.err), a, c);
    ++turn;
    return a;
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
      const ull s = sum_weights<T>(sh, row, mis, p.V, m, p.inv_t);
      const ull sq = qrow ? sum_weights<T>(sh, qrow, mis, p.V, mq, p.inv_t) : 0;
      ull a, c;
      total(exchange(sm, turn, rank, s, sq, p.err), a, c);
      ++turn;
      left = a;
      z = unfixed(a);
      zq = unfixed(c);
      summed = true;
    };
    if (p.stats) {
      m = sm.m[cur];
      z = sm.z[cur];
      if (qrow) { mq = sm.mq[cur]; zq = sm.zq[cur]; }
      left = (ull)((double)z * kFix);
    } else {
      const ull a = max_of<T>(sh, row, mis, p.V);
      const ull c = qrow ? max_of<T>(sh, qrow, mis, p.V) : __float_as_uint(-INFINITY);
      const Part* in = exchange(sm, turn, rank, a, c, p.err);
      ++turn;
      m = -INFINITY;
      int ix = INT_MAX;
#pragma unroll
      for (int i = 0; i < kCluster * kWarps / 32; ++i) {  // (ascending indexes)
        const Part o = in[lane * (kCluster * kWarps / 32) + i];
        const float x = __uint_as_float((uint32_t)o.a);
        if (x > m) { m = x; ix = (int)(o.a >> 32); }
        mq = fmaxf(mq, __uint_as_float((uint32_t)o.b));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oi = __shfl_xor_sync(0xffffffffu, ix, o);
        if (om > m || (om == m && oi < ix)) { m = om; ix = oi; }
      }
      mq = warp_max(mq);
      best = m > -INFINITY ? ix : -1;
      if (!p.greedy) sums();
    }
    // p and q of child i's token, after nst rejections
    auto p_of = [&](int i) {
      float pv = share(weight(sm.lt[i], m, p.inv_t), z);
      const float qv = share(weight(sm.qt[i], mq, p.inv_t), zq);
      for (int k = 0; k < nst; ++k)
        if (sm.stage[k] > 0.f) pv = __fdiv_rn(fmaxf(pv - qv, 0.f), sm.stage[k]);
      return pv;
    };
    auto uq_of = [&](int i) {
      return __fmul_rn(sm.u[i], share(weight(sm.qt[i], mq, p.inv_t), zq));
    };
    auto next_child = [&](int after) {
      for (int base = (after + 1) & ~31; base < p.T; base += 32) {
        const int j = base + lane;
        const unsigned hit = __ballot_sync(0xffffffffu, j > after && j < p.T && sm.par[j] == cur);
        if (hit) return base + __ffs(hit) - 1;
      }
      return p.T;
    };
    // whether an earlier child had node i's token (and so took its weight)
    auto seen = [&](int i) {
      bool s = false;
      for (int j = cur + 1 + lane; j < i; j += 32) s |= sm.par[j] == cur && sm.tok[j] == sm.tok[i];
      return __any_sync(0xffffffffu, s) != 0;
    };
    // ---- the children, in index order ----
    bool down = false;
    for (int i = next_child(last); i < p.T; i = next_child(last)) {
      last = i;
      const int t = sm.tok[i];
      bool ok = false;
      if (p.greedy) {
        ok = t == best && best >= 0;
      } else if (with_q) {
        if (t >= 0) {
          float uq = uq_of(i), pt = p_of(i);
          if (!summed && fabsf(uq - pt) <= 3.f * kSumError * fmaxf(uq, pt)) {
            sums();
            uq = uq_of(i);
            pt = p_of(i);
          }
          ok = uq < pt;
        }
        if (!ok) {
          if (!summed) sums();
          if (nst == 0) shares<T>(sh, row, mis, p.V, m, z, p.inv_t, cache);
          const ull r = sum1(reject<T>(sh, qrow, mis, p.V, mq, zq, p.inv_t, over, cache));
          sm.stage[nst] = unfixed(r);  // (all threads write the same)
          if (r > 0) {
            over = unfixed(r);
          } else {  // nothing left: p stays as it was, rebuilt stage by stage
            shares<T>(sh, row, mis, p.V, m, z, p.inv_t, cache);
            float s = 0.f;
            for (int k = 0; k < nst; ++k)
              if (sm.stage[k] > 0.f) {
                reject<T>(sh, qrow, mis, p.V, mq, zq, p.inv_t, s, cache);
                s = sm.stage[k];
              }
          }
          ++nst;
        }
      } else {
        const ull w = t >= 0 && !seen(i) ? fixed(weight(sm.lt[i], m, p.inv_t)) : 0;
        const double u = (double)sm.u[i];
        if (!summed && fabs(u * (double)left - (double)w) <= u * kSumError * kFix * (double)z) {
          sums();
          for (int j = next_child(cur); j < i; j = next_child(j))
            if (sm.tok[j] >= 0 && !seen(j)) left -= fixed(weight(sm.lt[j], m, p.inv_t));
        }
        ok = u * (double)left < (double)w;
        if (!ok) left -= min(left, w);
      }
      if (ok) {
        if (rank == 0 && tid == 0) path[n] = i;
        ++n;
        cur = i;
        down = true;
        break;
      }
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
        for (int j = next_child(cur); j < p.T; j = next_child(j))
          if (sm.tok[j] >= 0 && !seen(j)) sm.out[nout++] = j;  // (all threads write the same)
      }
      // the parts of the last exchange, less the rejected tokens
      const Part* in = sm.in[(turn - 1) & 1];
      const int me = rank * kWarps + warp;
      ull all = 0, before = 0, mine = in[me].a;
#pragma unroll
      for (int i = 0; i < kCluster * kWarps / 32; ++i) {
        const int e = lane + 32 * i;
        all += in[e].a;
        if (e < me) before += in[e].a;
      }
      all = warp_sum_u64(all);
      before = warp_sum_u64(before);
      for (int j = 0; j < nout; ++j) {
        const int i = sm.out[j], k = (sm.tok[i] + mis) / VE;
        const ull w = fixed(weight(sm.lt[i], m, p.inv_t));
        const int e = k / gc * kWarps + k % gc / gw;
        all -= w;
        if (e < me) before -= w;
        if (e == me) mine -= w;
      }
      if (all > 0) {
        ull at = (ull)((double)sm.u[0] * (double)all);
        if (at >= all) at = all - 1;
        owner = false;
        if (at >= before && at < before + mine) {  // in this warp's part
          if (with_q) {
            next = find_at<VE>(sh, mis, before, at, [&](int k, ull* w) {
              const float* c = cache + (k - sh.first) * VE;
#pragma unroll
              for (int j = 0; j < VE; ++j) w[j] = fixed(scaled(c[j], over));
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
    for (int i = n + tid; i < p.T; i += kThreads) path[i] = -1;
  }
  cluster.sync();  // a CTA's shared memory outlives its writers
}

// Rows are read ahead of the walk where all of them are at most this many bytes:
// measured (8 CTAs a sequence): see the launch below.
constexpr int64_t kStatsBytes = 32 << 20;

int stats_slices(int64_t V, int64_t item) {
  return (int)((V * item / 16 + 1 + kSlice) / kSlice);  // whatever the rows' alignment
}
int64_t stats_limit() { const char* e = getenv("TSTATS"); return e ? atoll(e) << 20 : kStatsBytes; }
bool use_stats(int64_t B, int64_t T, int64_t V, int with_q, int64_t item) {
  const int64_t rows = B * (T + (with_q ? T - 1 : 0));
  return T > 1 && rows <= 65535 && rows * V * item <= stats_limit();
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int64_t tpp_verify_tree_workspace(int64_t B, int64_t T, int64_t V, int with_draft,
                                             double temperature, int dtype) {
  const int64_t item = dtype == TPP_F32 ? 4 : 2;
  if (B <= 0 || T <= 0 || V <= 0 || temperature <= 0.0) return 0;
  if (!use_stats(B, T, V, with_draft, item)) return 0;
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
  a.err = device_error_flag();
  // the cache of what is left of p, a CTA's part of a row (with a draft)
  const int64_t ve = dtype == TPP_F32 ? 4 : 8;
  const size_t cache = draft_logits && !a.greedy
      ? ((V + 2 * ve - 2) / ve + kCluster - 1) / kCluster * ve * sizeof(float) : 0;
  TPP_REQUIRE(cache <= 200 * 1024, TPP_ERR_UNSUPPORTED,
              "draft logits need a vocabulary of at most 409600 tokens");
  auto go = [&](auto stats, auto walk) -> int {
    if (need) {
      const int64_t rows = B * (T + (draft_logits ? T - 1 : 0));
      const int rc = launch("verify_stats_kernel", stats, dim3((unsigned)a.slices, (unsigned)rows),
                            dim3(256), 0, as_stream(stream), 0u, a);
      if (rc != TPP_OK) return rc;
    }
    if (cache > 32 * 1024 &&
        cudaFuncSetAttribute(walk, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cache) !=
            cudaSuccess) {
      set_error("verify_tree_kernel: cannot reserve shared memory");
      return TPP_ERR_LAUNCH;
    }
    return launch("verify_tree_kernel", walk, dim3(kCluster, (unsigned)B), dim3(kThreads), cache,
                  as_stream(stream), 0u, a);
  };
  if (dtype == TPP_F16) return go(verify_stats_kernel<__half>, verify_tree_kernel<__half>);
  if (dtype == TPP_BF16)
    return go(verify_stats_kernel<__nv_bfloat16>, verify_tree_kernel<__nv_bfloat16>);
  return go(verify_stats_kernel<float>, verify_tree_kernel<float>);
}
