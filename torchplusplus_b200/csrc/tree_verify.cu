// Verification of a drafted tree against the target's logits (tpp_verify_tree).
//
// One cluster of 8 CTAs walks one sequence's tree from the root.  At a node it
// needs the softmax of one row of logits (and of the draft's row, where the
// children were drawn from one); only the rows on the accepted path are read.
// Every CTA of the cluster holds an eighth of the row, every thread makes the
// same decisions from the exchanged sums.
//
// Weights are exp((l - max) / temperature) in fp32; sums and cumulative sums of
// weights run over 64-bit integers, round(w * 2^40), so they are exact and a
// result does not depend on the order or the split of a row (fp32 cumulative
// sums over 150k tokens move the boundaries of a draw by about 1e-6).
#include <limits.h>
#include <math.h>
#include <cooperative_groups.h>
#include "common.cuh"

namespace cg = cooperative_groups;

namespace tpp {
namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxNodes = 256;
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
  int T; int V;
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

// Elements [e0, e0 + VE) of a row of V, -inf outside it.
template <typename T>
__device__ __forceinline__ void load_group(const T* row, int e0, int V, float* f) {
  constexpr int VE = 16 / sizeof(T);
  const T* a = row + e0;
  if (e0 >= 0 && e0 + VE <= V && (reinterpret_cast<uintptr_t>(a) & 15) == 0) {
    unpack_group<T>(__ldg(reinterpret_cast<const uint4*>(a)), f);
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      f[j] = (e0 + j >= 0 && e0 + j < V) ? to_f32(a[j]) : -INFINITY;
  }
}

// exp((l - m) / temperature), 0 where that is NaN (NaN logits; no finite max).
__device__ __forceinline__ float weight(float l, float m, float inv_t) {
  const float w = expf((l - m) * inv_t);
  return w == w ? w : 0.f;
}
__device__ __forceinline__ ull fixed(float w) { return __double2ull_rn((double)w * kFix); }
__device__ __forceinline__ float unfixed(ull s) { return (float)((double)s / kFix); }
__device__ __forceinline__ float share(float w, float z) { return z > 0.f ? __fdiv_rn(w, z) : 0.f; }

__device__ __forceinline__ ull warp_sum_u64(ull v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Slot { ull a, b; float x, y; int ix; };

struct Shared {
  Slot slot[2];            // this CTA's part of an exchange, by its parity
  ull wa[kWarps], wb[kWarps];
  float wx[kWarps], wy[kWarps];
  int wi[kWarps];
  ull tot[kWarps];         // each warp's part of the weights to draw from
  float stage[kMaxNodes];  // sums of the residual after each rejection
  int rejected[kMaxNodes];
  int par[kMaxNodes];
  long long tok[kMaxNodes];
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) __cluster_dims__(kCluster, 1, 1)
    verify_tree_kernel(VerifyArgs p) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ Shared sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool with_q = p.draft != nullptr && !p.greedy;
  pdl_wait();
  pdl_trigger();
  for (int i = tid; i < p.T; i += kThreads) {
    sm.par[i] = p.parents[b * p.par_sb + i];
    sm.tok[i] = p.tokens[b * p.tok_sb + i];
  }
  __syncthreads();
  int turn = 0;  // exchanges so far

  // Sum of (a, b) over the cluster; the warps' parts of a stay in sm.tot, the
  // CTAs' in slot[.].a of the exchange just made.
  auto sum2 = [&](ull& a, ull& c) {
    a = warp_sum_u64(a);
    c = warp_sum_u64(c);
    if (lane == 0) { sm.wa[warp] = a; sm.wb[warp] = c; }
    __syncthreads();
    if (tid == 0) {
      ull sa = 0, sb = 0;
      for (int w = 0; w < kWarps; ++w) { sa += sm.wa[w]; sb += sm.wb[w]; sm.tot[w] = sm.wa[w]; }
      sm.slot[turn & 1].a = sa;
      sm.slot[turn & 1].b = sb;
    }
    cluster.sync();
    a = c = 0;
    for (int r = 0; r < kCluster; ++r) {
      const Slot* s = cluster.map_shared_rank(&sm.slot[turn & 1], r);
      a += s->a;
      c += s->b;
    }
    ++turn;
  };
  // Maximum of x (with the lowest index that has it) and of y over the cluster.
  auto max2 = [&](float& x, int& ix, float& y) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ox = __shfl_xor_sync(0xffffffffu, x, o);
      const int oi = __shfl_xor_sync(0xffffffffu, ix, o);
      if (ox > x || (ox == x && oi < ix)) { x = ox; ix = oi; }
      y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, o));
    }
    if (lane == 0) { sm.wx[warp] = x; sm.wi[warp] = ix; sm.wy[warp] = y; }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) {
        if (sm.wx[w] > x || (sm.wx[w] == x && sm.wi[w] < ix)) { x = sm.wx[w]; ix = sm.wi[w]; }
        y = fmaxf(y, sm.wy[w]);
      }
      sm.slot[turn & 1].x = x;
      sm.slot[turn & 1].ix = ix;
      sm.slot[turn & 1].y = y;
    }
    cluster.sync();
    x = y = -INFINITY;
    ix = INT_MAX;
    for (int r = 0; r < kCluster; ++r) {
      const Slot* s = cluster.map_shared_rank(&sm.slot[turn & 1], r);
      const float ox = s->x;
      const int oi = s->ix;
      if (ox > x || (ox == x && oi < ix)) { x = ox; ix = oi; }
      y = fmaxf(y, s->y);
    }
    ++turn;
  };

  const T* lb = static_cast<const T*>(p.logits) + b * p.l_sb;
  const T* db = with_q ? static_cast<const T*>(p.draft) + b * p.d_sb : nullptr;
  const float* ub = p.greedy ? nullptr : p.u + b * p.u_sb;
  int32_t* path = p.path + (int64_t)b * p.T;
  int cur = 0, last = 0, n = 1, best = -1, nst = 0, nrej = 0;
  float m = 0.f, mq = 0.f, z = 0.f, zq = 0.f;
  ull left = 0;

  // Where this warp's groups of a row lie.
  auto range = [&](const Row<T>& row, int& g0, int& g1) {
    const int gc = (row.groups + kCluster - 1) / kCluster, gw = (gc + kWarps - 1) / kWarps;
    const int c0 = rank * gc, c1 = min(c0 + gc, row.groups);
    g0 = min(c0 + warp * gw, c1);
    g1 = min(g0 + gw, c1);
  };
  // What is left of p at an element, after the rejections so far.
  auto residual = [&](float l, float lq) {
    float pv = share(weight(l, m, p.inv_t), z);
    if (nst > 0) {
      const float qv = share(weight(lq, mq, p.inv_t), zq);
      for (int i = 0; i < nst; ++i) {
        const float s = sm.stage[i];
        if (s > 0.f) pv = __fdiv_rn(fmaxf(pv - qv, 0.f), s);
      }
    }
    return pv;
  };
  // The integer weights of group k to draw from.
  auto left_of = [&](const Row<T>& row, const T* qrow, int k, ull* w) {
    const int e0 = k * VE - row.mis;
    float f[VE], fq[VE];
    load_group<T>(row.p, e0, p.V, f);
    if (with_q) {
      if (nst > 0) load_group<T>(qrow, e0, p.V, fq);
#pragma unroll
      for (int j = 0; j < VE; ++j) w[j] = fixed(residual(f[j], nst > 0 ? fq[j] : 0.f));
    } else {
      for (int i = 0; i < nrej; ++i) {
        const int d = sm.rejected[i] - e0;
#pragma unroll
        for (int j = 0; j < VE; ++j)
          if (d == j) f[j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < VE; ++j) w[j] = fixed(weight(f[j], m, p.inv_t));
    }
  };

  for (;;) {
    const Row<T> row(lb + cur * p.l_st, p.V);
    const T* qrow = with_q && cur < p.T - 1 ? db + cur * p.d_st : nullptr;
    int g0, g1;
    range(row, g0, g1);
    // ---- maximum, then the sum of the weights ----
    m = mq = -INFINITY;
    int ix = INT_MAX;
    for (int k = g0 + lane; k < g1; k += 32) {
      const int e0 = k * VE - row.mis;
      float f[VE];
      load_group<T>(row.p, e0, p.V, f);
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (f[j] > m) { m = f[j]; ix = e0 + j; }
      if (qrow) {
        load_group<T>(qrow, e0, p.V, f);
#pragma unroll
        for (int j = 0; j < VE; ++j) mq = fmaxf(mq, f[j]);
      }
    }
    max2(m, ix, mq);
    best = m > -INFINITY ? ix : -1;
    nst = nrej = 0;
    if (!p.greedy) {
      ull s = 0, sq = 0;
      for (int k = g0 + lane; k < g1; k += 32) {
        const int e0 = k * VE - row.mis;
        float f[VE];
        load_group<T>(row.p, e0, p.V, f);
#pragma unroll
        for (int j = 0; j < VE; ++j) s += fixed(weight(f[j], m, p.inv_t));
        if (qrow) {
          load_group<T>(qrow, e0, p.V, f);
#pragma unroll
          for (int j = 0; j < VE; ++j) sq += fixed(weight(f[j], mq, p.inv_t));
        }
      }
      sum2(s, sq);
      left = s;
      z = unfixed(s);
      zq = unfixed(sq);
    }
    // ---- the children, in index order ----
    bool down = false;
    for (;;) {
      int i = p.T;
      for (int base = (last + 1) & ~31; base < p.T && i == p.T; base += 32) {
        const int j = base + lane;
        const unsigned hit = __ballot_sync(0xffffffffu, j > last && j < p.T && sm.par[j] == cur);
        if (hit) i = base + __ffs(hit) - 1;
      }
      if (i == p.T) break;
      last = i;
      const long long t = sm.tok[i];
      const bool known = t >= 0 && t < p.V;
      bool ok = false;
      if (p.greedy) {
        ok = t == best && best >= 0;
      } else if (with_q) {
        const float pt = known ? residual(to_f32(row.p[t]), to_f32(qrow[t])) : 0.f;
        const float qt = known ? share(weight(to_f32(qrow[t]), mq, p.inv_t), zq) : 0.f;
        ok = known && __fmul_rn(ub[i], qt) < pt;
        if (!ok) {
          ull s = 0, none = 0;
          __syncthreads();
          if (tid == 0) sm.stage[nst] = 1.f;  // p - q first, over 1
          __syncthreads();
          ++nst;
          for (int k = g0 + lane; k < g1; k += 32) {
            ull w[VE];
            left_of(row, qrow, k, w);
#pragma unroll
            for (int j = 0; j < VE; ++j) s += w[j];
          }
          sum2(s, none);
          __syncthreads();
          if (tid == 0) sm.stage[nst - 1] = unfixed(s);
          __syncthreads();
        }
      } else {
        bool seen = false;  // an earlier child with the same token took its weight
        for (int j = 0; j < nrej; ++j) seen |= sm.rejected[j] == (int)t;
        const ull w = known && !seen ? fixed(weight(to_f32(row.p[t]), m, p.inv_t)) : 0;
        ok = (double)ub[i] * (double)left < (double)w;
        if (!ok && known && !seen) {
          left -= w;
          __syncthreads();
          if (tid == 0) sm.rejected[nrej] = (int)t;
          __syncthreads();
          ++nrej;
        }
      }
      if (ok) {
        if (rank == 0 && tid == 0) path[n] = i;
        ++n;
        cur = i;
        down = true;
        break;
      }
    }
    if (!down) break;
  }

  // ---- the draw from what is left at the last node ----
  long long next = -1;
  bool owner = rank == 0 && tid == 0;
  if (p.greedy) {
    next = best;
  } else {
    const Row<T> row(lb + cur * p.l_st, p.V);
    const T* qrow = with_q && cur < p.T - 1 ? db + cur * p.d_st : nullptr;
    int g0, g1;
    range(row, g0, g1);
    ull s = 0, none = 0;
    for (int k = g0 + lane; k < g1; k += 32) {
      ull w[VE];
      left_of(row, qrow, k, w);
#pragma unroll
      for (int j = 0; j < VE; ++j) s += w[j];
    }
    sum2(s, none);
    __syncthreads();
    if (s > 0) {
      ull at = (ull)((double)ub[0] * (double)s);
      if (at >= s) at = s - 1;
      ull before = 0;
      for (int r = 0; r < rank; ++r) before += cluster.map_shared_rank(&sm.slot[(turn - 1) & 1], r)->a;
      for (int w = 0; w < warp; ++w) before += sm.tot[w];
      owner = false;
      if (at >= before && at < before + sm.tot[warp]) {  // in this warp's part
        for (int k0 = g0; k0 < g1; k0 += 32) {
          const int k = k0 + lane;
          ull w[VE], sum = 0;
          if (k < g1) {
            left_of(row, qrow, k, w);
#pragma unroll
            for (int j = 0; j < VE; ++j) sum += w[j];
          }
          ull incl = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const ull up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
          }
          const ull mine = before + incl - sum;
          if (at >= mine && at < mine + sum) {
            ull c = mine;
            int j = 0;  // elements whose cumulative weight does not pass `at`
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              c += w[e];
              j += c <= at;
            }
            next = (long long)k * VE - row.mis + j;
            owner = true;
          }
          before = __shfl_sync(0xffffffffu, before + incl, 31);
        }
      }
    }
  }
  if (owner) p.next[b] = next;
  if (rank == 0) {
    if (tid == 0) { path[0] = 0; p.count[b] = n; }
    for (int i = n + tid; i < p.T; i += kThreads) path[i] = -1;
  }
  cluster.sync();  // a CTA's shared memory outlives its readers
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int tpp_verify_tree(const void* logits, int64_t l_sb, int64_t l_st,
                               const void* draft_logits, int64_t d_sb, int64_t d_st,
                               const int64_t* tokens, int64_t tok_sb, const int32_t* parents,
                               int64_t par_sb, const float* u, int64_t u_sb, double temperature,
                               int32_t* path, int32_t* count, int64_t* next_token, int64_t B,
                               int64_t T, int64_t V, int dtype, void* stream) {
  if (B == 0) return TPP_OK;
  TPP_REQUIRE(logits && tokens && parents && path && count && next_token, TPP_ERR_SHAPE,
              "null pointer");
  TPP_REQUIRE(temperature >= 0.0 && temperature <= 1e30, TPP_ERR_SHAPE,
              "temperature must be finite and not negative");
  TPP_REQUIRE(temperature == 0.0 || (u != nullptr && temperature >= 1e-30), TPP_ERR_SHAPE,
              "temperature > 0 needs the uniform numbers");
  TPP_REQUIRE(B > 0 && B <= 65535 && T > 0 && T <= kMaxNodes && V > 0 && V <= (1 << 22),
              TPP_ERR_SHAPE, "need 1..65535 sequences, 1..256 nodes and 1..2^22 tokens");
  VerifyArgs a;
  a.logits = logits; a.l_sb = l_sb; a.l_st = l_st;
  a.draft = draft_logits; a.d_sb = d_sb; a.d_st = d_st;
  a.tokens = tokens; a.tok_sb = tok_sb; a.parents = parents; a.par_sb = par_sb;
  a.u = u; a.u_sb = u_sb;
  a.greedy = temperature == 0.0;
  a.inv_t = a.greedy ? 1.f : (float)(1.0 / temperature);
  a.path = path; a.count = count; a.next = next_token;
  a.T = (int)T; a.V = (int)V;
  const dim3 grid(kCluster, (unsigned)B);
  auto go = [&](auto kern) {
    return launch("verify_tree_kernel", kern, grid, dim3(kThreads), 0, as_stream(stream), 0u, a);
  };
  switch (dtype) {
    case TPP_F16: return go(verify_tree_kernel<__half>);
    case TPP_BF16: return go(verify_tree_kernel<__nv_bfloat16>);
    case TPP_F32: return go(verify_tree_kernel<float>);
    default:
      set_error("tpp_verify_tree: dtype must be f16, bf16 or f32");
      return TPP_ERR_DTYPE;
  }
}
