// Log probabilities of given tokens (and each row's entropy) straight from the LM head's
// operands: softmax statistics of x W^T in the product's epilogue, the logits never
// written.
//
// Persistent CTAs over tiles of 128 tokens x BN vocabulary rows, tokens first (a tile row of W
// stays in L2 meanwhile), the accumulators double-buffered in TMEM: a thread reads half a
// token's logits of a tile and leaves (largest, sum of weights, sum of weights times
// difference), 12 bytes for BN logits, which join_logprobs_kernel adds up.  Measured, bf16:
// 4096 x 1024 x 151936 800-825 us in bursts, 1546-1590 TFLOP/s (950 in long runs at the power
// limit's clock); 4096 x 2048 x 32003 338-349, as fast; to 128 tokens 62-64, 5.0 TB/s of
// weights.  Bound by the tensor core (95 % of its cycles); for few tokens by HBM (5.5 TB/s in
// mid-course) and some 7 us of start and join.  (Stages of 128 or 256 columns for few
// tokens, for longer requests, gave nothing: the same time, and 12 us more.)
#include <math.h>
#include "tc_issue.cuh"

namespace tpp {
namespace {

constexpr int BM = 128;        // tokens a tile
constexpr int BK = 64;         // a ring stage: one 128-byte swizzle row of the operands
constexpr int kMaxBN = 256;    // vocabulary rows a tile at most (a multiple of 16)
constexpr int kMaxStages = 8;
constexpr int kThreads = 384;  // 4 control warps, 8 of the epilogue
constexpr int kEpiWarp0 = 4;
// Stages a chain of products sums in the tensor core; longer ones are parts that the epilogue
// adds.  The tensor core's sums do not round to nearest, so a chain's logits are biased
// the more the longer it is: of 2048 columns in one chain (32003 vocabulary rows, temperature
// 0.8) the entropies were 2.8e-6 off, relative, in chains of 512 6e-7, 384 4e-7, 256 2.4e-7.  At
// 4096 x 1024 x 151936 one chain takes 814 us, of 512 816, 384 838, 256 925.  A single chain's
// logits go straight from TMEM to the weights (PARTS false), which is faster where the epilogue
// counts: 2000 x 256 x 50000 68 us, 85 through registers.
constexpr int kChain = 8;
// registers of a control and an epilogue thread that holds its logits meanwhile: 168 at launch
constexpr int kCtrlRegs = 72, kEpiRegs = 216;
static_assert(128 * kCtrlRegs + 256 * kEpiRegs == kThreads * 168, "");
constexpr size_t kRing = 216 * 1024;
constexpr size_t kSmem = kRing + 2 * 3 * BM * 4 + 1024 + 256;
static_assert(kSmem <= 227 * 1024, "shared memory plan exceeds 227 KB");

struct HeadArgs {
  const int64_t* tokens;
  float* part;    // [tiles of the vocabulary][3][rows]: m, S, E of token_logprobs
  float* target;  // [rows]: the token's logit
  int N, V, E, BN;
  int64_t rows;   // N rounded up to whole tiles
  // Ring stages, as many as fit: 4 for whole tiles, 8 for a few tokens, where the rest of
  // a tile's 128 rows is left unloaded (rows of x do not mix) and the weights are all that
  // counts.  a_rows: rows of x loaded.
  int stages, a_rows;
  float c;        // log2(e) / temperature
  int* err;
};

template <typename T, bool PARTS>
__global__ void __launch_bounds__(kThreads, 1)
    linear_logprobs_kernel(const __grid_constant__ CUtensorMap tm_x,
                           const __grid_constant__ CUtensorMap tm_w, HeadArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  float* half1 = reinterpret_cast<float*>(smem + kRing);  // [2 tiles][3][BM]
  uint64_t* full = reinterpret_cast<uint64_t*>(half1 + 2 * 3 * BM);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int BN = p.BN;
  const int ntm = (p.N + BM - 1) / BM;
  const int64_t ntiles = (int64_t)ntm * ((p.V + BN - 1) / BN);
  const int nk = (p.E + BK - 1) / BK, stages = p.stages;
  // a stage: x rows (whole 1 KB), then W rows
  const uint32_t a_bytes = (uint32_t)p.a_rows * 128, b_bytes = (uint32_t)BN * 128;
  const uint32_t stage = a_bytes + b_bytes;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_w);
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8);
    }
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  bool ok = true;
  if (warp < kEpiWarp0) {
  if constexpr (PARTS)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
  if ((warp == 0 || warp == 2) && lane == 0) {
    // ---------------- TMA producers: x by one thread, W by another ----------------
    // (a thread takes some 0.2 us a request, and a stage's products 0.3)
    int s = 0;
    uint32_t turn = 1;
    bool first = true;
    for (int64_t t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
      const int m0 = (int)(t % ntm) * BM, n0 = (int)(t / ntm) * BN;
      for (int kb = 0; kb < nk; ++kb) {
        if (!first) ok = ok && wait_short(&empty[s], turn, p.err, 51);
        if (!ok) break;
        uint8_t* at = smem + s * stage;
        if (warp == 0) {
          mbar_arrive_expect_tx(&full[s], a_bytes);
          tma_load_2d(at, &tm_x, &full[s], kb * BK, m0);
        } else {
          mbar_arrive_expect_tx(&full[s], b_bytes);
          tma_load_2d(at + a_bytes, &tm_w, &full[s], kb * BK, n0);
        }
        if (++s == stages) {
          s = 0;
          turn ^= 1;
          first = false;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the whole warp, see tc_issue.cuh) ----------------
    const uint32_t idesc = make_idesc_f16(BM, BN, IsBf16<T>::value, 0, 0);
    const uint32_t tm = (uint32_t)same((int)tmem);
    const uint32_t at = desc_lo(smem_u32(smem), 16);
    const bool on = elect_lane();
    int s = 0, j = 0;
    uint32_t turn = 0;
#pragma unroll 1
    for (int64_t t = blockIdx.x; t < ntiles; t += gridDim.x) {
#pragma unroll 1
      for (int kb = 0; kb < nk; ++j) {  // chain by chain
        const int buf = j & 1, end = min(kb + kChain, nk);
        if (ok && j >= 2) ok = wait_short(&tempty[buf], ((j >> 1) & 1) ^ 1, p.err, 52);
        tc_fence_after();
        const uint32_t acc = tm + (uint32_t)(buf * kMaxBN);
        bool more = false;
#pragma unroll 1
        for (; kb < end; ++kb) {
          if (ok) ok = wait_short(&full[s], turn, p.err, 53);
          tc_fence_after();
          const uint32_t a0 = at + s * (stage >> 4), b0 = a0 + (a_bytes >> 4);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_ss(on, acc, a0 + (k * 32 >> 4), b0 + (k * 32 >> 4), idesc, more || k != 0);
          more = true;
          commit(on, &empty[s]);
          if (++s == stages) {
            s = 0;
            turn ^= 1;
          }
        }
        commit(on, &tfull[buf]);
      }
      if (!__all_sync(0xffffffffu, ok)) break;
    }
  }
  } else {
    if constexpr (PARTS)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    // ---------------- epilogue: one row and half the tile's columns a thread ----------------
    const int quarter = warp & 3, hf = (warp - kEpiWarp0) >> 2;
    const int rl = quarter * 32 + lane;
    const int c_first = hf ? (BN / 16 + 1) / 2 * 16 : 0;  // this half's columns
    const int half = hf ? BN - c_first : (BN / 16 + 1) / 2 * 16;
    const float c = p.c;
    const uint64_t c2 = f2_pack(c, c);
    int j = 0, tile = 0;
    for (int64_t t = blockIdx.x; t < ntiles; t += gridDim.x, ++tile) {
      const int row = (int)(t % ntm) * BM + rl, vt = (int)(t / ntm);
      const int n0 = vt * BN + c_first;
      const int nv = max(0, min(half, p.V - n0));  // columns inside the vocabulary
      const int64_t at = row < p.N ? p.tokens[row] - n0 : -1;
      const int tl = at >= 0 && at < nv ? (int)at : -1;  // the token's column here
      const bool mine = __any_sync(0xffffffffu, tl >= 0);
      float ref = -INFINITY, S = 0.f, En = 0.f;
      auto arrived = [&]() {
        // (after a wait that ran out the loop goes on, for the barrier below)
        ok = ok && wait_short(&tfull[j & 1], (j >> 1) & 1, p.err, 54);
        __syncwarp();
        tc_fence_after();
        return tmem + (uint32_t)((j & 1) * kMaxBN + c_first) + ((uint32_t)(quarter * 32) << 16);
      };
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[j & 1]);
        ++j;
      };
      // C columns from c0 on, of which the first n weigh anything
      auto take = [&](const float* x, int c0, auto size, int n) {
        constexpr int C = decltype(size)::value;
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 4; i < C; i += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            mx[u] = i + 4 + u < C ? fmax3(mx[u], x[i + u], x[i + 4 + u]) : fmaxf(mx[u], x[i + u]);
        const float cm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (c0 == 0) ref = cm;
        if ((cm - ref) * c > 8.f) {  // (rare)
          const float d = ref - cm, f = exp2f(c * d);
          En = f == 0.f ? 0.f : (En + S * d) * f;
          S *= f;
          ref = cm;
        }
        const uint64_t r2 = f2_pack(-ref, -ref);
        uint64_t s2[2] = {0ull, 0ull}, e2[2] = {0ull, 0ull};
#pragma unroll
        for (int i = 0; i < C; i += 2) {
          const uint64_t q2 = f2_add(f2_pack(x[i], x[i + 1]), r2);
          float d0, d1;
          f2_unpack(f2_mul(q2, c2), d0, d1);
          const uint64_t w2 = f2_pack(i < n ? ex2_ftz(d0) : 0.f, i + 1 < n ? ex2_ftz(d1) : 0.f);
          s2[(i >> 1) & 1] = f2_add(s2[(i >> 1) & 1], w2);
          e2[(i >> 1) & 1] = f2_fma(w2, q2, e2[(i >> 1) & 1]);
        }
        float a0, a1;
        f2_unpack(f2_add(s2[0], s2[1]), a0, a1);
        S += a0 + a1;
        f2_unpack(f2_add(e2[0], e2[1]), a0, a1);
        En += a0 + a1;
        if (mine) {
#pragma unroll
          for (int i = 0; i < C; ++i)
            if (tl == c0 + i) p.target[row] = x[i];
        }
      };
      constexpr std::integral_constant<int, 32> k32{};
      constexpr std::integral_constant<int, 16> k16{};
      if constexpr (PARTS) {
        // the logits stay in registers: the parts, added in 32 bits
        float x[kMaxBN / 2];
#pragma unroll 1
        for (int kb = 0; kb < nk; kb += kChain) {
          const uint32_t from = arrived();
          if (kb == 0) {
#pragma unroll
            for (int c0 = 0; c0 < kMaxBN / 2; c0 += 32)
              if (c0 < half) tmem_ld32(from + c0, reinterpret_cast<uint32_t*>(x) + c0);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int c0 = 0; c0 < kMaxBN / 2; c0 += 32) {
              if (c0 >= half) break;
              uint32_t r[32];
              tmem_ld32(from + c0, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; i += 2)
                f2_unpack(f2_add(f2_pack(x[c0 + i], x[c0 + i + 1]),
                                 f2_pack(__uint_as_float(r[i]), __uint_as_float(r[i + 1]))),
                          x[c0 + i], x[c0 + i + 1]);
            }
          }
          release();
        }
#pragma unroll
        for (int c0 = 0; c0 < kMaxBN / 2; c0 += 32) {
          if (c0 + 32 <= nv) {
            take(x + c0, c0, k32, 32);
          } else if (c0 < nv) {
            // (behind the vocabulary: a logit of the row again, so that nothing moves, without
            // weight; a number of its own would weigh at high temperatures, or overflow)
#pragma unroll
            for (int i = 1; i < 32; ++i)
              if (c0 + i >= nv) x[c0 + i] = x[c0];
            take(x + c0, c0, k16, nv - c0);
            if (c0 + 16 < nv) take(x + c0 + 16, c0 + 16, k16, nv - c0 - 16);
          }
        }
      } else {
        const uint32_t trow = arrived();
        // a block's transfer runs beside the one before's weights
        auto as_f = [](const uint32_t* r) { return reinterpret_cast<const float*>(r); };
        int c0 = 0;
        if (nv >= 32) {
          uint32_t r[2][32];
          tmem_ld32(trow, r[0]);
          for (; c0 + 64 <= nv; c0 += 64) {
            tmem_wait_ld();
            tmem_ld32(trow + c0 + 32, r[1]);
            take(as_f(r[0]), c0, k32, 32);
            tmem_wait_ld();
            if (c0 + 96 <= nv) tmem_ld32(trow + c0 + 64, r[0]);
            take(as_f(r[1]), c0 + 32, k32, 32);
          }
          if (c0 + 32 <= nv) {
            tmem_wait_ld();
            take(as_f(r[0]), c0, k32, 32);
            c0 += 32;
          }
        }
        if (c0 + 16 <= nv) {
          uint32_t r[16];
          tmem_ld16(trow + c0, r);
          tmem_wait_ld();
          take(as_f(r), c0, k16, 16);
          c0 += 16;
        }
#pragma unroll 1
        for (; c0 < nv; ++c0) {  // the vocabulary's end
          uint32_t r;
          asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(trow + c0));
          tmem_wait_ld();
          const float x = __uint_as_float(r);
          if (c0 == 0) ref = x;
          if ((x - ref) * c > 8.f) {
            const float d = ref - x, f = exp2f(c * d);
            En = f == 0.f ? 0.f : (En + S * d) * f;
            S *= f;
            ref = x;
          }
          const float q = x - ref, w = ex2_ftz(q * c);
          S += w;
          En += w * q;
          if (tl == c0) p.target[row] = x;
          __syncwarp();
        }
        release();
      }
      // the row's two halves, joined by the first
      float* h1 = half1 + (tile & 1) * 3 * BM;
      if (hf == 1) {
        h1[rl] = ref;
        h1[BM + rl] = S;
        h1[2 * BM + rl] = En;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (hf == 0) {
        const float rb = h1[rl], Sb = h1[BM + rl], Eb = h1[2 * BM + rl];
        float* out = p.part + (int64_t)vt * 3 * p.rows + row;
        float M = ref, S0 = S, E0 = En;
        if (!(Sb == 0.f)) {  // (the second half may lie behind the vocabulary)
          M = fmaxf(ref, rb);
          const float da = ref - M, db = rb - M, fa = exp2f(c * da), fb = exp2f(c * db);
          S0 = S * fa + Sb * fb;
          E0 = (fa == 0.f ? 0.f : (En + S * da) * fa) + (fb == 0.f ? 0.f : (Eb + Sb * db) * fb);
        }
        out[0] = M;
        out[p.rows] = S0;
        out[2 * p.rows] = E0;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the vocabulary's tiles: 32 rows a block, a tile a warp at a time, kJoinAhead tiles'
// loads in flight (for a few tokens there is one block, and latency is all it costs).
constexpr int kJoinWarps = 32, kJoinAhead = 8;  // (32: a warp a row in the end)
__global__ void __launch_bounds__(32 * kJoinWarps)
    join_logprobs_kernel(const float* part, const float* target, const int64_t* tokens,
                         int64_t rows, int nt, int N, int V, float c, float inv_t,
                         float* logprobs, float* entropy) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sm[3][kJoinWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int row = blockIdx.x * 32 + lane;
  float M = -INFINITY, S = 0.f, E = 0.f;
  auto add = [&](float m, float s, float e) {
    const float big = fmaxf(M, m);
    // (nothing so far: not -inf - -inf)
    const float da = S == 0.f ? 0.f : M - big, db = s == 0.f ? 0.f : m - big;
    const float fa = exp2f(c * da), fb = exp2f(c * db);
    E = (fa == 0.f ? 0.f : (E + S * da) * fa) + (fb == 0.f ? 0.f : (e + s * db) * fb);
    S = S * fa + s * fb;
    M = big;
  };
  for (int t0 = warp; t0 < nt; t0 += kJoinWarps * kJoinAhead) {
    float m[kJoinAhead], s[kJoinAhead], e[kJoinAhead];
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const int t = t0 + u * kJoinWarps;
      const float* at = part + (int64_t)min(t, nt - 1) * 3 * rows + row;
      m[u] = at[0];
      s[u] = t < nt ? at[rows] : 0.f;
      e[u] = t < nt ? at[2 * rows] : 0.f;
    }
    // (one exponential a tile, where add() takes two)
    float big = M;
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) big = fmaxf(big, m[u]);
    const float d0 = S == 0.f ? 0.f : M - big, f0 = ex2_ftz(c * d0);
    E = f0 == 0.f ? 0.f : (E + S * d0) * f0;
    S *= f0;
    M = big;
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const float d = s[u] == 0.f ? 0.f : m[u] - big, f = ex2_ftz(c * d);
      E += f == 0.f ? 0.f : (e[u] + s[u] * d) * f;
      S += s[u] * f;
    }
  }
  sm[0][warp][lane] = M;
  sm[1][warp][lane] = S;
  sm[2][warp][lane] = E;
  __syncthreads();
  // a row a warp, a part a lane
  row = blockIdx.x * 32 + warp;
  if (row >= N) return;
  M = sm[0][lane][warp];
  S = sm[1][lane][warp];
  E = sm[2][lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_down_sync(0xffffffffu, M, o), t = __shfl_down_sync(0xffffffffu, S, o),
                e = __shfl_down_sync(0xffffffffu, E, o);
    add(m, t, e);
  }
  if (lane != 0) return;
  constexpr float kLn2 = 0.69314718055994531f;
  const float lz = log2f(S);
  const int64_t tok = tokens[row];
  // (not in bits, where the farthest logits' would overflow)
  logprobs[row] = tok >= 0 && tok < V ? (target[row] - M) * inv_t - lz * kLn2 : 0.f;
  entropy[row] = (lz - E / S * c) * kLn2;
}

// Vocabulary rows a tile: of the widths that fill the tensor core (a multiple of 16, at
// least 128), the one whose tiles go evenly onto the SMs -- 151936 rows are 594 tiles of
// 256, five rounds of 148 CTAs where four would nearly do, but five full rounds of 208.
// Measured (bf16, us; widths 128, 208, 224, 240, 256, then the choice): 7 x 1024 x 151936 63.7,
// 59.9, 57.7, 59.8, 60.4: 208; 4096 x 1024 x 32003 244, 183, 181, 177, 181: 240; 2000 x 256 x
// 50000 73, 63, 61, 61, 60: 240.  Not always the best: 1000 x 1024 x 32003 66.6, 49.8, 47.7, 48.9,
// 46.3, and it takes 176, 52.8 (a tile's own cost of 16 columns would give 256 there, and the
// same widths in the other cases).
int tile_width(int64_t N, int64_t V) {
  const int64_t ntm = (N + BM - 1) / BM, sms = num_sms();
  int best = kMaxBN;
  int64_t cost = -1;
  for (int bn = kMaxBN; bn >= 128; bn -= 16) {
    const int64_t tiles = ntm * ((V + bn - 1) / bn), rounds = (tiles + sms - 1) / sms;
    const int64_t c = rounds * (bn + 8);  // 8: a tile's own cost
    if (cost < 0 || c < cost) {
      cost = c;
      best = bn;
    }
  }
  return best;
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int64_t tpp_linear_logprobs_workspace(int64_t N, int64_t V, int64_t E) {
  if (N <= 0 || V <= 0 || E <= 0) return 0;
  const int64_t rows = (N + BM - 1) / BM * BM, bn = tile_width(N, V);
  return 4 * rows * (3 * ((V + bn - 1) / bn) + 1);
}

extern "C" int tpp_linear_logprobs(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                   const int64_t* tokens, int64_t N, int64_t V, int64_t E,
                                   double temperature, float* logprobs, float* entropy,
                                   void* workspace, int64_t workspace_bytes, int dtype,
                                   void* stream) {
  if (N == 0) return TPP_OK;
  TPP_REQUIRE(x && w && tokens && logprobs && entropy, TPP_ERR_SHAPE, "null pointer");
  TPP_REQUIRE(N > 0 && N < (1ll << 31) - BM && V > 0 && V < (1ll << 31) - kMaxBN && E > 0 &&
                  E < (1ll << 31) - BK && ldx >= E && ldw >= E,
              TPP_ERR_SHAPE, "bad sizes");
  TPP_REQUIRE(temperature >= 1e-6 && isfinite(temperature), TPP_ERR_SHAPE,
              "temperature must be positive");
  TPP_REQUIRE(E % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && aligned16(x) && aligned16(w),
              TPP_ERR_ALIGN, "rows must be 16-byte aligned and E a multiple of 8");
  TPP_REQUIRE(workspace && workspace_bytes >= tpp_linear_logprobs_workspace(N, V, E) &&
                  reinterpret_cast<uintptr_t>(workspace) % 4 == 0,
              TPP_ERR_WORKSPACE, "workspace missing or too small");
  HeadArgs a;
  a.tokens = tokens;
  a.N = (int)N; a.V = (int)V; a.E = (int)E;
  a.BN = tile_width(N, V);
  a.rows = (N + BM - 1) / BM * BM;
  const int nt = (int)((V + a.BN - 1) / a.BN);
  a.part = static_cast<float*>(workspace);
  a.target = a.part + 3 * a.rows * nt;
  a.a_rows = (int)(N < BM ? (N + 7) / 8 * 8 : BM);
  const int64_t stage = (int64_t)(a.a_rows + a.BN) * 128;
  a.stages = (int)((int64_t)kRing / stage < kMaxStages ? (int64_t)kRing / stage : kMaxStages);
  a.c = (float)(1.4426950408889634 / temperature);
  a.err = device_error_flag();
  CUtensorMap tx, tw;
  auto map = [&](CUtensorMap* m, const void* base, int64_t rows, int64_t ld, int box_rows) {
    const uint64_t dims[2] = {(uint64_t)E, (uint64_t)rows};
    const uint64_t strides[1] = {(uint64_t)ld * 2};
    const uint32_t box[2] = {BK, (uint32_t)box_rows};
    return make_tmap(m, base, dtype, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  return TPP_DISPATCH_HALF(dtype, T, [&] {
    int rc = map(&tx, x, N, ldx, a.a_rows);
    if (rc == TPP_OK) rc = map(&tw, w, V, ldw, a.BN);
    if (rc != TPP_OK) return rc;
    const bool parts = E > kChain * BK;
    auto kern = parts ? linear_logprobs_kernel<T, true> : linear_logprobs_kernel<T, false>;
    static std::atomic<bool> reserved[2][64];
    rc = reserve_smem(reinterpret_cast<const void*>(kern), reserved[parts], kSmem,
                      "linear_logprobs_kernel");
    if (rc != TPP_OK) return rc;
    const int64_t tiles = (a.rows / BM) * nt;
    const unsigned grid = (unsigned)(tiles < num_sms() ? tiles : num_sms());
    rc = launch("linear_logprobs_kernel", kern, dim3(grid), dim3(kThreads), kSmem,
                as_stream(stream), 0u, tx, tw, a);
    if (rc != TPP_OK) return rc;
    return launch("join_logprobs_kernel", join_logprobs_kernel, dim3((unsigned)((N + 31) / 32)),
                  dim3(32 * kJoinWarps), 0, as_stream(stream), 0u, (const float*)a.part,
                  (const float*)a.target, tokens, a.rows, nt, (int)N, (int)V, a.c,
                  (float)(1 / temperature), logprobs, entropy);
  });
}
