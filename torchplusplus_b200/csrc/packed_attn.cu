// Attention over whole prompts of different lengths packed into one row dimension
// (self-attention of each sequence: causal, or full, with an optional sliding window),
// grouped heads, on the 5th-generation tensor cores.
//
// Persistent: one CTA per SM walks work items.  An item is 2 x TT consecutive tokens of
// one sequence and all G = Hq / Hkv query heads of one kv head, TT = 128 / G: a query
// tile's 128 rows are (token, head of the group), so short prompts and wide groups fill
// it, and each K/V tile is read once for two query tiles.  512 threads:
//   warps 0-3, 4-7 : softmax of query tile 0, 1: a thread owns a row, a step's scores in registers
//                    (running maximum that only moves, and O with it, when it grows by
//                    more than 2^8, sums in 32 bits), P in TMEM in the storage type, as the
//                    product with V takes it (off by at most half a step, see kLift).
//   warps 8-11     : write O / l at an item's end, while the next one runs.
//   warps 12, 13   : products of query tile 0, 1: O_i += P_i V_j, then S_i = Q_i K^T of step
//                    j + 2, across items too: a softmax finds the next S done when it has
//                    written P.
//   warp 14        : hands out the items, blocks with the most keys first, and loads: Q
//                    tiles, and K and V tiles through one ring.
//   warp 15        : makes V tiles finite that some row sees only a part of.
//
// What a row does not see has no effect on it, NaN and infinities included: masked
// scores are -inf, and in tiles that any row sees a part of, V rows behind the sequence
// are zeros and non-finite values are cleared (0 * NaN is NaN) and added to the
// rows that see them at the end.
//
// Measured (bf16, heads over kv heads, D 128 unless said otherwise): one prompt of 32768,
// 16/8: 3.2-3.4 ms, 1300-1360 TFLOP/s of the visible pairs' products (3.8 in long runs at the
// power limit's clock); 6 to 8191, 32/8, f16: 1.7-1.8 ms; 32 to 512, 16/8: 52-56 us (their bytes:
// 22); one of 130: 9-11 us; 64-dim heads, one of 16384, 16/8: 0.77-0.9 ms by clock.  In long prompts a step
// of both tiles (80 keys) takes some 2250 clocks, its products 1280: the tiles' softmaxes run
// side by side, and their exponentials (1450 for both; the units' own rate gives 1280) are
// followed by 800 to 950 of barriers, transfers and maxima.  Taking turns, so that one tile's
// fill the other's gaps, is slower (2430 to 2560: a warp alone takes 11 clocks an
// exponential, two together 9 each).  In short prompts an item's start, its masked steps (3300
// clocks) and its output count.
#include <math.h>
#include "tc_issue.cuh"
#include "mma_common.cuh"

namespace tpp {
namespace {

constexpr int BQ = 128;
constexpr int kThreads = 512;
constexpr int kOutWarp0 = 8, kMmaWarp = 12, kTmaWarp = 14;  // (products: warps 12 and 13)
constexpr int kItems = 8;
constexpr float kMoves = 8.0f;  // growth of a row's maximum (log2) that moves its reference
// A row's reference lies kLift (log2) below the maximum that set it.  f16 numbers end at 2^-24, and
// thousands of keys that weigh less each may weigh something together: with 2^7, P stays
// below 2^(kMoves + 7) = 2^15, and a weight loses at most 2^-32 of the row's largest (2^-25 without,
// in one prompt of 6000 rows up to all of an output).  bf16 has the range of 32 bits.  Maxima
// from kFar on are their own references: where steps of float32 come near to 1, the room that
// is left up to 2^16 is for roundings.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
constexpr float kFar = 1048576.0f;  // 2^20

// TMEM (512 columns): O of both query tiles, then for each S (BKV columns) and, apart from
// it, P (half as many), so that S of a later step is under way while a step's softmax runs:
// that leaves 80 keys a step for 128 dims.  (With P over S, 128 keys a step, each tile's products
// and softmax take turns.)  For 64 dims 128 keys would fit, and 96 are faster: one prompt of
// 16384, 64: 912 us, 96: 770, 112: 850, 128: 832.
template <int D>
struct Plan {
  static constexpr int BKV = D == 128 ? 80 : 96;      // keys a step
  static constexpr int kBoxes = D / 64;               // 128-byte swizzle boxes a row
  static constexpr uint32_t kQBox = BQ * 128;         // bytes of a box of a Q or output tile
  static constexpr uint32_t kQTile = kBoxes * kQBox;
  static constexpr uint32_t kBox = BKV * 128;         // of a K or V tile
  static constexpr uint32_t kTile = kBoxes * kBox;
  static constexpr int kStages = D == 128 ? 6 : 8;
  static constexpr uint32_t tO = 0, tS = 2 * D, kSCols = 96,
                            tP = tS + kSCols + BKV, kPCols = BKV / 2;
  static_assert(tP + 2 * kPCols <= 512, "TMEM plan exceeds 512 columns");
  // registers of a softmax, an output and a control thread: 4 x 128 are the launch's
  static constexpr int kSoftRegs = 152, kOutRegs = 120, kCtrlRegs = 88;
  static_assert(2 * kSoftRegs + kOutRegs + kCtrlRegs == 512, "");
  static constexpr size_t kSmem =
      1024 + 3 * kQTile + kStages * kTile + 2 * BQ * 4 + kItems * 48 + 640;
  static_assert(kSmem <= 227 * 1024, "shared memory plan exceeds 227 KB");
};

struct PackedAttnArgs {
  const int32_t* cu;
  int B, N, Hkv, G, TT;
  int tok_w;  // tokens of 32 rows of a query tile (0: not a whole number)
  int inv_g;  // ceil(2^16 / G): r * inv_g >> 16 is r / G for r < 128
  int causal;
  int window;  // at most N; -1: none
  float scale_log2;
  int sign;  // of the scale: scores are negated (-1) or all equal (0) first
  void* o;
  int64_t o_sn, o_sh;
  const void* v;
  int64_t v_sn, v_sh;
  int* err;
};

// An item as the scheduler hands it out.  Its key tiles are counted from kb: query tile 0
// reads [0, end0), query tile 1 (none if end1 is 0) [start1, end1); some row may see
// only a part of those below `low` and from `high` on.
struct Work {
  int first, len, t0, kvh;
  int kb, nt, start1, end0;
  int end1, low, high, unused;

  __device__ __forceinline__ int start(int i) const { return i ? start1 : 0; }
  __device__ __forceinline__ int end(int i) const { return i ? end1 : end0; }
  __device__ __forceinline__ bool part(int j) const { return j < low || j >= high; }
};
template <int BKV>
__device__ __forceinline__ Work work_of(const int4& it, const PackedAttnArgs& p) {
  Work w{};
  w.first = it.x; w.len = it.y; w.t0 = it.z; w.kvh = it.w;
  w.high = 1 << 30;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = w.t0 + i * p.TT, n = min(p.TT, w.len - tok);
    if (n <= 0) continue;
    const int kb = p.window >= 0 ? max(0, tok - p.window) / BKV : 0;
    if (i == 0) w.kb = kb;
    const int end = ((p.causal ? tok + n : w.len) + BKV - 1) / BKV - w.kb;
    if (i == 0) w.end0 = end;
    else w.start1 = kb - w.kb, w.end1 = end;
    w.nt = max(w.nt, end);
    // key tile t: partly hidden behind the sequence, by causality, by the window
    w.high = min(w.high, (p.causal ? (tok + 1) / BKV : w.len / BKV) - w.kb);
    if (p.window >= 0 && tok + n - 1 > p.window)
      w.low = max(w.low, (tok + n - 1 - p.window + BKV - 1) / BKV - w.kb);
  }
  return w;
}

// A CTA's steps (key tiles) are numbered on over its items.  K runs two steps ahead of V in
// the ring: K_0, K_1, V_0, K_2, V_1, K_3 ..: the load of a step's K or V, by number.
__device__ __forceinline__ int k_load(int g) { return g < 2 ? g : 2 * g - 1; }
__device__ __forceinline__ int v_load(int g) { return 2 * g + 2; }

// Walks the items in order: blocks of 2 TT tokens, the last ones of the longest
// sequences first (a causal block's keys grow with its number), each for all kv heads.
struct Walk {
  const int32_t* cu;
  int B, N, per, Hkv;  // per: tokens a block
  int level;           // the blocks' number
  uint32_t base;       // items before this level (there are fewer than 2^31)
  int count;           // sequences that have it
  int seek, before;    // the last item's: of 32 sequences the first, those with it before

  // sequence b's first row and length (whatever cu holds, inside [0, N])
  __device__ __forceinline__ int2 span(int b) const {
    const int a = min(max(__ldg(cu + b), 0), N), e = min(max(__ldg(cu + b + 1), 0), N);
    return make_int2(a, max(e - a, 0));
  }
  __device__ __forceinline__ bool has(int b) const {
    return b < B && span(b).y > (int64_t)level * per;
  }
  __device__ void recount(int lane) {
    count = seek = before = 0;
#pragma unroll 1
    for (int b = 0; b < B; b += 32)
      count += __popc(__ballot_sync(0xffffffffu, has(b + lane)));
  }
  __device__ void init(int lane) {
    int most = 0;
#pragma unroll 1
    for (int b = lane; b < B; b += 32) most = max(most, span(b).y);
    most = __reduce_max_sync(0xffffffffu, most);
    level = (most + per - 1) / per - 1;
    base = 0;
    if (level >= 0) recount(lane);
  }
  // item number `at` (not before the last one asked for): first row, length, first
  // token of the block, kv head; length -1 behind the last
  __device__ int4 item(uint32_t at, int lane) {
#pragma unroll 1
    while (level >= 0 && at >= base + (uint32_t)(count * Hkv)) {
      base += (uint32_t)(count * Hkv);
      if (--level >= 0) recount(lane);
    }
    if (level < 0) return make_int4(0, -1, 0, 0);
    const uint32_t in = at - base;
    const int nth = (int)(in / (uint32_t)Hkv);
    const int kvh = (int)(in - (uint32_t)nth * Hkv);
#pragma unroll 1
    for (; seek < B; seek += 32) {  // (items ascend, so the last one's place is a start)
      const uint32_t set = __ballot_sync(0xffffffffu, has(seek + lane));
      const int n = __popc(set);
      if (nth < before + n) {
        const bool me =
            (set >> lane & 1) && before + __popc(set & ((1u << lane) - 1)) == nth;
        const int src = __ffs(__ballot_sync(0xffffffffu, me)) - 1;
        const int2 s = span(seek + src);
        return make_int4(s.x, s.y, level * per, kvh);
      }
      before += n;
    }
    return make_int4(0, -1, 0, 0);
  }
};

// Maxima that NaN passes through.
__device__ __forceinline__ float nanmax(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float nanmax(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

template <typename T>
__device__ __forceinline__ uint32_t times_zero_plus(uint32_t w, uint32_t acc) {
  if constexpr (std::is_same<T, __half>::value) {
    __half2 r = __hfma2(*reinterpret_cast<__half2*>(&w), __float2half2_rn(0.f),
                        *reinterpret_cast<__half2*>(&acc));
    return *reinterpret_cast<uint32_t*>(&r);
  } else {
    __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&w), __float2bfloat162_rn(0.f),
                               *reinterpret_cast<__nv_bfloat162*>(&acc));
    return *reinterpret_cast<uint32_t*>(&r);
  }
}

// Adds the non-finite values that were cleared to the output row of query tile i's row rl,
// as far as that row sees them (never but for broken inputs, hence apart).
template <typename T, int D>
__device__ __forceinline__ void add_hidden(const Work& w, int i, int rl, const PackedAttnArgs& p) {
  constexpr int BKV = Plan<D>::BKV;
  const int tl = rl / p.G, g = rl - tl * p.G, tok = w.t0 + i * p.TT + tl;
  if (tl >= p.TT || tok >= w.len) return;
  T* out = static_cast<T*>(p.o) + (int64_t)(w.first + tok) * p.o_sn +
           (int64_t)(w.kvh * p.G + g) * p.o_sh;
#pragma unroll 1
  for (int j = w.start(i); j < w.end(i); ++j) {
    if (!w.part(j)) continue;
#pragma unroll 1
    for (int k = 0; k < BKV; ++k) {
      const int key = (w.kb + j) * BKV + k;
      if (key >= w.len || (p.causal && key > tok) || (p.window >= 0 && key < tok - p.window))
        continue;
      const T* v = static_cast<const T*>(p.v) + (int64_t)(w.first + key) * p.v_sn +
                   (int64_t)w.kvh * p.v_sh;
#pragma unroll 1
      for (int c = 0; c < D; ++c) {
        const float e = to_f32(v[c]);
        if (!isfinite(e)) out[c] = from_f32<T>(to_f32(out[c]) + e);
      }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attn_kernel(const __grid_constant__ CUtensorMap tm_q,
                       const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ CUtensorMap tm_o,
                       const __grid_constant__ PackedAttnArgs p) {
  using P = Plan<D>;
  constexpr int S = P::kStages, BKV = P::BKV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint8_t* sQ = smem;                   // 2 tiles
  uint8_t* stage = sQ + 2 * P::kQTile;  // an output tile
  uint8_t* sKV = stage + P::kQTile;     // ring of K and V tiles
  float* sums = reinterpret_cast<float*>(sKV + S * P::kTile);  // [2][BQ]
  Work* items = reinterpret_cast<Work*>(sums + 2 * BQ);
  uint64_t* bars = reinterpret_cast<uint64_t*>(items + kItems);
  uint64_t* q_full = bars;           // 2 each, of the query tiles:
  uint64_t* q_empty = bars + 2;      // the item's last S_i is done
  uint64_t* s_full = bars + 4;       // S_i is done
  uint64_t* s_read = bars + 6;       // and in the softmax's registers
  uint64_t* p_ready = bars + 8;      // P_i written
  uint64_t* pv_done = bars + 10;     // P_i V done
  uint64_t* l_full = bars + 12;      // the item's sums
  uint64_t* l_empty = bars + 14;
  uint64_t* o_full = bars + 16;      // the item's last P_i V is done
  uint64_t* o_empty = bars + 18;     // its O_i has been read
  uint64_t* it_full = bars + 20;     // kItems
  uint64_t* it_empty = it_full + kItems;
  uint64_t* kv_full = it_empty + kItems;  // S
  uint64_t* kv_empty = kv_full + S;       // S
  uint64_t* v_sent = kv_empty + S;        // S: a masked V tile is on its way
  uint64_t* v_ok = v_sent + S;            // S: it is finite
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_ok + S);
  int* odd_v = reinterpret_cast<int*>(tmem_slot + 1);  // [kItems]: item whose V had non-finite values
  static_assert(S / 2 + 2 < kItems, "odd_v's places");
  static_assert((20 + 2 * kItems + 4 * S) * 8 + 4 + 4 * kItems <= 640, "barriers exceed their room");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_read[i], 4);
      mbar_init(&p_ready[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&l_full[i], 4);
      mbar_init(&l_empty[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&it_full[i], 1);
      mbar_init(&it_empty[i], 17);  // 8 + 4 warps, 2 twice, 1
    }
    for (int s = 0; s < S; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 2);
      mbar_init(&v_sent[s], 1);
      mbar_init(&v_ok[s], 1);
    }
    for (int s = 0; s < kItems; ++s) odd_v[s] = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  bool ok = true;
  // the n-th item (the same for the warp; every reader reads each once)
  auto take = [&](int n) {
    const int s = n % kItems;
    ok = ok && wait_short(&it_full[s], (n / kItems) & 1, p.err, 81);
    Work w{};
    w.len = -1;
    if (ok) w = items[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(&it_empty[s]);
    return w;
  };

  // (one instruction for a whole warpgroup)
  if (warp >= kMmaWarp) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kCtrlRegs));
  if (warp == kTmaWarp) {
    // ---------------- items and loads ----------------
    // Step gk of the K's, (wk, jk), runs two ahead of step gv of the V's, (wv, jv); an item is
    // handed out when the K's come to it.
    Walk walk{p.cu, p.B, p.N, 2 * p.TT, p.Hkv, 0, 0, 0, 0, 0};
    walk.init(lane);
    int nk = 0;
    auto next_item = [&]() {
      // there and back: a CTA's early and late items of two rounds balance
      const uint32_t at = nk * gridDim.x + (nk & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      const Work w = work_of<BKV>(walk.item(at, lane), p);
      const int s = nk % kItems;
      if (nk >= kItems) ok = ok && wait_short(&it_empty[s], ((nk / kItems) & 1) ^ 1, p.err, 82);
      if (lane == 0 && ok) {
        items[s] = w;
        mbar_arrive(&it_full[s]);
      }
      __syncwarp();
      ++nk;
      return w;
    };
    uint32_t nq = 0;  // loads of each Q tile: bit i their parity, bit 2 + i whether any
    const uint32_t q_box = (uint32_t)(p.G * p.TT) * 128;
    Work wk = next_item(), wv = wk;
    int nv = 0, jk = 0, jv = 0;
#pragma unroll 1
    for (int g = 0; (wk.len >= 0 || wv.len >= 0) && __all_sync(0xffffffffu, ok); ++g) {
      // V of step g - 2, then K of step g
#pragma unroll 1
      for (int k = g < 2 ? 1 : 0; k < 2; ++k) {
        Work& w = k ? wk : wv;
        int& j = k ? jk : jv;
        if (w.len < 0) continue;
        if (lane == 0) {
          const int r = k ? k_load(g) : v_load(g - 2), s = r % S;
          if (r >= S) ok = ok && wait_short(&kv_empty[s], ((r / S) & 1) ^ 1, p.err, 83);
          if (ok) {
            mbar_arrive_expect_tx(&kv_full[s], P::kTile);
            tma_load_4d(sKV + s * P::kTile, k ? &tm_k : &tm_v, &kv_full[s], 0,
                        w.first + (w.kb + j) * BKV, 0, w.kvh);
            if (!k && w.part(j)) mbar_arrive(&v_sent[s]);
          }
          if (k && j == 0) {
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
              if (w.end(i) <= w.start(i)) continue;
              if (nq >> (2 + i) & 1)
                ok = ok && wait_short(&q_empty[i], (nq >> i & 1) ^ 1, p.err, 84);
              if (!ok) break;
              mbar_arrive_expect_tx(&q_full[i], P::kBoxes * q_box);
              for (int b = 0; b < P::kBoxes; ++b)
                tma_load_3d(sQ + i * P::kQTile + b * P::kQBox, &tm_q, &q_full[i], b * 64,
                            w.kvh * p.G, w.first + w.t0 + i * p.TT);
              nq = (nq ^ 1u << i) | 4u << i;
            }
          }
        }
        __syncwarp();
        if (++j < w.nt) continue;
        j = 0;
        if (k) {
          wk = next_item();
        } else {
          wv = items[++nv % kItems];  // (at most three behind the items handed out)
        }
      }
    }
  } else if (warp < kTmaWarp) {
    // ---------------- products of query tile i ----------------
    constexpr uint32_t idesc_s = make_idesc_f16(BQ, BKV, IsBf16<T>::value, 0, 0);
    constexpr uint32_t idesc_o = make_idesc_f16(BQ, D, IsBf16<T>::value, 0, 1);
    const int i = same(warp - kMmaWarp);
    const bool on = elect_lane();
    const uint32_t tm = (uint32_t)same((int)tmem);
    const uint32_t kv_at = desc_lo(smem_u32(sKV), 0), qa = desc_lo(smem_u32(sQ) + i * P::kQTile, 16);
    const uint32_t tS = tm + P::tS + i * P::kSCols, tPi = tm + P::tP + i * P::kPCols,
                   tO = tm + P::tO + i * D;
    // a wait that ran out ends the loop with its item, not at once
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
      if (ok) ok = wait_short(bar, parity & 1, p.err, code);
    };
    // what this warp needs of an item
    struct Mine { int nt, start, end, low, high; };
    auto mine = [&](int n) {
      const Work w = take(n);
      const bool go = __all_sync(0xffffffffu, ok) && same(w.len) >= 0;
      return Mine{go ? same(w.nt) : 0, same(w.start(i)), same(w.end(i)), same(w.low), same(w.high)};
    };
    // S of step (ws, js) runs two ahead of P V of step (wp, jp)
    Mine ws = mine(0), wp = mine(0);
    int n_s = 0, n_p = 0, js = 0, jp = 0;
    uint32_t nq = 0, ns = 1, np = 0, no = 1;  // parities of the next waits
    bool s_any = false, o_any = false;
    uint32_t seen = 0;                        // of the clearings of each ring slot's V
    int sk = 0, sv = 2;                       // ring slots of the next K and V
    uint32_t hk = 0, hv = 0;                  // and their parities
    auto issue_s = [&]() {  // (K has landed)
      if (js >= ws.start && js < ws.end) {
        if (js == ws.start) {
          wait(&q_full[i], nq, 85);
          nq ^= 1;
        }
        if (s_any) wait(&s_read[i], ns, 86);  // the last S_i is in registers
        s_any = true;
        ns ^= 1;
        tc_fence_after();
        const uint32_t ka = kv_at + (16 >> 4 << 16) + sk * (P::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ss(on, tS, qa + (((kk >> 2) * P::kQBox + (kk & 3) * 32) >> 4),
                 ka + (((kk >> 2) * P::kBox + (kk & 3) * 32) >> 4), idesc_s, kk != 0);
        commit(on, &s_full[i]);
        if (js == ws.end - 1) commit(on, &q_empty[i]);
      }
      commit(on, &kv_empty[sk]);
      if (++js == ws.nt) {
        ws = mine(++n_s);
        js = 0;
      }
    };
    for (int g = 0; g < 2 && ws.nt > 0; ++g) {
      wait(&kv_full[g], 0, 87);
      issue_s();
      sk = g == 0 ? 1 : 3;
    }
    sk = 3;
    while (wp.nt > 0) {
      // V of this step, K of the one after the next: in time for the softmax, as a rule
      const bool part = jp < wp.low || jp >= wp.high;
      wait(&kv_full[sv], hv, 88);
      if (part) wait(&v_ok[sv], seen >> sv, 89);
      if (ws.nt > 0) wait(&kv_full[sk], hk, 90);
      if (jp >= wp.start && jp < wp.end) {
        if (jp == wp.start) {
          if (o_any) wait(&o_empty[i], no, 91);
          o_any = true;
          no ^= 1;
        }
        wait(&p_ready[i], np, 92);
        np ^= 1;
        tc_fence_after();
        const uint32_t va = kv_at + (P::kBox >> 4 << 16) + sv * (P::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < BKV / 16; ++kk)
          mma_ts(on, tO, tPi + kk * 8, va + kk * (2048 >> 4), idesc_o,
                 jp > wp.start || kk != 0);
        commit(on, &pv_done[i]);
        if (jp == wp.end - 1) commit(on, &o_full[i]);
      }
      if (part) seen ^= 1u << sv;
      commit(on, &kv_empty[sv]);
      sv += 2;
      if (sv >= S) sv -= S, hv ^= 1;
      if (ws.nt > 0) {
        issue_s();
        sk += 2;
        if (sk >= S) sk -= S, hk ^= 1;
      }
      if (++jp == wp.nt) {
        wp = mine(++n_p);
        jp = 0;
      }
    }
  } else {
    // ---------------- masked V tiles: zeros behind the sequence, elsewhere finite ----------------
    // (this warp skips the other tiles, so a slot's phases could pass it by: that the load is
    // on its way says that the slot's last phase is over, and the next one waits for v_ok)
    int g = 0;          // the step
    uint32_t seen = 0;  // bit: parity of the clearings of a ring slot's V
    for (int n = 0; ok; ++n) {
      const Work w = take(n);
      if (!ok || w.len < 0) break;
      for (int j = 0; j < w.nt && ok; ++j, ++g) {
        if (!w.part(j)) continue;
        const int r = v_load(g), s = r % S;
        ok = ok && wait_short(&v_sent[s], seen >> s & 1, p.err, 93);
        seen ^= 1u << s;
        ok = ok && wait_short(&kv_full[s], (r / S) & 1, p.err, 94);
        if (!ok) break;
        // rows of the sequence, then rows behind it (each 128 bytes a box)
        const int valid = min(BKV, w.len - (w.kb + j) * BKV);
        uint8_t* at = sKV + s * P::kTile;
        bool wrote = valid < BKV;
        uint32_t acc[4] = {0, 0, 0, 0};  // 0 or NaN
#pragma unroll 1
        for (int b = 0; b < P::kBoxes; ++b, at += P::kBox) {
          constexpr int kAtOnce = 10;
#pragma unroll 1
          for (int e0 = lane * 16; e0 < valid * 128; e0 += kAtOnce * 512) {
            uint4 u[kAtOnce];
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q)
              u[q] = e0 + q * 512 < valid * 128 ? *reinterpret_cast<const uint4*>(at + e0 + q * 512)
                                                : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) {
              acc[0] = times_zero_plus<T>(u[q].x, acc[0]);
              acc[1] = times_zero_plus<T>(u[q].y, acc[1]);
              acc[2] = times_zero_plus<T>(u[q].z, acc[2]);
              acc[3] = times_zero_plus<T>(u[q].w, acc[3]);
            }
          }
#pragma unroll 1
          for (int e0 = valid * 128 + lane * 16; e0 < (int)P::kBox; e0 += 512)
            *reinterpret_cast<uint4*>(at + e0) = make_uint4(0, 0, 0, 0);
        }
        if (__any_sync(0xffffffffu, ((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7fff7fffu) != 0)) {
          at = sKV + s * P::kTile;
#pragma unroll 1
          for (int e0 = lane; e0 < P::kBoxes * valid * 64; e0 += 32) {
            const int b = e0 / (valid * 64);
            T* e = reinterpret_cast<T*>(at + b * P::kBox) + (e0 - b * valid * 64);
            if (!isfinite(to_f32(*e))) *e = from_f32<T>(0.f);
          }
          wrote = true;
          atomicExch(odd_v + n % kItems, n + 1);
        }
        if (wrote) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[s]);
      }
    }
  }
  } else if (warp < kOutWarp0) {
    // ---------------- softmax ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::kSoftRegs));
    const int i = warp >> 2, rl = (warp & 3) * 32 + lane;
    const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tS = at + P::tS + i * P::kSCols, tP = at + P::tP + i * P::kPCols,
                   tO = at + P::tO + i * D;
    int ns = 0, nl = 0;
    for (int n = 0; ok; ++n) {
      const Work w = take(n);
      if (!ok || w.len < 0) break;
      if (w.end(i) <= w.start(i)) continue;
      const int qpos = w.t0 + i * p.TT + rl / p.G;
      float m_ref = -INFINITY, l = 0.f;
      for (int j = w.start(i); j < w.end(i); ++j) {
        ok = ok && wait_short(&s_full[i], ns & 1, p.err, 95);
        ++ns;
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        float sv[BKV];
        {
          uint32_t* r = reinterpret_cast<uint32_t*>(sv);
#pragma unroll
          for (int k = 0; k + 32 <= BKV; k += 32) tmem_ld32(tS + k, r + k);
          if (BKV % 32) tmem_ld16(tS + BKV - 16, r + BKV - 16);
          tmem_wait_ld();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_read[i]);
        if (p.sign <= 0) {
#pragma unroll
          for (int k = 0; k < BKV; ++k) sv[k] = p.sign < 0 ? -sv[k] : 0.f;
        }
        if (w.part(j)) {
          const int key0 = (w.kb + j) * BKV;
          const int hi = (p.causal ? min(qpos, w.len - 1) : w.len - 1) - key0;
          const int lo = p.window >= 0 ? max(0, qpos - p.window - key0) : 0;
#pragma unroll
          for (int k0 = 0; k0 < BKV; k0 += 16) {
            // the visible keys lo .. hi of these 16 as bits
            const int h = min(max(hi - k0 + 1, 0), 16), b = min(max(lo - k0, 0), 16);
            const uint32_t see = ((1u << h) - 1) & ~((1u << b) - 1);
            if (__all_sync(0xffffffffu, see == 0xffffu)) continue;
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (!(see & 1u << k)) sv[k0 + k] = -INFINITY;
          }
        }
        float pm[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) pm[u] = nanmax(sv[u], sv[8 + u]);
#pragma unroll
        for (int k = 16; k < BKV; k += 16)
#pragma unroll
          for (int u = 0; u < 8; ++u) pm[u] = nanmax(pm[u], sv[k + u], sv[k + 8 + u]);
        const float mx = nanmax(nanmax(pm[0], pm[1], pm[2]), nanmax(pm[3], pm[4], pm[5]),
                                nanmax(pm[6], pm[7])) * p.scale_log2;
        // P_i V of the last step is done: P_i may be written, and O_i is at rest
        if (ns > 1) ok = ok && wait_short(&pv_done[i], ns & 1, p.err, 96);
        if (!ok) break;
        tc_fence_after();
        const float lift = fabsf(mx) < kFar ? kLift<T> : 0.f;
        const bool moves = !(mx <= m_ref + (kMoves + lift));  // (the first finite one too; NaN)
        if (__any_sync(0xffffffffu, moves)) {
          const float to = mx - lift;
          const float f = !moves ? 1.f : m_ref == -INFINITY ? 0.f : exp2f(m_ref - to);
          l *= f;
          m_ref = moves ? to + (mx - mx) : m_ref;  // (infinite scores make a row NaN)
          __syncwarp();  // (the transfers below are the whole warp's)
          if (j > w.start(i)) {
#pragma unroll 1
            for (int c = 0; c < D; c += 8) {
              uint32_t r[8];
              tmem_ld8(tO + c, r);
              tmem_wait_ld();
#pragma unroll
              for (int q = 0; q < 8; ++q) r[q] = __float_as_uint(__uint_as_float(r[q]) * f);
              tmem_st8(tO + c, r);
            }
          }
        }
        const float nm = m_ref == -INFINITY ? 0.f : -m_ref;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nm2 = f2_pack(nm, nm);
        uint64_t ps[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int k0 = 0; k0 < BKV; k0 += 16) {
          uint32_t pk[8];
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            float a0, a1;
            f2_unpack(f2_fma(f2_pack(sv[k0 + k], sv[k0 + k + 1]), sc2, nm2), a0, a1);
            a0 = ex2_ftz(a0);
            a1 = ex2_ftz(a1);
            ps[(k >> 1) & 3] = f2_add(ps[(k >> 1) & 3], f2_pack(a0, a1));
            pk[k / 2] = pack2<T>(a0, a1);
          }
          tmem_st8(tP + k0 / 2, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[i]);
        float a0, a1;
        f2_unpack(f2_add(f2_add(ps[0], ps[1]), f2_add(ps[2], ps[3])), a0, a1);
        l += a0 + a1;
      }
      if (!ok) break;
      if (nl > 0) ok = ok && wait_short(&l_empty[i], (nl & 1) ^ 1, p.err, 97);
      ++nl;
      if (!ok) break;
      sums[i * BQ + rl] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full[i]);
    }
  } else {
    // ---------------- O ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kOutRegs));
    const int rl = (warp & 3) * 32 + lane;
    const uint32_t tO = tmem + P::tO + ((uint32_t)((warp & 3) * 32) << 16);
    uint32_t no = 0;  // parity of the items of each query tile, bit i
    for (int n = 0; ok; ++n) {
      const Work w = take(n);
      if (!ok || w.len < 0) break;
      // the sums, both at once, so that the next item's softmax can go on
      float inv0 = 0.f, inv1 = 0.f;
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (w.end(i) <= w.start(i)) continue;
        ok = ok && wait_short(&l_full[i], no >> i & 1, p.err, 98);
        if (!ok) break;
        const float l = sums[i * BQ + rl];
        (i ? inv1 : inv0) = l == 0.f ? 0.f : 1.f / l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_empty[i]);
      }
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (w.end(i) <= w.start(i)) continue;
        ok = ok && wait_short(&o_full[i], no >> i & 1, p.err, 99);
        no ^= 1u << i;
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        const float inv = i ? inv1 : inv0;
        // through this warp's part of the staging tile, so that a store covers whole rows
        const int tok0 = w.t0 + i * p.TT, rows = min(p.TT, w.len - tok0);
        uint8_t* st = stage + (warp & 3) * 4096;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int c = 0; c < D; c += 64) {
          uint32_t r[64];
          tmem_ld32(tO + i * D + c, r);
          tmem_ld32(tO + i * D + c + 32, r + 32);
          tmem_wait_ld();
          if (c + 64 == D) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty[i]);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(r[q * 8 + e]) * inv;
            *reinterpret_cast<uint4*>(st + (c >> 6) * P::kQBox + lane * 128 +
                                      (q ^ (lane & 7)) * 16) = pack8<T>(f);
          }
        }
        // this warp's tokens: all of them in one request a box, or their rows one by one
        const int t_lo = p.tok_w * (warp & 3);
        if (p.tok_w > 0 && t_lo + p.tok_w <= rows) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            for (int b = 0; b < P::kBoxes; ++b)
              asm volatile(
                  "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                  ::"l"(reinterpret_cast<uint64_t>(&tm_o)), "r"(b * 64), "r"(w.kvh * p.G),
                  "r"(w.first + tok0 + t_lo), "r"(smem_u32(st + b * P::kQBox))
                  : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          __syncwarp();
          T* out = static_cast<T*>(p.o) + (int64_t)(w.first + tok0) * p.o_sn +
                   (int64_t)w.kvh * p.G * p.o_sh + (lane & 7) * 8;
#pragma unroll 2
          for (int q = 0; q < 8 * P::kBoxes; ++q) {
            const int r = (q & 7) * 4 + (lane >> 3), row = (warp & 3) * 32 + r;
            const int tl = row * p.inv_g >> 16;
            const uint4 u = *reinterpret_cast<const uint4*>(st + (q >> 3) * P::kQBox + r * 128 +
                                                            ((lane ^ r) & 7) * 16);
            if (tl < rows)
              *reinterpret_cast<uint4*>(out + tl * p.o_sn + (row - tl * p.G) * p.o_sh +
                                        (q >> 3) * 64) = u;
          }
        }
        // (set, if at all, before the last P V could be issued; O of the next item but one
        // waits for this warp, so at most the ring's V tiles of later items are looked at
        // meanwhile, fewer items than share a place)
        if (*reinterpret_cast<volatile int*>(odd_v + n % kItems) == n + 1) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
          __syncwarp();
          add_hidden<T, D>(w, i, rl, p);
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int tpp_attention_packed(const void* q, int64_t q_sn, int64_t q_sh, const void* k,
                                    int64_t k_sn, int64_t k_sh, const void* v, int64_t v_sn,
                                    int64_t v_sh, const int32_t* cu_seqlens, int64_t B, void* o,
                                    int64_t o_sn, int64_t o_sh, int64_t N, int64_t Hq,
                                    int64_t Hkv, int64_t D, int causal, int64_t window_left,
                                    float scale, int dtype, void* stream) {
  if (N == 0 || B == 0) return TPP_OK;
  TPP_REQUIRE(q && k && v && cu_seqlens && o, TPP_ERR_SHAPE, "null pointer");
  TPP_REQUIRE(N > 0 && N < (1ll << 30) && B > 0 && B < (1ll << 30) && Hkv > 0 && Hq > 0 &&
                  Hq < (1ll << 24) && Hq % Hkv == 0,
              TPP_ERR_SHAPE, "bad sizes (Hq must be a multiple of Hkv)");
  TPP_REQUIRE(D == 64 || D == 128, TPP_ERR_UNSUPPORTED, "head dim must be 64 or 128");
  TPP_REQUIRE(Hq / Hkv <= BQ, TPP_ERR_UNSUPPORTED, "at most 128 query heads a kv head");
  TPP_REQUIRE(((q_sn | q_sh | k_sn | k_sh | v_sn | v_sh | o_sn | o_sh) & 7) == 0 &&
                  aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o),
              TPP_ERR_ALIGN, "rows must be 16-byte aligned");
  TPP_REQUIRE(isfinite(scale), TPP_ERR_SHAPE, "scale must be finite");
  PackedAttnArgs a;
  a.cu = cu_seqlens;
  a.B = (int)B; a.N = (int)N; a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.TT = BQ / a.G;
  a.inv_g = (65536 + a.G - 1) / a.G;
  a.tok_w = 32 % a.G == 0 ? 32 / a.G : 0;
  a.causal = causal != 0;
  a.window = (int)(window_left < 0 ? -1 : window_left < N ? window_left : N);
  a.sign = scale > 0 ? 1 : scale < 0 ? -1 : 0;
  a.scale_log2 = scale == 0 ? 1.f : fabsf(scale) * 1.4426950408889634f;
  a.o = o; a.o_sn = o_sn; a.o_sh = o_sh;
  a.v = v; a.v_sn = v_sn; a.v_sh = v_sh;
  a.err = device_error_flag();
  // items at most: a block of 2 TT tokens each, one more a sequence
  const int64_t items = (N / (2 * a.TT) + B) * Hkv;
  TPP_REQUIRE(items < (1ll << 30), TPP_ERR_SHAPE, "too many rows, sequences and heads");
  const unsigned grid = (unsigned)(items < num_sms() ? items : num_sms());
  CUtensorMap tq, tk, tv, to;
  const uint64_t qd[3] = {(uint64_t)D, (uint64_t)Hq, (uint64_t)N};
  const uint64_t qs[2] = {(uint64_t)q_sh * 2, (uint64_t)q_sn * 2};
  const uint32_t qb[3] = {64, (uint32_t)a.G, (uint32_t)a.TT};
  int rc = make_tmap(&tq, q, dtype, 3, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B);
  // K and V: {64 dims, rows, halves of a row, heads}, a tile in one request
  auto kv_map = [&](CUtensorMap* m, const void* base, int64_t sn, int64_t sh) {
    const uint64_t d[4] = {64, (uint64_t)N, (uint64_t)(D / 64), (uint64_t)Hkv};
    const uint64_t s[3] = {(uint64_t)sn * 2, 128, (uint64_t)sh * 2};
    const uint32_t b[4] = {64, (uint32_t)(D == 128 ? Plan<128>::BKV : Plan<64>::BKV),
                           (uint32_t)(D / 64), 1};
    return make_tmap(m, base, dtype, 4, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  const uint64_t os[2] = {(uint64_t)o_sh * 2, (uint64_t)o_sn * 2};
  const uint32_t ob[3] = {64, (uint32_t)(a.tok_w ? a.G : 1), (uint32_t)(a.tok_w ? a.tok_w : 1)};
  if (rc == TPP_OK) rc = make_tmap(&to, o, dtype, 3, qd, os, ob, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == TPP_OK) rc = kv_map(&tk, k, k_sn, k_sh);
  if (rc == TPP_OK) rc = kv_map(&tv, v, v_sn, v_sh);
  if (rc != TPP_OK) return rc;
  auto go = [&](auto tag, auto dim) -> int {
    using T = decltype(tag);
    constexpr int DH = decltype(dim)::value;
    auto kern = packed_attn_kernel<T, DH>;
    static std::atomic<bool> reserved[64];
    const int e = reserve_smem(reinterpret_cast<const void*>(kern), reserved, Plan<DH>::kSmem,
                               "packed_attn_kernel");
    if (e != TPP_OK) return e;
    return launch("packed_attn_kernel", kern, dim3(grid), dim3(kThreads), Plan<DH>::kSmem,
                  as_stream(stream), 0u, tq, tk, tv, to, a);
  };
  return TPP_DISPATCH_HALF(dtype, T, [&] {
    return D == 128 ? go(T(), std::integral_constant<int, 128>{})
                    : go(T(), std::integral_constant<int, 64>{});
  });
}
