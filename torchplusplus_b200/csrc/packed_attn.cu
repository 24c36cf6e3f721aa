// Attention over whole prompts of different lengths packed into one row dimension
// (self-attention of each sequence: causal, or full, with an optional sliding window),
// grouped heads, on the 5th-generation tensor cores.
//
// Persistent: one CTA per SM walks work items.  An item is 2 x TT consecutive tokens of
// one sequence and all G = Hq / Hkv query heads of one kv head, TT = 128 / G: a query
// tile's 128 rows are (token, head of the group), so short prompts and wide groups fill
// it, and each K/V tile is read once for two query tiles.  512 threads:
//   warps 0-3, 4-7 : softmax of query tile 0, 1: a thread owns a row, 128 scores a step
//                    (running maximum that only moves, and O with it, when it grows by
//                    more than 2^8, sums in 32 bits), P over S in TMEM in the storage type.
//   warps 8-11     : write O / l at an item's end, while the next one runs.
//   warp 12        : MMA issuer.  S_i = Q_i K_j^T and O_i += P_i V_j, in the order
//                    PV_0, S_0, PV_1, S_1: while one tile's softmax runs the tensor
//                    core has the other tile's products, across items too.
//   warp 13        : TMA: Q tiles, and K and V tiles of 128 keys through one ring.
//   warp 14        : hands out the items, blocks with the most keys first.
//   warp 15        : makes V tiles finite that some row sees only a part of.
// TMEM: S/P 0 and 1 in columns [0, 256), O 0 and 1 in [256, 512).
//
// What a row does not see has no effect on it, NaN and infinities included: masked
// scores are -inf, and in tiles that any row sees a part of, V rows behind the sequence
// are zeros and non-finite values are cleared (0 * NaN is NaN) and added to the
// rows that see them at the end.
#include <math.h>
#include "tc_issue.cuh"
#include "mma_common.cuh"

namespace tpp {
namespace {

constexpr int BQ = 128;
constexpr int BKV = 128;
constexpr int kThreads = 512;
constexpr int kCorrWarp0 = 8, kMmaWarp = 12, kTmaWarp = 13, kSchedWarp = 14;
constexpr int kItems = 4;
constexpr float kMoves = 8.0f;  // growth of a row's maximum (log2) that moves its reference

template <int D>
struct Plan {
  static constexpr int kBoxes = D / 64;             // 128-byte swizzle boxes a row
  static constexpr uint32_t kBox = 128 * 128;       // bytes of a box of 128 rows
  static constexpr uint32_t kTile = kBoxes * kBox;  // a Q, K or V tile
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr uint32_t kStage = kTile;         // an output tile's
  static constexpr size_t kSmem = 1024 + (2 + kStages) * kTile + kStage + 2 * BQ * 4 + kItems * 48 + 512;
  static_assert(kSmem <= 227 * 1024, "shared memory plan exceeds 227 KB");
};

struct PackedAttnArgs {
  const int32_t* cu;
  int B, N, Hkv, G, TT;
  int inv_g;  // ceil(2^16 / G): r * inv_g >> 16 is r / G for r < 128
  int causal;
  int64_t window;
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
  __device__ __forceinline__ bool active(int i, int j) const {
    return j >= start(i) && j < end(i);
  }
  __device__ __forceinline__ bool part(int j) const { return j < low || j >= high; }
};
__device__ __forceinline__ Work work_of(const int4& it, const PackedAttnArgs& p) {
  Work w{};
  w.first = it.x; w.len = it.y; w.t0 = it.z; w.kvh = it.w;
  w.high = 1 << 30;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = w.t0 + i * p.TT, n = min(p.TT, w.len - tok);
    if (n <= 0) continue;
    const int64_t lo = p.window >= 0 ? max((int64_t)0, tok - p.window) : 0;
    const int kb = (int)(lo / BKV);
    if (i == 0) w.kb = kb;
    const int end = ((p.causal ? tok + n : w.len) + BKV - 1) / BKV - w.kb;
    if (i == 0) w.end0 = end;
    else w.start1 = kb - w.kb, w.end1 = end;
    w.nt = max(w.nt, end);
    // key tile t: partly hidden behind the sequence, by causality, by the window
    w.high = min(w.high, (p.causal ? (tok + 1) / BKV : w.len / BKV) - w.kb);
    if (p.window >= 0 && tok + n - 1 > p.window)
      w.low = max(w.low, (int)((tok + n - 1 - p.window + BKV - 1) / BKV) - w.kb);
  }
  return w;
}

// Walks the items in order: blocks of 2 TT tokens, the last ones of the longest
// sequences first (a causal block's keys grow with its number), each for all kv heads.
struct Walk {
  const int32_t* cu;
  int B, N, per, Hkv;  // per: tokens a block
  int level;           // the blocks' number
  int64_t base;        // items before this level
  int count;           // sequences that have it

  // sequence b's first row and length (whatever cu holds, inside [0, N])
  __device__ __forceinline__ int2 span(int b) const {
    const int a = min(max(__ldg(cu + b), 0), N), e = min(max(__ldg(cu + b + 1), 0), N);
    return make_int2(a, max(e - a, 0));
  }
  __device__ __forceinline__ bool has(int b) const {
    return b < B && span(b).y > (int64_t)level * per;
  }
  __device__ void recount(int lane) {
    count = 0;
    for (int b = 0; b < B; b += 32)
      count += __popc(__ballot_sync(0xffffffffu, has(b + lane)));
  }
  __device__ void init(int lane) {
    int most = 0;
    for (int b = lane; b < B; b += 32) most = max(most, span(b).y);
    most = __reduce_max_sync(0xffffffffu, most);
    level = (most + per - 1) / per - 1;
    base = 0;
    if (level >= 0) recount(lane);
  }
  // item number `at` (not before the last one asked for): first row, length, first
  // token of the block, kv head; length -1 behind the last
  __device__ int4 item(int64_t at, int lane) {
    while (level >= 0 && at >= base + (int64_t)count * Hkv) {
      base += (int64_t)count * Hkv;
      if (--level >= 0) recount(lane);
    }
    if (level < 0) return make_int4(0, -1, 0, 0);
    const int64_t in = at - base;
    int nth = (int)(in / Hkv);
    const int kvh = (int)(in - (int64_t)nth * Hkv);
    for (int b = 0; b < B; b += 32) {
      const uint32_t set = __ballot_sync(0xffffffffu, has(b + lane));
      const int n = __popc(set);
      if (nth < n) {
        const bool me = (set >> lane & 1) && __popc(set & ((1u << lane) - 1)) == nth;
        const int src = __ffs(__ballot_sync(0xffffffffu, me)) - 1;
        const int2 s = span(b + src);
        return make_int4(s.x, s.y, level * per, kvh);
      }
      nth -= n;
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
                       const __grid_constant__ PackedAttnArgs p) {
  using P = Plan<D>;
  constexpr int S = P::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint8_t* sQ = smem;                      // 2 tiles
  uint8_t* sKV = smem + 2 * P::kTile;      // ring: K_0, V_0, K_1, V_1, ... across items
  uint8_t* stage = sKV + S * P::kTile;
  float* sums = reinterpret_cast<float*>(stage + P::kStage);  // [2][BQ]
  Work* items = reinterpret_cast<Work*>(sums + 2 * BQ);
  uint64_t* bars = reinterpret_cast<uint64_t*>(items + kItems);
  uint64_t* q_full = bars;             // 2
  uint64_t* q_empty = q_full + 2;      // 2: the item's last S_i is done
  uint64_t* s_full = q_empty + 2;      // 2: S_i (and every product before it) is done
  uint64_t* p_ready = s_full + 2;      // 2: P_i written
  uint64_t* l_full = p_ready + 2;      // 2: the item's sums
  uint64_t* l_empty = l_full + 2;      // 2
  uint64_t* o_full = l_empty + 2;      // 2: the item's last P_i V is done
  uint64_t* o_empty = o_full + 2;      // 2: its O_i has been read
  uint64_t* it_full = o_empty + 2;      // kItems
  uint64_t* it_empty = it_full + kItems;
  uint64_t* kv_full = it_empty + kItems;  // S
  uint64_t* kv_empty = kv_full + S;       // S
  uint64_t* v_sent = kv_empty + S;        // S: a masked V tile is on its way
  uint64_t* v_ok = v_sent + S;            // S: it is finite
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_ok + S);
  int* odd_v = reinterpret_cast<int*>(tmem_slot + 1);  // [2]: item whose V had non-finite values

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
      mbar_init(&p_ready[i], 4);
      mbar_init(&l_full[i], 4);
      mbar_init(&l_empty[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&it_full[i], 1);
      mbar_init(&it_empty[i], 15);
    }
    for (int s = 0; s < S; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
      mbar_init(&v_sent[s], 1);
      mbar_init(&v_ok[s], 1);
    }
    odd_v[0] = odd_v[1] = 0;
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
  // the n-th item (warp-uniform; every warp but the scheduler's reads each once)
  auto take = [&](int n) {
    const int s = n % kItems;
    ok = ok && mbar_wait(&it_full[s], (n / kItems) & 1, p.err, 61);
    Work w{};
    w.len = -1;
    if (ok) w = items[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(&it_empty[s]);
    return w;
  };

  // (one instruction for a whole warpgroup; 2 x 176 + 96 + 64 = 4 x 128, what the launch has)
  if (warp >= kMmaWarp) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == kSchedWarp) {
    // ---------------- items ----------------
    Walk w{p.cu, p.B, p.N, 2 * p.TT, p.Hkv, 0, 0, 0};
    w.init(lane);
    for (int n = 0; ok; ++n) {
      // there and back: a CTA's early and late items of two rounds balance
      const int64_t at = (int64_t)n * gridDim.x +
                         (n & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
      const int4 it = w.item(at, lane);
      const int s = n % kItems;
      if (n >= kItems) ok = ok && mbar_wait(&it_empty[s], ((n / kItems) & 1) ^ 1, p.err, 62);
      if (!ok) break;
      if (lane == 0) {
        items[s] = work_of(it, p);
        mbar_arrive(&it_full[s]);
      }
      if (it.y < 0) break;
    }
  } else if (warp == kTmaWarp) {
    // ---------------- loads ----------------
    uint32_t nq = 0;  // loads of each Q tile: bit i its parity, bit 2 + i whether any
    int ring = 0;
    const uint32_t q_box = (uint32_t)(p.G * p.TT) * 128;
    for (int n = 0; ok; ++n) {
      const Work w = take(n);
      if (!ok || w.len < 0) break;
      if (lane != 0) continue;
      auto load = [&](const CUtensorMap* map, int j) {
        const int s = ring % S;
        if (ring >= S) ok = ok && mbar_wait(&kv_empty[s], ((ring / S) & 1) ^ 1, p.err, 63);
        if (!ok) return;
        mbar_arrive_expect_tx(&kv_full[s], P::kTile);
        tma_load_4d(sKV + s * P::kTile, map, &kv_full[s], 0, w.first + (w.kb + j) * BKV, 0,
                    w.kvh);
        ++ring;
      };
      load(&tm_k, 0);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (w.end(i) <= w.start(i)) continue;
        if (nq >> (2 + i) & 1) ok = ok && mbar_wait(&q_empty[i], (nq >> i & 1) ^ 1, p.err, 64);
        if (!ok) break;
        mbar_arrive_expect_tx(&q_full[i], P::kBoxes * q_box);
        for (int b = 0; b < P::kBoxes; ++b)
          tma_load_3d(sQ + i * P::kTile + b * P::kBox, &tm_q, &q_full[i], b * 64, w.kvh * p.G,
                      w.first + w.t0 + i * p.TT);
        nq = (nq ^ 1u << i) | 4u << i;
      }
      for (int j = 0; j < w.nt && ok; ++j) {
        load(&tm_v, j);
        if (ok && w.part(j)) mbar_arrive(&v_sent[(ring - 1) % S]);
        if (j + 1 < w.nt && ok) load(&tm_k, j + 1);
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------- products ----------------
    constexpr uint32_t idesc_s = make_idesc_f16(BQ, BKV, IsBf16<T>::value, 0, 0);
    constexpr uint32_t idesc_o = make_idesc_f16(BQ, D, IsBf16<T>::value, 0, 1);
    const bool on = elect_lane();
    const uint32_t q_at = smem_u32(sQ), kv_at = smem_u32(sKV), tm = (uint32_t)same((int)tmem);
    // a wait that ran out ends the loops at the next step, not at once
    auto wait = [&](uint64_t* bar, int parity, int code) {
      if (ok) ok = mbar_wait(bar, (uint32_t)parity & 1, p.err, code);
    };
    int ring = 1;  // the next V tile's number
    // parities, a bit each: Q_i's loads, P_i's steps, the clearings of a ring slot's V
    uint32_t nq = 0, np = 0, seen = 0;
    uint32_t no = 0;  // items of each query tile: bit i their parity, bit 2 + i whether any
    // S_i of the item's key tile in ring slot s, which has landed; `last`: of this item and
    // query tile
    auto issue_s = [&](int i, int s, bool first, bool last) {
      if (first) {
        wait(&q_full[i], (int)(nq >> i), 65);
        nq ^= 1u << i;
        tc_fence_after();
      }
      const uint32_t qa = desc_lo(q_at + i * P::kTile, 16), ka = desc_lo(kv_at + s * P::kTile, 16);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t o = ((kk >> 2) * P::kBox + (kk & 3) * 32) >> 4;
        mma_ss(on, tm + i * 128, qa + o, ka + o, idesc_s, kk != 0);
      }
      commit(on, &s_full[i]);
      if (last) commit(on, &q_empty[i]);
    };
    // what this warp needs of an item
    auto tiles = [&](int n) {
      Work w = take(n);
      w.len = same(w.len);
      w.nt = same(w.nt);
      w.start1 = same(w.start1);
      w.end0 = same(w.end0);
      w.end1 = same(w.end1);
      w.low = same(w.low);
      w.high = same(w.high);
      return w;
    };
    Work cur = tiles(0);
    bool more = __all_sync(0xffffffffu, ok) && cur.len >= 0;
    if (more) {
      wait(&kv_full[0], 0, 66);
      tc_fence_after();
#pragma unroll 1
      for (int i = 0; i < 2; ++i)
        if (cur.active(i, 0)) issue_s(i, 0, true, cur.end(i) == 1);
      commit(on, &kv_empty[0]);
    }
    for (int n = 1; more; ++n) {
      const Work nxt = tiles(n);
      const bool follows = nxt.len >= 0;
      more = follows;
      for (int j = 0; j < cur.nt; ++j) {
        // V_j, then K_{j+1} or the next item's K_0.  Their waits, and all else that does not
        // hang on the softmax, come here, while the last step's products run: any wait
        // takes 200 clocks (the softmax warps' exponentials fill the queue that barriers go
        // through too)
        const int rv = ring, rk = ring + 1, s = rv % S, sk = rk % S;
        const bool part = cur.part(j), goes = j + 1 < cur.nt || follows;
        wait(&kv_full[s], rv / S, 68);
        if (goes) wait(&kv_full[sk], rk / S, 66);
        if (part) wait(&v_ok[s], (int)(seen >> s), 69);
        if (!__all_sync(0xffffffffu, ok)) {
          more = false;
          break;
        }
        const uint32_t va = desc_lo(kv_at + s * P::kTile, P::kBox);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          if (cur.active(i, j)) {
            if (j == cur.start(i)) {
              if (no >> (2 + i) & 1) wait(&o_empty[i], (int)(no >> i) ^ 1, 78);
              no = (no ^ 1u << i) | 4u << i;
            }
            wait(&p_ready[i], (int)(np >> i), 67);
            tc_fence_after();
            const uint32_t pa = tm + i * 128, oa = tm + 256 + i * 128;
#pragma unroll
            for (int kk = 0; kk < BKV / 16; ++kk)
              mma_ts(on, oa, pa + kk * 8, va + kk * (2048 >> 4), idesc_o,
                     j > cur.start(i) || kk != 0);
            np ^= 1u << i;
            if (j == cur.end(i) - 1) commit(on, &o_full[i]);
          }
          if (j + 1 < cur.nt) {
            if (cur.active(i, j + 1)) issue_s(i, sk, j + 1 == cur.start(i), j + 2 == cur.end(i));
          } else if (follows && nxt.active(i, 0)) {
            issue_s(i, sk, true, nxt.end(i) == 1);
          }
        }
        if (part) seen ^= 1u << s;
        commit(on, &kv_empty[s]);
        ring = rk;
        if (goes) {
          commit(on, &kv_empty[sk]);
          ring = rk + 1;
        }
      }
      cur = nxt;
    }
  } else {
    // ---------------- masked V tiles: zeros behind the sequence, elsewhere finite ----------------
    // (this warp skips the other tiles, so a slot's phases could pass it by: that the load is
    // on its way says that the slot's last phase is over, and the next one waits for v_ok)
    int ring = 1;       // V_0's number
    uint32_t seen = 0;  // bit: parity of the clearings of a ring slot's V
    for (int n = 0; ok; ++n) {
      const Work w = take(n);
      if (!ok || w.len < 0) break;
      for (int j = 0; j < w.nt && ok; ++j, ring += 2) {
        if (!w.part(j)) continue;
        const int s = ring % S;
        ok = ok && mbar_wait(&v_sent[s], seen >> s & 1, p.err, 77);
        seen ^= 1u << s;
        ok = ok && mbar_wait(&kv_full[s], (ring / S) & 1, p.err, 73);
        if (!ok) break;
        bool wrote = false;
#pragma unroll 1
        for (int rl = lane; rl < BKV; rl += 32) {
          uint8_t* at = sKV + s * P::kTile + rl * 128;
          // (chunks in the order that keeps eight rows on different banks)
          if ((w.kb + j) * BKV + rl >= w.len) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              *reinterpret_cast<uint4*>(at + (c >> 3) * P::kBox + ((c ^ rl) & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
            wrote = true;
            continue;
          }
          uint32_t acc[4] = {0, 0, 0, 0};  // 0 or NaN
#pragma unroll
          for (int c = 0; c < D / 8; ++c) {
            const uint4 u =
                *reinterpret_cast<const uint4*>(at + (c >> 3) * P::kBox + ((c ^ rl) & 7) * 16);
            acc[0] = times_zero_plus<T>(u.x, acc[0]);
            acc[1] = times_zero_plus<T>(u.y, acc[1]);
            acc[2] = times_zero_plus<T>(u.z, acc[2]);
            acc[3] = times_zero_plus<T>(u.w, acc[3]);
          }
          if (((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7fff7fffu) != 0) {
#pragma unroll 1
            for (int c = 0; c < D; ++c) {
              T* e = reinterpret_cast<T*>(at + (c >> 6) * P::kBox) + (c & 63);
              if (!isfinite(to_f32(*e))) *e = from_f32<T>(0.f);
            }
            wrote = true;
            atomicExch(odd_v + (n & 1), n + 1);
          }
        }
        if (wrote) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ok[s]);
      }
    }
  }
  } else if (warp < kCorrWarp0) {
    // ---------------- softmax ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int i = warp >> 2, rl = (warp & 3) * 32 + lane;
    const uint32_t tS = tmem + i * 128 + ((uint32_t)((warp & 3) * 32) << 16), tO = tS + 256;
    int ns = 0, nl = 0;
    for (int n = 0; ok; ++n) {
      const Work w = take(n);
      if (!ok || w.len < 0) break;
      if (w.end(i) <= w.start(i)) continue;
      const int qpos = w.t0 + i * p.TT + rl / p.G;
      float m_ref = -INFINITY, l = 0.f;
      for (int j = w.start(i); j < w.end(i); ++j) {
        ok = ok && mbar_wait(&s_full[i], ns & 1, p.err, 70);
        ++ns;
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        float sv[BKV];
        {
          uint32_t* r = reinterpret_cast<uint32_t*>(sv);
          tmem_ld32(tS, r);
          tmem_ld32(tS + 32, r + 32);
          tmem_ld32(tS + 64, r + 64);
          tmem_ld32(tS + 96, r + 96);
          tmem_wait_ld();
        }
        if (p.sign <= 0) {
#pragma unroll
          for (int k = 0; k < BKV; ++k) sv[k] = p.sign < 0 ? -sv[k] : 0.f;
        }
        if (w.part(j)) {
          const int key0 = (w.kb + j) * BKV;
          const int hi = (p.causal ? min(qpos, w.len - 1) : w.len - 1) - key0;
          const int lo = p.window >= 0 ? (int)max((int64_t)0, qpos - p.window - key0) : 0;
#pragma unroll
          for (int k0 = 0; k0 < BKV; k0 += 32) {
            // the visible keys lo .. hi of these 32 as bits
            const int h = min(max(hi - k0 + 1, 0), 32), b = min(max(lo - k0, 0), 32);
            const uint32_t see = (uint32_t)((1ull << h) - 1) & ~(uint32_t)((1ull << b) - 1);
#pragma unroll
            for (int k = 0; k < 32; ++k)
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
        const bool moves = !(mx <= m_ref + kMoves);  // (the first finite one too; NaN)
        if (__any_sync(0xffffffffu, moves)) {
          const float f = !moves ? 1.f : m_ref == -INFINITY ? 0.f : exp2f(m_ref - mx);
          l *= f;
          m_ref = moves ? mx + (mx - mx) : m_ref;  // (infinite scores make a row NaN)
          __syncwarp();  // (the transfers below are the whole warp's)
          // S_i of this step was issued behind P_i V of the last: O_i is at rest
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
        for (int k0 = 0; k0 < BKV; k0 += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float a0, a1;
            f2_unpack(f2_fma(f2_pack(sv[k0 + k], sv[k0 + k + 1]), sc2, nm2), a0, a1);
            a0 = ex2_ftz(a0);
            a1 = ex2_ftz(a1);
            ps[(k >> 1) & 3] = f2_add(ps[(k >> 1) & 3], f2_pack(a0, a1));
            pk[k / 2] = pack2<T>(a0, a1);
          }
          tmem_st16(tS + k0 / 2, pk);
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
      if (nl > 0) ok = ok && mbar_wait(&l_empty[i], (nl & 1) ^ 1, p.err, 72);
      ++nl;
      if (!ok) break;
      sums[i * BQ + rl] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full[i]);
    }
  } else {
    // ---------------- O ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    const int rl = (warp & 3) * 32 + lane;
    const uint32_t tO = tmem + 256 + ((uint32_t)((warp & 3) * 32) << 16);
    uint32_t no = 0;  // parity of the items of each query tile, bit i
    for (int n = 0; ok; ++n) {
      const Work w = take(n);
      if (!ok || w.len < 0) break;
      // the sums, both at once, so that the next item's softmax can go on
      float inv0 = 0.f, inv1 = 0.f;
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (w.end(i) <= w.start(i)) continue;
        ok = ok && mbar_wait(&l_full[i], no >> i & 1, p.err, 75);
        if (!ok) break;
        const float l = sums[i * BQ + rl];
        (i ? inv1 : inv0) = l == 0.f ? 0.f : 1.f / l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_empty[i]);
      }
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (w.end(i) <= w.start(i)) continue;
        ok = ok && mbar_wait(&o_full[i], no >> i & 1, p.err, 76);
        no ^= 1u << i;
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        const float inv = i ? inv1 : inv0;
        const int tok0 = w.t0 + i * p.TT, rows = min(p.TT, w.len - tok0);
        T* out = static_cast<T*>(p.o) + (int64_t)(w.first + tok0) * p.o_sn +
                 (int64_t)w.kvh * p.G * p.o_sh + (lane & 7) * 8;
        // through this warp's part of the staging tile, so that a store covers whole rows
        uint8_t* st = stage + (warp & 3) * 4096;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t r[32];
          tmem_ld32(tO + i * 128 + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(r[q * 8 + e]) * inv;
            *reinterpret_cast<uint4*>(st + (c >> 6) * P::kBox + lane * 128 +
                                      (((c & 63) / 8 + q) ^ (lane & 7)) * 16) = pack8<T>(f);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[i]);
#pragma unroll 4
        for (int q = 0; q < 8 * P::kBoxes; ++q) {
          const int r = (q & 7) * 4 + (lane >> 3), row = (warp & 3) * 32 + r;
          const int tl = row * p.inv_g >> 16;
          const uint4 u = *reinterpret_cast<const uint4*>(st + (q >> 3) * P::kBox + r * 128 +
                                                          ((lane ^ r) & 7) * 16);
          if (tl < rows)
            *reinterpret_cast<uint4*>(out + tl * p.o_sn + (row - tl * p.G) * p.o_sh +
                                      (q >> 3) * 64) = u;
        }
        // (set, if at all, before the last P V could be issued)
        if (*reinterpret_cast<volatile int*>(odd_v + (n & 1)) == n + 1) {
          __syncwarp();
          add_hidden<T, D>(w, i, rl, p);
        }
      }
    }
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
  a.causal = causal != 0;
  a.window = window_left < 0 ? -1 : window_left < N ? window_left : N;
  a.sign = scale > 0 ? 1 : scale < 0 ? -1 : 0;
  a.scale_log2 = scale == 0 ? 1.f : fabsf(scale) * 1.4426950408889634f;
  a.o = o; a.o_sn = o_sn; a.o_sh = o_sh;
  a.v = v; a.v_sn = v_sn; a.v_sh = v_sh;
  a.err = device_error_flag();
  CUtensorMap tq, tk, tv;
  const uint64_t qd[3] = {(uint64_t)D, (uint64_t)Hq, (uint64_t)N};
  const uint64_t qs[2] = {(uint64_t)q_sh * 2, (uint64_t)q_sn * 2};
  const uint32_t qb[3] = {64, (uint32_t)a.G, (uint32_t)a.TT};
  int rc = make_tmap(&tq, q, dtype, 3, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B);
  // K and V: {64 dims, rows, halves of a row, heads}, a tile in one request
  auto kv_map = [&](CUtensorMap* m, const void* base, int64_t sn, int64_t sh) {
    const uint64_t d[4] = {64, (uint64_t)N, (uint64_t)(D / 64), (uint64_t)Hkv};
    const uint64_t s[3] = {(uint64_t)sn * 2, 128, (uint64_t)sh * 2};
    const uint32_t b[4] = {64, BKV, (uint32_t)(D / 64), 1};
    return make_tmap(m, base, dtype, 4, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if (rc == TPP_OK) rc = kv_map(&tk, k, k_sn, k_sh);
  if (rc == TPP_OK) rc = kv_map(&tv, v, v_sn, v_sh);
  if (rc != TPP_OK) return rc;
  // items at most: a block of 2 TT tokens each, one more a sequence
  const int64_t items = (N / (2 * a.TT) + B) * Hkv;
  const unsigned grid = (unsigned)(items < num_sms() ? items : num_sms());
  auto go = [&](auto tag, auto dim) -> int {
    using T = decltype(tag);
    constexpr int DH = decltype(dim)::value;
    auto kern = packed_attn_kernel<T, DH>;
    static std::atomic<bool> reserved[64];
    const int e = reserve_smem(reinterpret_cast<const void*>(kern), reserved, Plan<DH>::kSmem,
                               "packed_attn_kernel");
    if (e != TPP_OK) return e;
    return launch("packed_attn_kernel", kern, dim3(grid), dim3(kThreads), Plan<DH>::kSmem,
                  as_stream(stream), 0u, tq, tk, tv, a);
  };
  return TPP_DISPATCH_HALF(dtype, T, [&] {
    return D == 128 ? go(T(), std::integral_constant<int, 128>{})
                    : go(T(), std::integral_constant<int, 64>{});
  });
}
