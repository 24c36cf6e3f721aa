// Attention of a drafted tree's nodes over the KV cache and the tree itself
// (tpp_attention_tree, tpp_attention_tree_paged).
//
// The T nodes x G query heads of one kv head are the rows of one unit (b, kv
// head, row tile): all of them read the same keys, so the cache is streamed
// once per 16 * RW rows.  Online softmax over tiles of 64 keys, first the cache's
// (masked only at the context's end and at a window's edge), then the tree's
// (one 64-bit mask word a row and tile).
//
// Split: the tiles of all units form one list, cut into equal parts, one for
// each CTA, whatever the lengths of the sequences.  A unit that lies within one
// part is finished there; the pieces of the others go to the workspace as
// (m, l, o) in fp32 and tree_combine_kernel joins them, in list order.  Where there
// are units enough and each is short, a CTA takes a unit instead: no pieces, and
// the next unit's start-up hides under its neighbours' work (32 x 8 nodes over up to
// 640 keys 25.2 us cut, 19.7 not; 64 x 8 46.0 and 34.6; but 8 x 8 over 2000 keys 21.4
// and 34.2).
//
// Threads 0 and 32 feed a ring of K and V tiles by TMA (one request a tile; an
// issuing thread spends about 0.2 us on each), on into the next piece; they refill
// a stage one tile after its use.  (A producer warp of
// its own makes 10 warps an SM, three on one scheduler, and so caps the
// registers of two CTAs at 168: the 64-row form spilled.)  The four warps are RW
// row groups of 16 rows x KW = 4 / RW key groups, each with its own running
// maximum and sum (mma.sync m16n8k16 on fragments from ldmatrix, fp32
// accumulators, exp2 domain); the key groups merge in shared memory at the end.
//
// Bound by HBM on the cache from some 8 tiles a unit on (16 query heads, 8 kv heads of
// 128 dims here and below, unless said otherwise): 64 x 4 nodes over 4096 keys each
// 172 us, 6.27 TB/s (96% of a copy's; 175 paged); 16 x 16 over 8192 (32 rows, the most
// of this form) 102 us, 5.3 TB/s.  Short calls are latency: 5 nodes over 130 keys 8.1
// us, of which 0.5 the lengths, 1.0 the first loads' issue, 1.0 their arrival, 3.6 four
// tiles, 1.1 the merge.  With room for many more keys than the lengths have, where
// tree_combine_kernel is launched to find nothing to do, 2 us more (32 x 8 over up to
// 640 in room for 4096 22.1 us, 20.0 in room for 640).
//
// Masked keys: the score becomes -inf and the value is cleared before the
// product, since 0 * NaN is NaN.  Values that some rows see and others do not
// (tree tiles, a window's edge) are cleared too where they are not finite, and
// added afterwards, element by element, to the rows that see them.
#include <limits.h>
#include <math.h>
#include <algorithm>
#include "mma_common.cuh"
#include "tc_common.cuh"

namespace tpp {
namespace {

constexpr int KT = 64;            // keys of a tile
constexpr int kThreads = 128;
constexpr int kMaxNodes = 256;
constexpr int kTcRows = 128;      // rows of a unit on tcgen05
constexpr float kRescale = 8.0f;  // log2: the base moves when the maximum grew by 2^8

struct TreeArgs {
  const void* q; int64_t q_sb, q_st, q_sh;
  const void* v_cache; int64_t c_sb, c_sh, c_ss;  // for values that are not finite
  const void* v_tree; int64_t vt_sb, vt_st, vt_sh;
  const int32_t* ctx_lens; int max_ctx;
  const uint64_t* mask; int64_t mask_sb;
  void* o; int64_t o_sb, o_st, o_sh;
  const int32_t* table; int64_t table_stride; int num_blocks;
  int64_t window_left;
  float scale_log2;
  float exp_scale;  // scale_log2 if that is positive, 1 otherwise
  int B, T, Hq, Hkv, G, W, R, RT, NT;  // W mask words a row, R = T * G rows, NT tree tiles
  int ctas, rows;                      // parts at most (0: a unit each), rows of a unit
  int whole_tiles;                     // a CTA takes a unit where none has more tiles
  int by_unit;                         // few wide units: try cutting each by itself
  int o_vec;                           // the output's rows start on 32 bytes
  float* ws;                           // pieces: two a part
  int* err;
};

// fp32 words of a piece: o [rows][D], m [rows], l [rows], whether a value that
// is not finite was met
__host__ __device__ constexpr int64_t slot_floats(int rows, int D) {
  return ((int64_t)rows * (D + 2) + 8) / 8 * 8;  // (a slot starts on 32 bytes)
}

__device__ __forceinline__ uint32_t sw_addr(uint32_t base, int r, int chunk) {
  return base + (uint32_t)((chunk >> 3) * KT * 128 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ void bar_compute() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool bar_compute_or(bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\t"
               "barrier.cta.red.or.pred b, 1, 128, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"((uint32_t)x) : "memory");
  return r != 0;
}

template <typename T> struct ExpMask;
template <> struct ExpMask<__half> { static constexpr uint32_t value = 0x7c00u; };
template <> struct ExpMask<__nv_bfloat16> { static constexpr uint32_t value = 0x7f80u; };

// Clears the halves of w that are not finite; `bad` collects whether any was.
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w, uint32_t& bad) {
  constexpr uint32_t E = ExpMask<T>::value;
  const uint32_t lo = (w & E) == E ? 0xffffu : 0u;
  const uint32_t hi = (w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u;
  bad |= lo | hi;
  return w & ~(lo | hi);
}

// One sequence's cache tiles: rows [64 * first, ctx), and the bounds below
// which a window hides rows from all (lo_all) or from some (lo_some) nodes.
struct Span {
  int ctx, first, tiles;
  int64_t lo_all, lo_some;
};
__device__ __forceinline__ Span span_of(const TreeArgs& p, int b) {
  Span s;
  s.ctx = min(max(p.ctx_lens[b], 0), p.max_ctx);
  s.lo_all = s.lo_some = 0;
  if (p.window_left >= 0) {
    s.lo_all = max((int64_t)0, (int64_t)s.ctx - 1 - p.window_left);
    s.lo_some = max((int64_t)0, (int64_t)s.ctx + p.T - 1 - p.window_left);
  }
  s.first = (int)(s.lo_all / KT);
  s.tiles = s.ctx > 0 ? (s.ctx + KT - 1) / KT - s.first : 0;
  return s;
}

// ---- the list of tiles -------------------------------------------------------
// Units in (b, kv head, row tile) order, each with its cache's tiles, then the
// tree's.  The first `more` of n parts hold each + 1 tiles, the others `each`.
struct Parts {
  int n, each, more;  // n = 0: a CTA a unit
  __device__ __forceinline__ int start(int c) const { return each * c + min(c, more); }
  __device__ __forceinline__ int of(int x) const {
    const int x1 = more * (each + 1);
    return x < x1 ? x / (each + 1) : more + (x - x1) / each;
  }
};
// The tiles of lane i's sequence (32 * round + i) and of all up to it, by one
// warp; `before` holds those of earlier rounds.
__device__ __forceinline__ int tiles_scan(const TreeArgs& p, int round, int& incl) {
  const int lane = threadIdx.x & 31, b = 32 * round + lane;
  const int n = b < p.B ? (span_of(p, b).tiles + p.NT) * p.Hkv * p.RT : 0;
  incl = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  return n;
}
// From all tiles and the longest unit's.
__device__ __forceinline__ Parts parts_of(const TreeArgs& p, int total, int longest) {
  Parts s;
  s.n = s.each = s.more = 0;
  if (longest <= p.whole_tiles) return s;
  s.n = max(1, min(p.ctas, total / 2));
  // a wide tree's piece is 64 KB of fp32 a part: below 8 tiles a part, one CTA an SM
  if (p.rows > 32 && total < 8 * p.ctas) s.n = min(s.n, max(p.ctas / 2, 1));
  s.each = total / s.n;
  s.more = total - s.each * s.n;
  return s;
}
// All tiles, those before sequence b, and the longest unit's.
__device__ __forceinline__ int tiles_before(const TreeArgs& p, int b, int& total, int& longest) {
  int before = 0;
  total = longest = 0;
  for (int r = 0; 32 * r < p.B; ++r) {
    int incl;
    const int n = tiles_scan(p, r, incl);
    if (b / 32 == r) before = total + __shfl_sync(0xffffffffu, incl - n, b % 32);
    total += __shfl_sync(0xffffffffu, incl, 31);
    longest = max(longest, __reduce_max_sync(0xffffffffu, n));
  }
  longest /= p.Hkv * p.RT;
  return before;
}
// A part of wide units that straddles two of them pays for two starts and two
// outputs of 64 KB (4 x 64 nodes over 32768 keys: 31 of 296 CTAs, 9 us after all
// others).  So where the longest part is then only a few tiles longer, each unit of
// sequence b is cut by itself, into n_b equal parts.  (Narrow units are not: their
// pieces are small, and the code cost their kernel more.)
__device__ __forceinline__ int unit_parts(const Parts& s, int total, int tiles) {
  return (int)((int64_t)s.n * tiles / total);
}
__device__ __forceinline__ bool cut_by_unit(const TreeArgs& p, const Parts& s, int total) {
  if (!p.by_unit || s.n == 0) return false;
  int worst = 0;
  for (int b = threadIdx.x & 31; b < p.B; b += 32) {
    const int n = span_of(p, b).tiles + p.NT, k = unit_parts(s, total, n);
    worst = max(worst, k == 0 ? INT_MAX : (n + k - 1) / k);
  }
  return __reduce_max_sync(0xffffffffu, worst) <= s.each + 5;
}
// Parts of the sequences before b, so cut.
__device__ __forceinline__ int unit_parts_before(const TreeArgs& p, const Parts& s, int total,
                                                 int b) {
  int n = 0;
  for (int i = threadIdx.x & 31; i < b; i += 32)
    n += unit_parts(s, total, span_of(p, i).tiles + p.NT) * p.Hkv * p.RT;
  return __reduce_add_sync(0xffffffffu, n);
}
// Walks the pieces of units in one CTA's part.
struct Piece {
  int pos, end, before;  // in the list; before: tiles of earlier sequences
  int b, unit, t0, t1;   // tiles [t0, t1) of the unit (kv head, row tile) of b
  Span sp;
  bool whole;
  template <bool WIDE>
  __device__ __forceinline__ bool start(const TreeArgs& p) {
    Parts s;
    s.n = 0;
    int incl = 0, total = 0, n = 0, longest = 0, rounds = (p.B + 31) / 32;
    if (p.ctas > 0) {
      for (int r = 0; r < rounds; ++r) {
        n = tiles_scan(p, r, incl);
        total += __shfl_sync(0xffffffffu, incl, 31);
        longest = max(longest, __reduce_max_sync(0xffffffffu, n));
      }
      s = parts_of(p, total, longest / (p.Hkv * p.RT));
    }
    if (s.n == 0) {
      const int u = p.Hkv * p.RT;
      b = blockIdx.x / u;
      if (b >= p.B) return false;
      sp = span_of(p, b);
      before = 0;  // a list of b's own
      pos = (int)(blockIdx.x % u) * (sp.tiles + p.NT);
      end = pos + sp.tiles + p.NT;
    } else if (WIDE && cut_by_unit(p, s, total)) {
      // one piece, in a list of b's own
      const int u = p.Hkv * p.RT, lane = threadIdx.x & 31;
      int base = 0, at = -1, tiles = 0, k = 0;
      for (int r = 0; r < rounds && at < 0; ++r) {
        const int i = 32 * r + lane, m = i < p.B ? span_of(p, i).tiles + p.NT : 0;
        const int parts = unit_parts(s, total, m);
        int scan = parts * u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, scan, o);
          if (lane >= o) scan += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, (int)blockIdx.x < base + scan);
        if (hit) {
          const int l = __ffs(hit) - 1;
          b = 32 * r + l;
          tiles = __shfl_sync(0xffffffffu, m, l);
          k = __shfl_sync(0xffffffffu, parts, l);
          at = (int)blockIdx.x - base - __shfl_sync(0xffffffffu, scan - parts * u, l);
        } else {
          base += __shfl_sync(0xffffffffu, scan, 31);
        }
      }
      if (at < 0) return false;
      sp = span_of(p, b);
      const int un = at / k, part = at - un * k;
      before = 0;
      pos = un * tiles + (int)((int64_t)tiles * part / k);
      end = un * tiles + (int)((int64_t)tiles * (part + 1) / k);
    } else {
      if ((int)blockIdx.x >= s.n) return false;
      pos = s.start(blockIdx.x);
      end = s.start(blockIdx.x + 1);
      // the sequence that pos belongs to; the scan of a single round is at hand
      b = p.B;
      before = 0;
      for (int r = 0; r < rounds && b == p.B; ++r) {
        if (rounds > 1) n = tiles_scan(p, r, incl);
        const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && pos < before + incl);
        const int l = hit ? __ffs(hit) - 1 : 31;
        if (hit) b = 32 * r + l;
        before += __shfl_sync(0xffffffffu, hit ? incl - n : incl, l);
      }
      if (b >= p.B) return false;
      sp = span_of(p, b);
    }
    locate(p);
    return pos < end;
  }
  __device__ __forceinline__ void locate(const TreeArgs& p) {
    const int n = sp.tiles + p.NT;
    unit = (pos - before) / n;
    t0 = pos - before - unit * n;
    t1 = min(n, t0 + (end - pos));
    whole = t0 == 0 && t1 == n;
  }
  __device__ __forceinline__ bool next(const TreeArgs& p) {
    pos += t1 - t0;
    if (pos >= end) return false;
    const int n = sp.tiles + p.NT;
    if (unit == p.Hkv * p.RT - 1 && t1 == n) {
      before += n * p.Hkv * p.RT;
      sp = span_of(p, ++b);
    }
    locate(p);
    return true;
  }
};
template <int D, int RW>
struct TreeSmem {
  static constexpr int KW = 4 / RW;
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr uint32_t kTile = KT * D * 2;
  static constexpr uint32_t kRing = kStages * 2 * kTile;
  static constexpr int kDims = RW == 1 ? D : 64;  // dims merged at a time
  static constexpr uint32_t kMerge = KW > 1 ? RW * 16 * kDims * 4 : 0;
  static constexpr uint32_t kMl = 4 * 16 * 2 * 4;  // (m, l) of each warp's rows
  static constexpr size_t kBytes = 1024 + kRing + kMerge + kMl + 2 * kStages * 8 + 2 * sizeof(Piece);
};

// Where part c keeps a piece: the one that starts its unit, or continues one.
__device__ __forceinline__ float* slot_of(const TreeArgs& p, int D, int c, bool starts) {
  return p.ws + (int64_t)(2 * c + (starts ? 1 : 0)) * slot_floats(p.rows, D);
}

// The first cache row that the node with mask row `row` sees.
__device__ __forceinline__ int64_t low_of(const TreeArgs& p, const Span& s, const uint64_t* row) {
  if (p.window_left < 0) return 0;
  int seen = 0;
  for (int w = 0; w < p.W; ++w) {
    const int n = p.T - 64 * w;
    seen += __popcll(row[w] & (n < 64 ? (1ull << n) - 1 : ~0ull));
  }
  return (int64_t)s.ctx + seen - 1 - p.window_left;
}

// Sum of the values at dim d that are not finite over the keys that node t sees
// in the tree and in the cache tiles that were cleared of them.
template <typename T, int D>
__device__ float odd_values(const TreeArgs& p, const Span& sp, int b, int kvh, int t, int d) {
  const uint64_t* row = p.mask + b * p.mask_sb + (int64_t)t * p.W;
  float acc = 0.f;
  auto add = [&](float x) { if (!isfinite(x)) acc += x; };
  for (int j = 0; j < p.T; ++j)
    if ((row[j / 64] >> (j % 64)) & 1)
      add(to_f32(static_cast<const T*>(p.v_tree)[b * p.vt_sb + j * p.vt_st + kvh * p.vt_sh + d]));
  for (int64_t k = max(low_of(p, sp, row), (int64_t)0); k < sp.ctx; ++k) {
    const int64_t k0 = k / KT * KT;
    if (k0 + KT <= sp.ctx && k0 >= sp.lo_some) { k = k0 + KT - 1; continue; }
    int64_t at = b * p.c_sb + kvh * p.c_sh + k * p.c_ss;
    if (p.table) {
      const int blk = p.table[b * p.table_stride + k / KT];
      if (blk < 0 || blk >= p.num_blocks) continue;
      at = (((int64_t)blk * p.Hkv + kvh) * KT + k % KT) * D;
    }
    add(to_f32(static_cast<const T*>(p.v_cache)[at + d]));
  }
  return acc;
}

template <typename T, int D, int RW>
__global__ void __launch_bounds__(kThreads, 2) tree_attn_kernel(
    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
    const __grid_constant__ CUtensorMap tm_kt, const __grid_constant__ CUtensorMap tm_vt,
    const __grid_constant__ TreeArgs p) {
  using SM = TreeSmem<D, RW>;
  constexpr int ST = SM::kStages, KW = SM::KW;
  constexpr int KPW = KT / KW;    // keys of a tile for each warp
  constexpr int NTL = KPW / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  float* mbuf = reinterpret_cast<float*>(smem + SM::kRing);
  float* ml = reinterpret_cast<float*>(smem + SM::kRing + SM::kMerge);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SM::kRing + SM::kMerge + SM::kMl);
  uint64_t* empty = full + ST;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    prefetch_tmap(&tm_kt);
    prefetch_tmap(&tm_vt);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 4);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  Piece pc;
  if (!pc.start<false>(p)) return;
  bool ok = true;
  int it = 0;  // tiles so far: the ring's position
  // The loads run ahead of pc; their threads keep the place in shared memory.
  const bool loader = threadIdx.x == 0 || threadIdx.x == 32;
  Piece* ahead = reinterpret_cast<Piece*>(empty + ST) + (warp & 1);
  const CUtensorMap* from = warp == 0 ? &tm_k : &tm_v;
  const CUtensorMap* from_tree = warp == 0 ? &tm_kt : &tm_vt;
  int issued = 0;
  auto issue = [&]() {  // the next tile of the part, if there is one
    if (issued < 0) return;
    const int i = ahead->t0, b = ahead->b, kvh = ahead->unit / p.RT;
    const int s = issued % ST, first = ahead->sp.first, tiles = ahead->sp.tiles;
    uint8_t* dst = smem + (s * 2 + (warp & 1)) * SM::kTile;
    mbar_arrive_expect_tx(&full[s], SM::kTile);
    if (i >= tiles) {
      tma_load_5d(dst, from_tree, &full[s], 0, (i - tiles) * KT, 0, kvh, b);
    } else if (p.table) {
      // a block outside the pool is out of the map's range: zeros
      int blk = p.table[b * p.table_stride + first + i];
      if (blk < 0 || blk >= p.num_blocks) blk = p.num_blocks;
      tma_load_5d(dst, from, &full[s], 0, 0, 0, kvh, blk);
    } else {
      tma_load_5d(dst, from, &full[s], 0, (first + i) * KT, 0, kvh, b);
    }
    ++issued;
    if (i + 1 < ahead->t1) {
      ahead->t0 = i + 1;
      ahead->pos += 1;
    } else if (!ahead->next(p)) {
      issued = -1;
    }
  };
  if (loader) {
    *ahead = pc;
    for (int s = 0; s < ST; ++s) issue();
  }
  __syncwarp();

  // ---------------- compute ----------------
  const int g = lane >> 2, c = lane & 3;
  const int rw = warp / KW, kw = warp % KW;
  const int kr0 = kw * KPW;
  do {
    const int b = pc.b, kvh = pc.unit / p.RT, rt = pc.unit % p.RT;
    const Span& sp = pc.sp;
    int node[2], head[2];
    bool live[2];
    const uint64_t* mrow[2];
    int64_t lo[2];
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      const int r = rt * 16 * RW + rw * 16 + g + 8 * hr;
      live[hr] = r < p.R;
      node[hr] = live[hr] ? r / p.G : 0;
      head[hr] = kvh * p.G + (live[hr] ? r % p.G : 0);
      mrow[hr] = p.mask + b * p.mask_sb + (int64_t)node[hr] * p.W;
      lo[hr] = low_of(p, sp, mrow[hr]);
    }
    // Q fragments straight from global memory: each value is used by one lane only
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          static_cast<const T*>(p.q) + b * p.q_sb + node[hr] * p.q_st + head[hr] * p.q_sh);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks][hr] = live[hr] ? src[ks * 8 + c] : 0u;
        qf[ks][hr + 2] = live[hr] ? src[ks * 8 + c + 4] : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_r[2] = {-INFINITY, -INFINITY}, l_r[2] = {0.f, 0.f};
    uint32_t bad = 0;

    for (int i = pc.t0; i < pc.t1; ++i, ++it) {
      const int s = it % ST;
      if (loader && it > 0 && ok && issued >= 0) {
        ok = mbar_wait(&empty[(it - 1) % ST], ((it - 1) / ST) & 1, p.err, 61);
        if (ok) issue();
      }
      if (ok) ok = mbar_wait(&full[s], (it / ST) & 1, p.err, 62);
      const uint32_t kb = smem_u32(smem + s * 2 * SM::kTile), vb = kb + SM::kTile;
      float sc[NTL][4];
#pragma unroll
      for (int j = 0; j < NTL; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int jp = 0; jp < NTL / 2; ++jp) {
          uint32_t bf[4];
          ldsm_x4(sw_addr(kb, kr0 + jp * 16 + (lane & 7) + (lane >> 4) * 8,
                          ks * 2 + ((lane >> 3) & 1)), bf);
          mma<T>(sc[2 * jp], qf[ks], bf[0], bf[1]);
          mma<T>(sc[2 * jp + 1], qf[ks], bf[2], bf[3]);
        }
      }
      const bool tree = i >= sp.tiles;
      const int64_t key0 = (int64_t)(sp.first + i) * KT;   // of a cache tile
      const bool careful = tree || key0 + KT > sp.ctx || key0 < sp.lo_some;
      if (tree) {
        const int n0 = (i - sp.tiles) * KT, n = p.T - n0;
        const uint64_t in = n < 64 ? (1ull << n) - 1 : ~0ull;
        const uint64_t w0 = mrow[0][i - sp.tiles] & in, w1 = mrow[1][i - sp.tiles] & in;
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = kr0 + j * 8 + 2 * c + (e & 1);
            sc[j][e] = (((e < 2 ? w0 : w1) >> k) & 1) ? sc[j][e] * p.scale_log2 : -INFINITY;
          }
      } else if (careful) {
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t k = key0 + kr0 + j * 8 + 2 * c + (e & 1);
            sc[j][e] = (k < sp.ctx && k >= lo[e >> 1]) ? sc[j][e] * p.scale_log2 : -INFINITY;
          }
      } else {
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[j][e] *= p.scale_log2;
      }
      // Online softmax with a lazy base: m_r moves, and o and l are rescaled,
      // only when a row's maximum grew by more than 2^8.
      float corr[2];
      bool grow = false;
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < NTL; ++j) mx = fmax3(mx, sc[j][2 * hr], sc[j][2 * hr + 1]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        corr[hr] = 1.f;
        if (mx > m_r[hr] + kRescale) {
          corr[hr] = ex2_ftz(m_r[hr] - mx);  // 0 when no key was seen yet
          m_r[hr] = mx;
          grow = true;
        }
        const float base = m_r[hr] == -INFINITY ? 0.f : m_r[hr];
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float pv = ex2_ftz(sc[j][2 * hr + e] - base);
            sc[j][2 * hr + e] = pv;
            sum += pv;
          }
        l_r[hr] = l_r[hr] * corr[hr] + sum;
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][0] *= corr[0]; o[d][1] *= corr[0];
          o[d][2] *= corr[1]; o[d][3] *= corr[1];
        }
      }
#pragma unroll
      for (int kk = 0; kk < KPW / 16; ++kk) {
        // the probabilities are rounded to T for the product: the same relative
        // error as the values themselves carry
        uint32_t pa[4];
        pa[0] = pack2<T>(sc[2 * kk][0], sc[2 * kk][1]);
        pa[1] = pack2<T>(sc[2 * kk][2], sc[2 * kk][3]);
        pa[2] = pack2<T>(sc[2 * kk + 1][0], sc[2 * kk + 1][1]);
        pa[3] = pack2<T>(sc[2 * kk + 1][2], sc[2 * kk + 1][3]);
        uint32_t keep0 = ~0u, keep1 = ~0u;  // values no row sees: stale rows of a cache
        if (careful && !tree) {
          const int64_t k = key0 + kr0 + kk * 16 + 2 * c;
          auto in = [&](int64_t x) { return x < sp.ctx && x >= sp.lo_all; };
          keep0 = (in(k) ? 0xffffu : 0u) | (in(k + 1) ? 0xffff0000u : 0u);
          keep1 = (in(k + 8) ? 0xffffu : 0u) | (in(k + 9) ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int dp = 0; dp < D / 16; ++dp) {
          uint32_t bf[4];
          ldsm_x4_t(sw_addr(vb, kr0 + kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8,
                            dp * 2 + (lane >> 4)), bf);
          if (careful) {
            bf[0] = finite2<T>(bf[0] & keep0, bad);
            bf[1] = finite2<T>(bf[1] & keep1, bad);
            bf[2] = finite2<T>(bf[2] & keep0, bad);
            bf[3] = finite2<T>(bf[3] & keep1, bad);
          }
          mma<T>(o[2 * dp], pa, bf[0], bf[1]);
          mma<T>(o[2 * dp + 1], pa, bf[2], bf[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    // ---------------- merge the key groups ----------------
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      l_r[hr] += __shfl_xor_sync(0xffffffffu, l_r[hr], 1);
      l_r[hr] += __shfl_xor_sync(0xffffffffu, l_r[hr], 2);
    }
    if (KW > 1) {
      if (c == 0) {
#pragma unroll
        for (int hr = 0; hr < 2; ++hr) {
          ml[(warp * 16 + g + 8 * hr) * 2] = m_r[hr];
          ml[(warp * 16 + g + 8 * hr) * 2 + 1] = l_r[hr];
        }
      }
      bar_compute();
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) M = fmaxf(M, ml[((rw * KW + w) * 16 + g + 8 * hr) * 2]);
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float* x = ml + ((rw * KW + w) * 16 + g + 8 * hr) * 2;
          L += x[1] * ex2_ftz(x[0] - base);
        }
        const float f = ex2_ftz(m_r[hr] - base);
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][2 * hr] *= f;
          o[d][2 * hr + 1] *= f;
        }
        m_r[hr] = M;
        l_r[hr] = L;
      }
      // group k hands its sum to group k - 1, in this order always
#pragma unroll
      for (int k = KW - 1; k > 0; --k)
#pragma unroll
        for (int d0 = 0; d0 < D / 8; d0 += SM::kDims / 8) {
          float2* buf = reinterpret_cast<float2*>(mbuf) + rw * 16 * SM::kDims / 2 + lane;
          if (kw == k) {
#pragma unroll
            for (int d = 0; d < SM::kDims / 8; ++d) {
              buf[(2 * d) * 32] = make_float2(o[d0 + d][0], o[d0 + d][1]);
              buf[(2 * d + 1) * 32] = make_float2(o[d0 + d][2], o[d0 + d][3]);
            }
          }
          bar_compute();
          if (kw == k - 1) {
#pragma unroll
            for (int d = 0; d < SM::kDims / 8; ++d) {
              const float2 x = buf[(2 * d) * 32], y = buf[(2 * d + 1) * 32];
              o[d0 + d][0] += x.x; o[d0 + d][1] += x.y;
              o[d0 + d][2] += y.x; o[d0 + d][3] += y.y;
            }
          }
          bar_compute();
        }
    }
    // ---------------- output ----------------
    float* slot = pc.whole ? nullptr : slot_of(p, D, blockIdx.x, pc.t0 == 0);
    if (kw == 0) {
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        if (!live[hr]) continue;
        if (pc.whole) {
          const float inv = l_r[hr] == 0.f ? 0.f : 1.f / l_r[hr];  // nothing seen: zeros
          uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + b * p.o_sb +
                                                      node[hr] * p.o_st + head[hr] * p.o_sh);
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            dst[d * 4 + c] = pack2<T>(o[d][2 * hr] * inv, o[d][2 * hr + 1] * inv);
        } else {
          const int r = rw * 16 + g + 8 * hr;
          float2* dst = reinterpret_cast<float2*>(slot + r * D);
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
            dst[d * 4 + c] = make_float2(o[d][2 * hr], o[d][2 * hr + 1]);
          if (c == 0) {
            slot[p.rows * D + r] = m_r[hr];
            slot[p.rows * (D + 1) + r] = l_r[hr];
          }
        }
      }
    }
    const bool odd = bar_compute_or(bad != 0);
    if (!pc.whole) {
      if (threadIdx.x == 0) slot[p.rows * (D + 2)] = odd ? 1.f : 0.f;
    } else if (odd) {
      const int n = min(16 * RW, p.R - rt * 16 * RW);
      for (int e = threadIdx.x; e < n * D; e += 128) {
        const int r = rt * 16 * RW + e / D, d = e % D;
        const int t = r / p.G, h = kvh * p.G + r % p.G;
        const float acc = odd_values<T, D>(p, sp, b, kvh, t, d);
        if (acc != 0.f) {
          T* dst = static_cast<T*>(p.o) + b * p.o_sb + t * p.o_st + h * p.o_sh + d;
          *dst = from_f32<T>(to_f32(*dst) + acc);
        }
      }
    }
  } while (pc.next(p));
}

// ---- wide trees: tcgen05 ------------------------------------------------------
// From 33 rows a unit on, the products outgrow mma.sync (64 rows over a 64-key
// tile are 1050 clocks of MMA an SM, about what the tile takes to arrive), so a
// unit is a 128-row tile on the 5th-generation tensor core.  Two CTAs an SM, each
// with its own S, P and O in 256 columns of TMEM: while one waits for its scores
// the other's softmax runs.
//   warps 0-3: softmax (a row a thread), output
//   warp 4:    Q, and K and V tiles into two rings, by TMA, ahead into the next
//              piece (a unit takes as many whole nodes as 128 rows hold, so that
//              its Q is one box of nodes x heads for each 64 dims)
//   warp 5:    S = Q K^T (M 128, N 64), O += P V (P read from TMEM)
// S and P share two 64-column buffers; S of tile j+1 is computed under the softmax
// of tile j.  Rows that a narrow unit (R < 128) lacks are skipped by whole warps.
// Two CTAs of 192 threads leave 168 registers a thread, of which the softmax warps
// spill 112 bytes.
// 4 x 64 nodes over 32768 keys: 114 us, 604 TFLOP/s, 4.74 TB/s; in mid-course a CTA
// takes 1.3 to 1.5 us a tile, which for all 296 is 7.4 to 6.5 TB/s; the rest is
// the start (5 us), the pieces' output (4) and the combine kernel (4).  Measured and
// not kept: P in shared memory, so that S of tile j+2 need not wait for the product
// of tile j (113 us, and 76 for 69 at 64 dims); two threads a row, 8 softmax warps a
// CTA (96 registers, spills, 185 us); polls that do not suspend (no change).
constexpr int kTcThreads = 192;
constexpr int kKSt = 2, kVSt = 3;

template <int D>
struct TcSmem {
  static constexpr uint32_t kQ = kTcRows * D * 2;
  static constexpr uint32_t kTile = KT * D * 2;
  static constexpr size_t kBytes = kQ + (kKSt + kVSt) * kTile + 1024;
};

__device__ __forceinline__ bool bar_softmax_or(bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\t"
               "barrier.cta.red.or.pred b, 2, 128, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"((uint32_t)x) : "memory");
  return r != 0;
}

// 32 bytes at once: a lane writes its own row, so narrower stores would leave half
// a sector each (a piece's 64 KB took 5 us).
__device__ __forceinline__ void store8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 2) tree_attn_tc_kernel(
    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
    const __grid_constant__ CUtensorMap tm_kt, const __grid_constant__ CUtensorMap tm_vt,
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ TreeArgs p) {
  using SM = TcSmem<D>;
  extern __shared__ __align__(1024) uint8_t tc_smem[];
  uint8_t* sQ = tc_smem;
  uint8_t* sK = sQ + SM::kQ;
  uint8_t* sV = sK + kKSt * SM::kTile;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sV + kVSt * SM::kTile);
  uint64_t* q_empty = q_full + 1;      // every S of a piece is complete
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + kKSt;
  uint64_t* v_full = k_empty + kKSt;
  uint64_t* v_empty = v_full + kVSt;
  uint64_t* s_full = v_empty + kVSt;   // S of a tile is in its buffer
  uint64_t* p_full = s_full + 2;       // P has replaced it
  uint64_t* pv_done = p_full + 2;      // P V is complete: the buffer is free
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    prefetch_tmap(&tm_kt);
    prefetch_tmap(&tm_vt);
    prefetch_tmap(&tm_q);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < kKSt; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
    for (int s = 0; s < kVSt; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  Piece pc;
  if (!pc.start<true>(p)) return;
  if (warp == 5) tmem_alloc(tmem_slot, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Only now: a dependent kernel that allocates TMEM ahead of its own wait could take
  // what this CTA still lacks, and keep it until this kernel has ended.
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp == 4) {
    // ---------------- K/V producer ----------------
    if (lane == 0) {
      Piece pv = pc;                 // where V is; pc: where K is
      bool more_k = true, more_v = true, new_piece = true;
      int nk = 0, nv = 0, nq = 0;
      uint32_t idle = 0;
      auto load = [&](Piece& at, const CUtensorMap* cache, const CUtensorMap* tree, uint8_t* dst,
                      uint64_t* full) {
        const int kvh = at.unit / p.RT, i = at.t0;
        mbar_arrive_expect_tx(full, SM::kTile);
        if (i >= at.sp.tiles) {
          tma_load_5d(dst, tree, full, 0, (i - at.sp.tiles) * KT, 0, kvh, at.b);
        } else if (p.table) {
          int blk = p.table[at.b * p.table_stride + at.sp.first + i];
          if (blk < 0 || blk >= p.num_blocks) blk = p.num_blocks;
          tma_load_5d(dst, cache, full, 0, 0, 0, kvh, blk);
        } else {
          tma_load_5d(dst, cache, full, 0, (at.sp.first + i) * KT, 0, kvh, at.b);
        }
        if (i + 1 < at.t1) { at.t0 = i + 1; at.pos += 1; return true; }
        return at.next(p);
      };
      while (ok && more_v) {
        bool moved = false;
        if (new_piece && (nq == 0 || mbar_try_wait(q_empty, (nq - 1) & 1))) {
          mbar_arrive_expect_tx(q_full, p.rows * D * 2);
          for (int bx = 0; bx < D / 64; ++bx)
            tma_load_5d(sQ + bx * (kTcRows * 128), &tm_q, q_full, 0, (pc.unit / p.RT) * p.G,
                        (pc.unit % p.RT) * (p.rows / p.G), bx, pc.b);
          ++nq;
          new_piece = false;
          moved = true;
        }
        if (more_k && !new_piece && (nk < kKSt || mbar_try_wait(&k_empty[nk % kKSt], ((nk / kKSt) & 1) ^ 1))) {
          const int s = nk % kKSt;
          new_piece = pc.t0 + 1 == pc.t1;
          more_k = load(pc, &tm_k, &tm_kt, sK + s * SM::kTile, &k_full[s]);
          new_piece = new_piece && more_k;
          ++nk;
          moved = true;
        }
        if (nv < nk && (nv < kVSt || mbar_try_wait(&v_empty[nv % kVSt], ((nv / kVSt) & 1) ^ 1))) {
          const int s = nv % kVSt;
          more_v = load(pv, &tm_v, &tm_vt, sV + s * SM::kTile, &v_full[s]);
          ++nv;
          moved = true;
        }
        if (moved) {
          idle = 0;
        } else if (++idle > (kWaitLimit << 2)) {
          if (p.err) atomicExch(p.err, 63);
          ok = false;
        }
      }
    }
  } else if (warp == 5) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_f16(kTcRows, KT, IsBf16<T>::value, 0, 0);
      constexpr uint32_t idesc_o = make_idesc_f16(kTcRows, D, IsBf16<T>::value, 0, 1);
      const uint32_t tO = tmem, tS = tmem + 128, qa = smem_u32(sQ);
      int ns = 0, npv = 0, piece = 0;
      do {
        // (O of the piece before is read by the time the first P is written)
        ok = mbar_wait(q_full, piece & 1, p.err, 64);
        ++piece;
        const int end = npv + (pc.t1 - pc.t0), begin = npv;
        tc_fence_after();
        uint32_t idle = 0;
        while (ok && npv < end) {
          bool moved = false;
          // buffer ns % 2 last held P of tile ns - 2
          if (ns < end && ns < npv + 2 &&
              (ns < 2 || mbar_try_wait(&pv_done[ns & 1], ((ns - 2) >> 1) & 1)) &&
              mbar_try_wait(&k_full[ns % kKSt], (ns / kKSt) & 1)) {
            tc_fence_after();
            const uint32_t ka = smem_u32(sK + (ns % kKSt) * SM::kTile);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              tc_mma_f16(tS + (ns & 1) * 64,
                         make_sdesc(qa + (kk >> 2) * (kTcRows * 128) + (kk & 3) * 32, 16, 1024, 2),
                         make_sdesc(ka + (kk >> 2) * (KT * 128) + (kk & 3) * 32, 16, 1024, 2),
                         idesc_s, kk != 0);
            tc_commit(&s_full[ns & 1]);
            tc_commit(&k_empty[ns % kKSt]);
            if (ns == end - 1) tc_commit(q_empty);
            ++ns;
            moved = true;
          }
          if (npv < ns && mbar_try_wait(&p_full[npv & 1], (npv >> 1) & 1) &&
              mbar_try_wait(&v_full[npv % kVSt], (npv / kVSt) & 1)) {
            tc_fence_after();
            const uint32_t va = smem_u32(sV + (npv % kVSt) * SM::kTile);
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk)
              // V is MN-major: 64-dim boxes KT * 128 bytes apart, 8-key groups
              // 1 KB apart; 16 keys are 2 KB
              tc_mma_f16_ts(tO, tS + (npv & 1) * 64 + kk * 8,
                            make_sdesc(va + kk * 2048, KT * 128, 1024, 2), idesc_o,
                            (npv != begin) || kk != 0);
            tc_commit(&pv_done[npv & 1]);
            tc_commit(&v_empty[npv % kVSt]);
            ++npv;
            moved = true;
          }
          if (moved) {
            idle = 0;
          } else if (++idle > (kWaitLimit << 2)) {
            if (p.err) atomicExch(p.err, 65);
            ok = false;
          }
        }
      } while (ok && pc.next(p));
    }
  } else {
    // ---------------- softmax and output: thread = row ----------------
    const int rl = threadIdx.x;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const uint32_t tO = tmem + lane_off, tS = tmem + 128 + lane_off;
    int it = 0;
    do {
      const int b = pc.b, kvh = pc.unit / p.RT, row0 = (pc.unit % p.RT) * p.rows;
      const Span& sp = pc.sp;
      const int row = row0 + rl;
      const bool live = rl < p.rows && row < p.R;
      const bool warp_live = row0 + warp * 32 < p.R;
      const int node = live ? row / p.G : 0, head = kvh * p.G + (live ? row % p.G : 0);
      const uint64_t* mrow = p.mask + b * p.mask_sb + (int64_t)node * p.W;
      const int64_t lo = low_of(p, sp, mrow);
      float m_ref = -INFINITY, l = 0.f;
      uint32_t bad = 0;
      for (int i = pc.t0; i < pc.t1; ++i, ++it) {
        const int buf = it & 1;
        if (ok) ok = mbar_wait(&s_full[buf], (it >> 1) & 1, p.err, 66);
        tc_fence_after();
        const bool tree = i >= sp.tiles;
        const int64_t key0 = (int64_t)(sp.first + i) * KT;
        const bool careful = tree || key0 + KT > sp.ctx || key0 < sp.lo_some;
        if (warp_live) {
          float sv[KT];
          {
            uint32_t r[KT];
            tmem_ld32(tS + buf * 64, r);
            tmem_ld32(tS + buf * 64 + 32, r + 32);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < KT; ++k) sv[k] = __uint_as_float(r[k]);
          }
          // The scale goes into the exponent's fma, behind the mask and the maximum,
          // which only a positive one leaves as they are: others are applied here.
          if (!(p.scale_log2 > 0.f)) {
#pragma unroll
            for (int k = 0; k < KT; ++k) sv[k] *= p.scale_log2;
          }
          if (careful) {
            uint64_t see;
            if (tree) {
              const int w = i - sp.tiles, n = p.T - 64 * w;
              see = mrow[w] & (n < 64 ? (1ull << n) - 1 : ~0ull);
            } else {
              const int64_t hi = sp.ctx - key0, from = lo - key0;  // seen: [from, hi)
              see = hi >= 64 ? ~0ull : (1ull << hi) - 1;
              if (from > 0) see &= from >= 64 ? 0ull : ~0ull << from;
            }
#pragma unroll
            for (int k = 0; k < KT; ++k)
              if (!((see >> k) & 1)) sv[k] = -INFINITY;
          }
          float pm[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) pm[u] = fmaxf(sv[u], sv[8 + u]);
#pragma unroll
          for (int k = 16; k < KT; k += 16)
#pragma unroll
            for (int u = 0; u < 8; ++u) pm[u] = fmax3(pm[u], sv[k + u], sv[k + 8 + u]);
          const float mx = fmax3(fmax3(pm[0], pm[1], pm[2]), fmax3(pm[3], pm[4], pm[5]),
                                 fmaxf(pm[6], pm[7])) * p.exp_scale;
          // lazy base, as above; O's rescale is warp-collective, so lanes that
          // keep their base use the factor 1
          const bool grow = mx > m_ref + kRescale;
          const float corr = grow ? ex2_ftz(m_ref - mx) : 1.f;
          if (grow) { l *= corr; m_ref = mx; }
          if (i > pc.t0 && __any_sync(0xffffffffu, grow)) {
            if (ok) ok = mbar_wait(&pv_done[(it - 1) & 1], ((it - 1) >> 1) & 1, p.err, 67);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              uint32_t r[32];
              tmem_ld32(tO + c, r);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * corr);
              tmem_st32(tO + c, r);
            }
            tmem_wait_st();
          }
          const float nm = m_ref == -INFINITY ? 0.f : -m_ref;
          const uint64_t sc2 = f2_pack(p.exp_scale, p.exp_scale), nm2 = f2_pack(nm, nm);
          uint64_t ps[4] = {0ull, 0ull, 0ull, 0ull};
          uint32_t pk[KT / 2];
#pragma unroll
          for (int k = 0; k < KT; k += 2) {
            float a0, a1;
            f2_unpack(f2_fma(f2_pack(sv[k], sv[k + 1]), sc2, nm2), a0, a1);
            const float p0 = ex2_ftz(a0), p1 = ex2_ftz(a1);
            ps[(k >> 1) & 3] = f2_add(ps[(k >> 1) & 3], f2_pack(p0, p1));
            pk[k / 2] = pack2<T>(p0, p1);
          }
          float t0, t1;
          f2_unpack(f2_add(f2_add(ps[0], ps[1]), f2_add(ps[2], ps[3])), t0, t1);
          l += t0 + t1;
          tmem_st32(tS + buf * 64, pk);
          tmem_wait_st();
        }
        if (careful) {
          // clear the values that no row may take from this tile's V
          if (ok) ok = mbar_wait(&v_full[it % kVSt], (it / kVSt) & 1, p.err, 68);
          uint8_t* v = sV + (it % kVSt) * SM::kTile;
          for (int e = rl; e < KT * (D / 8); e += 128) {
            const int64_t key = key0 + (e / 8) % KT;
            uint4* w = reinterpret_cast<uint4*>(v) + e;   // [box][key][8 chunks]
            uint4 x = *w;
            if (!tree && (key >= sp.ctx || key < sp.lo_all)) {
              x = make_uint4(0, 0, 0, 0);
            } else {
              x.x = finite2<T>(x.x, bad); x.y = finite2<T>(x.y, bad);
              x.z = finite2<T>(x.z, bad); x.w = finite2<T>(x.w, bad);
            }
            *w = x;
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      // ---- the piece's output ----
      if (ok) ok = mbar_wait(&pv_done[(it - 1) & 1], ((it - 1) >> 1) & 1, p.err, 69);
      tc_fence_after();
      float* slot = pc.whole ? nullptr : slot_of(p, D, blockIdx.x, pc.t0 == 0);
      if (warp_live) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* dst = static_cast<T*>(p.o) + b * p.o_sb + node * p.o_st + head * p.o_sh;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t r[32];
          __syncwarp();
          tmem_ld32(tO + c, r);
          tmem_wait_ld();
          if (!live) {
          } else if (!pc.whole) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) store8(slot + rl * D + c + k, r + k);
          } else {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; ++k)
              w[k] = pack2<T>(__uint_as_float(r[2 * k]) * inv, __uint_as_float(r[2 * k + 1]) * inv);
            if (p.o_vec) {
#pragma unroll
              for (int k = 0; k < 16; k += 8) store8(dst + c + 2 * k, w + k);
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k) *reinterpret_cast<uint32_t*>(dst + c + 2 * k) = w[k];
            }
          }
        }
        if (!pc.whole && live) {
          slot[p.rows * D + rl] = m_ref;
          slot[p.rows * (D + 1) + rl] = l;
        }
      }
      const bool odd = bar_softmax_or(bad != 0);
      if (!pc.whole) {
        if (rl == 0) slot[p.rows * (D + 2)] = odd ? 1.f : 0.f;
      } else if (odd && live) {
        T* dst = static_cast<T*>(p.o) + b * p.o_sb + node * p.o_st + head * p.o_sh;
        for (int d = 0; d < D; ++d) {
          const float acc = odd_values<T, D>(p, sp, b, kvh, node, d);
          if (acc != 0.f) dst[d] = from_f32<T>(to_f32(dst[d]) + acc);
        }
      }
    } while (pc.next(p));
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, 256);
}

// Joins the pieces of the units that more than one part holds.  WPR warps a row
// take every WPR-th piece each: the few units of one long sequence have up to 37
// pieces (narrow trees over 8192 keys; wide ones 18), on which one warp a row would
// wait several round trips long.
template <typename T, int D, int WPR>
__global__ void __launch_bounds__(256) tree_combine_kernel(const __grid_constant__ TreeArgs p) {
  constexpr int PER = D / 32;
  __shared__ float part[WPR > 1 ? 8 : 1][D + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w0 = warp % WPR;
  const int item = blockIdx.x * (8 / WPR) + warp / WPR;
  // which pieces: from the lengths alone, which the kernel before this one
  // only reads
  const bool in = item < p.B * p.Hkv * p.R;
  const int row = item % p.R;
  const int kvh = item / p.R % p.Hkv, b = in ? item / p.R / p.Hkv : 0;
  const Span sp = span_of(p, b);
  int total, longest;
  const int before = tiles_before(p, b, total, longest);
  const Parts s = parts_of(p, total, longest);
  if (s.n == 0) {
    pdl_wait();
    pdl_trigger();
    return;
  }
  const int n = sp.tiles + p.NT;
  const int unit = kvh * p.RT + row / p.rows;
  int c0, c1;
  if (cut_by_unit(p, s, total)) {
    const int k = unit_parts(s, total, n);
    c0 = unit_parts_before(p, s, total, b) + unit * k;
    c1 = c0 + k - 1;
  } else {
    c0 = s.of(before + unit * n);
    c1 = s.of(before + unit * n + n - 1);
  }
  pdl_wait();
  pdl_trigger();
  const bool work = in && c0 != c1;
  const int r = row % p.rows;
  float M = -INFINITY, L = 0.f, odd = 0.f, o[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = 0.f;
  // 32 pieces at a time: a lane takes the weight of one, all take its values
  for (int k0 = c0 + w0; work && k0 <= c1; k0 += 32 * WPR) {
    const int k = k0 + lane * WPR, cnt = min(32, (c1 - k0) / WPR + 1);
    float m = -INFINITY, l = 0.f;
    if (k <= c1) {
      const float* sl = slot_of(p, D, k, k == c0);
      m = sl[p.rows * D + r];
      l = sl[p.rows * (D + 1) + r];
      odd += sl[p.rows * (D + 2)];
    }
    const float mx = fmaxf(M, warp_max(m));
    const float base = mx == -INFINITY ? 0.f : mx;
    const float w = ex2_ftz(m - base), corr = ex2_ftz(M - base);
    M = mx;
    L = L * corr + warp_sum(l * w);
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] *= corr;
#pragma unroll 8
    for (int j = 0; j < cnt; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const int kj = k0 + j * WPR;
      const float* sl = slot_of(p, D, kj, kj == c0) + r * D + lane * PER;
      float v[PER];
      if constexpr (PER == 4) {
        const float4 x = *reinterpret_cast<const float4*>(sl);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(sl);
        v[0] = x.x; v[1] = x.y;
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = fmaf(wj, v[i], o[i]);
    }
  }
  bool any_odd = __any_sync(0xffffffffu, odd != 0.f);
  if (WPR > 1) {  // the row's warps, in order
    if (lane == 0) {
      part[warp][D] = M;
      part[warp][D + 1] = L;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) part[warp][lane * PER + i] = o[i];
    any_odd = __syncthreads_or(any_odd);
    if (w0 != 0) return;
    float mx = M;
    for (int w = 1; w < WPR; ++w) mx = fmaxf(mx, part[warp + w][D]);
    const float base = mx == -INFINITY ? 0.f : mx;
    const float f0 = ex2_ftz(M - base);
    L *= f0;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] *= f0;
    for (int w = 1; w < WPR; ++w) {
      const float f = ex2_ftz(part[warp + w][D] - base);
      L += part[warp + w][D + 1] * f;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] += part[warp + w][lane * PER + i] * f;
    }
  }
  if (!work) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int t = row / p.G, h = kvh * p.G + row % p.G;
  T* dst = static_cast<T*>(p.o) + b * p.o_sb + t * p.o_st + h * p.o_sh + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    o[i] *= inv;
    if (any_odd) o[i] += odd_values<T, D>(p, sp, b, kvh, t, lane * PER + i);
  }
#pragma unroll
  for (int i = 0; i < PER; i += 2)
    *reinterpret_cast<uint32_t*>(dst + i) = pack2<T>(o[i], o[i + 1]);
}

struct TreeCall {
  const void* q; int64_t q_sb, q_st, q_sh;
  const void* k; const void* v; int64_t c_sb, c_sh, c_ss;
  int64_t num_blocks; const int32_t* table; int64_t table_stride;
  const void* kt; int64_t kt_sb, kt_st, kt_sh;
  const void* vt; int64_t vt_sb, vt_st, vt_sh;
  const int32_t* ctx_lens; int64_t max_ctx;
  const uint64_t* mask; int64_t mask_sb;
  void* o; int64_t o_sb, o_st, o_sh;
  int64_t B, T, Hq, Hkv, D, window_left;
  float scale;
  void* ws; int64_t ws_bytes;
};

std::atomic<bool> g_reserved[12][64];  // by kernel

// How a call is cut: the row groups of a CTA (0: tcgen05), a unit's rows and row
// tiles, and the parts at most (0: a CTA takes a unit, whatever the lengths).
struct Plan { int rw, rows, rt, whole_tiles, ctas, grid; };
Plan plan_of(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t max_ctx, int64_t D,
             int64_t window_left) {
  const int64_t R = T * (Hq / Hkv);
  Plan pl;
  const int64_t G = Hq / Hkv;
  // (more than 128 query heads a kv head: no whole node fits a tcgen05 tile)
  pl.rw = R <= 16 ? 1 : R <= 32 || G > kTcRows ? 2 : 0;
  pl.rows = pl.rw ? 16 * pl.rw : (int)(kTcRows / G * G);
  pl.rt = (int)((R + pl.rows - 1) / pl.rows);
  int64_t keys = max_ctx;
  if (window_left >= 0 && window_left < keys - 1) keys = window_left + KT;
  const int64_t tiles = (keys + KT - 1) / KT + (T + 63) / 64;
  const int64_t units = B * Hkv * pl.rt, ctas = 2 * sm_budget();
  // A unit a CTA up to so many tiles (us, whole / cut).  Few units: a narrow tree's 5
  // (4 x 5 nodes over 400 keys, 8 tiles, 12.1 / 10.5), a wide one's 12 (64 nodes over
  // 500 keys, 9 tiles, 15.3 / 18.0; over 2000, 33 tiles, 37.0 / 20.5); 64 units, 16 (8 x
  // 5 over 400 keys 12.1 / 12.8; 16 x 8 over 2000 36.6 / 30.5).  Narrow units that fill
  // most of the slots, 32 (32 x 8 over 2000 keys 43.5 / 46.5; 64 x 4 over ragged lengths
  // up to 4096 140 / 126).  Wide ones, whose pieces cost more, 100 (32 x 32 over 4000 81
  // / 90; 64 x 13 of 32 query heads over ragged lengths up to 4096 146 / 153), but 40 where the last wave of CTAs is nearly empty (48 x 32
  // over 5000 159 / 143; 40 x 32 over 1500 55 / 63) or the keys are narrow (64 x 32 over
  // 6000 keys of 64 dims 156 / 142).
  const bool last_full = units <= ctas || units >= 3 * ctas || units % ctas * 10 >= 7 * ctas;
  if (units < 64) pl.whole_tiles = pl.rw ? 5 : 12;
  else if (2 * units < ctas) pl.whole_tiles = 16;
  else if (pl.rw) pl.whole_tiles = 10 * units >= 8 * ctas ? 32 : 16;
  else pl.whole_tiles = last_full && D == 128 ? 100 : 40;
  pl.ctas = tiles <= pl.whole_tiles ? 0 : (int)std::min<int64_t>(ctas, std::max<int64_t>(units * tiles / 2, 1));
  // (the lengths are on the device: they may turn out short, so each unit has a CTA)
  pl.grid = (int)std::max<int64_t>(units, pl.ctas);
  return pl;
}

// {64 columns, row, column box (D/64), kv head, batch or block}
int kv_map(CUtensorMap* m, const void* base, int dtype, int64_t D, int64_t rows, int64_t heads,
           int64_t outer, int64_t s_row, int64_t s_head, int64_t s_outer) {
  // a dim of one needs a valid stride all the same
  auto st = [&](int64_t n, int64_t s) { return (uint64_t)(n > 1 ? s : D) * 2; };
  const uint64_t dims[5] = {64, (uint64_t)rows, (uint64_t)(D / 64), (uint64_t)heads,
                            (uint64_t)outer};
  const uint64_t strides[4] = {st(rows, s_row), 128, st(heads, s_head), st(outer, s_outer)};
  const uint32_t box[5] = {64, KT, (uint32_t)(D / 64), 1, 1};
  return make_tmap(m, base, dtype, 5, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int64_t workspace_of(const Plan& pl, int64_t D) {
  return pl.ctas ? 2 * pl.ctas * slot_floats(pl.rows, (int)D) * 4 : 0;
}

int tree_attention(TreeCall c, int dtype, cudaStream_t st) {
  if (c.B == 0 || c.T == 0) return TPP_OK;
  if (c.max_ctx == 0 && !c.table) {  // no rows are read: an empty cache has no address
    c.k = c.kt;
    c.v = c.vt;
    c.c_sb = c.c_sh = c.c_ss = c.D;
  }
  // a window that reaches past every row is none (and cannot overflow below)
  if (c.window_left >= c.max_ctx + c.T) c.window_left = -1;
  TPP_REQUIRE(c.q && c.k && c.v && c.kt && c.vt && c.ctx_lens && c.mask && c.o, TPP_ERR_SHAPE,
              "null pointer");
  TPP_REQUIRE(c.B > 0 && c.B <= 65535 && c.T > 0 && c.T <= kMaxNodes && c.Hq > 0 && c.Hkv > 0 &&
                  c.Hq <= 65535 && c.max_ctx >= 0 && c.max_ctx < (1ll << 31) - 2 * KT &&
                  c.num_blocks >= 0 && c.num_blocks < (1ll << 31),
              TPP_ERR_SHAPE, "bad sizes (1..256 nodes, at most 65535 sequences and heads)");
  TPP_REQUIRE(c.Hq % c.Hkv == 0, TPP_ERR_SHAPE, "Hq must be a multiple of Hkv");
  TPP_REQUIRE(c.D == 64 || c.D == 128, TPP_ERR_UNSUPPORTED, "head dim must be 64 or 128");
  TPP_REQUIRE(dtype == TPP_F16 || dtype == TPP_BF16, TPP_ERR_DTYPE,
              "dtype must be f16 (0) or bf16 (1)");
  TPP_REQUIRE(((c.q_sb | c.q_st | c.q_sh | c.kt_sb | c.kt_st | c.kt_sh | c.vt_sb | c.vt_st |
                c.vt_sh) & 7) == 0 &&
                  ((c.o_sb | c.o_st | c.o_sh) & 1) == 0 && aligned16(c.q) && aligned16(c.k) &&
                  aligned16(c.v) && aligned16(c.kt) && aligned16(c.vt) &&
                  (reinterpret_cast<uintptr_t>(c.o) & 3) == 0,
              TPP_ERR_ALIGN, "rows must be 16-byte aligned (the output's: 4-byte)");
  CUtensorMap tk, tv, tkt, tvt;
  const int64_t rows = c.max_ctx > 0 ? c.max_ctx : 1;
  int rc;
  if (c.table) {
    rc = kv_map(&tk, c.k, dtype, c.D, KT, c.Hkv, c.num_blocks, c.D, KT * c.D, c.Hkv * KT * c.D);
    if (rc == TPP_OK)
      rc = kv_map(&tv, c.v, dtype, c.D, KT, c.Hkv, c.num_blocks, c.D, KT * c.D, c.Hkv * KT * c.D);
  } else {
    rc = kv_map(&tk, c.k, dtype, c.D, rows, c.Hkv, c.B, c.c_ss, c.c_sh, c.c_sb);
    if (rc == TPP_OK) rc = kv_map(&tv, c.v, dtype, c.D, rows, c.Hkv, c.B, c.c_ss, c.c_sh, c.c_sb);
  }
  if (rc == TPP_OK) rc = kv_map(&tkt, c.kt, dtype, c.D, c.T, c.Hkv, c.B, c.kt_st, c.kt_sh, c.kt_sb);
  if (rc == TPP_OK) rc = kv_map(&tvt, c.vt, dtype, c.D, c.T, c.Hkv, c.B, c.vt_st, c.vt_sh, c.vt_sb);
  if (rc != TPP_OK) return rc;
  TreeArgs a;
  a.q = c.q; a.q_sb = c.q_sb; a.q_st = c.q_st; a.q_sh = c.q_sh;
  a.v_cache = c.v; a.c_sb = c.c_sb; a.c_sh = c.c_sh; a.c_ss = c.c_ss;
  a.v_tree = c.vt; a.vt_sb = c.vt_sb; a.vt_st = c.vt_st; a.vt_sh = c.vt_sh;
  a.ctx_lens = c.ctx_lens; a.max_ctx = (int)c.max_ctx;
  a.mask = c.mask; a.mask_sb = c.mask_sb;
  a.o = c.o; a.o_sb = c.o_sb; a.o_st = c.o_st; a.o_sh = c.o_sh;
  a.table = c.table; a.table_stride = c.table_stride; a.num_blocks = (int)c.num_blocks;
  a.window_left = c.window_left;
  a.scale_log2 = c.scale * 1.4426950408889634f;
  a.exp_scale = a.scale_log2 > 0.f ? a.scale_log2 : 1.f;
  a.B = (int)c.B; a.T = (int)c.T; a.Hq = (int)c.Hq; a.Hkv = (int)c.Hkv;
  a.G = (int)(c.Hq / c.Hkv); a.W = (a.T + 63) / 64; a.R = a.T * a.G; a.NT = a.W;
  a.err = device_error_flag();
  const Plan pl = plan_of(c.B, c.T, c.Hq, c.Hkv, c.max_ctx, c.D, c.window_left);
  const int rw = pl.rw;
  a.RT = pl.rt; a.ctas = pl.ctas; a.rows = pl.rows;
  a.o_vec = (reinterpret_cast<uintptr_t>(c.o) & 31) == 0 && ((c.o_sb | c.o_st | c.o_sh) & 15) == 0;
  a.whole_tiles = pl.whole_tiles;
  a.by_unit = pl.rw == 0 && 4 * c.B * c.Hkv * pl.rt <= pl.ctas;
  a.ws = static_cast<float*>(c.ws);
  TPP_REQUIRE(pl.ctas == 0 || (c.ws && c.ws_bytes >= workspace_of(pl, c.D) &&
                                (reinterpret_cast<uintptr_t>(c.ws) & 31) == 0),
              TPP_ERR_WORKSPACE, "workspace missing, too small or not 32-byte aligned");
  const int64_t units = c.B * c.Hkv * pl.rt;
  TPP_REQUIRE(units < (1ll << 31) && units * (c.max_ctx / KT + a.NT + 1) < (1ll << 31) &&
                  c.B * c.Hkv * a.R < (1ll << 29) - 8,
              TPP_ERR_SHAPE, "too many rows or tiles");
  const dim3 grid((unsigned)pl.grid);
  CUtensorMap tq;
  if (pl.rw == 0) {
    // {64 columns, head, node, column box, batch}
    auto sb = [&](int64_t n, int64_t s) { return (uint64_t)(n > 1 ? s : c.D) * 2; };
    const uint64_t dims[5] = {64, (uint64_t)c.Hq, (uint64_t)c.T, (uint64_t)(c.D / 64), (uint64_t)c.B};
    const uint64_t strides[4] = {sb(c.Hq, c.q_sh), sb(c.T, c.q_st), 128, sb(c.B, c.q_sb)};
    const uint32_t box[5] = {64, (uint32_t)a.G, (uint32_t)(pl.rows / a.G), 1, 1};
    rc = make_tmap(&tq, c.q, dtype, 5, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != TPP_OK) return rc;
  }
  auto go_tc = [&](auto kern, int id, size_t smem) -> int {
    if (const int e = reserve_smem(reinterpret_cast<const void*>(kern), g_reserved[id], smem,
                                   "tree_attn_tc_kernel"))
      return e;
    return launch("tree_attn_tc_kernel", kern, grid, dim3(kTcThreads), smem, st, 0u, tk, tv, tkt,
                  tvt, tq, a);
  };
  auto go = [&](auto kern, int id, size_t smem) -> int {
    if (const int e = reserve_smem(reinterpret_cast<const void*>(kern), g_reserved[id], smem,
                                   "tree_attn_kernel"))
      return e;
    return launch("tree_attn_kernel", kern, grid, dim3(kThreads), smem, st, 0u, tk, tv, tkt, tvt,
                  a);
  };
  rc = TPP_DISPATCH_HALF(dtype, T, [&]() -> int {
    const int id = 6 * IsBf16<T>::value;
    if (c.D == 64) {
      if (rw == 1) return go(tree_attn_kernel<T, 64, 1>, id, TreeSmem<64, 1>::kBytes);
      if (rw == 2) return go(tree_attn_kernel<T, 64, 2>, id + 1, TreeSmem<64, 2>::kBytes);
      return go_tc(tree_attn_tc_kernel<T, 64>, id + 2, TcSmem<64>::kBytes);
    }
    if (rw == 1) return go(tree_attn_kernel<T, 128, 1>, id + 3, TreeSmem<128, 1>::kBytes);
    if (rw == 2) return go(tree_attn_kernel<T, 128, 2>, id + 4, TreeSmem<128, 2>::kBytes);
    return go_tc(tree_attn_tc_kernel<T, 128>, id + 5, TcSmem<128>::kBytes);
  });
  if (rc != TPP_OK || pl.ctas == 0) return rc;
  const int wpr = pl.ctas >= 4 * units ? 4 : 1;  // four pieces a unit and more
  const int64_t blocks = (c.B * c.Hkv * a.R * wpr + 7) / 8;
  return TPP_DISPATCH_HALF(dtype, T, [&]() -> int {
    auto kern = c.D == 64 ? (wpr == 4 ? tree_combine_kernel<T, 64, 4> : tree_combine_kernel<T, 64, 1>)
                          : (wpr == 4 ? tree_combine_kernel<T, 128, 4> : tree_combine_kernel<T, 128, 1>);
    return launch("tree_combine_kernel", kern, dim3((unsigned)blocks), dim3(256), 0, st, 0u, a);
  });
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int64_t tpp_attention_tree_workspace(int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                                                int64_t max_ctx, int64_t D,
                                                int64_t window_left) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || max_ctx < 0) return 0;
  return workspace_of(plan_of(B, T, Hq, Hkv, max_ctx, D, window_left), D);
}

extern "C" int tpp_attention_tree(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                  const void* k_cache, const void* v_cache, int64_t c_sb,
                                  int64_t c_sh, int64_t c_ss, const void* k_tree, int64_t kt_sb,
                                  int64_t kt_st, int64_t kt_sh, const void* v_tree,
                                  int64_t vt_sb, int64_t vt_st, int64_t vt_sh,
                                  const int32_t* ctx_lens, int64_t max_ctx, const uint64_t* mask,
                                  int64_t mask_sb, void* o, int64_t o_sb, int64_t o_st,
                                  int64_t o_sh, int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                                  int64_t D, int64_t window_left, float scale, void* workspace,
                                  int64_t workspace_bytes, int dtype, void* stream) {
  TPP_REQUIRE(((c_sb | c_sh | c_ss) & 7) == 0, TPP_ERR_ALIGN,
              "cache strides must be multiples of 8 elements");
  const TreeCall c{q, q_sb, q_st, q_sh, k_cache, v_cache, c_sb, c_sh, c_ss, 0, nullptr, 0,
                   k_tree, kt_sb, kt_st, kt_sh, v_tree, vt_sb, vt_st, vt_sh, ctx_lens, max_ctx,
                   mask, mask_sb, o, o_sb, o_st, o_sh, B, T, Hq, Hkv, D, window_left, scale,
                   workspace, workspace_bytes};
  return tree_attention(c, dtype, as_stream(stream));
}

extern "C" int tpp_attention_tree_paged(
    const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k_pool,
    const void* v_pool, int64_t num_blocks, const int32_t* block_table, int64_t table_stride,
    const void* k_tree, int64_t kt_sb, int64_t kt_st, int64_t kt_sh, const void* v_tree,
    int64_t vt_sb, int64_t vt_st, int64_t vt_sh, const int32_t* ctx_lens, int64_t max_ctx,
    const uint64_t* mask, int64_t mask_sb, void* o, int64_t o_sb, int64_t o_st, int64_t o_sh,
    int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window_left, float scale,
    void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  TPP_REQUIRE(block_table != nullptr && num_blocks > 0, TPP_ERR_SHAPE,
              "null block table or empty pools");
  const TreeCall c{q, q_sb, q_st, q_sh, k_pool, v_pool, 0, 0, 0, num_blocks, block_table,
                   table_stride, k_tree, kt_sb, kt_st, kt_sh, v_tree, vt_sb, vt_st, vt_sh,
                   ctx_lens, max_ctx, mask, mask_sb, o, o_sb, o_st, o_sh, B, T, Hq, Hkv, D,
                   window_left, scale, workspace, workspace_bytes};
  return tree_attention(c, dtype, as_stream(stream));
}
