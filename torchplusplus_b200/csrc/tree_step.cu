// The two bandwidth kernels of a draft-tree step: q/k RMSNorm + RoPE at each
// node's own position, and the copy of the accepted path's K/V rows of every
// layer into the cache.
#include "common.cuh"

namespace tpp {
namespace {

template <typename CS>
__device__ __forceinline__ void load_table8(const CS* p, float* f) {
  unpack8<CS>(__ldg(reinterpret_cast<const uint4*>(p)), f);
}
template <>
__device__ __forceinline__ void load_table8<float>(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

struct RopeTreeArgs {
  const void* qkv; int64_t qkv_sb, qkv_st;
  const void* qn; const void* kn; float eps;
  const void* cosp; const void* sinp; int64_t cs_stride, table_rows;
  const int32_t* positions;
  void* q_out; void* k_out;
  int64_t tokens;  // B * T
  int T, Hq, Hkv;
};

// y = rope(x * rsqrt(mean(x^2) + eps) * w) of a token's head rows: a group of G =
// D/8 lanes owns HPG head rows of one token, lane l elements [8l, 8l+8) of each; the
// rotate-half partner chunk lives in lane l ^ (G/2).  fp32 throughout, one rounding
// at the store.  Bound by HBM at many tokens, so a group keeps the loads of HPG rows
// in flight and takes the token's table rows and the norm weights once for all of
// them; at few tokens by latency, where HPG = 1 spreads the rows.
template <typename T, typename CS, int G, int HPG>
__global__ void __launch_bounds__(256) qk_norm_rope_tree_kernel(RopeTreeArgs p) {
  pdl_wait();
  pdl_trigger();
  constexpr int D = G * 8;
  const int heads = p.Hq + p.Hkv, per = (heads + HPG - 1) / HPG;
  const int64_t item = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  const bool valid = item < p.tokens * per;  // (lanes past the end take part in the shuffles)
  const int64_t tok = valid ? item / per : 0;
  const int h0 = valid ? (int)(item - tok * per) * HPG : 0;
  const int64_t b = tok / p.T, t = tok - b * p.T;
  const T* row = static_cast<const T*>(p.qkv) + b * p.qkv_sb + t * p.qkv_st + lane * 8;
  uint4 raw[HPG];
#pragma unroll
  for (int i = 0; i < HPG; ++i) raw[i] = ldg_nc_v4(row + (int64_t)min(h0 + i, heads - 1) * D);
  const int64_t pos = p.positions[tok];
  // a position outside the tables: zero rows, from zero inputs
  const bool known = pos >= 0 && pos < p.table_rows;
  float c8[8], s8[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c8[j] = s8[j] = 0.f;
  if (known) {
    load_table8<CS>(static_cast<const CS*>(p.cosp) + pos * p.cs_stride + lane * 8, c8);
    load_table8<CS>(static_cast<const CS*>(p.sinp) + pos * p.cs_stride + lane * 8, s8);
#pragma unroll
    for (int j = 0; j < 8; ++j) s8[j] = lane < G / 2 ? -s8[j] : s8[j];
  } else {
#pragma unroll
    for (int i = 0; i < HPG; ++i) raw[i] = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const int h = min(h0 + i, heads - 1);
    const bool is_q = h < p.Hq;
    float v[8];
    unpack8<T>(raw[i], v);
    const void* nw = is_q ? p.qn : p.kn;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += v[j] * v[j];
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (nw != nullptr) {
      const float inv = known ? rsqrtf(ss / (float)D + p.eps) : 0.f;  // (eps may be 0)
      float g[8];
      unpack8<T>(__ldg(static_cast<const uint4*>(nw) + lane), g);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] * inv * g[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float r = __shfl_xor_sync(0xffffffffu, v[j], G / 2);
      v[j] = fmaf(v[j], c8[j], r * s8[j]);
    }
    if (valid && h0 + i < heads) {
      T* dst = is_q ? static_cast<T*>(p.q_out) + (tok * p.Hq + h) * D
                    : static_cast<T*>(p.k_out) + (tok * p.Hkv + h - p.Hq) * D;
      *reinterpret_cast<uint4*>(dst + lane * 8) = pack8<T>(v);
    }
  }
}

template <typename T, typename CS>
int rope_tree_launch(const RopeTreeArgs& a, int64_t D, cudaStream_t st) {
  auto go = [&](auto tag) -> int {
    constexpr int G = decltype(tag)::value;
    // four rows a group from where they fill the SMs' threads (148 * 2048) on
    const int64_t heads = a.Hq + a.Hkv;
    const int hpg = a.tokens * heads * G >= 4 * 2048 * (int64_t)num_sms() ? 4 : 1;
    const int64_t grid = (a.tokens * ((heads + hpg - 1) / hpg) + 256 / G - 1) / (256 / G);
    TPP_REQUIRE(grid < (1ll << 31), TPP_ERR_SHAPE, "too many rows");
    return launch("qk_norm_rope_tree_kernel",
                  hpg == 4 ? qk_norm_rope_tree_kernel<T, CS, G, 4>
                           : qk_norm_rope_tree_kernel<T, CS, G, 1>,
                  dim3((unsigned)grid), dim3(256), 0, st, 0u, a);
  };
  switch (D) {
    case 16: return go(std::integral_constant<int, 2>{});
    case 32: return go(std::integral_constant<int, 4>{});
    case 64: return go(std::integral_constant<int, 8>{});
    case 128: return go(std::integral_constant<int, 16>{});
    case 256: return go(std::integral_constant<int, 32>{});
    default:
      set_error("tpp_qk_norm_rope_tree: head dim must be 16, 32, 64, 128 or 256");
      return TPP_ERR_UNSUPPORTED;
  }
}

constexpr int kMaxPath = 256;

struct CommitArgs {
  const uint4* src[2];                       // k, v trees
  int64_t s_sl[2], s_sb[2], s_st[2], s_sh[2];  // in 16-byte words
  uint4* dst[2];
  int64_t c_sl, c_sb, c_sh, c_ss;            // in 16-byte words
  int64_t rows, num_blocks;
  const int32_t* path; int64_t path_sb;
  const int32_t* count;
  const int32_t* ctx_lens;
  const int32_t* table; int64_t table_stride;
  int B, T, Hkv, words;                      // words: 16-byte words of a row
};

// One block copies the rows of one (layer, sequence, k or v), four words a thread
// in flight.  One sequence: 2.2 us, the latency of the chain count -> path -> row ->
// store.  28 layers of 64 sequences, 4.5 rows each: 15.9 us, 4.15 TB/s (64% of a
// copy's), issue slots 64% busy: two divisions a word, four dependent loads a block, the
// destination's rows of 256 bytes 16 KB apart; their shares are not known.  (Four layers a
// block, so that all blocks start at once, 17.3; a thread for each word of a row
// instead of divisions, 16.9.)
__global__ void __launch_bounds__(256) kv_commit_kernel(CommitArgs p) {
  constexpr int U = 4;
  pdl_wait();
  pdl_trigger();
  const int l = blockIdx.x / p.B, b = blockIdx.x - l * p.B;
  const int kv = blockIdx.y;
  __shared__ int64_t from[kMaxPath], to[kMaxPath];  // words, of head 0
  const int n = min(p.count[b], p.T);
  const int64_t ctx = p.ctx_lens[b];
  const uint4* src = p.src[kv] + l * p.s_sl[kv] + b * p.s_sb[kv];
  uint4* dst = p.dst[kv] + l * p.c_sl + (p.table ? 0 : b * p.c_sb);
  const int per = p.Hkv * p.words;
  const int64_t head = p.table ? 64 * p.words : p.c_sh;
  for (int i0 = 0; i0 < n; i0 += kMaxPath) {
    const int m = min(kMaxPath, n - i0);
    if (i0 > 0) __syncthreads();
    for (int i = threadIdx.x; i < m; i += blockDim.x) {
      const int node = p.path[b * p.path_sb + i0 + i];
      const int64_t row = ctx + i0 + i;
      int64_t at = -1;
      if (node >= 0 && node < p.T && row >= 0 && row < p.rows) {
        if (p.table) {
          const int64_t blk = p.table[b * p.table_stride + row / 64];
          if (blk >= 0 && blk < p.num_blocks) at = (blk * p.Hkv * 64 + row % 64) * p.words;
        } else {
          at = row * p.c_ss;
        }
      }
      from[i] = node * p.s_st[kv];
      to[i] = at;
    }
    __syncthreads();
    for (int e0 = threadIdx.x; e0 < m * per; e0 += U * blockDim.x) {
      uint4 x[U];
      int64_t at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = e0 + u * blockDim.x;
        at[u] = -1;
        if (e >= m * per) continue;
        const int i = e / per, r = e - i * per;
        const int h = r / p.words, w = r - h * p.words;
        if (to[i] < 0) continue;
        at[u] = to[i] + h * head + w;
        x[u] = src[from[i] + h * p.s_sh[kv] + w];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (at[u] >= 0) dst[at[u]] = x[u];
    }
  }
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int tpp_qk_norm_rope_tree(const void* qkv, int64_t qkv_sb, int64_t qkv_st,
                                     const void* qn_w, const void* kn_w, float eps,
                                     const void* cos, const void* sin, int64_t cs_stride,
                                     int64_t table_rows, int cs_dtype, const int32_t* positions,
                                     void* q_out, void* k_out, int64_t B, int64_t T, int64_t Hq,
                                     int64_t Hkv, int64_t D, int dtype, void* stream) {
  if (B == 0 || T == 0) return TPP_OK;
  TPP_REQUIRE(qkv && cos && sin && positions && q_out && k_out, TPP_ERR_SHAPE, "null pointer");
  TPP_REQUIRE(B > 0 && T > 0 && Hq > 0 && Hkv > 0 && D > 0 && table_rows >= 0 &&
                  T < (1ll << 31) && Hq + Hkv < (1ll << 31),
              TPP_ERR_SHAPE, "bad sizes");
  TPP_REQUIRE(qkv_sb % 8 == 0 && qkv_st % 8 == 0 && cs_stride % 8 == 0, TPP_ERR_ALIGN,
              "row strides must be multiples of 8 elements");
  TPP_REQUIRE(aligned16(qkv) && aligned16(q_out) && aligned16(k_out) && aligned16(cos) &&
                  aligned16(sin) && aligned16(qn_w) && aligned16(kn_w),
              TPP_ERR_ALIGN, "pointers must be 16-byte aligned");
  const RopeTreeArgs a{qkv, qkv_sb, qkv_st, qn_w, kn_w, eps, cos, sin, cs_stride, table_rows,
                       positions, q_out, k_out, B * T, (int)T, (int)Hq, (int)Hkv};
  return TPP_DISPATCH_HALF(dtype, T_, [&] {
    switch (cs_dtype) {
      case TPP_F16: return rope_tree_launch<T_, __half>(a, D, as_stream(stream));
      case TPP_BF16: return rope_tree_launch<T_, __nv_bfloat16>(a, D, as_stream(stream));
      case TPP_F32: return rope_tree_launch<T_, float>(a, D, as_stream(stream));
      default:
        set_error("tpp_qk_norm_rope_tree: cos/sin dtype must be f16, bf16 or f32");
        return (int)TPP_ERR_DTYPE;
    }
  });
}

extern "C" int tpp_kv_commit(const void* k_tree, int64_t kt_sl, int64_t kt_sb, int64_t kt_st,
                             int64_t kt_sh, const void* v_tree, int64_t vt_sl, int64_t vt_sb,
                             int64_t vt_st, int64_t vt_sh, const int32_t* path, int64_t path_sb,
                             const int32_t* count, const int32_t* ctx_lens, void* k_cache,
                             void* v_cache, int64_t c_sl, int64_t c_sb, int64_t c_sh,
                             int64_t c_ss, int64_t rows, int64_t num_blocks,
                             const int32_t* block_table, int64_t table_stride, int64_t L,
                             int64_t B, int64_t T, int64_t Hkv, int64_t D, int dtype,
                             void* stream) {
  if (L == 0 || B == 0 || T == 0) return TPP_OK;
  TPP_REQUIRE(k_tree && v_tree && path && count && ctx_lens && k_cache && v_cache, TPP_ERR_SHAPE,
              "null pointer");
  TPP_REQUIRE(L > 0 && B > 0 && T > 0 && Hkv > 0 && D > 0 && rows >= 0 && num_blocks >= 0,
              TPP_ERR_SHAPE, "bad sizes");
  TPP_REQUIRE(L * B < (1ll << 31) && T * Hkv * D < (1ll << 31), TPP_ERR_SHAPE, "too many rows");
  TPP_REQUIRE(dtype == TPP_F16 || dtype == TPP_BF16, TPP_ERR_DTYPE,
              "dtype must be f16 (0) or bf16 (1)");
  TPP_REQUIRE(D % 8 == 0 && ((kt_sl | kt_sb | kt_st | kt_sh | vt_sl | vt_sb | vt_st | vt_sh |
                              c_sl | c_sb | c_sh | c_ss) & 7) == 0 &&
                  aligned16(k_tree) && aligned16(v_tree) && aligned16(k_cache) &&
                  aligned16(v_cache),
              TPP_ERR_ALIGN, "rows must be 16-byte aligned and D a multiple of 8");
  CommitArgs a;
  a.src[0] = static_cast<const uint4*>(k_tree);
  a.src[1] = static_cast<const uint4*>(v_tree);
  a.s_sl[0] = kt_sl / 8; a.s_sb[0] = kt_sb / 8; a.s_st[0] = kt_st / 8; a.s_sh[0] = kt_sh / 8;
  a.s_sl[1] = vt_sl / 8; a.s_sb[1] = vt_sb / 8; a.s_st[1] = vt_st / 8; a.s_sh[1] = vt_sh / 8;
  a.dst[0] = static_cast<uint4*>(k_cache);
  a.dst[1] = static_cast<uint4*>(v_cache);
  a.c_sl = c_sl / 8; a.c_sb = c_sb / 8; a.c_sh = c_sh / 8; a.c_ss = c_ss / 8;
  a.rows = rows; a.num_blocks = num_blocks;
  a.path = path; a.path_sb = path_sb; a.count = count; a.ctx_lens = ctx_lens;
  a.table = block_table; a.table_stride = table_stride;
  a.B = (int)B; a.T = (int)T; a.Hkv = (int)Hkv; a.words = (int)(D / 8);
  return launch("kv_commit_kernel", kv_commit_kernel, dim3((unsigned)(L * B), 2), dim3(256), 0,
                as_stream(stream), 0u, a);
}
