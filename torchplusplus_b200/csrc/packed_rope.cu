// q/k RMSNorm + RoPE of prompts packed into one row dimension, each row at its
// own position in its sequence, with the K and V rows written into the cache.
#include "common.cuh"

namespace tpp {
namespace {

template <typename CS>
__device__ __forceinline__ void table8(const CS* p, float* f) {
  unpack8<CS>(__ldg(reinterpret_cast<const uint4*>(p)), f);
}
template <>
__device__ __forceinline__ void table8<float>(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

struct PackedRopeArgs {
  const void* qkv; int64_t qkv_sn;
  const void* qn; const void* kn; float eps;
  const void* cosp; const void* sinp; int64_t cs_stride, table_rows;
  const int32_t* cu; int B;
  void* q_out; void* k_out;
  void* k_cache; void* v_cache;
  int64_t c_sb, c_sh, c_ss, rows, num_blocks;
  const int32_t* table; int64_t table_stride;
  uint32_t units;
  int Hq, Hkv;
};

constexpr int kBlock = 128;  // (blocks are short: 96 threads 216 us where 128 take 211, 256: 238, 512: 252)

// y = rope(x * rsqrt(mean(x^2) + eps) * w): a unit is R head rows of one kind (q, k
// or, with a cache, v) of one token.  G = D/16 lanes own it, lane l elements
// [8l, 8l+8) of both halves of each row, so rotate-half stays inside a lane and only
// the sum of squares crosses lanes; the norm's weight is folded into the lane's cos and
// sin once for all R rows.  fp32 throughout, one rounding at the store.  Bound by HBM
// at many tokens (R rows' loads in flight a lane), by latency at few (R = 1).  Measured, bf16,
// D 128: 64 prompts to 1024, 32 + 2 x 8 heads into a paged cache 211 us, 5.8 TB/s, 88 % of a
// copy's rate (R = 2: 236, 8: 224); one of 130, 16 + 2 x 8 heads: 4.3 us.
template <typename T, typename CS, int G, int R>
__global__ void __launch_bounds__(kBlock) qk_norm_rope_packed_kernel(PackedRopeArgs p) {
  pdl_wait();
  pdl_trigger();
  constexpr int D = G * 16;
  const uint32_t unit = blockIdx.x * (kBlock / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  const bool valid = unit < p.units;  // (lanes past the end take part in the shuffles)
  const int gq = (p.Hq + R - 1) / R, gk = (p.Hkv + R - 1) / R;
  const uint32_t per = gq + (p.k_cache ? 2 : 1) * gk;
  const uint32_t tok = valid ? unit / per : 0;
  int grp = valid ? (int)(unit - tok * per) : 0;
  const int kind = grp < gq ? 0 : grp < gq + gk ? 1 : 2;  // q, k, v
  grp -= kind == 0 ? 0 : kind == 1 ? gq : gq + gk;
  const int heads = kind == 0 ? p.Hq : p.Hkv, h0 = grp * R;
  const T* src = static_cast<const T*>(p.qkv) + (int64_t)tok * p.qkv_sn + lane * 8 +
                 (int64_t)(kind == 0 ? 0 : kind == 1 ? p.Hq : p.Hq + p.Hkv) * D;
  uint4 lo[R], hi[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const T* r = src + (int64_t)min(h0 + i, heads - 1) * D;
    lo[i] = ldg_nc_v4(r);
    hi[i] = ldg_nc_v4(r + D / 2);
  }
  // the token's sequence: the first whose end lies behind it
  int b = 0;
  for (int end = p.B; b < end;) {
    const int mid = (b + end) >> 1;
    if (__ldg(p.cu + mid + 1) <= (int64_t)tok) b = mid + 1;
    else end = mid;
  }
  const int64_t first = b < p.B ? __ldg(p.cu + b) : (int64_t)tok + 1;
  const int64_t pos = (int64_t)tok - first;
  const bool mine = valid && pos >= 0 && first >= 0;  // rows of no sequence stay as they are
  T* cache = nullptr;  // this lane's words of the row of head 0
  int64_t c_sh = p.c_sh;
  if (mine && kind != 0 && p.k_cache != nullptr && pos < p.rows) {
    T* base = static_cast<T*>(kind == 1 ? p.k_cache : p.v_cache) + lane * 8;
    if (p.table != nullptr) {
      const int64_t blk = p.table[b * p.table_stride + pos / 64];
      c_sh = 64 * D;
      if (blk >= 0 && blk < p.num_blocks) cache = base + blk * p.Hkv * c_sh + (pos % 64) * D;
    } else {
      cache = base + b * p.c_sb + pos * p.c_ss;
    }
  }
  if (kind == 2) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (cache == nullptr || h0 + i >= heads) break;
      T* dst = cache + (int64_t)(h0 + i) * c_sh;
      *reinterpret_cast<uint4*>(dst) = lo[i];
      *reinterpret_cast<uint4*>(dst + D / 2) = hi[i];
    }
  }
  // y_lo = inv (x_lo a - x_hi b), y_hi = inv (x_hi c + x_lo d)
  const bool known = mine && pos < p.table_rows;  // beyond the tables: zero rows
  float a[8], bb[8], c[8], d[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = bb[j] = c[j] = d[j] = 0.f;
  if (known && kind != 2) {
    const CS* cs = static_cast<const CS*>(p.cosp) + pos * p.cs_stride + lane * 8;
    const CS* sn = static_cast<const CS*>(p.sinp) + pos * p.cs_stride + lane * 8;
    table8<CS>(cs, a);
    table8<CS>(sn, bb);
    table8<CS>(cs + D / 2, c);
    table8<CS>(sn + D / 2, d);
  }
  const T* nw = static_cast<const T*>(kind == 0 ? p.qn : p.kn);
  if (nw != nullptr) {
    float g1[8], g2[8];
    unpack8<T>(__ldg(reinterpret_cast<const uint4*>(nw + lane * 8)), g1);
    unpack8<T>(__ldg(reinterpret_cast<const uint4*>(nw + D / 2 + lane * 8)), g2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      a[j] *= g1[j];
      bb[j] *= g2[j];
      c[j] *= g2[j];
      d[j] *= g1[j];
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float x[8], y[8];
    if (!known) lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
    unpack8<T>(lo[i], x);
    unpack8<T>(hi[i], y);
    float inv = 1.f;
    {
      // (a warp's units are of several kinds, of which only one may have a norm: every lane takes
      // part in the shuffles, whatever its own; a branch round all of it took 122 registers
      // for 96, and 228 us for 213)
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s0 = fmaf(x[j], x[j], s0);
        s1 = fmaf(y[j], y[j], s1);
      }
      s0 += s1;
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      if (nw != nullptr) inv = known ? rsqrtf(s0 / (float)D + p.eps) : 0.f;  // (eps may be 0)
    }
    float u[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = inv * fmaf(-y[j], bb[j], x[j] * a[j]);
      v[j] = inv * fmaf(x[j], d[j], y[j] * c[j]);
    }
    if (!mine || kind == 2 || h0 + i >= heads) continue;
    T* dst = static_cast<T*>(kind == 0 ? p.q_out : p.k_out) +
             ((int64_t)tok * heads + h0 + i) * D + lane * 8;
    const uint4 w0 = pack8<T>(u), w1 = pack8<T>(v);
    *reinterpret_cast<uint4*>(dst) = w0;
    *reinterpret_cast<uint4*>(dst + D / 2) = w1;
    if (cache != nullptr) {
      T* cd = cache + (int64_t)(h0 + i) * c_sh;
      *reinterpret_cast<uint4*>(cd) = w0;
      *reinterpret_cast<uint4*>(cd + D / 2) = w1;
    }
  }
}

template <typename T, typename CS>
int packed_rope_launch(PackedRopeArgs a, int64_t N, int64_t D, cudaStream_t st) {
  auto go = [&](auto tag) -> int {
    constexpr int G = decltype(tag)::value;
    const int64_t kv = a.k_cache ? 2 : 1;
    // four rows a unit from where they fill the SMs' threads (148 * 2048) on
    const bool four = N * (a.Hq + kv * a.Hkv) * G >= 4 * 2048 * (int64_t)num_sms();
    const int r = four ? 4 : 1;
    const int64_t units = N * ((a.Hq + r - 1) / r + kv * ((a.Hkv + r - 1) / r));
    TPP_REQUIRE(units < (1ll << 31), TPP_ERR_SHAPE, "too many rows");
    a.units = (uint32_t)units;
    return launch("qk_norm_rope_packed_kernel",
                  four ? qk_norm_rope_packed_kernel<T, CS, G, 4>
                       : qk_norm_rope_packed_kernel<T, CS, G, 1>,
                  dim3((unsigned)((units + kBlock / G - 1) / (kBlock / G))), dim3(kBlock), 0, st, 0u, a);
  };
  switch (D) {
    case 16: return go(std::integral_constant<int, 1>{});
    case 32: return go(std::integral_constant<int, 2>{});
    case 64: return go(std::integral_constant<int, 4>{});
    case 128: return go(std::integral_constant<int, 8>{});
    case 256: return go(std::integral_constant<int, 16>{});
    default:
      set_error("tpp_qk_norm_rope_packed: head dim must be 16, 32, 64, 128 or 256");
      return TPP_ERR_UNSUPPORTED;
  }
}

}  // namespace
}  // namespace tpp

using namespace tpp;

extern "C" int tpp_qk_norm_rope_packed(const void* qkv, int64_t qkv_sn, const void* qn_w,
                                       const void* kn_w, float eps, const void* cos,
                                       const void* sin, int64_t cs_stride, int64_t table_rows,
                                       int cs_dtype, const int32_t* cu_seqlens, int64_t B,
                                       void* q_out, void* k_out, void* k_cache, void* v_cache,
                                       int64_t c_sb, int64_t c_sh, int64_t c_ss, int64_t rows,
                                       int64_t num_blocks, const int32_t* block_table,
                                       int64_t table_stride, int64_t N, int64_t Hq, int64_t Hkv,
                                       int64_t D, int dtype, void* stream) {
  if (N == 0 || B == 0) return TPP_OK;
  TPP_REQUIRE(qkv && cos && sin && cu_seqlens && q_out && k_out, TPP_ERR_SHAPE, "null pointer");
  TPP_REQUIRE((k_cache == nullptr) == (v_cache == nullptr), TPP_ERR_SHAPE,
              "k_cache and v_cache go together");
  TPP_REQUIRE(N > 0 && N < (1ll << 31) && B > 0 && B < (1ll << 31) && Hq > 0 && Hkv > 0 &&
                  Hq + Hkv < (1ll << 31) && D > 0 && table_rows >= 0 && rows >= 0 &&
                  num_blocks >= 0,
              TPP_ERR_SHAPE, "bad sizes");
  TPP_REQUIRE(((qkv_sn | cs_stride | c_sb | c_sh | c_ss) & 7) == 0, TPP_ERR_ALIGN,
              "row strides must be multiples of 8 elements");
  TPP_REQUIRE(aligned16(qkv) && aligned16(q_out) && aligned16(k_out) && aligned16(cos) &&
                  aligned16(sin) && aligned16(qn_w) && aligned16(kn_w) && aligned16(k_cache) &&
                  aligned16(v_cache),
              TPP_ERR_ALIGN, "pointers must be 16-byte aligned");
  const PackedRopeArgs a{qkv, qkv_sn, qn_w, kn_w, eps, cos, sin, cs_stride, table_rows,
                         cu_seqlens, (int)B, q_out, k_out, k_cache, v_cache, c_sb, c_sh, c_ss,
                         rows, num_blocks, block_table, table_stride, 0u, (int)Hq, (int)Hkv};
  return TPP_DISPATCH_HALF(dtype, T_, [&] {
    switch (cs_dtype) {
      case TPP_F16: return packed_rope_launch<T_, __half>(a, N, D, as_stream(stream));
      case TPP_BF16: return packed_rope_launch<T_, __nv_bfloat16>(a, N, D, as_stream(stream));
      case TPP_F32: return packed_rope_launch<T_, float>(a, N, D, as_stream(stream));
      default:
        set_error("tpp_qk_norm_rope_packed: cos/sin dtype must be f16, bf16 or f32");
        return (int)TPP_ERR_DTYPE;
    }
  });
}
