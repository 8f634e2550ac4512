// Norms of queries and keys head by head with their rotation, and the write into the KV cache, in one pass over the rows
// of a fused qkv projection.
//
//   y = x rsqrt(mean(x^2) + eps) w,   out_j = y_j cos_j - y_{j + D/2} sin_j,   out_{j + D/2} = y_{j + D/2} cos_{j + D/2} +
//   y_j sin_{j + D/2},   j < D / 2
//
// for every query and key head (w: a weight of the D dims for all query heads, one for all key heads); values are copied.
// Everything is fp32 until the one rounding of the result: the norm's and the rotation's intermediate roundings of
// lsk_rmsnorm and lsk_rope_append (the reference's, whose models have no such norms) would only add error here.
#include "lsk_common.h"
#include "../include/lsk.h"

namespace {

template <typename T>
struct NormRopeArgs {
  const T* qkv;           // rows of [(Hq + 2 Hkv) D] elements, `ld` apart
  long ld;
  const T *wq, *wk;
  float eps;
  const float *cos_tab, *sin_tab;
  int tab_len;
  const int32_t *rows, *pos;
  T *q_out, *k_out;       // [N, Hq, D], [N, Hkv, D] (NULL: K and V go into the caches)
  T *kc, *vc;
  int N, Hq, Hkv, max_batch, max_seq;
};

// N consecutive elements at any address that aligns one of them, at most 16 bytes a load or store
template <int N>
__device__ __forceinline__ void load_f(const uint16_t* p, float* x) {
  constexpr int W = N < 8 ? N : 8;
  typedef uint16_t V __attribute__((ext_vector_type(W), aligned(2)));
#pragma unroll
  for (int i = 0; i < N; i += W) {
    const V v = *(const V*)(p + i);
#pragma unroll
    for (int j = 0; j < W; ++j) x[i + j] = bf2f(v[j]);
  }
}
template <int N>
__device__ __forceinline__ void load_f(const float* p, float* x) {
  constexpr int W = N < 4 ? N : 4;
  typedef float V __attribute__((ext_vector_type(W), aligned(4)));
#pragma unroll
  for (int i = 0; i < N; i += W) {
    const V v = *(const V*)(p + i);
#pragma unroll
    for (int j = 0; j < W; ++j) x[i + j] = v[j];
  }
}
template <int N>
__device__ __forceinline__ void store_f(uint16_t* p, const float* x) {
  constexpr int W = N < 8 ? N : 8;
  typedef uint16_t V __attribute__((ext_vector_type(W), aligned(2)));
  typedef __bf16 B __attribute__((ext_vector_type(W)));
#pragma unroll
  for (int i = 0; i < N; i += W) {
    B v;
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = (__bf16)x[i + j];
    *(V*)(p + i) = __builtin_bit_cast(V, v);
  }
}
template <int N>
__device__ __forceinline__ void store_f(float* p, const float* x) {
  constexpr int W = N < 4 ? N : 4;
  typedef float V __attribute__((ext_vector_type(W), aligned(4)));
#pragma unroll
  for (int i = 0; i < N; i += W) {
    V v;
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = x[i + j];
    *(V*)(p + i) = v;
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, false));
}
// the sum over 16 lanes, in each of them
__device__ __forceinline__ float row_sum(float x) {
  x += dpp<0x128>(x);                                // row_ror:8, 4, 2, 1
  x += dpp<0x124>(x);
  x += dpp<0x122>(x);
  x += dpp<0x121>(x);
  return x;
}

}  // namespace

#define NORM_ROPE_THREADS 256
#define NORM_ROPE_HEADS (NORM_ROPE_THREADS / 16)  // heads of a pass
#define NORM_ROPE_TOKENS 32                       // tokens of a workgroup of values

// The values of up to 32 tokens of one KV head.  The cache holds a dim's 32 positions of a block side by side: a run of
// positions of one cache row (a prompt's tokens) is turned in LDS and written in 16-byte pieces where they are whole;
// other tokens element by element, lanes side by side over the tokens.
template <typename T, int D>
__device__ __forceinline__ void norm_rope_values(const NormRopeArgs<T>& A, int t0, int h) {
  constexpr int NT = NORM_ROPE_TOKENS, PP = 16 / (int)sizeof(T), SLOTS = NT + PP;
  constexpr int LD = SLOTS + 4 / (int)sizeof(T);     // (an odd number of dwords)
  typedef T Piece __attribute__((ext_vector_type(PP)));
  __shared__ __attribute__((aligned(16))) T s_v[D * LD];
  const int nt = min(NT, A.N - t0), tid = threadIdx.x, l = tid & 31;
  const T* x = A.qkv + (long)t0 * A.ld + (long)(A.Hq + A.Hkv + h) * D;
  const int i = min(l, nt - 1), r = A.rows[t0 + i], p = A.pos[t0 + i];
  const int r0 = __shfl(r, 0, 32), p0 = __shfl(p, 0, 32);
  const bool ok = r >= 0 && r < A.max_batch && p >= 0 && p < A.max_seq && p < A.tab_len;
  const bool run = __builtin_amdgcn_ballot_w64(ok && r == r0 && (uint32_t)p - (uint32_t)p0 == (uint32_t)i) == ~0ull;
  const int sh = run ? p0 % PP : 0;                  // the tile's first token stands at sh
  if constexpr (sizeof(T) == 2) {                    // two slots at a time
    constexpr int CH = D / 8;
    for (int e = tid; e < (sh + nt + 1) / 2 * CH; e += NORM_ROPE_THREADS) {
      const int u = e / CH, d = 8 * (e - u * CH), t = 2 * u - sh;
      const lsk_u32x4_u lo = *(const lsk_u32x4_u*)(x + (long)min(max(t, 0), nt - 1) * A.ld + d);
      const lsk_u32x4_u hi = *(const lsk_u32x4_u*)(x + (long)min(max(t + 1, 0), nt - 1) * A.ld + d);
      uint32_t* to = (uint32_t*)(s_v + d * LD) + u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        to[(2 * j) * (LD / 2)] = __builtin_amdgcn_perm(hi[j], lo[j], 0x05040100);
        to[(2 * j + 1) * (LD / 2)] = __builtin_amdgcn_perm(hi[j], lo[j], 0x07060302);
      }
    }
  } else {
    for (int e = tid; e < nt * (D / 4); e += NORM_ROPE_THREADS) {
      const int t = e / (D / 4), d = 4 * (e - t * (D / 4));
      const lsk_f32x4_u v = *(const lsk_f32x4_u*)(x + (long)t * A.ld + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) s_v[(d + j) * LD + sh + t] = v[j];
    }
  }
  __syncthreads();
  if (!run) {
    if (l >= nt || !ok) return;
    T* dst = A.vc + ((long)r * A.Hkv + h) * (long)D * A.max_seq + (long)(p >> 5) * 32 * D + (p & 31);
    for (int d = tid >> 5; d < D; d += NORM_ROPE_THREADS / 32) dst[(long)d * 32] = s_v[d * LD + sh + l];
    return;
  }
  T* base = A.vc + ((long)r0 * A.Hkv + h) * (long)D * A.max_seq;
  const int pieces = (sh + nt + PP - 1) / PP, q0 = p0 - sh;
  for (int e = tid; e < D * (SLOTS / PP); e += NORM_ROPE_THREADS) {
    const int d = e / (SLOTS / PP), w = e - d * (SLOTS / PP), q = q0 + w * PP;
    if (w >= pieces) continue;
    T* dst = base + (long)(q >> 5) * 32 * D + d * 32 + (q & 31);
    const T* src = s_v + d * LD + w * PP;
    if (w * PP >= sh && w * PP + PP <= sh + nt && ((uintptr_t)dst & 15) == 0) {
      Piece x;
      __builtin_memcpy(&x, src, 16);
      *(Piece*)dst = x;
    } else {
#pragma unroll
      for (int j = 0; j < PP; ++j)
        if (w * PP + j >= sh && w * PP + j < sh + nt) dst[j] = src[j];
    }
  }
}

// The first `nv` workgroups write values; each other takes heads of one token: 16 lanes a head, PER = D / 16 consecutive
// dims a lane, whose rotation partners are eight lanes on; PASSES heads a group of lanes (a token's table rows are loaded
// once for them).  Each XCD has a run of consecutive tokens, so that the pieces of K that neighbours write meet in one L2
// (4001 tokens of 32 / 8 heads of 128: without 26.8 us, with 23.5).  Bound by HBM: those 98 MB, cold, 27 us.
// 32 tokens 3.5 us, a chain of loads, sums and stores.
template <typename T, int D, int PASSES>
__global__ __launch_bounds__(NORM_ROPE_THREADS) void norm_rope_kernel(const NormRopeArgs<T> A, int nv, int splits) {
  constexpr int PER = D / 16;
  const int Hq = A.Hq, Hkv = A.Hkv, heads = Hq + (A.k_out || nv > 0 ? Hkv : 2 * Hkv);
  if ((int)blockIdx.x < nv) {
    norm_rope_values<T, D>(A, (blockIdx.x / Hkv) * NORM_ROPE_TOKENS, blockIdx.x % Hkv);
    return;
  }
  const int b = blockIdx.x - nv, each = (A.N * splits + 7) >> 3, at = (b & 7) * each + (b >> 3);
  if ((b >> 3) >= each || at >= A.N * splits) return;
  const int t = at / splits, l = threadIdx.x & 15, j = l * PER;
  const int h0 = (at - t * splits) * PASSES * NORM_ROPE_HEADS + (int)threadIdx.x / 16;
  const T* x = A.qkv + (long)t * A.ld + j;
  float v[PASSES][PER];
#pragma unroll
  for (int k = 0; k < PASSES; ++k)                   // (heads past the last one: copies, not stored)
    load_f<PER>(x + (long)min(h0 + k * NORM_ROPE_HEADS, heads - 1) * D, v[k]);
  const int p = A.pos[t], row = A.k_out ? 0 : A.rows[t];
  if (p < 0 || p >= A.tab_len) return;
  if (!A.k_out && (row < 0 || row >= A.max_batch || p >= A.max_seq)) return;
  float c[PER], s[PER];
  load_f<PER>(A.cos_tab + (long)p * D + j, c);
  load_f<PER>(A.sin_tab + (long)p * D + j, s);
#pragma unroll
  for (int i = 0; i < PER; ++i) s[i] = l < 8 ? -s[i] : s[i];
#pragma unroll
  for (int k = 0; k < PASSES; ++k) {
    const int h = h0 + k * NORM_ROPE_HEADS;
    if (h >= heads) break;                           // (16 lanes at a time)
    if (h >= Hq + Hkv) {                             // a value of few tokens
      T* dst = A.vc + ((long)row * Hkv + (h - Hq - Hkv)) * (long)D * A.max_seq + (long)(p >> 5) * 32 * D + (p & 31);
#pragma unroll
      for (int i = 0; i < PER; ++i) Elem<T>::st(dst + (long)(j + i) * 32, v[k][i]);
      continue;
    }
    float ss = 0.f, w[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) ss = __builtin_fmaf(v[k][i], v[k][i], ss);
    const float r = rsqrtf(row_sum(ss) * (1.f / D) + A.eps);
    load_f<PER>((h < Hq ? A.wq : A.wk) + j, w);
#pragma unroll
    for (int i = 0; i < PER; ++i) v[k][i] = v[k][i] * r * w[i];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float y = dpp<0x128>(v[k][i]);           // (row_ror:8)
      w[i] = __builtin_fmaf(v[k][i], c[i], y * s[i]);
    }
    T* dst;
    if (h < Hq) dst = A.q_out + ((long)t * Hq + h) * D + j;
    else if (A.k_out) dst = A.k_out + ((long)t * Hkv + (h - Hq)) * D + j;
    else dst = A.kc + ((long)row * Hkv + (h - Hq)) * (long)A.max_seq * D;
    if (h < Hq || A.k_out) {
      store_f<PER>(dst, w);
    } else {                                         // (bf16: pieces of 8 dims are consecutive)
      constexpr int W = PER < 8 ? PER : 8;
#pragma unroll
      for (int i = 0; i < PER; i += W) store_f<W>(dst + k_cache_offset<T>(p, j + i, D), w + i);
    }
  }
}

template <typename T>
static int norm_rope_launch(const char* what, const NormRopeArgs<T>& a, int head_dim, hipStream_t s) {
  const bool many = a.N >= 64;
  const int heads = a.Hq + (a.k_out || many ? a.Hkv : 2 * a.Hkv), passes = a.N >= 512 ? 3 : 1;
  const int splits = (heads + passes * NORM_ROPE_HEADS - 1) / (passes * NORM_ROPE_HEADS);
  const int nv = a.k_out || !many ? 0 : (a.N + NORM_ROPE_TOKENS - 1) / NORM_ROPE_TOKENS * a.Hkv;
  const unsigned grid = (unsigned)(nv + (a.N * splits + 7) / 8 * 8);
#define NORM_ROPE(DD)                                                                                  \
  do {                                                                                                 \
    if (passes == 3) norm_rope_kernel<T, DD, 3><<<grid, NORM_ROPE_THREADS, 0, s>>>(a, nv, splits);      \
    else norm_rope_kernel<T, DD, 1><<<grid, NORM_ROPE_THREADS, 0, s>>>(a, nv, splits);                  \
  } while (0)
  switch (head_dim) {
    case 32: NORM_ROPE(32); break;
    case 64: NORM_ROPE(64); break;
    case 128: NORM_ROPE(128); break;
    default: NORM_ROPE(256); break;
  }
#undef NORM_ROPE
  return lsk_check_launch(what);
}

extern "C" int lsk_qk_norm_rope(int dtype, const void* qkv, long ld, const void* wq, const void* wk, float eps,
                                const float* cos_tab, const float* sin_tab, int tab_len, const int32_t* rows,
                                const int32_t* pos, int n_tokens, int n_heads, int n_kv_heads, int head_dim, void* q_out,
                                void* k_out, void* kcache, void* vcache, int max_batch, int max_seq, void* stream) {
  const char* what = "lsk_qk_norm_rope";
  LSK_REQUIRE(qkv && wq && wk && cos_tab && sin_tab && pos && q_out, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(k_out ? !kcache && !vcache : kcache && vcache && rows, LSK_EARG,
              "%s: either k_out, or rows and both caches", what);
  LSK_REQUIRE(dtype == LSK_DTYPE_BF16 || dtype == LSK_DTYPE_F32, LSK_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  LSK_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256, LSK_EUNSUPPORTED,
              "%s: head_dim %d (supported: 32, 64, 128, 256)", what, head_dim);
  LSK_REQUIRE(n_tokens >= 0 && n_tokens <= (1 << 20) && n_heads > 0 && n_kv_heads > 0 && n_heads <= 1024 &&
                  n_heads % n_kv_heads == 0 && tab_len > 0 && ld >= (long)(n_heads + 2 * n_kv_heads) * head_dim &&
                  (k_out || (max_batch > 0 && max_seq > 0 && max_seq % 32 == 0)),
              LSK_ESHAPE, "%s: bad shape", what);
  LSK_REQUIRE(eps >= 0.f, LSK_EARG, "%s: eps %g (not negative)", what, (double)eps);
  if (n_tokens == 0) return 0;
  if (dtype == LSK_DTYPE_BF16) {
    const NormRopeArgs<uint16_t> a = {(const uint16_t*)qkv, ld, (const uint16_t*)wq, (const uint16_t*)wk, eps, cos_tab,
                                      sin_tab, tab_len, rows, pos, (uint16_t*)q_out, (uint16_t*)k_out,
                                      (uint16_t*)kcache, (uint16_t*)vcache, n_tokens, n_heads, n_kv_heads, max_batch,
                                      max_seq};
    return norm_rope_launch(what, a, head_dim, (hipStream_t)stream);
  }
  const NormRopeArgs<float> a = {(const float*)qkv, ld, (const float*)wq, (const float*)wk, eps, cos_tab, sin_tab,
                                 tab_len, rows, pos, (float*)q_out, (float*)k_out, (float*)kcache, (float*)vcache,
                                 n_tokens, n_heads, n_kv_heads, max_batch, max_seq};
  return norm_rope_launch(what, a, head_dim, (hipStream_t)stream);
}
