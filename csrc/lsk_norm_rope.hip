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

template <int N, typename T>
__device__ __forceinline__ void load_f(const T* p, float* x) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = Elem<T>::ld(p + i);
}
template <int N, typename T>
__device__ __forceinline__ void store_f(T* p, const float* x) {
#pragma unroll
  for (int i = 0; i < N; ++i) Elem<T>::st(p + i, x[i]);
}

}  // namespace

#define NORM_ROPE_THREADS 256
// 16 lanes a vector, PER = D / 32 dims of each half a lane.
template <typename T, int D>
__global__ __launch_bounds__(NORM_ROPE_THREADS) void norm_rope_kernel(const NormRopeArgs<T> A) {
  constexpr int PER = D / 32, HALF = D / 2;
  const int t = blockIdx.x, h = blockIdx.y * (NORM_ROPE_THREADS / 16) + threadIdx.x / 16, j = (threadIdx.x & 15) * PER;
  const int Hq = A.Hq, Hkv = A.Hkv;
  if (h >= Hq + (A.k_out ? Hkv : 2 * Hkv)) return;   // (16 lanes at a time)
  const T* x = A.qkv + (long)t * A.ld + (long)h * D;
  float a[PER], b[PER];
  load_f<PER>(x + j, a);
  load_f<PER>(x + j + HALF, b);
  const int p = A.pos[t], row = A.k_out ? 0 : A.rows[t];
  if (p < 0 || p >= A.tab_len) return;
  if (!A.k_out && (row < 0 || row >= A.max_batch || p >= A.max_seq)) return;
  if (h >= Hq + Hkv) {
    T* dst = A.vc + ((long)row * Hkv + (h - Hq - Hkv)) * (long)D * A.max_seq + (long)(p >> 5) * 32 * D + (p & 31);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      dst[(long)(j + i) * 32] = x[j + i];
      dst[(long)(j + i + HALF) * 32] = x[j + i + HALF];
    }
    return;
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 16);
  const float r = rsqrtf(ss * (1.f / D) + A.eps);
  const T* w = h < Hq ? A.wq : A.wk;
  float wa[PER], wb[PER], c1[PER], c2[PER], s1[PER], s2[PER];
  load_f<PER>(w + j, wa);
  load_f<PER>(w + j + HALF, wb);
  const float *ct = A.cos_tab + (long)p * D + j, *st = A.sin_tab + (long)p * D + j;
  load_f<PER>(ct, c1);
  load_f<PER>(ct + HALF, c2);
  load_f<PER>(st, s1);
  load_f<PER>(st + HALF, s2);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float y1 = a[i] * r * wa[i], y2 = b[i] * r * wb[i];
    a[i] = y1 * c1[i] - y2 * s1[i];
    b[i] = y2 * c2[i] + y1 * s2[i];
  }
  T *lo, *hi;
  if (h < Hq) {
    lo = A.q_out + ((long)t * Hq + h) * D + j;
    hi = lo + HALF;
  } else if (A.k_out) {
    lo = A.k_out + ((long)t * Hkv + (h - Hq)) * D + j;
    hi = lo + HALF;
  } else {
    T* dst = A.kc + ((long)row * Hkv + (h - Hq)) * (long)A.max_seq * D;
    lo = dst + k_cache_offset<T>(p, j, D);
    hi = dst + k_cache_offset<T>(p, j + HALF, D);
  }
  store_f<PER>(lo, a);
  store_f<PER>(hi, b);
}

template <typename T>
static int norm_rope_launch(const char* what, const NormRopeArgs<T>& a, int head_dim, hipStream_t s) {
  const int heads = a.Hq + (a.k_out ? a.Hkv : 2 * a.Hkv), per = NORM_ROPE_THREADS / 16;
  const dim3 grid(a.N, (heads + per - 1) / per);
  switch (head_dim) {
    case 32: norm_rope_kernel<T, 32><<<grid, NORM_ROPE_THREADS, 0, s>>>(a); break;
    case 64: norm_rope_kernel<T, 64><<<grid, NORM_ROPE_THREADS, 0, s>>>(a); break;
    case 128: norm_rope_kernel<T, 128><<<grid, NORM_ROPE_THREADS, 0, s>>>(a); break;
    default: norm_rope_kernel<T, 256><<<grid, NORM_ROPE_THREADS, 0, s>>>(a); break;
  }
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
  LSK_REQUIRE(n_tokens >= 0 && n_heads > 0 && n_kv_heads > 0 && n_heads <= 65535 && n_kv_heads <= 65535 &&
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
