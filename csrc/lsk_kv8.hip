// The 8-bit KV cache: quantisation as tokens are written, and reading them back.
//
// Each token's K (and V) of one KV head is D e4m3 codes and one power-of-two scale 2^e, held as the biased exponent
// e + 127 in a byte:
//   amax = the largest finite |x|,  e = the smallest integer >= -117 with amax <= 448 * 2^e  (448: e4m3's largest value),
//   code = rne_e4m3(x * 2^-e),  the cache stands for code * 2^e.  NaN and infinities become NaN codes; amax = 0: e = 0.
// With e >= -117 every value is zero or a normal number (e4m3's smallest is 2^-9), in bf16 as in fp32.
// The product x * 2^-e is exact (a value far below amax may underflow, where its code is 0 anyway), so the only rounding
// is the one to e4m3: at most 2^-4 of the value, or 2^-10 * 2^e for values below 2^-6 * 2^e.
//
// Storage of one (row, KV head) stripe of S positions (S a multiple of 64), 64-position blocks of 64 D bytes:
//   K  fragments (a, j) of 16 positions x 64 d, 1 KiB in lane order: lane 16 lg + l16 holds position
//      16 (l16 / 4) + 4 a + l16 % 4 of the block and d = 64 j + 16 lg .. + 15 (kv8_k_offset);
//   V  transposed: position p, dim d at d * 64 + p % 64;
//   exponents [S].
#include "lsk_common.h"
#include "../include/lsk.h"

namespace {

__device__ __forceinline__ long kv8_k_offset(int p, int d, int D) {
  const int pp = p & 63;
  const int a = (pp >> 2) & 3, l16 = ((pp >> 4) << 2) | (pp & 3);
  const int j = d >> 6, lg = (d >> 4) & 3;
  return (long)(p >> 6) * 64 * D + (long)((a * (D >> 6) + j) * 64 + lg * 16 + l16) * 16 + (d & 15);
}

// e + 127 of a vector whose largest finite magnitude has the bits `m` (>= 0): 448 = 1.75 * 2^8
__device__ __forceinline__ int biased_exponent(uint32_t m) {
  if (m == 0u) return 127;
  const int e = (int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);  // (subnormals end at the floor as well)
  return e < 10 ? 10 : e;
}

// four floats -> four e4m3 codes, after the exact scaling by inv; non-finite values -> NaN codes
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, (int)r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, (int)r, true);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if ((__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u) r |= 0x7fu << (8 * i);
  return r;
}

__device__ __forceinline__ void values4(uint32_t c, float scale, float* o) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const f2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  o[0] = a[0] * scale; o[1] = a[1] * scale; o[2] = b[0] * scale; o[3] = b[1] * scale;
}

#define KV8_TOKENS 16  // tokens of a workgroup: 16 threads each
#define KV8_THREADS 256

}  // namespace

// A workgroup quantises 16 tokens of one KV head, K then V; 16 threads hold a token's vector, D / 16 consecutive
// elements each, and find its largest magnitude by shuffles.  K goes straight to its place; V is turned in LDS so that
// a dim's positions land side by side.
template <typename T, int D>
__global__ __launch_bounds__(KV8_THREADS) void kv8_append_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                                 long st_t, long st_h, uint8_t* __restrict__ kc,
                                                                 uint8_t* __restrict__ vc, uint8_t* __restrict__ ks,
                                                                 uint8_t* __restrict__ vs,
                                                                 const int32_t* __restrict__ rows,
                                                                 const int32_t* __restrict__ pos, int N, int Hkv,
                                                                 int max_batch, int S) {
  constexpr int PER = D / 16;
  __shared__ uint8_t s_v[KV8_TOKENS][D + 4];
  const int t0 = blockIdx.x * KV8_TOKENS, h = blockIdx.y;
  const int j = threadIdx.x >> 4, part = threadIdx.x & 15;
  const int t = t0 + j;
  const int row = t < N ? rows[t] : -1, p = t < N ? pos[t] : -1;
  const bool ok = row >= 0 && row < max_batch && p >= 0 && p < S;
  const long stripe = ((long)row * Hkv + h) * (long)S;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    float x[PER];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      x[i] = ok ? Elem<T>::ld((kv ? v : k) + (long)t * st_t + (long)h * st_h + part * PER + i) : 0.f;
      const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
      m = u < 0x7f800000u && u > m ? u : m;
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
      const uint32_t y = (uint32_t)__shfl_xor((int)m, o, 16);
      m = y > m ? y : m;
    }
    const int e = biased_exponent(m);
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
    if (ok) {
      if (part == 0) (kv ? vs : ks)[stripe + p] = (uint8_t)e;
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        const uint32_t c = codes4(x + i, inv);
        if (kv == 0) *(uint32_t*)(kc + stripe * D + kv8_k_offset(p, part * PER + i, D)) = c;
        else *(uint32_t*)(&s_v[j][part * PER + i]) = c;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < KV8_TOKENS * D; i += KV8_THREADS) {
    const int tj = i % KV8_TOKENS, d = i / KV8_TOKENS, tt = t0 + tj;
    if (tt >= N) continue;
    const int r = rows[tt], pp = pos[tt];
    if (r < 0 || r >= max_batch || pp < 0 || pp >= S) continue;
    vc[((long)r * Hkv + h) * (long)S * D + (long)(pp >> 6) * 64 * D + d * 64 + (pp & 63)] = s_v[tj][d];
  }
}

template <typename T, int D>
__global__ __launch_bounds__(KV8_THREADS) void kv8_read_kernel(const uint8_t* __restrict__ kc,
                                                               const uint8_t* __restrict__ vc,
                                                               const uint8_t* __restrict__ ks,
                                                               const uint8_t* __restrict__ vs,
                                                               const int32_t* __restrict__ rows,
                                                               const int32_t* __restrict__ pos, T* __restrict__ k,
                                                               T* __restrict__ v, int N, int Hkv, int max_batch,
                                                               int S) {
  constexpr int PER = D / 16;
  __shared__ uint8_t s_v[KV8_TOKENS][D + 4];
  const int t0 = blockIdx.x * KV8_TOKENS, h = blockIdx.y;
  for (int i = threadIdx.x; i < KV8_TOKENS * D; i += KV8_THREADS) {
    const int tj = i % KV8_TOKENS, d = i / KV8_TOKENS, tt = t0 + tj;
    if (tt >= N) continue;
    const int r = rows[tt], pp = pos[tt];
    if (r < 0 || r >= max_batch || pp < 0 || pp >= S) continue;
    s_v[tj][d] = vc[((long)r * Hkv + h) * (long)S * D + (long)(pp >> 6) * 64 * D + d * 64 + (pp & 63)];
  }
  __syncthreads();
  const int j = threadIdx.x >> 4, part = threadIdx.x & 15;
  const int t = t0 + j;
  if (t >= N) return;
  const int row = rows[t], p = pos[t];
  const bool ok = row >= 0 && row < max_batch && p >= 0 && p < S;
  const long stripe = ((long)row * Hkv + h) * (long)S;
  const float sk = ok ? __uint_as_float((uint32_t)ks[stripe + p] << 23) : 0.f;
  const float sv = ok ? __uint_as_float((uint32_t)vs[stripe + p] << 23) : 0.f;
#pragma unroll
  for (int i = 0; i < PER; i += 4) {
    const int d = part * PER + i;
    const long o = ((long)t * Hkv + h) * D + d;
    float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    if (ok) {
      values4(*(const uint32_t*)(kc + stripe * D + kv8_k_offset(p, d, D)), sk, a);
      values4(*(const uint32_t*)(&s_v[j][d]), sv, b);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      Elem<T>::st(k + o + q, a[q]);
      Elem<T>::st(v + o + q, b[q]);
    }
  }
}

static int kv8_args(const char* what, int dtype, const void* k, const void* v, const void* kc, const void* vc,
                    const void* ks, const void* vs, const void* rows, const void* pos, int n, int hkv, int d, int b,
                    int s) {
  LSK_REQUIRE(k && v && kc && vc && ks && vs && rows && pos, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(dtype == LSK_DTYPE_BF16 || dtype == LSK_DTYPE_F32, LSK_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  LSK_REQUIRE(d == 64 || d == 128, LSK_EUNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", what, d);
  LSK_REQUIRE(n >= 0 && hkv > 0 && hkv <= 65535 && b > 0 && s > 0 && s % 64 == 0, LSK_ESHAPE,
              "%s: bad shape (max_seq %% 64 == 0)", what);
  LSK_REQUIRE((((uintptr_t)kc | (uintptr_t)vc) & 15) == 0, LSK_EARG, "%s: the cache tensors start at multiples of 16 bytes",
              what);
  return 0;
}

#define KV8_LAUNCH(KERNEL, T, ...)                                            \
  do {                                                                        \
    if (head_dim == 128) KERNEL<T, 128><<<grid, KV8_THREADS, 0, st>>>(__VA_ARGS__); \
    else KERNEL<T, 64><<<grid, KV8_THREADS, 0, st>>>(__VA_ARGS__);            \
  } while (0)

extern "C" int lsk_kv8_append(int dtype, const void* k, const void* v, long stride_t, long stride_h, void* k8, void* v8,
                              void* k_exp, void* v_exp, const int32_t* rows, const int32_t* pos, int n_tokens,
                              int n_kv_heads, int head_dim, int max_batch, int max_seq, void* stream) {
  const char* what = "lsk_kv8_append";
  if (int rc = kv8_args(what, dtype, k, v, k8, v8, k_exp, v_exp, rows, pos, n_tokens, n_kv_heads, head_dim, max_batch,
                        max_seq)) return rc;
  LSK_REQUIRE(stride_t >= 0 && stride_h >= 0, LSK_ESHAPE, "%s: negative strides", what);
  if (n_tokens == 0) return 0;
  const dim3 grid((n_tokens + KV8_TOKENS - 1) / KV8_TOKENS, n_kv_heads);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LSK_DTYPE_BF16)
    KV8_LAUNCH(kv8_append_kernel, uint16_t, (const uint16_t*)k, (const uint16_t*)v, stride_t, stride_h, (uint8_t*)k8,
               (uint8_t*)v8, (uint8_t*)k_exp, (uint8_t*)v_exp, rows, pos, n_tokens, n_kv_heads, max_batch, max_seq);
  else
    KV8_LAUNCH(kv8_append_kernel, float, (const float*)k, (const float*)v, stride_t, stride_h, (uint8_t*)k8,
               (uint8_t*)v8, (uint8_t*)k_exp, (uint8_t*)v_exp, rows, pos, n_tokens, n_kv_heads, max_batch, max_seq);
  return lsk_check_launch(what);
}

extern "C" int lsk_kv8_read(int dtype, const void* k8, const void* v8, const void* k_exp, const void* v_exp,
                            const int32_t* rows, const int32_t* pos, void* k, void* v, int n_tokens, int n_kv_heads,
                            int head_dim, int max_batch, int max_seq, void* stream) {
  const char* what = "lsk_kv8_read";
  if (int rc = kv8_args(what, dtype, k, v, k8, v8, k_exp, v_exp, rows, pos, n_tokens, n_kv_heads, head_dim, max_batch,
                        max_seq)) return rc;
  if (n_tokens == 0) return 0;
  const dim3 grid((n_tokens + KV8_TOKENS - 1) / KV8_TOKENS, n_kv_heads);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LSK_DTYPE_BF16)
    KV8_LAUNCH(kv8_read_kernel, uint16_t, (const uint8_t*)k8, (const uint8_t*)v8, (const uint8_t*)k_exp,
               (const uint8_t*)v_exp, rows, pos, (uint16_t*)k, (uint16_t*)v, n_tokens, n_kv_heads, max_batch, max_seq);
  else
    KV8_LAUNCH(kv8_read_kernel, float, (const uint8_t*)k8, (const uint8_t*)v8, (const uint8_t*)k_exp,
               (const uint8_t*)v_exp, rows, pos, (float*)k, (float*)v, n_tokens, n_kv_heads, max_batch, max_seq);
  return lsk_check_launch(what);
}
#undef KV8_LAUNCH
