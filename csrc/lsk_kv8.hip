// The 8-bit KV cache: quantisation as tokens are written, and reading them back.
//
// Each token's K (and V) of one KV head is D e4m3 codes and one power-of-two scale 2^e, held as the biased exponent
// e + 127 in a byte:
//   amax = the largest finite |x|,  e = the smallest integer >= -117 with amax <= 448 * 2^e  (448 is e4m3's largest),
//   code = rne_e4m3(x * 2^-e),  the cache stands for code * 2^e.  NaN and infinities become NaN codes; amax = 0: e = 0.
// At the largest e, 120, a code is at most 240 (the next one, 256, would stand for 2^128; still within 2^-4 of x).
// With e >= -117 every value is zero or a normal number (e4m3's smallest is 2^-9), in bf16 as in fp32.
// The product x * 2^-e is exact (a value far below amax may underflow, where its code is 0 anyway), so the only
// rounding is the one to e4m3: at most 2^-4 of the value, or 2^-10 * 2^e for values below 2^-6 * 2^e.
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

// four floats -> four e4m3 codes, after the exact scaling by 2^(127 - e); non-finite values -> NaN codes
__device__ __forceinline__ uint32_t codes4(const float* x, int e) {
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23), top = e == 247 ? 240.f : 448.f;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -top, top);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], (int)r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)r, true);
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

// 4 consecutive elements at any address that aligns one of them
__device__ __forceinline__ void load4(const uint16_t* p, float* x) {
  const lsk_u32x2_u u = *(const lsk_u32x2_u*)p;
  x[0] = __uint_as_float(u[0] << 16); x[1] = __uint_as_float(u[0] & 0xffff0000u);
  x[2] = __uint_as_float(u[1] << 16); x[3] = __uint_as_float(u[1] & 0xffff0000u);
}
__device__ __forceinline__ void load4(const float* p, float* x) {
  const lsk_f32x4_u u = *(const lsk_f32x4_u*)p;
  x[0] = u[0]; x[1] = u[1]; x[2] = u[2]; x[3] = u[3];
}
__device__ __forceinline__ void store4(uint16_t* p, const float* x) {
  lsk_u32x2_u u;
  u[0] = (uint32_t)f2bf(x[0]) | ((uint32_t)f2bf(x[1]) << 16);
  u[1] = (uint32_t)f2bf(x[2]) | ((uint32_t)f2bf(x[3]) << 16);
  *(lsk_u32x2_u*)p = u;
}
__device__ __forceinline__ void store4(float* p, const float* x) {
  *(lsk_f32x4_u*)p = (lsk_f32x4_u){x[0], x[1], x[2], x[3]};
}

// Four dwords of four bytes, turned: byte j of a[i] <-> byte i of a[j]
__device__ __forceinline__ void turn4(uint32_t* a) {
  const uint32_t l0 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400), h0 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602);
  const uint32_t l1 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400), h1 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602);
  a[0] = __builtin_amdgcn_perm(l1, l0, 0x05040100);
  a[1] = __builtin_amdgcn_perm(l1, l0, 0x07060302);
  a[2] = __builtin_amdgcn_perm(h1, h0, 0x05040100);
  a[3] = __builtin_amdgcn_perm(h1, h0, 0x07060302);
}

// the largest finite magnitude (bits) of the vector that 16 threads hold
template <int PER>
__device__ __forceinline__ uint32_t vector_max(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
    m = u < 0x7f800000u && u > m ? u : m;
  }
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)m, o, 16);
    m = y > m ? y : m;
  }
  return m;
}

#define KV8_THREADS 256
#define KV8_TOKENS 64  // tokens of a workgroup of V, and of four workgroups of K: 16 threads hold a token's vector
#define KV8_LD 17      // dwords of a dim's row of the V tile in LDS (64 tokens from any position: 17 dwords of slots)

// Whether the V workgroup's nt tokens are a run of one cache row (consecutive positions, inside the cache), from every
// wave's own look at them.
__device__ __forceinline__ bool kv8_run(const int32_t* rows, const int32_t* pos, int t0, int nt, int max_batch, int S) {
  const int l = threadIdx.x & 63, i = min(l, nt - 1);
  const int r = rows[t0 + i], p = pos[t0 + i];
  const int r0 = __shfl(r, 0, 64), p0 = __shfl(p, 0, 64);
  const bool ok = r >= 0 && r < max_batch && p >= 0 && p < S && r == r0 &&
                  (uint32_t)p - (uint32_t)p0 == (uint32_t)i;
  return __builtin_amdgcn_ballot_w64(ok) == ~0ull;
}

// A workgroup's tokens one by one: f(d, token, address of its byte in the V codes), lanes side by side over the tokens.
template <int D, typename F>
__device__ __forceinline__ void kv8_each(const int32_t* rows, const int32_t* pos, int t0, int nt, int h, int Hkv,
                                         int max_batch, int S, F f) {
  const int lg = nt > 1 ? 32 - __builtin_clz(nt - 1) : 0;              // 2^lg >= nt
  const int tj = threadIdx.x & ((1 << lg) - 1);
  if (tj >= nt) return;
  const int r = rows[t0 + tj], p = pos[t0 + tj];
  if (r < 0 || r >= max_batch || p < 0 || p >= S) return;
  const long at = ((long)r * Hkv + h) * (long)S * D + (long)(p >> 6) * 64 * D + (p & 63);
  for (int d = threadIdx.x >> lg; d < D; d += KV8_THREADS >> lg) f(d, tj, at + d * 64);
}

// A run's dwords of V codes: f(d, its index in the LDS row, address), over the 64-position blocks that it touches.
template <int D, typename F>
__device__ __forceinline__ void kv8_dwords(long stripe, int p0, int nt, F f) {
  const int q0 = p0 & ~3, n = (p0 + nt - q0 + 3) >> 2;                 // <= 17
  for (int i = threadIdx.x; i < D * 16; i += KV8_THREADS) {
    const int d = i >> 4, w = i & 15, q = q0 + 4 * w;
    if (w < n) f(d, w, stripe * D + (long)(q >> 6) * 64 * D + d * 64 + (q & 63));
  }
  if (n == 17 && threadIdx.x < D) {
    const int d = threadIdx.x, q = q0 + 64;
    f(d, 16, stripe * D + (long)(q >> 6) * 64 * D + d * 64 + (q & 63));
  }
}

}  // namespace

// Workgroup 0 of blockIdx.z quantises 64 tokens' V of one KV head (it takes longest and starts first), workgroups 1 to
// 4 quantise 16 tokens' K each.  16 threads hold a token's vector, D / 16 consecutive elements each, and find its
// largest magnitude by shuffles.  K goes straight to its place.  V is turned, 4 x 4 in registers and the rest in LDS: a
// run of positions (a prompt's tokens) is written a dword at a time, whole 64-byte sectors from one workgroup; other
// tokens byte by byte.
// Bound by a workgroup's chain of loading, reducing, converting, turning and storing: 6.9 us for a decode step's
// tokens, whose V asks for rows and positions behind the conversion and is stored byte by byte; a prompt moves 3 D
// bytes a token and head (4001 tokens of 8 heads of 128: 11.3 us, 4.8 by their bytes; with the V workgroups last 13.4;
// with 16 tokens to every workgroup, so that four share a sector of V, 16.9).
template <typename T, int D>
__global__ __launch_bounds__(KV8_THREADS) void kv8_append_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                                 long st_t, long st_h, uint8_t* __restrict__ kc,
                                                                 uint8_t* __restrict__ vc, uint8_t* __restrict__ ks,
                                                                 uint8_t* __restrict__ vs,
                                                                 const int32_t* __restrict__ rows,
                                                                 const int32_t* __restrict__ pos, int N, int Hkv,
                                                                 int max_batch, int S) {
  constexpr int PER = D / 16;
  __shared__ uint32_t s_v[D * KV8_LD];
  const int h = blockIdx.y, j = threadIdx.x >> 4, part = threadIdx.x & 15;
  if (blockIdx.z > 0) {
    const int t = blockIdx.x * KV8_TOKENS + (blockIdx.z - 1) * 16 + j;
    if (t >= N) return;                              // (16 threads at a time)
    float x[PER];
    const T* src = k + (long)t * st_t + (long)h * st_h + part * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 4) load4(src + i, x + i);
    const int row = rows[t], p = pos[t];
    const int e = biased_exponent(vector_max<PER>(x));
    if (row < 0 || row >= max_batch || p < 0 || p >= S) return;
    const long stripe = ((long)row * Hkv + h) * (long)S;
    uint32_t* dst = (uint32_t*)(kc + stripe * D + kv8_k_offset(p, part * PER, D));
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) dst[i] = codes4(x + 4 * i, e);
    if (part == 0) ks[stripe + p] = (uint8_t)e;
    return;
  }
  const int t0 = blockIdx.x * KV8_TOKENS, nt = min(KV8_TOKENS, N - t0);
  float x[4][PER];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int tj = min(4 * j + c, nt - 1);           // (tokens behind the last one: its copies, never written)
    const T* src = v + (long)(t0 + tj) * st_t + (long)h * st_h + part * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 4) load4(src + i, &x[c][i]);
  }
  uint32_t w[PER / 4][4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int e = biased_exponent(vector_max<PER>(x[c]));
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) w[i][c] = codes4(&x[c][4 * i], e);
    if (part == 0 && 4 * j + c < nt) {
      const int row = rows[t0 + 4 * j + c], p = pos[t0 + 4 * j + c];
      if (row >= 0 && row < max_batch && p >= 0 && p < S) vs[((long)row * Hkv + h) * (long)S + p] = (uint8_t)e;
    }
  }
#pragma unroll
  for (int i = 0; i < PER / 4; ++i) {
    turn4(w[i]);
#pragma unroll
    for (int c = 0; c < 4; ++c) s_v[(part * PER + 4 * i + c) * KV8_LD + j] = w[i][c];
  }
  const bool run = kv8_run(rows, pos, t0, nt, max_batch, S);
  __syncthreads();
  if (!run) {
    kv8_each<D>(rows, pos, t0, nt, h, Hkv, max_batch, S, [&](int d, int tj, long at) {
      vc[at] = (uint8_t)(s_v[d * KV8_LD + (tj >> 2)] >> (8 * (tj & 3)));
    });
    return;
  }
  const int p0 = pos[t0], sh = p0 & 3;
  kv8_dwords<D>(((long)rows[t0] * Hkv + h) * (long)S, p0, nt, [&](int d, int i, long at) {
    const uint32_t* r = s_v + d * KV8_LD;            // slots 4 i .. + 3 of the run's: tokens 4 i - sh .. + 3
    const uint32_t u = sh == 0 ? r[i] : __builtin_amdgcn_alignbyte(r[i], r[max(i - 1, 0)], 4 - sh);
    const int tj = 4 * i - sh;
    if (tj >= 0 && tj + 3 < nt) {
      *(uint32_t*)(vc + at) = u;
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (tj + b >= 0 && tj + b < nt) vc[at + b] = (uint8_t)(u >> (8 * b));
    }
  });
}

// The way back, in the same shape and bound alike (4001 tokens of 8 heads of 128: 10.2 us).
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
  __shared__ uint32_t s_v[D * KV8_LD];
  const int h = blockIdx.y, j = threadIdx.x >> 4, part = threadIdx.x & 15;
  if (blockIdx.z > 0) {
    const int t = blockIdx.x * KV8_TOKENS + (blockIdx.z - 1) * 16 + j;
    if (t >= N) return;
    const int row = rows[t], p = pos[t];
    const bool ok = row >= 0 && row < max_batch && p >= 0 && p < S;
    const long stripe = ((long)row * Hkv + h) * (long)S;
    const uint32_t* src = (const uint32_t*)(kc + stripe * D + kv8_k_offset(p, part * PER, D));
    T* dst = k + ((long)t * Hkv + h) * D + part * PER;
    const float scale = ok ? __uint_as_float((uint32_t)ks[stripe + p] << 23) : 0.f;
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
      float o[4];
      values4(ok ? src[i] : 0u, scale, o);
      store4(dst + 4 * i, o);
    }
    return;
  }
  const int t0 = blockIdx.x * KV8_TOKENS, nt = min(KV8_TOKENS, N - t0);
  const bool run = kv8_run(rows, pos, t0, nt, max_batch, S);
  int sh = 0;
  if (run) {
    const int p0 = pos[t0];
    sh = p0 & 3;
    kv8_dwords<D>(((long)rows[t0] * Hkv + h) * (long)S, p0, nt,
                  [&](int d, int i, long at) { s_v[d * KV8_LD + i] = *(const uint32_t*)(vc + at); });
  } else {
    kv8_each<D>(rows, pos, t0, nt, h, Hkv, max_batch, S,
                [&](int d, int tj, long at) { ((uint8_t*)(s_v + d * KV8_LD))[tj] = vc[at]; });
  }
  __syncthreads();
  uint32_t w[PER / 4][4];
#pragma unroll
  for (int i = 0; i < PER / 4; ++i) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t* r = s_v + (part * PER + 4 * i + c) * KV8_LD + j;
      w[i][c] = __builtin_amdgcn_alignbyte(r[1], r[0], sh);
    }
    turn4(w[i]);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int t = t0 + 4 * j + c;
    if (4 * j + c >= nt) break;
    const int row = rows[t], p = pos[t];
    const bool ok = row >= 0 && row < max_batch && p >= 0 && p < S;
    const float scale = ok ? __uint_as_float((uint32_t)vs[((long)row * Hkv + h) * (long)S + p] << 23) : 0.f;
    T* dst = v + ((long)t * Hkv + h) * D + part * PER;
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
      float o[4];
      values4(ok ? w[i][c] : 0u, scale, o);
      store4(dst + 4 * i, o);
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
  LSK_REQUIRE((((uintptr_t)kc | (uintptr_t)vc) & 15) == 0, LSK_EARG,
              "%s: the cache tensors start at multiples of 16 bytes", what);
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
  const dim3 grid((n_tokens + KV8_TOKENS - 1) / KV8_TOKENS, n_kv_heads, 5);
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
  const dim3 grid((n_tokens + KV8_TOKENS - 1) / KV8_TOKENS, n_kv_heads, 5);
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
