// The 4-bit KV cache: quantisation as tokens are written, reading them back, and the compaction of accepted paths.
//
// 32 consecutive dims of a token's K (or V) of one KV head are 32 e2m1 codes and one power-of-two scale 2^e, held as the
// biased exponent e + 127 in a byte:
//   amax = the largest |x|,  e = the smallest integer >= -125 with amax <= 7 * 2^e  (6 is e2m1's largest value; what lies
//   between 6 and 7 becomes 6, off by no more than a value between 4 and 6 may be, and every other value of the 32 is
//   held twice as finely as with the next e),
//   code = rne_e2m1(x * 2^-e), at most 6;  the cache stands for code * 2^e.  amax = 0: e = 0.
// At the largest e, 126, a code is at most 3 (4 would stand for 2^128).  With e >= -125 every value is zero or a normal
// number (e2m1's smallest is 0.5).  x * 2^-e is exact, so the only rounding is the one to e2m1: by at most 2^e for
// values above 4 * 2^e, 2^e / 2 above 2 * 2^e and 2^e / 4 below.
// 32 dims that hold a NaN or an infinity are NaN as a whole: the exponent byte 255 and zero codes.
//
// Storage of one (row, KV head) stripe of S positions (S a multiple of 64), 64-position blocks of 32 D bytes, D / 32
// fragments of 1 KiB in lane order; the lower half of a byte is the dim (V: the position) that comes first:
//   K  lane 16 lg + l16 holds position 16 (l16 / 4) + 4 a + l16 % 4 of the block and d = D / 4 lg .. + D / 4 - 1: 16 bytes
//      of fragment a for D = 128, half a % 2 of those of fragment a / 2 for D = 64 (kv4_k_offset);
//   V  transposed: half h of lane 16 lg + l16's bytes of fragment c holds dim 32 c + 16 h + l16 at positions 16 lg .. + 15
//      (kv4_v_offset);
//   exponents, 64 bytes for each 32 dims of a block: K's [l16][a], V's [position].
#include "lsk_common.h"
#include "../include/lsk.h"

namespace {

__device__ __forceinline__ long kv4_k_offset(int p, int d, int D) {
  const int pp = p & 63, h = 128 / D, per = D >> 2;
  const int a = (pp >> 2) & 3, l16 = ((pp >> 4) << 2) | (pp & 3);
  return (long)(p >> 6) * 32 * D + ((a / h) * 64 + (d / per) * 16 + l16) * 16 + (a % h) * (16 / h) + (d % per) / 2;
}
__device__ __forceinline__ long kv4_v_offset(int p, int d, int D) {
  const int pp = p & 63;
  return (long)(p >> 6) * 32 * D + ((d >> 5) * 64 + (pp >> 4) * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + ((pp & 15) >> 1);
}
__device__ __forceinline__ long kv4_ks_offset(int p, int d, int D) {
  const int pp = p & 63;
  return ((long)(p >> 6) * (D >> 5) + (d >> 5)) * 64 + ((pp >> 4) * 4 + (pp & 3)) * 4 + ((pp >> 2) & 3);
}
__device__ __forceinline__ long kv4_vs_offset(int p, int d, int D) {
  return ((long)(p >> 6) * (D >> 5) + (d >> 5)) * 64 + (p & 63);
}

// e + 127 of 32 values whose largest magnitude has the bits `m` (>= 0): 7 = 1.75 * 2^2.  255: one is not finite.
__device__ __forceinline__ int kv4_exponent(uint32_t m) {
  if (m >= 0x7f800000u) return 255;
  if (m == 0u) return 127;
  const int e = (int)(m >> 23) - 2 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);  // (subnormals end at the floor as well)
  return e < 2 ? 2 : e;
}

// two floats -> a byte of two e2m1 codes (nearest even, at most 6), after the exact scaling by 2^(127 - e)
__device__ __forceinline__ uint32_t kv4_byte(float x0, float x1, int e) {
  if (e == 255) return 0u;
  if (e == 253) {                                    // (4 * 2^126 would be 2^128)
    const float top = 0x1.8p127f;
    x0 = __builtin_amdgcn_fmed3f(x0, -top, top);
    x1 = __builtin_amdgcn_fmed3f(x1, -top, top);
  }
  return (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x0, x1, __uint_as_float((uint32_t)e << 23), 0) & 255u;
}

__device__ __forceinline__ void kv4_values(uint32_t byte, uint32_t e, float* o) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(byte, __uint_as_float(e << 23), 0);
  o[0] = a[0];
  o[1] = a[1];
}

__device__ __forceinline__ void load2(const uint16_t* p, float* x) { x[0] = bf2f(p[0]); x[1] = bf2f(p[1]); }
__device__ __forceinline__ void load2(const float* p, float* x) { x[0] = p[0]; x[1] = p[1]; }
__device__ __forceinline__ void store2(uint16_t* p, const float* x) { p[0] = f2bf(x[0]); p[1] = f2bf(x[1]); }
__device__ __forceinline__ void store2(float* p, const float* x) { p[0] = x[0]; p[1] = x[1]; }

// The bits of `mask` of a dword become those of x: other threads may be replacing others of its bits.
__device__ __forceinline__ void put_bits(uint32_t* w, uint32_t x, uint32_t mask) {
  const uint32_t old = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if ((old ^ x) & mask) __hip_atomic_fetch_xor(w, (old ^ x) & mask, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put_nibble(uint8_t* codes, long at, int odd, uint32_t code) {
  const int sh = 8 * (int)(at & 3) + 4 * odd;
  put_bits((uint32_t*)(codes + (at & ~3l)), code << sh, 15u << sh);
}

// 32 consecutive elements (at any address that aligns one of them): their largest magnitude's exponent and their codes
__device__ __forceinline__ void load32(const uint16_t* p, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const lsk_u32x4_u u = *(const lsk_u32x4_u*)(p + 8 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
      x[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void load32(const float* p, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const lsk_f32x4_u u = *(const lsk_f32x4_u*)(p + 4 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 * i + j] = u[j];
  }
}
template <typename T>
__device__ __forceinline__ int quantise32(const T* p, uint32_t* codes) {
  float x[32];
  load32(p, x);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  const int e = kv4_exponent(m);
  const float scale = __uint_as_float((uint32_t)e << 23);
  if (e == 253) {                                    // (as kv4_byte)
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __builtin_amdgcn_fmed3f(x[i], -0x1.8p127f, 0x1.8p127f);
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[8 * w], x[8 * w + 1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[8 * w + 2], x[8 * w + 3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[8 * w + 4], x[8 * w + 5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[8 * w + 6], x[8 * w + 7], scale, 3);
    codes[w] = e == 255 ? 0u : c;
  }
  return e;
}

// 8 codes (pairs in bytes) -> values, stored (at any address that aligns one of them)
__device__ __forceinline__ void store8(uint16_t* p, uint32_t c, float scale) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
  const bf2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
  *(lsk_u32x4_u*)p = __builtin_bit_cast(lsk_u32x4_u, (lsk_bf16x8){a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]});
}
__device__ __forceinline__ void store8(float* p, uint32_t c, float scale) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
  const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
  *(lsk_f32x4_u*)p = (lsk_f32x4_u){a[0], a[1], b[0], b[1]};
  *(lsk_f32x4_u*)(p + 4) = (lsk_f32x4_u){d[0], d[1], e[0], e[1]};
}

}  // namespace

#define KV4_THREADS 256
// Tokens times KV heads from which the kernels for many tokens run (8 heads of 128, a prompt of 1024 / 4001 tokens, append:
// 5.7 / 7.7 us against 6.2 / 22; single tokens of 32 rows 8.5 us against 3.2)
#define KV4_MANY 8192

// Few tokens: D / 2 threads a token and head, two dims each; 16 of them find their 32 dims' largest magnitude.
template <typename T, int D>
__global__ __launch_bounds__(KV4_THREADS) void kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                                 long st_t, long st_h, uint8_t* __restrict__ kc,
                                                                 uint8_t* __restrict__ vc, uint8_t* __restrict__ ks,
                                                                 uint8_t* __restrict__ vs,
                                                                 const int32_t* __restrict__ rows,
                                                                 const int32_t* __restrict__ pos, int N, int Hkv,
                                                                 int max_batch, int S) {
  constexpr int PER = KV4_THREADS / (D / 2);         // tokens of a workgroup
  const int t = blockIdx.x * PER + threadIdx.x / (D / 2), h = blockIdx.y, d = 2 * (threadIdx.x % (D / 2));
  if (t >= N) return;                                // (16 threads at a time)
  const T* src = (blockIdx.z ? v : k) + (long)t * st_t + (long)h * st_h + d;
  float x[2];
  load2(src, x);
  const int row = rows[t], p = pos[t];
  uint32_t m = max(__float_as_uint(x[0]) & 0x7fffffffu, __float_as_uint(x[1]) & 0x7fffffffu);
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 16));
  if (row < 0 || row >= max_batch || p < 0 || p >= S) return;
  const int e = kv4_exponent(m);
  const uint32_t b = kv4_byte(x[0], x[1], e);
  const long stripe = ((long)row * Hkv + h) * (long)S;
  if (blockIdx.z == 0) {
    kc[stripe * (D / 2) + kv4_k_offset(p, d, D)] = (uint8_t)b;
    if ((d & 31) == 0) ks[stripe * (D / 32) + kv4_ks_offset(p, d, D)] = (uint8_t)e;
  } else {
    uint8_t* to = vc + stripe * (D / 2);
    put_nibble(to, kv4_v_offset(p, d, D), p & 1, b & 15u);
    put_nibble(to, kv4_v_offset(p, d + 1, D), p & 1, b >> 4);
    if ((d & 31) == 0) vs[stripe * (D / 32) + kv4_vs_offset(p, d, D)] = (uint8_t)e;
  }
}

// A workgroup's tokens as groups: runs of positions within 16 aligned ones of a cache row.  first[g] .. first[g + 1] - 1
// are group g's tokens; returns the number of groups.  row and pos: this thread's token (row -1: outside the cache), held
// by the first of its NB threads.
template <int TOK, int NB>
struct Kv4Groups {
  int row[TOK], pos[TOK], first[TOK + 1], n;
  __device__ __forceinline__ void put(int tj, int b, int row_, int pos_) {
    if (b == 0) {
      row[tj] = row_;
      pos[tj] = pos_;
    }
  }
  __device__ __forceinline__ void find(int nt) {     // after put and a barrier, before another; the first wave's work
    const int l = threadIdx.x;
    if (l >= 64) return;
    int at = 0;
#pragma unroll
    for (int u = 0; u < TOK; u += 64) {
      const int j = u + l;
      const bool begins = j < nt && (j == 0 || row[j] != row[j - 1] || pos[j] != pos[j - 1] + 1 || (pos[j] & 15) == 0);
      const uint64_t m = __builtin_amdgcn_ballot_w64(begins);
      if (begins) first[at + __builtin_popcountll(m & ((1ull << l) - 1))] = j;
      at += __builtin_popcountll(m);
    }
    if (l == 0) {
      first[at] = nt;
      n = at;
    }
  }
};

// Many tokens: a thread takes 32 dims of a token.  K's codes go straight to their place, 16 bytes (D = 64: twice 8).  V's
// go through LDS: a workgroup's tokens fall into groups, runs of positions within 16 aligned ones of a cache row (a
// prompt's groups are whole, a decode step's single tokens), and a wave writes a group at a time, a lane the bytes of two
// dims.  A dword that other tokens share is put together by an atomic xor of the bits that change.
template <typename T, int D>
__global__ __launch_bounds__(KV4_THREADS) void kv4_append_many_kernel(
    const T* __restrict__ k, const T* __restrict__ v, long st_t, long st_h, uint8_t* __restrict__ kc,
    uint8_t* __restrict__ vc, uint8_t* __restrict__ ks, uint8_t* __restrict__ vs, const int32_t* __restrict__ rows,
    const int32_t* __restrict__ pos, int N, int Hkv, int max_batch, int S) {
  constexpr int NB = D / 32, TOK = KV4_THREADS / NB;  // blocks of 32 dims of a token, tokens of a workgroup
  constexpr int LD = D / 8 + 1;                       // dwords of a token's codes in LDS
  __shared__ uint32_t s_c[TOK * LD];
  __shared__ Kv4Groups<TOK, NB> s_g;
  const int tid = threadIdx.x, tj = tid / NB, b = tid % NB, h = blockIdx.y, t0 = blockIdx.x * TOK, t = t0 + tj;
  const int nt = min(TOK, N - t0);
  int row = -1, p = -1, e = 0;
  uint32_t c[4] = {0, 0, 0, 0};
  if (t < N) {
    row = rows[t];
    p = pos[t];
    e = quantise32((blockIdx.z ? k : v) + (long)t * st_t + (long)h * st_h + 32 * b, c);
  }
  const bool ok = row >= 0 && row < max_batch && p >= 0 && p < S;
  const long stripe = ((long)row * Hkv + h) * (long)S;
  if (blockIdx.z) {                                  // (V's workgroups take longer and start first)
    if (!ok) return;
    uint8_t* to = kc + stripe * (D / 2) + kv4_k_offset(p, 32 * b, D);
    if constexpr (D == 128) {
      *(lsk_i32x4*)to = (lsk_i32x4){(int)c[0], (int)c[1], (int)c[2], (int)c[3]};
    } else {                                         // (the next lane group's 16 dims lie 256 bytes on)
      *(uint2*)to = make_uint2(c[0], c[1]);
      *(uint2*)(to + 256) = make_uint2(c[2], c[3]);
    }
    ks[stripe * NB + kv4_ks_offset(p, 32 * b, D)] = (uint8_t)e;
    return;
  }
  if (ok) vs[stripe * NB + kv4_vs_offset(p, 32 * b, D)] = (uint8_t)e;
#pragma unroll
  for (int w = 0; w < 4; ++w) s_c[tj * LD + 4 * b + w] = c[w];
  s_g.put(tj, b, ok ? row : -1, p);
  __syncthreads();
  s_g.find(nt);
  __syncthreads();
  constexpr int LANES = D / 2, PER = 64 / LANES;      // lanes of a group, groups of a wave at a time
  const int lane = tid & 63, l = lane % LANES, fr = l >> 4, l16 = l & 15;
  for (int g = (tid >> 6) * PER + lane / LANES; g < s_g.n; g += KV4_THREADS / LANES) {
    const int j0 = s_g.first[g], n = s_g.first[g + 1] - j0, r = s_g.row[j0], q = s_g.pos[j0];
    if (r < 0) continue;
    // dims 32 fr + l16 and 16 more: positions q % 16 .. of 16, four bits each
    uint64_t lo = 0, hi = 0;
    const uint8_t* src = (const uint8_t*)(s_c + j0 * LD) + 16 * fr + (l16 >> 1);
    const int odd = 4 * (l16 & 1);
    for (int i = 0; i < n; ++i, src += 4 * LD) {
      const int sh = 4 * ((q & 15) + i);
      lo |= (uint64_t)(src[0] >> odd & 15u) << sh;
      hi |= (uint64_t)(src[8] >> odd & 15u) << sh;
    }
    uint8_t* to = vc + ((long)r * Hkv + h) * (long)S * (D / 2) + kv4_v_offset(q & ~15, 32 * fr + l16, D);
    if (n == 16) {
      *(lsk_i32x4*)to = (lsk_i32x4){(int)(uint32_t)lo, (int)(lo >> 32), (int)(uint32_t)hi, (int)(hi >> 32)};
    } else {
      const uint64_t mask = ((1ull << (4 * n)) - 1) << (4 * (q & 15));
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t mw = (uint32_t)(mask >> (32 * w)), x = (uint32_t)(lo >> (32 * w)), y = (uint32_t)(hi >> (32 * w));
        uint32_t* at = (uint32_t*)to + w;
        if (mw == 0xffffffffu) {
          at[0] = x;
          at[2] = y;
        } else if (mw) {
          put_bits(at, x, mw);
          put_bits(at + 2, y, mw);
        }
      }
    }
  }
}

// The way back: eight dims of a token a thread, so that a token's are written side by side.  V's groups go through LDS, two
// lanes exchanging a dim each so that a byte there holds two neighbouring dims.  (4001 tokens of 8 heads of 128, K and V: 8.5
// us, 2.4 TB/s of the bytes read and written; appended 8.3: every workgroup is resident and loads, turns and stores once.)
template <typename T, int D>
__global__ __launch_bounds__(KV4_THREADS) void kv4_read_many_kernel(
    const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const uint8_t* __restrict__ ks,
    const uint8_t* __restrict__ vs, const int32_t* __restrict__ rows, const int32_t* __restrict__ pos, T* __restrict__ k,
    T* __restrict__ v, int N, int Hkv, int max_batch, int S) {
  constexpr int NB = D / 32, TOK = KV4_THREADS / NB, LD = D / 8 + 1;
  constexpr int PARTS = D / 8, TP = KV4_THREADS / PARTS, PASSES = TOK / TP;
  __shared__ uint32_t s_c[TOK * LD];
  __shared__ Kv4Groups<TOK, 1> s_g;
  const int tid = threadIdx.x, h = blockIdx.y, t0 = blockIdx.x * TOK, nt = min(TOK, N - t0), d = 8 * (tid % PARTS);
  const bool is_k = blockIdx.z != 0;
  uint32_t c[PASSES], e[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int tj = tid / PARTS + i * TP, row = tj < nt ? rows[t0 + tj] : -1, p = tj < nt ? pos[t0 + tj] : -1;
    const bool ok = row >= 0 && row < max_batch && p >= 0 && p < S;
    const long stripe = ((long)row * Hkv + h) * (long)S;
    c[i] = 0;
    e[i] = 127;
    if (ok && is_k) {
      c[i] = *(const uint32_t*)(kc + stripe * (D / 2) + kv4_k_offset(p, d, D));
      e[i] = ks[stripe * NB + kv4_ks_offset(p, d, D)];
    } else if (ok) {
      e[i] = vs[stripe * NB + kv4_vs_offset(p, d, D)];
    }
    if (!is_k) {
      if (!ok) s_c[tj * LD + (d >> 3)] = 0;          // (outside the cache: zeros)
      s_g.put(tj, tid % PARTS, ok ? row : -1, p);
    }
  }
  if (!is_k) {
    __syncthreads();
    s_g.find(nt);
    __syncthreads();
    constexpr int LANES = D / 2, PER = 64 / LANES;
    const int lane = tid & 63, l = lane % LANES, fr = l >> 4, l16 = l & 15;
    for (int g = (tid >> 6) * PER + lane / LANES; g < s_g.n; g += KV4_THREADS / LANES) {
      const int j0 = s_g.first[g], n = s_g.first[g + 1] - j0, r = s_g.row[j0], q = s_g.pos[j0];
      if (r < 0) continue;                           // (LANES lanes at a time)
      const lsk_i32x4 u = *(const lsk_i32x4*)(vc + ((long)r * Hkv + h) * (long)S * (D / 2) +
                                              kv4_v_offset(q & ~15, 32 * fr + l16, D));
      // an even lane takes dims 32 fr + l16 and the next, the odd one beside it those 16 on
      uint32_t bytes[2][2];                          // [positions 0 .. 7, 8 .. 15][even, odd]
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t mine = (uint32_t)(l16 & 1 ? u[2 + w] : u[w]), give = (uint32_t)(l16 & 1 ? u[w] : u[2 + w]);
        const uint32_t got = __builtin_amdgcn_mov_dpp(give, 0xb1, 0xf, 0xf, false);  // quad_perm [1, 0, 3, 2]
        const uint32_t lo = l16 & 1 ? got : mine, hi = l16 & 1 ? mine : got;
        bytes[w][0] = (lo & 0x0f0f0f0fu) | (hi & 0x0f0f0f0fu) << 4;
        bytes[w][1] = (lo >> 4 & 0x0f0f0f0fu) | (hi & 0xf0f0f0f0u);
      }
      uint8_t* to = (uint8_t*)(s_c + j0 * LD) + 16 * fr + 8 * (l16 & 1) + (l16 >> 1);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = i - (q & 15);
        if (j >= 0 && j < n) to[j * 4 * LD] = (uint8_t)(bytes[i >> 3][i & 1] >> (8 * ((i & 7) >> 1)));
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PASSES; ++i) c[i] = s_c[(tid / PARTS + i * TP) * LD + (d >> 3)];
  }
  T* to = (is_k ? k : v) + ((long)(t0 + tid / PARTS) * Hkv + h) * D + d;
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
    if (tid / PARTS + i * TP < nt) store8(to + (long)i * TP * Hkv * D, c[i], __uint_as_float(e[i] << 23));
}

// The way back for few tokens.
template <typename T, int D>
__global__ __launch_bounds__(KV4_THREADS) void kv4_read_kernel(const uint8_t* __restrict__ kc,
                                                               const uint8_t* __restrict__ vc,
                                                               const uint8_t* __restrict__ ks,
                                                               const uint8_t* __restrict__ vs,
                                                               const int32_t* __restrict__ rows,
                                                               const int32_t* __restrict__ pos, T* __restrict__ k,
                                                               T* __restrict__ v, int N, int Hkv, int max_batch,
                                                               int S) {
  constexpr int PER = KV4_THREADS / (D / 2);
  const int t = blockIdx.x * PER + threadIdx.x / (D / 2), h = blockIdx.y, d = 2 * (threadIdx.x % (D / 2));
  if (t >= N) return;
  const int row = rows[t], p = pos[t];
  float o[2] = {0.f, 0.f};
  if (row >= 0 && row < max_batch && p >= 0 && p < S) {
    const long stripe = ((long)row * Hkv + h) * (long)S;
    if (blockIdx.z == 0) {
      kv4_values(kc[stripe * (D / 2) + kv4_k_offset(p, d, D)], ks[stripe * (D / 32) + kv4_ks_offset(p, d, D)], o);
    } else {
      const uint8_t* from = vc + stripe * (D / 2);
      const uint32_t lo = from[kv4_v_offset(p, d, D)], hi = from[kv4_v_offset(p, d + 1, D)];
      const int sh = 4 * (p & 1);
      kv4_values((lo >> sh & 15u) | (hi >> sh & 15u) << 4, vs[stripe * (D / 32) + kv4_vs_offset(p, d, D)], o);
    }
  }
  store2((blockIdx.z ? v : k) + ((long)t * Hkv + h) * D + d, o);
}

// Accepted paths to consecutive slots (lsk_kv_compact): a thread moves one dim of V, or two of K, slot after slot.  A
// source never lies before its destination, and the sources increase, so none is overwritten before it is read.
template <int D>
__global__ __launch_bounds__(2 * D) void kv4_compact_kernel(uint8_t* __restrict__ kc, uint8_t* __restrict__ vc,
                                                            uint8_t* __restrict__ ks, uint8_t* __restrict__ vs,
                                                            const int32_t* __restrict__ rows,
                                                            const int32_t* __restrict__ pos0,
                                                            const int64_t* __restrict__ acc,
                                                            const int32_t* __restrict__ path, int max_nodes,
                                                            int max_batch, int Hkv, int S) {
  const int b = blockIdx.x, h = blockIdx.y, layer = blockIdx.z, i = threadIdx.x;
  const int row = rows[b], p0 = pos0[b];
  const int n = (int)min(max(acc[b], (int64_t)0), (int64_t)(max_nodes - 1));
  if (row < 0 || row >= max_batch || p0 < 0 || p0 >= S) return;
  const long stripe = (((long)layer * max_batch + row) * Hkv + h) * (long)S;
  uint8_t *k = kc + stripe * (D / 2), *v = vc + stripe * (D / 2), *ke = ks + stripe * (D / 32), *ve = vs + stripe * (D / 32);
  for (int j = 1; j <= n; ++j) {
    const int node = path[(long)b * max_nodes + j];
    if (node <= j || node >= S - p0) continue;       // (it stays where it is; outside the cache)
    const int from = p0 + node, to = p0 + j;
    if (i < D) {
      const long at = kv4_v_offset(to, i, D);
      const uint32_t c = v[kv4_v_offset(from, i, D)] >> (4 * (from & 1)) & 15u;
      v[at] = (uint8_t)((v[at] & (to & 1 ? 0x0fu : 0xf0u)) | c << (4 * (to & 1)));
    } else if (i < D + D / 2) {
      const int d = 2 * (i - D);
      k[kv4_k_offset(to, d, D)] = k[kv4_k_offset(from, d, D)];
    } else if (i < D + D / 2 + D / 32) {
      const int d = 32 * (i - D - D / 2);
      ke[kv4_ks_offset(to, d, D)] = ke[kv4_ks_offset(from, d, D)];
      ve[kv4_vs_offset(to, d, D)] = ve[kv4_vs_offset(from, d, D)];
    }
  }
}

static int kv4_args(const char* what, int dtype, const void* k, const void* v, const void* kc, const void* vc,
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

#define KV4_LAUNCH(NAME, T, ...)                                                               \
  do {                                                                                         \
    if (head_dim == 128 && many) NAME##_many_kernel<T, 128><<<grid, KV4_THREADS, 0, st>>>(__VA_ARGS__); \
    else if (head_dim == 128) NAME##_kernel<T, 128><<<grid, KV4_THREADS, 0, st>>>(__VA_ARGS__); \
    else if (many) NAME##_many_kernel<T, 64><<<grid, KV4_THREADS, 0, st>>>(__VA_ARGS__);        \
    else NAME##_kernel<T, 64><<<grid, KV4_THREADS, 0, st>>>(__VA_ARGS__);                       \
  } while (0)

extern "C" int lsk_kv4_append(int dtype, const void* k, const void* v, long stride_t, long stride_h, void* k4, void* v4,
                              void* k_exp, void* v_exp, const int32_t* rows, const int32_t* pos, int n_tokens,
                              int n_kv_heads, int head_dim, int max_batch, int max_seq, void* stream) {
  const char* what = "lsk_kv4_append";
  if (int rc = kv4_args(what, dtype, k, v, k4, v4, k_exp, v_exp, rows, pos, n_tokens, n_kv_heads, head_dim, max_batch,
                        max_seq)) return rc;
  LSK_REQUIRE(stride_t >= 0 && stride_h >= 0, LSK_ESHAPE, "%s: negative strides", what);
  if (n_tokens == 0) return 0;
  const bool many = (long)n_tokens * n_kv_heads >= KV4_MANY;
  const int per = KV4_THREADS / (many ? head_dim / 32 : head_dim / 2);
  const dim3 grid((n_tokens + per - 1) / per, n_kv_heads, 2);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LSK_DTYPE_BF16)
    KV4_LAUNCH(kv4_append, uint16_t, (const uint16_t*)k, (const uint16_t*)v, stride_t, stride_h, (uint8_t*)k4,
               (uint8_t*)v4, (uint8_t*)k_exp, (uint8_t*)v_exp, rows, pos, n_tokens, n_kv_heads, max_batch, max_seq);
  else
    KV4_LAUNCH(kv4_append, float, (const float*)k, (const float*)v, stride_t, stride_h, (uint8_t*)k4,
               (uint8_t*)v4, (uint8_t*)k_exp, (uint8_t*)v_exp, rows, pos, n_tokens, n_kv_heads, max_batch, max_seq);
  return lsk_check_launch(what);
}

extern "C" int lsk_kv4_read(int dtype, const void* k4, const void* v4, const void* k_exp, const void* v_exp,
                            const int32_t* rows, const int32_t* pos, void* k, void* v, int n_tokens, int n_kv_heads,
                            int head_dim, int max_batch, int max_seq, void* stream) {
  const char* what = "lsk_kv4_read";
  if (int rc = kv4_args(what, dtype, k, v, k4, v4, k_exp, v_exp, rows, pos, n_tokens, n_kv_heads, head_dim, max_batch,
                        max_seq)) return rc;
  if (n_tokens == 0) return 0;
  const bool many = (long)n_tokens * n_kv_heads >= KV4_MANY;
  const int per = KV4_THREADS / (many ? head_dim / 32 : head_dim / 2);
  const dim3 grid((n_tokens + per - 1) / per, n_kv_heads, 2);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LSK_DTYPE_BF16)
    KV4_LAUNCH(kv4_read, uint16_t, (const uint8_t*)k4, (const uint8_t*)v4, (const uint8_t*)k_exp,
               (const uint8_t*)v_exp, rows, pos, (uint16_t*)k, (uint16_t*)v, n_tokens, n_kv_heads, max_batch, max_seq);
  else
    KV4_LAUNCH(kv4_read, float, (const uint8_t*)k4, (const uint8_t*)v4, (const uint8_t*)k_exp,
               (const uint8_t*)v_exp, rows, pos, (float*)k, (float*)v, n_tokens, n_kv_heads, max_batch, max_seq);
  return lsk_check_launch(what);
}
#undef KV4_LAUNCH

int lsk_kv4_compact(void* kc, void* vc, void* ks, void* vs, int n_layers, const int32_t* rows, const int32_t* pos0,
                    const int64_t* acc, const int32_t* path, int nb, int max_nodes, int n_kv_heads, int head_dim,
                    int max_batch, int max_seq, hipStream_t s) {
  const dim3 grid(nb, n_kv_heads, n_layers);
#define KV4_COMPACT(DD)                                                                                             \
  kv4_compact_kernel<DD><<<grid, 2 * DD, 0, s>>>((uint8_t*)kc, (uint8_t*)vc, (uint8_t*)ks, (uint8_t*)vs, rows, pos0, \
                                                 acc, path, max_nodes, max_batch, n_kv_heads, max_seq)
  if (head_dim == 128) KV4_COMPACT(128);
  else KV4_COMPACT(64);
#undef KV4_COMPACT
  return lsk_check_launch("lsk_kv_compact");
}
