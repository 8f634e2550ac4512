// 8-bit integer projections: activations quantised row by row, weights output channel by output channel, multiplied by
// the integer matrix instructions.
//
//   a row of x [M, K]: amax = max |x|, r = fl(127 fl(1 / amax)), s = fl(amax / 127), code = rne(x r), -127 .. 127
//   (r as an array program computes 127 / amax: a reciprocal, then a product);
//   C[m][n] = epilogue(s_m sw_n sum_k code_m[k] codew_n[k])
//
// x r is rounded once, to an integer (fma with 1.5 * 2^23), so codes do not depend on how the product would round in
// fp32.  Sums of products are exact (32-bit integers; K <= 131072 keeps them below 2^31), so a result depends neither on
// the tile nor on the order of additions nor on what else is in the launch.  The epilogues are fp32 with one rounding at
// the end:
//   NONE s_m sw_n sum;   RESIDUAL that + R;   SILU_MUL silu(g) u, g and u the rows n and ffn + n of the weight.
// A row that holds a NaN or an infinity has the scale NaN; one with amax < 2^-100 the scale 0 (r would overflow).
//
// Codes of both sides are stored as the matrix instruction v_mfma_i32_16x16x64_i8 reads them: fragment (g, j) of 1 KiB
// holds rows 16 g .. + 15 and k = 64 j .. + 63, lane 16 lg + l16 the 16 bytes of row 16 g + l16 from k = 64 j + 16 lg;
// fragments ordered [g][j], zeros past K and (weights) past the rows.
#include <type_traits>

#include "lsk_common.h"
#include "lsk_gemm.h"
#include "../include/lsk.h"

namespace {

// sum * s * w for a token's scale s and a channel's w.  From 2^90 on, where sum * s alone could pass fp32's range, s goes in
// without 2^32, which comes back at the end (bits are the same: powers of two).
struct TokenScale {
  float s, up;
  __device__ __forceinline__ TokenScale(float x) : s(x > 0x1p90f ? x * 0x1p-32f : x), up(x > 0x1p90f ? 0x1p32f : 1.f) {}
  __device__ __forceinline__ float times(int sum, float w) const { return (float)sum * s * w * up; }
};

__device__ __forceinline__ uint32_t code_bits(float x, float r) {
  return __float_as_uint(__builtin_fmaf(x, r, 0x1.8p23f)) & 255u;
}

// 16 consecutive values of a row, as loaded (at any address that aligns one of them); zeros past K
template <typename T>
struct Raw16;
template <>
struct Raw16<uint16_t> {
  lsk_u32x4_u u[2];
  __device__ __forceinline__ void load(const uint16_t* p, int k, int K) {
    if (k + 16 <= K) {
      u[0] = *(const lsk_u32x4_u*)(p + k);
      u[1] = *(const lsk_u32x4_u*)(p + k + 8);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t lo = k + 2 * i < K ? p[k + 2 * i] : 0u, hi = k + 2 * i + 1 < K ? p[k + 2 * i + 1] : 0u;
        u[i >> 2][i & 3] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = u[i >> 3][(i >> 1) & 3];
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
};
template <>
struct Raw16<float> {
  lsk_f32x4_u u[4];
  __device__ __forceinline__ void load(const float* p, int k, int K) {
    if (k + 16 <= K) {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = *(const lsk_f32x4_u*)(p + k + 4 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) u[i >> 2][i & 3] = k + i < K ? p[k + i] : 0.f;
    }
  }
  __device__ __forceinline__ float get(int i) const { return u[i >> 2][i & 3]; }
};

// 4 consecutive outputs of a row, of which the first `left` exist (at any address that aligns one of them).  R may be C, here
// and below: the thread that writes an element has read it before, and no other does.
template <int EPI>
__device__ __forceinline__ void store_out(uint16_t* c, const uint16_t* r, float* o, int left) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  if (left >= 4) {
    if constexpr (EPI == LSK_EPI_RESIDUAL) {
      const lsk_u32x2_u u = *(const lsk_u32x2_u*)r;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
    }
    const bf16x4 b = {(__bf16)o[0], (__bf16)o[1], (__bf16)o[2], (__bf16)o[3]};
    *(lsk_u32x2_u*)c = __builtin_bit_cast(lsk_u32x2_u, b);
    return;
  }
  for (int i = 0; i < 4; ++i)
    if (i < left) c[i] = f2bf(EPI == LSK_EPI_RESIDUAL ? o[i] + bf2f(r[i]) : o[i]);
}
template <int EPI>
__device__ __forceinline__ void store_out(float* c, const float* r, float* o, int left) {
  if (left >= 4) {
    lsk_f32x4_u v = {o[0], o[1], o[2], o[3]};
    if constexpr (EPI == LSK_EPI_RESIDUAL) v += *(const lsk_f32x4_u*)r;
    *(lsk_f32x4_u*)c = v;
    return;
  }
  for (int i = 0; i < 4; ++i)
    if (i < left) c[i] = EPI == LSK_EPI_RESIDUAL ? o[i] + r[i] : o[i];
}

}  // namespace

#define QUANT_THREADS 256
// A workgroup a row: the largest magnitude, then the codes.  NC: 16-value pieces of a thread, held in registers between
// the two (0: longer rows, read again).  The 16 rows of a fragment go to one XCD, whose L2 puts their 16-byte stores
// together.  Bound by HBM: 2001 bf16 rows of 14336 22 us (86 MB read and written, 4.0 TB/s); one row of 2048 2.4.
template <typename T, int NC>
__global__ __launch_bounds__(QUANT_THREADS) void quant_rows_kernel(const T* __restrict__ x, long ldx,
                                                                   uint8_t* __restrict__ codes,
                                                                   float* __restrict__ scales, int M, int K, int nks) {
  __shared__ uint32_t s_m[QUANT_THREADS / 64];
  const int b = blockIdx.x >> 3, m = ((b >> 4) * 8 + (blockIdx.x & 7)) * 16 + (b & 15);
  if (m >= M) return;
  const T* row = x + (long)m * ldx;
  Raw16<T> v[NC > 0 ? NC : 1];
  uint32_t top = 0;
  auto look = [&](const Raw16<T>& r) {
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(r.get(i)) & 0x7fffffffu);
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i].load(row, 16 * ((int)threadIdx.x + i * QUANT_THREADS), K);
#pragma unroll
    for (int i = 0; i < NC; ++i) look(v[i]);
  } else {
    for (int c = threadIdx.x; c < 4 * nks; c += QUANT_THREADS) {
      v[0].load(row, 16 * c, K);
      look(v[0]);
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < QUANT_THREADS / 64; ++w) top = max(top, s_m[w]);
  const float amax = __uint_as_float(top);
  const bool finite = top < 0x7f800000u, some = finite && amax >= 0x1p-100f;
  const float r = some ? 127.f * (1.f / amax) : 0.f;
  if (threadIdx.x == 0) scales[m] = !finite ? __builtin_nanf("") : some ? amax / 127.f : 0.f;
  uint8_t* to = codes + (long)(m >> 4) * nks * 1024 + (m & 15) * 16;
  auto put = [&](const Raw16<T>& q, int c) {
    lsk_i32x4 u;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t y = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) y |= code_bits(q.get(4 * w + i), r) << (8 * i);
      u[w] = finite ? (int)y : 0;
    }
    *(lsk_i32x4*)(to + (long)(c >> 2) * 1024 + (c & 3) * 256) = u;
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = threadIdx.x + i * QUANT_THREADS;
      if (c < 4 * nks) put(v[i], c);
    }
  } else {
    for (int c = threadIdx.x; c < 4 * nks; c += QUANT_THREADS) {
      v[0].load(row, 16 * c, K);
      put(v[0], c);
    }
  }
}

// Codes [N, K] (row-major, ld) <-> fragments; zeros past N and K.
template <bool PACK>
__global__ __launch_bounds__(256) void pack_i8_kernel(const int8_t* __restrict__ src, int8_t* __restrict__ dst, long ld,
                                                      int N, int K, int nks, long n_lanes) {
  const long o = (long)blockIdx.x * 256 + threadIdx.x;
  if (o >= n_lanes) return;
  const int l = (int)(o & 63);
  const long f = o >> 6;
  const long row = f / nks * 16 + (l & 15), k = f % nks * 64 + 16 * (l >> 4);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const bool in = row < N && k + i < K;
    if constexpr (PACK) dst[o * 16 + i] = in ? src[row * ld + k + i] : (int8_t)0;
    else if (in) dst[row * ld + k + i] = src[o * 16 + i];
  }
}

// Few tokens: a workgroup of four waves owns 16 NS weight rows (silu-mul: of gate and of up) x 16 MS tokens; the waves
// take the k-steps round robin, U at a time with the next U in flight, both operands straight from memory as fragments,
// and add their sums up in LDS (integers: in any order).  Bound by the weights' bytes: 32 tokens of the 8B shape's gate and
// up projection 22 us (117 MB, 5.3 TB/s); one token of the 1B shape's o projection (4 MB) 4.3.
template <int NS, int MS, int EPI, typename T>
__global__ __launch_bounds__(256) void gemm_i8_kernel(const uint8_t* __restrict__ A, const float* __restrict__ sa,
                                                      const uint8_t* __restrict__ W, const float* __restrict__ sw,
                                                      T* __restrict__ C, long ldc, const T* __restrict__ R, long ldr,
                                                      int M, int N, int nks, int ffn) {
  constexpr bool SILU = EPI == LSK_EPI_SILU_MUL;
  constexpr int NW = 4, NT = SILU ? 2 * NS : NS, E = NT * MS * 256;
  constexpr int U = NT + MS <= 3 ? 8 : NT + MS <= 4 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) int red[E];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g0 = blockIdx.x * NS, t0 = blockIdx.y * MS;
  const int ng = (N + 15) >> 4, mg = (M + 15) >> 4;
  const long step_bytes = (long)nks * 1024;          // of a group
  // (rows and tokens past the last group: zeros)
  auto rsrc = [&](const uint8_t* p, int groups) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, groups * (int)step_bytes, LSK_BUFFER_RSRC_WORD3);
  };
  const __amdgpu_buffer_rsrc_t wr = rsrc(W + (long)g0 * step_bytes, min(NS, ng - g0));
  const __amdgpu_buffer_rsrc_t ur = rsrc(W + (long)(SILU ? (ffn >> 4) + g0 : g0) * step_bytes, min(NS, ng - g0));
  const __amdgpu_buffer_rsrc_t ar = rsrc(A + (long)t0 * step_bytes, min(MS, mg - t0));
  for (int e = tid; e < E; e += 64 * NW) red[e] = 0;
  lsk_i32x4 acc[NT][MS], wA[U][NT], aA[U][MS], wB[U][NT], aB[U][MS];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int t = 0; t < MS; ++t) acc[a][t] = (lsk_i32x4){0, 0, 0, 0};
  auto ld = [&](__amdgpu_buffer_rsrc_t r, int i, int so, auto nt) {
    return __builtin_bit_cast(lsk_i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, 16 * lane + i * (int)step_bytes, so,
                                                                               decltype(nt)::value));
  };
  const std::integral_constant<int, 2> stream;       // (a weight is read once)
  const std::integral_constant<int, 0> keep;
  auto load = [&](lsk_i32x4 (&w)[U][NT], lsk_i32x4 (&x)[U][MS], int j) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = j + u * NW, so = k < nks ? k * 1024 : 0x7fffffff;  // (past the last k-step: zeros)
#pragma unroll
      for (int i = 0; i < NT; ++i) w[u][i] = ld(i < NS ? wr : ur, i % NS, so, stream);
#pragma unroll
      for (int i = 0; i < MS; ++i) x[u][i] = ld(ar, i, so, keep);
    }
  };
  auto mul = [&](const lsk_i32x4 (&w)[U][NT], const lsk_i32x4 (&x)[U][MS]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int t = 0; t < MS; ++t)
          acc[a][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][a], x[u][t], acc[a][t], 0, 0, 0);
  };
  load(wA, aA, wave);
  for (int j = wave; j < nks; j += 2 * U * NW) {
    load(wB, aB, j + U * NW);
    mul(wA, aA);
    load(wA, aA, j + 2 * U * NW);
    mul(wB, aB);
  }
  __syncthreads();
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int t = 0; t < MS; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) atomicAdd(&red[((a * MS + t) * 4 + i) * 64 + lane], acc[a][t][i]);
  __syncthreads();
  // (row 16 a + w of the tile, token 16 t + l of it)
  auto sum = [&](int a, int t, int w, int l) { return red[((a * MS + t) * 4 + (w & 3)) * 64 + (w >> 2) * 16 + l]; };
  for (int o = tid; o < NS * MS * 256; o += 64 * NW) {
    const int nl = o % (16 * NS), ml = o / (16 * NS);
    const int n = 16 * g0 + nl, m = 16 * t0 + ml;
    if (n >= N || m >= M) continue;
    const TokenScale s(sa[m]);
    float v = s.times(sum(nl >> 4, ml >> 4, nl & 15, ml & 15), sw[n]);
    if constexpr (SILU) {
      const float u = s.times(sum((nl >> 4) + NS, ml >> 4, nl & 15, ml & 15), sw[ffn + n]);
      v = silu_f(v) * u;
    } else if constexpr (EPI == LSK_EPI_RESIDUAL) {
      v += Elem<T>::ld(R + (long)m * ldr + n);
    }
    Elem<T>::st(C + (long)m * ldc + n, v);
  }
}

// Many tokens: a workgroup of four waves owns 256 weight rows (silu-mul: 128 of gate and of up), 64 a wave, read straight
// into registers three k-steps ahead (no other wave needs them), x MG 16-token groups, staged through LDS half a chunk of
// four k-steps at a time and shared by the waves.  KP > 1: that many such sets of four waves share the k-steps.  Bound by
// the matrix instructions at the clock that they leave: 2001 tokens of the 8B shape's w2 110 us, 2.1 POP/s.
template <int NG, int MG, int KP, int EPI, typename T>
__global__ __launch_bounds__(256 * KP, NG * MG == 32 || KP > 1 ? 1 : 2) void gemm_i8_deep_kernel(
    const uint8_t* __restrict__ A, const float* __restrict__ sa, const uint8_t* __restrict__ W,
    const float* __restrict__ sw, T* __restrict__ C, long ldc, const T* __restrict__ R, long ldr, int M, int N, int nks,
    int ffn, int n_tiles, int m_blocks) {
  constexpr bool SILU = EPI == LSK_EPI_SILU_MUL;
  constexpr int WN = SILU ? NG / 2 : NG;             // output row groups of a wave
  constexpr int PU = MG / 2;                         // 16-byte pieces per thread of half a staged chunk
  constexpr int UNIT = MG * 2 * 1024;                // bytes of half a chunk: MG groups x 2 k-steps
  static_assert(MG % 2 == 0 && MG <= 8, "staging split");
  static_assert(KP == 1 || NG * (KP - 1) <= KP, "the parts' sums fit the staging buffers");
  __shared__ __attribute__((aligned(16))) uint8_t s_a[KP][2][UNIT];
  const int tid = threadIdx.x & 255, lane = tid & 63;
  const int part = KP > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t *const al0 = s_a[part][0], *const al1 = s_a[part][1];
  const int l16 = lane & 15, lg = lane >> 4;
  // pieces ordered 8 token blocks at a time, row tiles within them, token blocks innermost; each XCD takes one run of that
  // order, so that its workgroups share a few row tiles and token blocks through its L2
  const int total = n_tiles * m_blocks, run = (total + 7) >> 3;
  const int lin = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= run || lin >= total) return;
  const int sup = lin / (8 * n_tiles), rem = lin - sup * 8 * n_tiles;
  const int mcount = min(8, m_blocks - 8 * sup);
  const int tn = rem / mcount, mb = 8 * sup + (rem - tn * mcount);
  const int gtot = (M + 15) >> 4, ng = (N + 15) >> 4;
  const int gq = gtot / m_blocks, gr = gtot - gq * m_blocks;  // token groups of the block, dealt evenly
  const int g0 = mb * gq + min(mb, gr), gn = gq + (mb < gr ? 1 : 0);
  const unsigned wbytes = (unsigned)((SILU ? 2 * ffn : 16 * ng) >> 4) * (unsigned)nks * 1024u;
  const __amdgpu_buffer_rsrc_t wr =
      __builtin_amdgcn_make_buffer_rsrc((void*)W, (short)0, (int)wbytes, LSK_BUFFER_RSRC_WORD3);
  const __amdgpu_buffer_rsrc_t ar = __builtin_amdgcn_make_buffer_rsrc(
      (void*)A, (short)0, (int)((unsigned)gtot * (unsigned)nks * 1024u), LSK_BUFFER_RSRC_WORD3);
  const int r0 = (4 * tn + wave) * WN;               // this wave's first output row group
  unsigned wofs[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g)
    wofs[g] = (unsigned)((g < WN ? min(r0 + g, ng - 1) : (ffn >> 4) + min(r0 + g - WN, ng - 1)) * nks) * 1024u;
  // half a chunk: k-steps 2 u, 2 u + 1 of every group; its fragment wave + 4 p is group (wave + 4 p) / 2, k-step 2 u + its
  // parity
  unsigned aofs[PU];
#pragma unroll
  for (int p = 0; p < PU; ++p)
    aofs[p] = (unsigned)(min(g0 + min((wave >> 1) + 2 * p, gn - 1), gtot - 1) * nks) * 1024u;
  const int lofs = 16 * lane;
  lsk_i32x4 acc[NG][MG], wf[4][NG], af[2][MG], st[2][PU];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int t = 0; t < MG; ++t) acc[g][t] = (lsk_i32x4){0, 0, 0, 0};
  const int chunks = ((nks + 3) / 4 + KP - 1) / KP, first = part * chunks;  // chunks of a part of K, and its first one
  const int last = min(4 * (first + chunks), nks);   // behind the part's last k-step
  // a k-step past the last one: weights of zero (an offset past the buffer), activations of the last one
  auto kw = [&](int c, int i) { return 4 * c + i < last ? (unsigned)(4 * c + i) * 1024u : wbytes; };
  auto ka = [&](int c, int u) { return (unsigned)min(4 * c + 2 * u + (wave & 1), nks - 1) * 1024u; };
  auto load_w1 = [&](lsk_i32x4 (&w)[NG], unsigned ko, int g) {
    w[g] = __builtin_bit_cast(lsk_i32x4,
                              __builtin_amdgcn_raw_buffer_load_b128(wr, lofs, (int)(ko == wbytes ? ko : wofs[g] + ko), 0));
  };
  auto load_st = [&](unsigned ko, int u, int p) {
    st[u][p] = __builtin_bit_cast(lsk_i32x4, __builtin_amdgcn_raw_buffer_load_b128(ar, lofs, (int)(aofs[p] + ko), 0));
  };
  auto put_st = [&](int u, int p) { *(lsk_i32x4*)((u ? al1 : al0) + (wave + 4 * p) * 1024 + lofs) = st[u][p]; };
  auto read_a = [&](int ksi, int t) {
    return *(const lsk_i32x4*)((ksi >= 2 ? al1 : al0) + (t * 2 + (ksi & 1)) * 1024 + lofs);
  };
#pragma unroll
  for (int p = 0; p < PU; ++p) load_st(ka(first, 0), 0, p);
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int g = 0; g < NG; ++g) load_w1(wf[i], kw(first, i), g);
#pragma unroll
  for (int p = 0; p < PU; ++p) put_st(0, p);
#pragma unroll
  for (int p = 0; p < PU; ++p) load_st(ka(first, 1), 1, p);
#pragma unroll
  for (int p = 0; p < PU; ++p) load_st(ka(first + 1, 0), 0, p);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < MG; ++t) af[0][t] = read_a(0, t);
  // A k-step in MG slots of NG products: a slot also reads one A fragment of the next step and issues one or two of the
  // step's loads (a W fragment per row group; with LU >= 0 the pieces of half chunk LU) and, with PUT >= 0, writes a piece
  // of half chunk PUT to LDS.
  using std::integral_constant;
  auto step = [&](lsk_i32x4 (&wn)[NG], unsigned kn, const lsk_i32x4 (&w)[NG], const lsk_i32x4 (&a)[MG],
                  lsk_i32x4 (&an)[MG], int rks, unsigned kp, auto put_c, auto lu_c) {
    constexpr int PUT = decltype(put_c)::value, LU = decltype(lu_c)::value;
    auto mf = [&](int f) {
      const int g = f / MG, t = f - g * MG;
      acc[g][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[g], a[t], acc[g][t], 0, 0, 0);
    };
    auto ld = [&](int l) {
      if (l < NG) load_w1(wn, kn, l);
      else if (LU >= 0 && l < NG + PU) load_st(kp, LU, l - NG);
    };
#pragma unroll
    for (int i = 0; i < MG; ++i) {
      an[i] = read_a(rks, i);
#pragma unroll
      for (int j = 0; j < NG / 2; ++j) mf(NG * i + j);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MG < 8) {
        ld(2 * i);
        ld(2 * i + 1);
      } else {
        ld(i);
      }
#pragma unroll
      for (int j = NG / 2; j < NG; ++j) {
        mf(NG * i + j);
        if (j == NG / 2 && PUT >= 0 && i >= MG - PU) put_st(PUT, i - (MG - PU));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const integral_constant<int, 0> u0;
  const integral_constant<int, 1> u1;
  const integral_constant<int, -1> no;
  for (int c = first; c < first + chunks; ++c) {
    __builtin_amdgcn_sched_barrier(0);
    step(wf[3], kw(c, 3), wf[0], af[0], af[1], 1, 0, u1, no);
    __syncthreads();
    step(wf[0], kw(c + 1, 0), wf[1], af[1], af[0], 2, ka(c + 1, 1), no, u1);
    step(wf[1], kw(c + 1, 1), wf[2], af[0], af[1], 3, 0, u0, no);
    __syncthreads();
    step(wf[2], kw(c + 1, 2), wf[3], af[1], af[0], 0, ka(c + 2, 0), no, u0);
  }
  if constexpr (KP > 1) {                            // the parts' sums to the first one
    lsk_i32x4* const sums = (lsk_i32x4*)s_a;
    __syncthreads();
    if (part > 0) {
#pragma unroll
      for (int f = 0; f < NG * MG; ++f) sums[((part - 1) * NG * MG + f) * 256 + tid] = acc[f / MG][f % MG];
    }
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int f = 0; f < NG * MG; ++f)
#pragma unroll
      for (int k = 1; k < KP; ++k) acc[f / MG][f % MG] += sums[((k - 1) * NG * MG + f) * 256 + tid];
  }
  float ws[NG][4];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = (r0 + (g < WN ? g : g - WN)) * 16 + 4 * lg + i;
      ws[g][i] = sw[min(n, N - 1) + (g < WN ? 0 : ffn)];
    }
#pragma unroll
  for (int t = 0; t < MG; ++t) {
    const int m = (g0 + t) * 16 + l16;
    if (t >= gn || m >= M) continue;
    const TokenScale s(sa[m]);
#pragma unroll
    for (int g = 0; g < WN; ++g) {
      const int n = (r0 + g) * 16 + 4 * lg;
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = s.times(acc[g][t][i], ws[g][i]);
        if constexpr (SILU) o[i] = silu_f(o[i]) * s.times(acc[g + WN][t][i], ws[g + WN][i]);
      }
      store_out<EPI>(C + (long)m * ldc + n, EPI == LSK_EPI_RESIDUAL ? R + (long)m * ldr + n : nullptr, o, N - n);
    }
  }
}

static bool i8_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
#define I8_MAX_K 131072

extern "C" int lsk_quant_rows_i8(int dtype, const void* x, long ldx, void* codes, float* scales, int M, int K,
                                 void* stream) {
  const char* what = "lsk_quant_rows_i8";
  LSK_REQUIRE(x && codes && scales, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(dtype == LSK_DTYPE_BF16 || dtype == LSK_DTYPE_F32, LSK_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  LSK_REQUIRE(M >= 0 && K > 0 && K <= I8_MAX_K && (ldx >= K || M <= 1), LSK_ESHAPE, "%s: bad shape (K <= %d)", what,
              I8_MAX_K);
  LSK_REQUIRE(i8_aligned(codes), LSK_EARG, "%s: codes start at a multiple of 16 bytes", what);
  if (M == 0) return 0;
  const int nks = (K + 63) / 64, pieces = (4 * nks + QUANT_THREADS - 1) / QUANT_THREADS;
  const unsigned grid = (unsigned)((M + 127) / 128) * 128;
  hipStream_t s = (hipStream_t)stream;
#define QUANT(T, NC) \
  quant_rows_kernel<T, NC><<<grid, QUANT_THREADS, 0, s>>>((const T*)x, ldx, (uint8_t*)codes, scales, M, K, nks)
#define QUANT_T(T)                \
  do {                            \
    if (pieces == 1) QUANT(T, 1); \
    else if (pieces == 2) QUANT(T, 2); \
    else if (pieces <= 4) QUANT(T, 4); \
    else QUANT(T, 0);             \
  } while (0)
  if (dtype == LSK_DTYPE_BF16) QUANT_T(uint16_t);
  else QUANT_T(float);
#undef QUANT_T
#undef QUANT
  return lsk_check_launch(what);
}

static int pack_i8(const char* what, bool pack, const void* src, void* dst, long ld, int N, int K, void* stream) {
  LSK_REQUIRE(src && dst, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(N > 0 && K > 0 && K <= I8_MAX_K && (ld >= K || N == 1), LSK_ESHAPE, "%s: bad shape (K <= %d)", what,
              I8_MAX_K);
  LSK_REQUIRE(i8_aligned(pack ? dst : src), LSK_EARG, "%s: packed codes start at a multiple of 16 bytes", what);
  const int nks = (K + 63) / 64;
  const long lanes = (long)((N + 15) / 16) * nks * 64;
  const unsigned grid = (unsigned)((lanes + 255) / 256);
  hipStream_t s = (hipStream_t)stream;
  if (pack) pack_i8_kernel<true><<<grid, 256, 0, s>>>((const int8_t*)src, (int8_t*)dst, ld, N, K, nks, lanes);
  else pack_i8_kernel<false><<<grid, 256, 0, s>>>((const int8_t*)src, (int8_t*)dst, ld, N, K, nks, lanes);
  return lsk_check_launch(what);
}

extern "C" int lsk_pack_i8(const void* codes, long ld, void* packed, int N, int K, void* stream) {
  return pack_i8("lsk_pack_i8", true, codes, packed, ld, N, K, stream);
}

extern "C" int lsk_unpack_i8(const void* packed, void* codes, long ld, int N, int K, void* stream) {
  return pack_i8("lsk_unpack_i8", false, packed, codes, ld, N, K, stream);
}

// The many-token kernel's configurations (NG row groups a wave, MG token groups, KP parts of K) and the time of a launch
// of each, fitted to the presets' projections at 65 to 4001 tokens (MI355X, cold weights; within 10 % rms): with n the
// workgroups of the busiest CU and c the chunks of 256 k that one walks, us = a + b n + c (d + e n).  The one with the
// least is taken: over those 207 launches 1.3 % slower than the best of them on average.
struct DeepI8 {
  int ng, mg, kp;
  float a, b, d, e;
};
static const DeepI8 kDeepI8[] = {{1, 4, 4, 2.7f, 1.6f, 0.0f, 1.73f}, {1, 4, 2, 2.4f, 0.96f, 0.25f, 0.69f},
                                 {2, 4, 1, 2.2f, 1.5f, 0.24f, 0.50f}, {2, 4, 2, 2.9f, 1.8f, 0.07f, 1.1f},
                                 {2, 8, 1, 4.3f, 2.1f, 0.0f, 0.90f}, {4, 4, 1, 3.0f, 1.9f, 0.02f, 0.97f},
                                 {4, 8, 1, 5.5f, 4.6f, -0.56f, 1.84f}};
static const DeepI8 kDeepI8Silu[] = {{2, 4, 1, -2.0f, -0.07f, 1.1f, 0.62f}, {2, 8, 1, -3.3f, 3.8f, 1.15f, 0.80f},
                                     {4, 4, 1, -6.0f, 2.2f, 1.52f, 0.95f}, {4, 8, 1, -10.f, 15.8f, 0.90f, 1.4f}};

template <typename T>
static int gemm_i8_launch(const char* what, const void* A, const float* sa, const void* W, const float* sw, void* C,
                          long ldc, const void* R, long ldr, int M, int N, int K, int epilogue, int ffn, hipStream_t s) {
  const int nks = (K + 63) / 64, ng = (N + 15) / 16, mg = (M + 15) / 16;
  const bool silu = epilogue == LSK_EPI_SILU_MUL;
#define GEMM_I8_ARGS \
  (const uint8_t*)A, sa, (const uint8_t*)W, sw, (T*)C, ldc, (const T*)R, ldr, M, N, nks, ffn
  // Up to 64 tokens (two 64-token tiles where the weight has at most 256 row groups: w2 of the 8B shape at 96 tokens 27 us
  // against 33, qkv 15 against 11): each weight is read once, two row groups a workgroup where one each makes more than
  // 256 of them (16 tokens: qkv of the 8B shape 7.6 us against 8.4, o 7.2 against 6.0).  Operands of 2 GiB, which the
  // many-token kernel's offsets do not reach, go here too.
  const double bytes = (double)(silu ? 2 * ng : ng) * nks * 1024, a_bytes = (double)mg * nks * 1024;
  const bool few = M <= 64 || (M <= 128 && !silu && ng <= 256);
  if (few || bytes >= 2147483648.0 || a_bytes >= 2147483648.0) {
    const int mt = (mg + 3) / 4, ns = (long)ng * mt > 256 ? 2 : 1;
    const dim3 grid((ng + ns - 1) / ns, mt);
#define GEMM_I8(NS, MS, EPI) gemm_i8_kernel<NS, MS, EPI, T><<<grid, 256, 0, s>>>(GEMM_I8_ARGS)
#define GEMM_I8_EPI(NS, MS)                                              \
  do {                                                                   \
    if (silu) GEMM_I8(NS, MS, LSK_EPI_SILU_MUL);                         \
    else if (epilogue == LSK_EPI_RESIDUAL) GEMM_I8(NS, MS, LSK_EPI_RESIDUAL); \
    else GEMM_I8(NS, MS, LSK_EPI_NONE);                                  \
  } while (0)
#define GEMM_I8_NS(MS)                  \
  do {                                  \
    if (ns == 1) GEMM_I8_EPI(1, MS);    \
    else GEMM_I8_EPI(2, MS);            \
  } while (0)
    if (mg == 1) GEMM_I8_NS(1);
    else if (mg == 2) GEMM_I8_NS(2);
    else if (mg == 3) GEMM_I8_NS(3);
    else GEMM_I8_NS(4);
#undef GEMM_I8_NS
#undef GEMM_I8_EPI
#undef GEMM_I8
    return lsk_check_launch(what);
  }
  const DeepI8* best = nullptr;
  float least = 0.f;
  const DeepI8* const list = silu ? kDeepI8Silu : kDeepI8;
  for (int i = 0; i < (silu ? 4 : 7); ++i) {
    const DeepI8& d = list[i];
    const int cols = (silu ? 32 : 64) * d.ng;
    const float n = (float)(((long)((N + cols - 1) / cols) * ((mg + d.mg - 1) / d.mg) + 255) / 256);
    const float c = (float)(((nks + 3) / 4 + d.kp - 1) / d.kp);
    const float us = d.a + d.b * n + c * (d.d + d.e * n);
    if (best == nullptr || us < least) {
      best = &d;
      least = us;
    }
  }
  const int cols = (silu ? 32 : 64) * best->ng, nt = (N + cols - 1) / cols, mb = (mg + best->mg - 1) / best->mg;
  const unsigned grid = (unsigned)((nt * mb + 7) / 8 * 8);
#define GEMM_I8_DEEP(NG, MG, KP, EPI) \
  gemm_i8_deep_kernel<NG, MG, KP, EPI, T><<<grid, 256 * KP, 0, s>>>(GEMM_I8_ARGS, nt, mb)
#define GEMM_I8_DEEP_EPI(NG, MG, KP)                                                      \
  do {                                                                                    \
    if (epilogue == LSK_EPI_RESIDUAL) GEMM_I8_DEEP(NG, MG, KP, LSK_EPI_RESIDUAL);         \
    else GEMM_I8_DEEP(NG, MG, KP, LSK_EPI_NONE);                                          \
  } while (0)
  const int cfg = best->ng * 100 + best->mg * 10 + best->kp;
  if (silu) {
    if (cfg == 241) GEMM_I8_DEEP(2, 4, 1, LSK_EPI_SILU_MUL);
    else if (cfg == 281) GEMM_I8_DEEP(2, 8, 1, LSK_EPI_SILU_MUL);
    else if (cfg == 441) GEMM_I8_DEEP(4, 4, 1, LSK_EPI_SILU_MUL);
    else GEMM_I8_DEEP(4, 8, 1, LSK_EPI_SILU_MUL);
  } else if (cfg == 144) GEMM_I8_DEEP_EPI(1, 4, 4);
  else if (cfg == 142) GEMM_I8_DEEP_EPI(1, 4, 2);
  else if (cfg == 241) GEMM_I8_DEEP_EPI(2, 4, 1);
  else if (cfg == 242) GEMM_I8_DEEP_EPI(2, 4, 2);
  else if (cfg == 281) GEMM_I8_DEEP_EPI(2, 8, 1);
  else if (cfg == 441) GEMM_I8_DEEP_EPI(4, 4, 1);
  else GEMM_I8_DEEP_EPI(4, 8, 1);
#undef GEMM_I8_DEEP_EPI
#undef GEMM_I8_DEEP
#undef GEMM_I8_ARGS
  return lsk_check_launch(what);
}

extern "C" int lsk_gemm_i8(int dtype, const void* A, const float* a_scales, const void* W, const float* w_scales, void* C,
                           long ldc, const void* R, long ldr, int M, int N, int K, int epilogue, int ffn,
                           void* stream) {
  const char* what = "lsk_gemm_i8";
  LSK_REQUIRE(A && a_scales && W && w_scales && C, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(dtype == LSK_DTYPE_BF16 || dtype == LSK_DTYPE_F32, LSK_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  LSK_REQUIRE(epilogue == LSK_EPI_NONE || epilogue == LSK_EPI_RESIDUAL || epilogue == LSK_EPI_SILU_MUL,
              LSK_EUNSUPPORTED, "%s: epilogue %d", what, epilogue);
  LSK_REQUIRE(M >= 0 && N > 0 && K > 0 && K <= I8_MAX_K && M <= (1 << 20) && (ldc >= N || M <= 1), LSK_ESHAPE,
              "%s: bad shape (K <= %d)", what, I8_MAX_K);
  LSK_REQUIRE(epilogue != LSK_EPI_RESIDUAL || (R && (ldr >= N || M <= 1)), LSK_EARG, "%s: residual without R", what);
  LSK_REQUIRE(epilogue != LSK_EPI_SILU_MUL || (ffn == N && N % 16 == 0), LSK_ESHAPE,
              "%s: silu-mul over ffn %d and N %d (equal, a multiple of 16)", what, ffn, N);
  LSK_REQUIRE(i8_aligned(A) && i8_aligned(W), LSK_EARG, "%s: codes start at multiples of 16 bytes", what);
  if (M == 0) return 0;
  if (dtype == LSK_DTYPE_BF16)
    return gemm_i8_launch<uint16_t>(what, A, a_scales, W, w_scales, C, ldc, R, ldr, M, N, K, epilogue, ffn,
                                    (hipStream_t)stream);
  return gemm_i8_launch<float>(what, A, a_scales, W, w_scales, C, ldc, R, ldr, M, N, K, epilogue, ffn,
                               (hipStream_t)stream);
}
