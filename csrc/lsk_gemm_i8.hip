// 8-bit integer projections: activations quantised row by row, weights output channel by output channel, multiplied by
// the integer matrix instructions.
//
//   a row of x [M, K]: amax = max |x|, r = fl(127 / amax), s = fl(amax / 127), code = rne(x r), -127 .. 127;
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
#include "lsk_common.h"
#include "lsk_gemm.h"
#include "../include/lsk.h"

namespace {

template <int N, typename T>
__device__ __forceinline__ void load_row(const T* p, long k, long K, float* x) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = k + i < K ? Elem<T>::ld(p + k + i) : 0.f;
}

__device__ __forceinline__ uint32_t code_bits(float x, float r) {
  return __float_as_uint(__builtin_fmaf(x, r, 0x1.8p23f)) & 255u;
}

}  // namespace

#define QUANT_THREADS 256
// A workgroup a row: the largest magnitude, then the codes (the row comes from L2 the second time).
template <typename T>
__global__ __launch_bounds__(QUANT_THREADS) void quant_rows_kernel(const T* __restrict__ x, long ldx,
                                                                   uint8_t* __restrict__ codes,
                                                                   float* __restrict__ scales, int K, int nks) {
  __shared__ uint32_t s_m[QUANT_THREADS / 64];
  const int m = blockIdx.x;
  const T* row = x + (long)m * ldx;
  uint32_t top = 0;
  for (int c = threadIdx.x; c < 4 * nks; c += QUANT_THREADS) {
    float v[16];
    load_row<16>(row, 16L * c, K, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < QUANT_THREADS / 64; ++w) top = max(top, s_m[w]);
  const float amax = __uint_as_float(top);
  const bool finite = top < 0x7f800000u, some = finite && amax >= 0x1p-100f;
  const float r = some ? 127.f / amax : 0.f;
  if (threadIdx.x == 0) scales[m] = !finite ? __builtin_nanf("") : some ? amax / 127.f : 0.f;
  uint8_t* to = codes + (long)(m >> 4) * nks * 1024 + (m & 15) * 16;
  for (int c = threadIdx.x; c < 4 * nks; c += QUANT_THREADS) {
    float v[16];
    load_row<16>(row, 16L * c, K, v);
    lsk_i32x4 u;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t b = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) b |= (some ? code_bits(v[4 * w + i], r) : 0u) << (8 * i);
      u[w] = (int)b;
    }
    *(lsk_i32x4*)(to + (long)(c >> 2) * 1024 + (c & 3) * 256) = u;
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

// A workgroup of four waves owns 16 NS weight rows (silu-mul: of gate and of up) x 16 MS tokens; the waves take the
// k-steps round robin, both operands straight from memory as fragments, and their sums are added through LDS.
template <int NS, int MS, int EPI, typename T>
__global__ __launch_bounds__(256) void gemm_i8_kernel(const uint8_t* __restrict__ A, const float* __restrict__ sa,
                                                      const uint8_t* __restrict__ W, const float* __restrict__ sw,
                                                      T* __restrict__ C, long ldc, const T* __restrict__ R, long ldr,
                                                      int M, int N, int nks, int ffn) {
  constexpr int NT = EPI == LSK_EPI_SILU_MUL ? 2 * NS : NS;
  constexpr int E = NT * MS * 256;
  __shared__ __attribute__((aligned(16))) int red[4 * E];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g0 = blockIdx.x * NS, t0 = blockIdx.y * MS;
  const int ng = (N + 15) >> 4, mg = (M + 15) >> 4;
  const uint8_t *wp[NT], *ap[MS];
#pragma unroll
  for (int i = 0; i < NT; ++i) {                     // (groups past the last one: its copies, never stored)
    const int g = min(g0 + i % NS, ng - 1) + (i < NS ? 0 : ffn >> 4);
    wp[i] = W + (long)g * nks * 1024 + 16 * lane;
  }
#pragma unroll
  for (int i = 0; i < MS; ++i) ap[i] = A + (long)min(t0 + i, mg - 1) * nks * 1024 + 16 * lane;
  lsk_i32x4 acc[NT][MS];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int t = 0; t < MS; ++t) acc[a][t] = (lsk_i32x4){0, 0, 0, 0};
  for (int j = wave; j < nks; j += 4) {
    lsk_i32x4 wf[NT], af[MS];
#pragma unroll
    for (int i = 0; i < NT; ++i) wf[i] = __builtin_nontemporal_load((const lsk_i32x4*)(wp[i] + (long)j * 1024));
#pragma unroll
    for (int i = 0; i < MS; ++i) af[i] = *(const lsk_i32x4*)(ap[i] + (long)j * 1024);
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int t = 0; t < MS; ++t) acc[a][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[a], af[t], acc[a][t], 0, 0, 0);
  }
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int t = 0; t < MS; ++t) *(lsk_i32x4*)(red + wave * E + ((a * MS + t) * 64 + lane) * 4) = acc[a][t];
  __syncthreads();
  // (row 16 a + w of the tile, token 16 t + l of it)
  auto sum = [&](int a, int t, int w, int l) {
    const int e = ((a * MS + t) * 64 + (w >> 2) * 16 + l) * 4 + (w & 3);
    return red[e] + red[E + e] + red[2 * E + e] + red[3 * E + e];
  };
  for (int o = tid; o < NS * MS * 256; o += 256) {
    const int nl = o % (16 * NS), ml = o / (16 * NS);
    const int n = 16 * g0 + nl, m = 16 * t0 + ml;
    if (n >= N || m >= M) continue;
    const float s = sa[m];
    float v = (float)sum(nl >> 4, ml >> 4, nl & 15, ml & 15) * s * sw[n];
    if constexpr (EPI == LSK_EPI_SILU_MUL) {
      const float u = (float)sum((nl >> 4) + NS, ml >> 4, nl & 15, ml & 15) * s * sw[ffn + n];
      v = silu_f(v) * u;
    } else if constexpr (EPI == LSK_EPI_RESIDUAL) {
      v += Elem<T>::ld(R + (long)m * ldr + n);
    }
    Elem<T>::st(C + (long)m * ldc + n, v);
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
  const int nks = (K + 63) / 64;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LSK_DTYPE_BF16)
    quant_rows_kernel<uint16_t><<<M, QUANT_THREADS, 0, s>>>((const uint16_t*)x, ldx, (uint8_t*)codes, scales, K, nks);
  else
    quant_rows_kernel<float><<<M, QUANT_THREADS, 0, s>>>((const float*)x, ldx, (uint8_t*)codes, scales, K, nks);
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

template <typename T>
static int gemm_i8_launch(const char* what, const void* A, const float* sa, const void* W, const float* sw, void* C,
                          long ldc, const void* R, long ldr, int M, int N, int K, int epilogue, int ffn, hipStream_t s) {
  const int nks = (K + 63) / 64, ng = (N + 15) / 16, mg = (M + 15) / 16;
#define GEMM_I8(NS, MS, EPI)                                                                                     \
  gemm_i8_kernel<NS, MS, EPI, T><<<dim3((ng + NS - 1) / NS, (mg + MS - 1) / MS), 256, 0, s>>>(                    \
      (const uint8_t*)A, sa, (const uint8_t*)W, sw, (T*)C, ldc, (const T*)R, ldr, M, N, nks, ffn)
#define GEMM_I8_EPI(NS, MS)                                           \
  do {                                                                \
    if (epilogue == LSK_EPI_SILU_MUL) GEMM_I8(NS, MS, LSK_EPI_SILU_MUL); \
    else if (epilogue == LSK_EPI_RESIDUAL) GEMM_I8(NS, MS, LSK_EPI_RESIDUAL); \
    else GEMM_I8(NS, MS, LSK_EPI_NONE);                               \
  } while (0)
  if (mg == 1) GEMM_I8_EPI(1, 1);
  else if (mg == 2) GEMM_I8_EPI(2, 2);
  else GEMM_I8_EPI(2, 4);
#undef GEMM_I8_EPI
#undef GEMM_I8
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
