// Verify / decode attention over an 8-bit KV cache, and over trees of drafted tokens.
//
// Rule: token t of a block {q_start, pos0, T, row} sits in slot pos0 + t of its cache row (this call's K / V already
// appended) and reads the slots 0 .. pos0 + t.  With a mask it reads, of the block's own slots pos0 .. pos0 + t, only
// those whose bit is set: bit j (word j / 32, bit j % 32) of token t's mask words says that it reads node j of its
// block.  A tree of drafted tokens sets the bits of a node's ancestors and of the node itself.  A row that reads
// nothing gets zeros.
//
//   out = sum_p w_p v_p / sum_p w_p,   w_p = exp2(s_p - max s),   s_p = scale log2(e) (q . k_p)
//
// Work items, their records and the splits of long contexts are lsk_cache_attn_plan's (below).  Two kernels walk them:
// cache_attn_kernel, whose waves share the positions of up to two row groups of 32 rows, and cache_tree_kernel for
// trees of more rows, whose waves share K and V.
//
// Both cache formats are read as 1 KiB fragments in lane order, 64 D bytes per block of STEP positions:
//   bf16   STEP = 32: K fragment (a, f), lane 16 lg + l16: position 8 (l16 / 4) + 4 a + l16 % 4,
//          d = 32 f + 8 lg .. + 7; V^T: row d, positions 8 lg .. + 7.
//   8-bit  STEP = 64: e4m3 codes; K fragment (a, j): position 16 (l16 / 4) + 4 a + l16 % 4, d = 64 j + 16 lg .. + 15
//          (two MFMA operands of 8 d each); V^T: row d, positions 16 lg .. + 15 (two operands of 8 positions each).
//          A position's K and V are its codes times 2^(ks - 127) and 2^(vs - 127).
// Per step of a wave (v_mfma_f32_16x16x32_bf16): S^T[pos][q] = K Q^T, whose rows are mapped to positions so that lane
// group lg ends up with the consecutive positions its V^T load needs; online softmax with fp32 statistics; O^T[d][q] +=
// V^T P^T.  e4m3 values times a power of two are bf16 values, so the conversions in registers are exact and K's scale
// costs nothing (the conversion takes one); V's scale, which differs per position, multiplies the weights.  The weights
// are rounded to bf16 for the second product, as the ragged attention's are (by at most 2^-8 each, independent of one
// another: with the bf16 output's rounding the error against 64 bits is 0.0021 to 0.0023 of the outputs' size, where
// fp32 weights leave 0.0017); the sum of the weights is taken before that rounding.
//
// The waves of a row group take the steps round robin and are merged in wave order.  Which wave takes a step and every
// order of additions depend on absolute positions only: a row's result never depends on what else is in the launch.  An
// fp32 chain (every ancestor's bit set) gives the ragged attention's bits.
#include <algorithm>
#include <exception>
#include <type_traits>
#include <utility>
#include <vector>

#include "lsk_attn.h"
#include "../include/lsk.h"

namespace {

struct CacheAttnArgs {
  const uint16_t* q;      // [N] x [Hq] x [D], strides below
  long q_st, q_sh;        // elements between tokens and between heads
  const void* kc;         // K and V cache of the layer
  const void* vc;
  const uint8_t* ks;      // [B, Hkv, S] biased exponents (8-bit cache)
  const uint8_t* vs;
  const uint32_t* mask;   // [N, W]
  int W;
  const int32_t* recs;
  int n_rounds;
  uint16_t* out;          // [N, Hq * D]
  float* o_part;          // split partials: [part][Hkv][part_rows][D], and (m, l) of each
  float* ml_part;
  int part_rows;
  int G, Hkv, S;
  float scale_log2;
};

// The mask bits of a token for its block's slots rel .. rel + 31, relative to pos0: slots before the block are read by
// every token; bits past the words are 0.
__device__ __forceinline__ uint32_t mask_window(const uint32_t* words, int W, int rel) {
  const int w = rel >> 5, sh = rel & 31;
  const uint32_t lo = (w >= 0 && w < W) ? words[w] : 0u;
  const uint32_t hi = (w + 1 >= 0 && w + 1 < W) ? words[w + 1] : 0u;
  uint32_t bits = (uint32_t)(((((uint64_t)hi) << 32) | lo) >> sh);
  if (rel < 0) bits |= rel <= -32 ? 0xffffffffu : (1u << -rel) - 1u;
  return bits;
}

// Whether token t of a block reads a slot at all: one before the block, or a node whose bit is set.
__device__ __forceinline__ bool reads_any(const uint32_t* words, int W, int t, int pos0) {
  uint32_t any = pos0 > 0 ? 1u : 0u;
  for (int w = 0; w < W && 32 * w <= t; ++w) any |= words[w] & (t - 32 * w >= 31 ? ~0u : (2u << (t - 32 * w)) - 1u);
  return any != 0u;
}

// 8 e4m3 codes -> bf16, times a power of two (exact)
__device__ __forceinline__ lsk_bf16x8 codes_to_bf16(uint32_t x, uint32_t y, float scale) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false);
  const bf2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true);
  const bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, false);
  const bf2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, true);
  return (lsk_bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float exp_bits(uint32_t byte) { return __uint_as_float(byte << 23); }

}  // namespace

#define ORDER() __builtin_amdgcn_sched_barrier(0)  // (keeps the loads and conversions where their registers are free)
#define LAG 8.0f
// A row's running maximum before its first score: finite, so that a score of -infinity gets the weight 0 also where the
// row has read no other (against a maximum of -infinity it would be exp2(NaN)); no finite score lies below it.
#define M_NONE (-3.4028234663852886e38f)

// K / V through buffer loads over an item's (row, KV head) stripe, whose range ends with the block that holds the
// item's last position: loads past it give zeros without touching memory, so the next step's are unconditional (under
// a branch the compiler would wait for them early).
struct Stripe {
  __amdgpu_buffer_rsrc_t k, v, ks, vs;
};
template <int D, bool KV8>
__device__ __forceinline__ Stripe cache_stripe(const CacheAttnArgs& A, int crow, int kvh, int kv_hi) {
  constexpr int STEP = KV8 ? 64 : 32;
  const long st = (long)crow * A.Hkv + kvh;
  const long bytes = (long)(A.S / STEP) * 64 * D;    // of a whole stripe
  const int end = min(A.S, (kv_hi + STEP - 1) / STEP * STEP);
  Stripe s;
  s.k = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)A.kc + st * bytes), (short)0, end / STEP * 64 * D,
                                          LSK_BUFFER_RSRC_WORD3);
  s.v = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)A.vc + st * bytes), (short)0, end / STEP * 64 * D,
                                          LSK_BUFFER_RSRC_WORD3);
  if constexpr (KV8) {
    s.ks = __builtin_amdgcn_make_buffer_rsrc((void*)(A.ks + st * A.S), (short)0, end, LSK_BUFFER_RSRC_WORD3);
    s.vs = __builtin_amdgcn_make_buffer_rsrc((void*)(A.vs + st * A.S), (short)0, end, LSK_BUFFER_RSRC_WORD3);
  }
  return s;
}

// A step's V as loaded (row d = 16 c + l16, this lane's slots): clears the values past the first nk slots and the
// non-finite ones; bit u of the result: slot u of the step holds a non-finite value.
template <bool KV8, int CT>
__device__ __forceinline__ uint64_t clear_odd(lsk_i32x4 (&vr)[CT], int nk) {
  constexpr int PER = KV8 ? 4 : 2, BITS = 32 / PER;  // slots of a dword, bits of a value
  constexpr int NE = 4 * PER;
  uint32_t any[4];                                   // the top bits of this lane's non-finite values
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int m = nk - PER * w;
    const uint32_t keep = m >= PER ? 0xffffffffu : m <= 0 ? 0u : (1u << (BITS * m)) - 1u;
    any[w] = 0;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const uint32_t x = (uint32_t)vr[c][w] & keep;
      const uint32_t nf = KV8 ? ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u
                              : ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
      vr[c][w] = (int)(x & ~((nf - (nf >> (BITS - 1))) | nf));
      any[w] |= nf;
    }
  }
  uint64_t odd = 0;
  if (__builtin_amdgcn_ballot_w64((any[0] | any[1] | any[2] | any[3]) != 0u) != 0ull) {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const uint64_t lanes = __builtin_amdgcn_ballot_w64((any[e / PER] >> (BITS * (e % PER) + BITS - 1)) & 1u);
#pragma unroll
      for (int g = 0; g < 4; ++g) odd |= ((lanes >> (16 * g)) & 0xffffull) ? 1ull << (NE * g + e) : 0ull;
    }
  }
  return odd;
}

// The non-finite values of V that clear_odd took out, for the rows that read them.
template <bool KV8, bool TREE, int QT, int CT>
__device__ __forceinline__ void add_odd(const CacheAttnArgs& A, __amdgpu_buffer_rsrc_t v, uint64_t odd, int sb,
                                        int q_start, int pos0, const int (&qpos)[QT], lsk_f32x4 (&oacc)[QT][CT],
                                        int wide = 0) {
  constexpr int STEP = KV8 ? 64 : 32, D = 16 * CT;
  const int lg = (threadIdx.x & 63) >> 4;
  while (odd != 0ull) {                              // (rare: one slot after the other, few registers)
    const int u = __builtin_ctzll(odd), kp = sb + u + (u & wide);  // (wide 0x18: groups of 8 slots, 16 apart)
    odd &= odd - 1;
    bool hit[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      hit[qt] = kp <= qpos[qt];
      if constexpr (TREE) {
        const int t = max(qpos[qt] - pos0, 0);
        hit[qt] = hit[qt] && (mask_window(A.mask + (long)(q_start + t) * A.W, A.W, kp - pos0) & 1u);
      }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ORDER();
        // V[kp][16 c + 4 lg + i]: a dim's slots of a block are 64 bytes in both formats
        const int so = kp / STEP * 64 * D + (16 * c + i) * 64 + kp % STEP * (KV8 ? 1 : 2);
        float x;
        if constexpr (KV8) {
          const uint32_t b = __builtin_amdgcn_raw_buffer_load_b8(v, 256 * lg, so, 0);
          x = (b & 0x7fu) == 0x7fu ? __builtin_nanf("") : 0.f;
        } else {
          x = bf2f((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(v, 256 * lg, so, 0));
          x = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? x : 0.f;
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          if (hit[qt]) oacc[qt][c][i] += x;
      }
  }
}

// The online softmax of one tile's 16 query columns over a step: s[a][e] are the scores of this lane's slots 4 a + e,
// of which `reads` says what the column reads (FULL: all), vsr V's exponents of the slots (8-bit); pb the weights for
// the second product.  A row's m only moves when a score passes it by more than LAG (weights up to 2^LAG; each row for
// itself, so the rows of a tile stay independent), which is seldom after the first step: then no maximum crosses lanes
// and nothing is rescaled.  Each lane sums its own slots' weights.
template <bool KV8, bool FULL, int NA, int CT, int HV>
__device__ __forceinline__ void softmax_tile(lsk_f32x4 (&s)[NA], uint32_t reads, lsk_i32x4 vsr, float scale_log2,
                                             float& m, float& l, lsk_f32x4 (&o)[CT], lsk_bf16x8 (&pb)[HV]) {
  float mt = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4 * NA; ++i) {
    if constexpr (!FULL) s[i >> 2][i & 3] = (reads >> i) & 1u ? s[i >> 2][i & 3] : -INFINITY;
    mt = fmaxf(mt, s[i >> 2][i & 3]);
  }
  mt *= scale_log2;
  if (__builtin_amdgcn_ballot_w64(mt > m + LAG) != 0ull) {
    mt = rows_max(mt);
    const bool up = mt > m + LAG;
    const float alpha = up ? fast_exp2(m - mt) : 1.f;
    m = up ? mt : m;
    l *= alpha;
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[c][i] *= alpha;
  }
  float rs = 0.f;
#pragma unroll
  for (int i = 0; i < 4 * NA; ++i) {
    float pe = fast_exp2(__builtin_fmaf(s[i >> 2][i & 3], scale_log2, -m));
    if constexpr (!FULL) pe = (reads >> i) & 1u ? pe : 0.f;
    rs += pe;
    float pv = pe;
    if constexpr (KV8) {
      pv = pe * exp_bits(((uint32_t)vsr[i >> 2] >> (8 * (i & 3))) & 255u);
      if constexpr (!FULL) pv = (reads >> i) & 1u ? pv : 0.f;  // (a slot never written: any exponent)
    }
    pb[i >> 3][i & 7] = static_cast<__bf16>(pv);
  }
  l += rs;
}

// A workgroup has four waves, and each CU two workgroups (n_slots): one's first loads and merge fall into the other's
// steps.  Against one workgroup of eight waves (8B heads, 8-bit, decode): 256 requests of 250 positions 28 us against
// 46, of 960 81 against 91, of 4000 313 against 311; 7B heads, 16 trees of 30 nodes and 960 positions 30 against 36;
// one request of 100000 positions, 1B heads, 25 against 23.
#define CACHE_WAVES 4
template <int D, int QT, bool KV8, bool TREE>
__global__ __launch_bounds__(64 * CACHE_WAVES, 2) void cache_attn_kernel(const CacheAttnArgs A) {
  constexpr int STEP = KV8 ? 64 : 32;                // positions per step of a wave
  constexpr int HV = STEP / 32;                      // 32-position halves of a step; a lane group has 8 slots of each
  constexpr int NE = 8 * HV;                         // slots of a lane group: NE consecutive ones
  constexpr uint32_t ALL = NE == 16 ? 0xffffu : 0xffu;
  constexpr int KF = D / 32;                         // K operands per 16-position tile
  constexpr int CT = D / 16;                         // 16-byte loads per lane of a step, for K and for V
  constexpr int NW = CACHE_WAVES;
  constexpr int GR = 16 * QT;                        // rows of a wave
  constexpr bool QREG = QT == 1;                     // one tile: Q fragments in registers (items of one row group)
  constexpr int MT = TREE || QT < ATTN_MERGE_TILES ? 1 : ATTN_MERGE_TILES;  // (two workgroups' LDS fits a CU's)
  constexpr int MR = 16 * MT;                        // rows of a wave merged per pass
  constexpr int QROWS = QREG ? 0 : TREE ? 2 * GR : GR;  // rows of an item at most
  constexpr int QLD = D + 8;                         // 16 rows' 16-byte reads hit distinct banks
  constexpr int QCH = D / 8;
  constexpr int QPT = QREG ? 1 : (QROWS * QCH + 64 * NW - 1) / (64 * NW);
  __shared__ __attribute__((aligned(16))) float s_o[NW][MR][D + 4];
  __shared__ __attribute__((aligned(16))) uint16_t s_q[QREG ? 1 : QROWS][QLD];
  __shared__ float s_ml[NW][2][GR];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int G = A.G, Hkv = A.Hkv, S = A.S, Hq = Hkv * G;
  const int32_t* my_recs = A.recs + (long)blockIdx.x * A.n_rounds * 8;

  // lr: log2 of the item's row groups; the waves of a row group share the item's steps
  struct Item {
    int q_start, row0, nrows, lr, kv_lo, kv_hi, part, pos0, crow, kvh;
  };
  auto fetch = [&](int r) {
    Item it;
    if (r >= A.n_rounds) {
      it.nrows = 0;
      return it;
    }
    const int32_t* wk = my_recs + (long)r * 8;
    it.q_start = wk[0]; it.row0 = wk[1]; it.nrows = wk[2] & 1023; it.lr = (wk[2] >> 10) & 3; it.kvh = wk[2] >> 12;
    it.kv_lo = wk[3]; it.kv_hi = wk[4]; it.part = wk[5]; it.pos0 = wk[6]; it.crow = wk[7];
    return it;
  };
  auto row_base = [&](const Item& it) { return TREE ? (wave & ((1 << it.lr) - 1)) * GR : 0; };  // the wave's first row
  // Q: row rl of an item -> 8 elements from d; operand f's k index 8 lg + e stands for d = q_dim(f) + e
  auto q_dim = [&](int f) { return KV8 ? 64 * (f >> 1) + 16 * lg + 8 * (f & 1) : 32 * f + 8 * lg; };
  auto q_ptr = [&](const Item& it, int rl) {
    const int r = it.row0 + rl, t = r / G, g = r - t * G;
    return A.q + (long)(it.q_start + t) * A.q_st + (long)(it.kvh * G + g) * A.q_sh;
  };
  auto ldq = [&](const uint16_t* p) { return __builtin_bit_cast(lsk_bf16x8, *(const lsk_u32x4_u*)p); };
  // Q of the next item waits in registers during the merge where they hold it (with 128 dims it spilled: 256 requests
  // of 1 to 9 tokens 199 us against 181 without; with 64 dims 53.9 against 55.2), else it comes after the merge
  constexpr bool QAHEAD = !TREE && D == 64;
  lsk_bf16x8 qst[QAHEAD ? QPT : 1];
  auto q_chunk = [&](const Item& it, int c) {        // 8 elements of a row, zeros past the rows
    const int row = c / QCH;
    return row < it.nrows ? ldq(q_ptr(it, row) + 8 * (c - row * QCH)) : (lsk_bf16x8){};
  };
  lsk_bf16x8 qreg[KF];
  auto q_load = [&](const Item& it) {
    if constexpr (QREG) {
      const bool valid = l16 < it.nrows;
      const uint16_t* p = q_ptr(it, valid ? l16 : 0);
#pragma unroll
      for (int f = 0; f < KF; ++f) qreg[f] = valid ? ldq(p + q_dim(f)) : (lsk_bf16x8){};
    } else if constexpr (QAHEAD) {
#pragma unroll
      for (int i = 0; i < QPT; ++i) qst[i] = q_chunk(it, tid + i * 64 * NW);
    }
  };
  auto q_store = [&](const Item& it) {
    if constexpr (!QREG) {
      int t0 = tid;
      asm volatile("" : "+v"(t0));                   // (the chunks' offsets, kept across the items, spilled)
#pragma unroll
      for (int i = 0; i < QPT; ++i) {
        const int c = t0 + i * 64 * NW, row = c / QCH;
        if (row < QROWS) *(lsk_bf16x8*)(&s_q[row][8 * (c - row * QCH)]) = QAHEAD ? qst[QAHEAD ? i : 0] : q_chunk(it, c);
      }
    }
  };
  auto stripe = [&](const Item& it) { return cache_stripe<D, KV8>(A, it.crow, it.kvh, it.kv_hi); };
  // Non-temporal where each byte is read once (32 trees of 16 nodes, 7B heads, 960 positions of bf16: 95 us against
  // 80); not where two row groups read it (39 nodes: 111 us against 118)
  constexpr int AUX = TREE && QT == 2 ? 0 : 2;
  auto ld = [&](__amdgpu_buffer_rsrc_t rs, int vo, int so) -> lsk_i32x4 {
    return __builtin_bit_cast(lsk_i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vo, so, AUX));
  };
  const int k_vo = 16 * lane, v_vo = 64 * l16 + 16 * lg;
  lsk_i32x4 kr[CT], vr[CT], ksr, vsr;                // this step's K and V as loaded
  constexpr int KL = CT / (2 * HV);                  // K loads of 16 slots
  auto load_k = [&](const Stripe& s, int sb, int a) {
#pragma unroll
    for (int i = a * KL; i < (a + 1) * KL; ++i) kr[i] = ld(s.k, k_vo, sb / STEP * 64 * D + i * 1024);
    if constexpr (KV8) {
      if (a == 2 * HV - 1) ksr = ld(s.ks, 16 * (l16 >> 2), sb);
    }
  };
  auto load_v = [&](const Stripe& s, int sb, int c) { vr[c] = ld(s.v, v_vo, sb / STEP * 64 * D + c * 1024); };
  auto load_vs = [&](const Stripe& s, int sb) {
    if constexpr (KV8) vsr = ld(s.vs, 16 * lg, sb);
  };
  // a wave without rows starts past the stripe
  auto first_step = [&](const Item& it) {
    return row_base(it) < it.nrows ? it.kv_lo + STEP * (TREE ? wave >> it.lr : wave) : S;
  };
  auto issue_first = [&](const Item& it) {
    q_load(it);
    const Stripe s = stripe(it);
    const int sb = first_step(it);
#pragma unroll
    for (int a = 0; a < 2 * HV; ++a) load_k(s, sb, a);
    load_vs(s, sb);
#pragma unroll
    for (int c = 0; c < CT; ++c) load_v(s, sb, c);
  };

  Item cur = fetch(0);
  if (cur.nrows == 0) return;
  issue_first(cur);
  Item nxt = fetch(1);
  if constexpr (!QREG) {
    q_store(cur);
    __syncthreads();
  }
  for (int r = 0; cur.nrows > 0; ++r) {
    const int kv_hi = cur.kv_hi, rb = row_base(cur);
    const int stride = STEP * (TREE ? NW >> cur.lr : NW);
    const Stripe sr = stripe(cur);
    int qpos[QT];                                    // the row's own slot; -1: no such row
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int rl = rb + 16 * qt + l16;
      qpos[qt] = rl < cur.nrows ? cur.pos0 + (cur.row0 + rl) / G : -1;
    }
    // slots that every row of the item reads
    const int full_lim = min(kv_hi - 1, TREE ? cur.pos0 - 1 : cur.pos0 + cur.row0 / G);
    lsk_f32x4 oacc[QT][CT];
    float m_run[QT], l_run[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m_run[qt] = M_NONE;
      l_run[qt] = 0.f;
#pragma unroll
      for (int c = 0; c < CT; ++c) oacc[qt][c] = (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
    }
    // bit e: row l16 of tile qt reads slot s0 + e, e < NE
    auto allow = [&](int qt, int s0) {
      const int n = min(kv_hi - 1, qpos[qt]) - s0 + 1;
      uint32_t bits = n >= NE ? ALL : n <= 0 ? 0u : (1u << n) - 1u;
      if constexpr (TREE) {
        const int t = max(qpos[qt] - cur.pos0, 0);
        bits &= mask_window(A.mask + (long)(cur.q_start + t) * A.W, A.W, s0 - cur.pos0);
      }
      return bits;
    };
    // One step.  FULL: every row reads all of its slots.  All QT tiles are computed,
    // also those without rows (copies of the loop for fewer tiles cost more in registers than they save).
    auto step = [&](auto full_, int sb) {
      constexpr bool FULL = decltype(full_)::value;
      // In a step that some row does not read whole, a slot whose V holds an infinity or NaN must not reach the rows
      // that do not read it (0 x NaN): the values past the item and the non-finite ones are cleared here, and the rows
      // that do read such a value get it after the products (below).
      uint64_t odd = 0;                              // bit u: slot sb + u holds a non-finite value
      if constexpr (!FULL) {
        odd = clear_odd<KV8>(vr, kv_hi - (sb + NE * lg));
      }
      // S^T = K Q^T, 16 slots at a time: sacc[qt][a][e] <-> slot s0 + 4 a + e.  The registers of a converted K take the
      // next step's at once.
      const int s0 = sb + NE * lg, sn = sb + stride;
      uint32_t reads[QT];                            // (the mask's words are asked for before the products)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) reads[qt] = FULL ? ALL : allow(qt, s0);
      lsk_f32x4 sacc[QT][2 * HV];
#pragma unroll
      for (int a = 0; a < 2 * HV; ++a) {
        if constexpr (KV8) ORDER();
        lsk_bf16x8 kf[KF];
        if constexpr (KV8) {
          const float sc = exp_bits(((uint32_t)ksr[a] >> (8 * (l16 & 3))) & 255u);
#pragma unroll
          for (int f = 0; f < KF; ++f) {
            const lsk_i32x4 x = kr[a * (KF / 2) + (f >> 1)];
            kf[f] = codes_to_bf16(x[2 * (f & 1)], x[2 * (f & 1) + 1], sc);
          }
          ORDER();
          load_k(sr, sn, a);
        } else {
#pragma unroll
          for (int f = 0; f < KF; ++f) kf[f] = __builtin_bit_cast(lsk_bf16x8, kr[a * KF + f]);
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          lsk_f32x4 acc = (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int f = 0; f < KF; ++f) {
            const lsk_bf16x8 qf =
                QREG ? qreg[f] : *(const lsk_bf16x8*)(&s_q[rb + 16 * qt + l16][q_dim(f)]);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[f], qf, acc, 0, 0, 0);
          }
          sacc[qt][a] = acc;
        }
      }
      ORDER();
      if constexpr (!KV8) {
#pragma unroll
        for (int a = 0; a < 2 * HV; ++a) load_k(sr, sn, a);
      }
      lsk_bf16x8 pb[QT][HV];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        if constexpr (KV8) ORDER();
        softmax_tile<KV8, FULL>(sacc[qt], reads[qt], vsr, A.scale_log2, m_run[qt], l_run[qt], oacc[qt], pb[qt]);
      }
      ORDER();
      load_vs(sr, sn);
      // O^T += V^T P^T; V's registers take the next step's V one by one
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        lsk_bf16x8 vf[HV];
        if constexpr (KV8) {
#pragma unroll
          for (int hv = 0; hv < HV; ++hv) vf[hv] = codes_to_bf16(vr[c][2 * hv], vr[c][2 * hv + 1], 1.f);
        } else {
          vf[0] = __builtin_bit_cast(lsk_bf16x8, vr[c]);
        }
#pragma unroll
        for (int hv = 0; hv < HV; ++hv)
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            oacc[qt][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[hv], pb[qt][hv], oacc[qt][c], 0, 0, 0);
        load_v(sr, sn, c);
        ORDER();
      }
      if constexpr (!FULL) {
        add_odd<KV8, TREE>(A, sr.v, odd, sb, cur.q_start, cur.pos0, qpos, oacc);
      }
    };
    int sb = first_step(cur);
    for (; sb + STEP - 1 <= full_lim; sb += stride) step(std::true_type{}, sb);
    for (; sb < kv_hi; sb += stride) step(std::false_type{}, sb);
    // the next item's Q and first K / V loads fly while this item is merged
    const Item done = cur;
    cur = nxt;
    if (cur.nrows > 0) {
      issue_first(cur);
      nxt = fetch(r + 2);
    }
    // merge a row group's waves in order: M = max m_w, e_w = exp2(m_w - M), L = sum e_w l_w, O = sum e_w O_w
    int tm = tid;
    asm volatile("" : "+v"(tm));                     // (no address of the merge is kept in registers across the steps)
    const int m16 = tm & 15, mg = (tm & 63) >> 4;
#pragma unroll
    for (int p0 = 0; p0 < QT; p0 += MT) {
      if (16 * p0 >= done.nrows) break;
#pragma unroll
      for (int qt = p0; qt < p0 + MT && qt < QT; ++qt) {
        const float l = rows_sum(l_run[qt]);
        if (mg == 0) {
          s_ml[wave][0][16 * qt + m16] = m_run[qt];
          s_ml[wave][1][16 * qt + m16] = l;
        }
        if (16 * qt < done.nrows - rb) {             // (a tile with rows)
#pragma unroll
          for (int c = 0; c < CT; ++c)
            *(float4*)(&s_o[wave][16 * (qt - p0) + m16][16 * c + 4 * mg]) =
                make_float4(oacc[qt][c][0], oacc[qt][c][1], oacc[qt][c][2], oacc[qt][c][3]);
        }
      }
      __syncthreads();
      // 4 consecutive d of one row per thread; RANKS waves hold a part of it
      auto merge = [&](auto ranks_) {
        constexpr int RANKS = decltype(ranks_)::value, NR = NW / RANKS;
        for (int e = tm; e < NR * MR * (D / 4); e += 64 * NW) {
          const int x = e / (D / 4), d = 4 * (e - x * (D / 4));
          const int rg = x / MR, ql = x - rg * MR, qr = 16 * p0 + ql;  // row group, row of the pass, row of the group
          const int row = rg * GR + qr;                                // row of the item
          if (qr >= GR || row >= done.nrows) continue;
          float M = M_NONE;
#pragma unroll
          for (int k = 0; k < RANKS; ++k) M = fmaxf(M, s_ml[k * NR + rg][0][qr]);
          float L = 0.f;
          float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int k = 0; k < RANKS; ++k) {
            const float mw = s_ml[k * NR + rg][0][qr];
            const float ew = mw == M ? 1.f : fast_exp2(mw - M);
            L = L + ew * s_ml[k * NR + rg][1][qr];
            const float4 ow = *(const float4*)(&s_o[k * NR + rg][ql][d]);
            O.x = O.x + ew * ow.x;
            O.y = O.y + ew * ow.y;
            O.z = O.z + ew * ow.z;
            O.w = O.w + ew * ow.w;
          }
          const int rr = done.row0 + row;
          const int tt = rr / G, gg = rr - tt * G;
          if (done.part < 0) {
            if constexpr (TREE) {                    // (0 / 0 stays where every score is -infinity)
              const uint32_t* words = A.mask + (long)(done.q_start + tt) * A.W;
              if (L == 0.f && !reads_any(words, A.W, tt, done.pos0)) L = 1.f;
            }
            lsk_u32x2_u pk;
            pk[0] = (uint32_t)f2bf(O.x / L) | ((uint32_t)f2bf(O.y / L) << 16);
            pk[1] = (uint32_t)f2bf(O.z / L) | ((uint32_t)f2bf(O.w / L) << 16);
            *(lsk_u32x2_u*)(A.out + ((long)(done.q_start + tt) * Hq + done.kvh * G + gg) * D + d) = pk;
          } else {
            const long slot = ((long)done.part * Hkv + done.kvh) * A.part_rows + row;
            *(float4*)(A.o_part + slot * D + d) = O;
            if (d == 0) {
              A.ml_part[slot * 2 + 0] = M;
              A.ml_part[slot * 2 + 1] = L;
            }
          }
        }
      };
      if (QREG || !TREE || done.lr == 0) merge(std::integral_constant<int, NW>{});
      else merge(std::integral_constant<int, NW / 2>{});
      if (p0 == 0 && cur.nrows > 0) q_store(cur);       // (every wave is past its steps)
      __syncthreads();
    }
  }
}

// Trees of more rows: an item of four row groups of 32 rows, a wave each, which read the same K and V.  These go
// through LDS, a step's at a time (8-bit: two steps'), in two buffers: a wave that reads them for itself takes its
// share of the CU's 64 bytes per clock (32 trees of 25 to 64 nodes, 8B heads, 128 to 1280 positions: 67 us without LDS,
// 42 with it). 8-bit codes become bf16 on the way, once for all the waves.  Q stays in registers.  Two workgroups fit a
// CU, so that one's waits fall into the other's steps (one of eight waves, merged at the end: 45 us).
// A CU is bound by the softmax's vector instructions beside the products and the reads of LDS: 32 positions of 256 rows
// take 1.3 us of it, of which the matrix instructions are 0.5.  The launch is bound by its fullest CU: every item is a
// workgroup of its own and all are resident at once (those 32 trees: 480 items, 23 to 28 us of such work a CU, 40 on
// the fullest).
#define TREE_WAVES 4
template <int D, bool KV8>
__global__ __launch_bounds__(64 * TREE_WAVES, 2) void cache_tree_kernel(const CacheAttnArgs A,
                                                                        const int32_t* __restrict__ items) {
  constexpr int KF = D / 32, CT = D / 16, NW = TREE_WAVES, QT = 2;
  constexpr int STEPS = KV8 ? 2 : 1, CHUNK = 32 * STEPS;  // steps and positions that go through LDS at a time
  constexpr int NE = 8;                              // slots of a lane in a step
  constexpr uint32_t ALL = 0xffu;
  constexpr int UNITS = 2 * CT;                      // 1 KiB bf16 fragments of a step: K's (a, f), then V's
  constexpr int UPW = UNITS / NW;                    // fragments of a chunk, as they are in the cache, per wave
  constexpr int HALF = UNITS * 1024, BUF = STEPS * HALF;
  __shared__ __attribute__((aligned(16))) char s_buf[2 * BUF];
  __shared__ __attribute__((aligned(16))) uint8_t s_vs[2][64];
  const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = A.G, Hkv = A.Hkv;
  const int32_t* wk = items + (long)blockIdx.x * 8;
  const int q_start = wk[0], row0 = wk[1], nrows = wk[2] & 1023, kvh = wk[2] >> 12;
  const int kv_lo = wk[3], kv_hi = wk[4], part = wk[5], pos0 = wk[6], crow = wk[7];
  const int rb = wave * 16 * QT;
  const Stripe sr = cache_stripe<D, KV8>(A, crow, kvh, kv_hi);
  lsk_i32x4 st[UPW];                                 // the wave's part of the next chunk, in flight
  uint32_t st_ks[UPW], st_vs;                        // 8-bit: exponents of this lane's K, and of position `lane`
  auto st_load = [&](int sb) {
#pragma unroll
    for (int i = 0; i < UPW; ++i) {                  // (a wave's fragments are all of K or all of V)
      const int w = wave * UPW + i;
      const int so = sb * (KV8 ? 1 : 2) * D + w % CT * 1024;
      st[i] = __builtin_bit_cast(lsk_i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                w < CT ? sr.k : sr.v, w < CT ? 16 * lane : 64 * l16 + 16 * lg, so, 0));
      if constexpr (KV8)
        st_ks[i] = __builtin_amdgcn_raw_buffer_load_b8(sr.ks, 16 * (l16 >> 2) + (l16 & 3),
                                                       sb + 4 * (w % CT / (KF / 2)), 0);
    }
    if constexpr (KV8) st_vs = __builtin_amdgcn_raw_buffer_load_b8(sr.vs, lane, sb, 0);
  };
  auto st_write = [&](int buf) {
    char* to = s_buf + buf * BUF + 16 * lane;
#pragma unroll
    for (int i = 0; i < UPW; ++i) {
      const int u = wave * UPW + i;
      if constexpr (KV8) {                           // codes -> bf16, K with its scale: once for all the waves
        const float sc = u < CT ? exp_bits(st_ks[i]) : 1.f;
        const int a = u / (KF / 2), f = 2 * (u % (KF / 2));
        char* lo = to + (u < CT ? (a >> 1) * HALF + ((a & 1) * KF + f) * 1024 : u * 1024);
        *(lsk_bf16x8*)lo = codes_to_bf16(st[i][0], st[i][1], sc);
        *(lsk_bf16x8*)(lo + (u < CT ? 1024 : HALF)) = codes_to_bf16(st[i][2], st[i][3], sc);
      } else {
        *(lsk_i32x4*)(to + u * 1024) = st[i];
      }
    }
    if constexpr (KV8) {
      if (wave == 0) s_vs[buf][lane] = (uint8_t)st_vs;
    }
  };
  st_load(kv_lo);
  lsk_bf16x8 qf[QT][KF];
  int qpos[QT];                                      // the row's own slot; -1: no such row
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int rl = rb + 16 * qt + l16, r = row0 + min(rl, nrows - 1), t = r / G, g = r - t * G;
    const uint16_t* q = A.q + (long)(q_start + t) * A.q_st + (long)(kvh * G + g) * A.q_sh;
    qpos[qt] = rl < nrows ? pos0 + t : -1;
#pragma unroll
    for (int f = 0; f < KF; ++f) {
      const int d = KV8 ? 64 * (f >> 1) + 16 * lg + 8 * (f & 1) : 32 * f + 8 * lg;
      qf[qt][f] = __builtin_bit_cast(lsk_bf16x8, *(const lsk_u32x4_u*)(q + d));
    }
  }
  lsk_f32x4 oacc[QT][CT];
  float m_run[QT], l_run[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m_run[qt] = M_NONE;
    l_run[qt] = 0.f;
#pragma unroll
    for (int c = 0; c < CT; ++c) oacc[qt][c] = (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
  }
  // Step j of the chunk at s2 (as in cache_attn_kernel): this lane's slots are s0 .. s0 + 7.
  auto step = [&](auto full_, int s2, int j, int buf) {
    constexpr bool FULL = decltype(full_)::value;
    const char* src = s_buf + buf * BUF + j * HALF + 16 * lane;
    const int s0 = s2 + (KV8 ? 16 * lg + 8 * j : 32 * j + 8 * lg);
    uint32_t reads[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      reads[qt] = ALL;
      if constexpr (!FULL) {
        const int n = min(kv_hi - 1, qpos[qt]) - s0 + 1, t = max(qpos[qt] - pos0, 0);
        reads[qt] = (n >= NE ? ALL : n <= 0 ? 0u : (1u << n) - 1u) &
                    mask_window(A.mask + (long)(q_start + t) * A.W, A.W, s0 - pos0);
      }
    }
    lsk_f32x4 sacc[QT][2];
    lsk_bf16x8 kf[2][KF];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int f = 0; f < KF; ++f) kf[a][f] = *(const lsk_bf16x8*)(src + (a * KF + f) * 1024);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) sacc[qt][a] = (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int f = 0; f < KF; ++f)                     // (four independent chains)
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          sacc[qt][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[a][f], qf[qt][f], sacc[qt][a], 0, 0, 0);
    ORDER();
    lsk_i32x4 vr[CT], vsr = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < CT; ++c) vr[c] = *(const lsk_i32x4*)(src + (CT + c) * 1024);
    if constexpr (KV8) {
      const uint2 e = *(const uint2*)(s_vs[buf] + 16 * lg + 8 * j);
      vsr[0] = (int)e.x;
      vsr[1] = (int)e.y;
    }
    lsk_bf16x8 pb[QT][1];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
      softmax_tile<KV8, FULL>(sacc[qt], reads[qt], vsr, A.scale_log2, m_run[qt], l_run[qt], oacc[qt], pb[qt]);
    uint64_t odd = 0;                                // (V is bf16 here in both formats)
    if constexpr (!FULL) odd = clear_odd<false>(vr, kv_hi - s0);
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        oacc[qt][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lsk_bf16x8, vr[c]), pb[qt][0],
                                                              oacc[qt][c], 0, 0, 0);
    if constexpr (!FULL)
      add_odd<KV8, true>(A, sr.v, odd, s2 + (KV8 ? 8 : 32) * j, q_start, pos0, qpos, oacc, KV8 ? 0x18 : 0);
  };
  st_write(0);
  st_load(kv_lo + CHUNK);
  int s2 = kv_lo, buf = 0;
  auto chunks = [&](auto full_, int end) {           // those that start before `end`
    for (; s2 < end; s2 += CHUNK, buf ^= 1) {
      __syncthreads();                               // (the other buffer's readers are done, this one is written)
#pragma nounroll
      for (int j = 0; j < STEPS; ++j) {
        if (s2 + 8 * j >= kv_hi || rb >= nrows) break;
        step(full_, s2, j, buf);
      }
      st_write(buf ^ 1);
      st_load(s2 + 2 * CHUNK);
    }
  };
  chunks(std::true_type{}, min(kv_hi, pos0) - CHUNK + 1);  // (every row reads them whole)
  chunks(std::false_type{}, kv_hi);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) l_run[qt] = rows_sum(l_run[qt]);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int rl = rb + 16 * qt + l16;
    if (rl >= nrows) continue;
    const int r = row0 + rl, t = r / G, g = r - t * G;
    float L = l_run[qt];
    if (L == 0.f && part < 0 && !reads_any(A.mask + (long)(q_start + t) * A.W, A.W, t, pos0)) L = 1.f;
    const long slot = ((long)part * Hkv + kvh) * A.part_rows + rl;
    uint16_t* o = A.out + ((long)(q_start + t) * G * Hkv + kvh * G + g) * D + 4 * lg;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const lsk_f32x4 v = oacc[qt][c];
      if (part < 0) {
        lsk_u32x2_u pk;
        pk[0] = (uint32_t)f2bf(v[0] / L) | ((uint32_t)f2bf(v[1] / L) << 16);
        pk[1] = (uint32_t)f2bf(v[2] / L) | ((uint32_t)f2bf(v[3] / L) << 16);
        *(lsk_u32x2_u*)(o + 16 * c) = pk;
      } else {
        *(lsk_f32x4*)(A.o_part + slot * D + 16 * c + 4 * lg) = v;
      }
    }
    if (part >= 0 && lg == 0) {
      A.ml_part[slot * 2 + 0] = m_run[qt];
      A.ml_part[slot * 2 + 1] = l_run[qt];
    }
  }
}

// Merge the splits of a row in split order: M = max_s m_s, w_s = exp2(m_s - M), out = sum w_s O_s / sum w_s l_s (zeros
// where the row reads nothing).  16 lanes per row: they take the splits' statistics side by side, then each D / 16 dims
// of the partial outputs, AHEAD splits' loads in flight, the first ones beside the statistics'.  (A wave per row with
// the loads behind the statistics: 32 trees of 64 nodes in three splits 57 us, now 20.)
#define COMBINE_ROWS 16
template <int D>
__global__ __launch_bounds__(256) void cache_combine_kernel(const int32_t* __restrict__ groups,
                                                            const float* __restrict__ o_part,
                                                            const float* __restrict__ ml_part,
                                                            const uint32_t* __restrict__ mask, int W,
                                                            uint16_t* __restrict__ out, int G, int Hkv, int part_rows) {
  constexpr int PER = D / 16, AHEAD = D == 64 ? 16 : 8, MS = ATTN_MAX_SPLITS / 16;
  const int32_t* gp = groups + (long)blockIdx.x * 8;
  const int q_start = gp[0], row0 = gp[1], nrows = gp[2], pf = gp[3], ns = gp[4], pos0 = gp[5];
  const int kvh = blockIdx.y, l16 = threadIdx.x & 15;
  const int rl = blockIdx.z * COMBINE_ROWS + (threadIdx.x >> 4);
  if (rl >= nrows) return;                           // (no barrier: a row's lanes are its own)
  const long slot0 = ((long)pf * Hkv + kvh) * part_rows + rl, step = (long)Hkv * part_rows;
  float m[MS], l[MS], w[MS], M = M_NONE;
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    m[i] = M_NONE;
    l[i] = 0.f;
    if (16 * i < ns && l16 + 16 * i < ns) {
      const float* p = ml_part + (slot0 + (l16 + 16 * i) * step) * 2;
      m[i] = p[0];
      l[i] = p[1];
    }
  }
  lsk_f32x4 v[AHEAD][PER / 4];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (s0 + j < ns)
#pragma unroll
        for (int i = 0; i < PER / 4; ++i)
          v[j][i] = *(const lsk_f32x4*)(o_part + (slot0 + (s0 + j) * step) * D + l16 * PER + 4 * i);
  };
  fetch(0);
#pragma unroll
  for (int i = 0; i < MS; ++i) M = fmaxf(M, m[i]);
#define COMBINE_ROR(N) \
  M = fmaxf(M, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(M), 0x120 + N, 0xf, 0xf, false)))
  COMBINE_ROR(8); COMBINE_ROR(4); COMBINE_ROR(2); COMBINE_ROR(1);
#undef COMBINE_ROR
#pragma unroll
  for (int i = 0; i < MS; ++i) w[i] = m[i] == M ? 1.f : fast_exp2(m[i] - M);
  float L = 0.f, O[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) O[i] = 0.f;
#pragma unroll
  for (int i = 0; i < MS; ++i) {
    if (16 * i >= ns) break;
    // lane j of the row to all of them
#define COMBINE_STEP(J)                                                                                             \
  if (16 * i + J < ns) {                                                                                            \
    const float wj = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(w[i]), 0x150 + J, 0xf, 0xf, false));  \
    const float lj = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(l[i]), 0x150 + J, 0xf, 0xf, false));  \
    L = L + wj * lj;                                                                                                \
    _Pragma("unroll") for (int d = 0; d < PER; ++d) O[d] = O[d] + wj * v[J % AHEAD][d / 4][d % 4];                  \
    if (J % AHEAD == AHEAD - 1) fetch(16 * i + J + 1);                                                              \
  }
    COMBINE_STEP(0) COMBINE_STEP(1) COMBINE_STEP(2) COMBINE_STEP(3) COMBINE_STEP(4) COMBINE_STEP(5) COMBINE_STEP(6)
    COMBINE_STEP(7) COMBINE_STEP(8) COMBINE_STEP(9) COMBINE_STEP(10) COMBINE_STEP(11) COMBINE_STEP(12)
    COMBINE_STEP(13) COMBINE_STEP(14) COMBINE_STEP(15)
#undef COMBINE_STEP
  }
  const int r = row0 + rl, t = r / G, g = r - t * G;
  if (L == 0.f && mask != nullptr && !reads_any(mask + (long)(q_start + t) * W, W, t, pos0)) L = 1.f;
  uint16_t* o = out + ((long)(q_start + t) * G * Hkv + kvh * G + g) * D + l16 * PER;
#pragma unroll
  for (int i = 0; i < PER; i += 4) {
    lsk_u32x2_u pk;
    pk[0] = (uint32_t)f2bf(O[i] / L) | ((uint32_t)f2bf(O[i + 1] / L) << 16);
    pk[1] = (uint32_t)f2bf(O[i + 2] / L) | ((uint32_t)f2bf(O[i + 3] / L) << 16);
    *(lsk_u32x2_u*)(o + i) = pk;
  }
}

// ----------------------------------------------------------------------------- fp32 trees
// The token-identity model's kernel: a wave per query row walks the row's slots in 64-position chunks (lane = slot,
// then lane = dim), in the ragged attention's order of additions (a chain gives its bits), skipping the slots the row
// does not read.  The four rows of a workgroup share the chunk's K and V in LDS, fetched in whole lines while the
// chunk before is worked on: a wave that reads K for itself touches 64 lines with every load, which bounded it (4
// trees of 12 nodes, 1B heads, 192 positions: 23.7 us against 11.3).  Bound by the chain of a row's additions.
#define F32_ROWS 4
// x[i] + x[i ^ 32], then ^ 16, 8, 4, 2, 1 (or the maxima): rotations by 8 and 4 within rows of 16 lanes equal the
// exchanges, the values having that period by then
template <typename F>
__device__ __forceinline__ float wave_reduce(float x, F f) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(b[0]), __uint_as_float(b[1]));
#define F32_DPP(CTRL) x = f(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CTRL, 0xf, 0xf, false)))
  F32_DPP(0x128);                                    // row_ror:8
  F32_DPP(0x124);                                    // row_ror:4
  F32_DPP(0x4e);                                     // quad_perm [2, 3, 0, 1]
  F32_DPP(0xb1);                                     // quad_perm [1, 0, 3, 2]
#undef F32_DPP
  return x;
}

template <int D>
__global__ __launch_bounds__(64 * F32_ROWS) void tree_attn_f32_kernel(
    const float* __restrict__ q, long q_st, long q_sh, const float* __restrict__ kc, const float* __restrict__ vc,
    const uint32_t* __restrict__ mask, int W, const int32_t* __restrict__ works, float* __restrict__ out, int G,
    int Hkv, int S, float scale) {
  constexpr int DPL = (D + 63) / 64;
  constexpr int KLD = D + 4, VLD = 68;               // floats of an LDS row of K (a position), of V (a dim)
  constexpr int NT = 64 * F32_ROWS, PER = 64 * D / 4 / NT;
  __shared__ __attribute__((aligned(16))) float s_k[64 * KLD];
  __shared__ __attribute__((aligned(16))) float s_v[D * VLD];
  __shared__ __attribute__((aligned(16))) float sp[F32_ROWS][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int kvh = blockIdx.y;
  const int32_t* wk = works + (long)blockIdx.x * 8;
  const int q_start = wk[0], row0 = wk[1], nrows = wk[2], pos0 = wk[6], crow = wk[7];
  const int first = blockIdx.z * F32_ROWS;
  if (first >= nrows) return;
  const bool active = first + wave < nrows;
  const int r = row0 + min(first + wave, nrows - 1), t = r / G, g = r - t * G;
  const int qpos = pos0 + t, qmax = pos0 + (row0 + min(first + F32_ROWS, nrows) - 1) / G;
  const float* qv = q + (long)(q_start + t) * q_st + (long)(kvh * G + g) * q_sh;
  const uint32_t* words = mask + (long)(q_start + t) * W;
  const long head_base = ((long)crow * Hkv + kvh) * (long)S * D;
  lsk_f32x4 ks[PER], vs[PER];
  uint32_t word;
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = 4 * ((int)threadIdx.x + i * NT);
      const bool in_k = base + e / D < S, in_v = base + 32 * (e / (32 * D)) < S;   // (S a multiple of 32)
      const lsk_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      ks[i] = in_k ? *(const lsk_f32x4_u*)(kc + head_base + (long)base * D + e) : zero;
      vs[i] = in_v ? *(const lsk_f32x4_u*)(vc + head_base + (long)base * D + e) : zero;
    }
    const int rel = base + lane - pos0;
    word = rel >= 0 && (rel >> 5) < W ? words[rel >> 5] >> (rel & 31) : 0u;
  };
  float m_run = -INFINITY, l_run = 0.f;
  float o[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) o[i] = 0.f;
  fetch(0);
  for (int base = 0; base <= qmax; base += 64) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = 4 * ((int)threadIdx.x + i * NT), f = e % (32 * D);
      *(lsk_f32x4*)&s_k[e / D * KLD + e % D] = ks[i];
      *(lsk_f32x4*)&s_v[f / 32 * VLD + 32 * (e / (32 * D)) + f % 32] = vs[i];
    }
    const int kp = base + lane;
    const bool reads = kp <= qpos && (kp < pos0 || (word & 1u));
    __syncthreads();
    if (base + 64 <= qmax) fetch(base + 64);
    if (!active || base > qpos) continue;
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < D; d += 4) {
      const lsk_f32x4 k4 = *(const lsk_f32x4*)&s_k[lane * KLD + d];
      s += qv[d] * k4[0];
      s += qv[d + 1] * k4[1];
      s += qv[d + 2] * k4[2];
      s += qv[d + 3] * k4[3];
    }
    s = reads ? s * scale : -INFINITY;
    const float mt = wave_reduce(s, [](float x, float y) { return fmaxf(x, y); });
    const float m_new = fmaxf(m_run, mt);
    const float alpha = (m_new == m_run) ? 1.f : lsk_exp(m_run - m_new);
    const float p = (s == -INFINITY) ? 0.f : lsk_exp(s - m_new);
    const float rs = wave_reduce(p, [](float x, float y) { return x + y; });
    l_run = l_run * alpha + rs;
    m_run = m_new;
    sp[wave][lane] = reads ? p : -1.f;               // (weights are never negative: -1 marks a slot not read)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      const float* vr = s_v + min(lane + 64 * i, D - 1) * VLD;
      float acc = o[i] * alpha;
      auto step = [&](float pj, float vj) { acc = pj < 0.f ? acc : acc + pj * vj; };
#pragma unroll
      for (int j = 0; j < 64; j += 4) {
        const lsk_f32x4 p4 = *(const lsk_f32x4*)&sp[wave][j], v4 = *(const lsk_f32x4*)&vr[j];
        step(p4[0], v4[0]);
        step(p4[1], v4[1]);
        step(p4[2], v4[2]);
        step(p4[3], v4[3]);
      }
      o[i] = acc;
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (!active) return;
  if (l_run == 0.f && !reads_any(words, W, t, pos0)) l_run = 1.f;
  float* orow = out + ((long)(q_start + t) * Hkv * G + kvh * G + g) * D;
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    const int d = lane + 64 * i;
    if (d < D) orow[d] = o[i] / l_run;
  }
}

// ----------------------------------------------------------------------------- host planner

// Work items of one launch: 32 rows (token x query head of the group) of a block per wave, 16 where no block has more,
// 48 for causal launches over 64 dims with larger blocks; the context in splits at absolute multiples of `split`.
//   causal  an item is one row group: 4 waves share its steps.
//   tree    a block of more than 32 rows gives an item 2 or 4 row groups (up to 128 rows), whose waves each walk more
//           of the positions: K / V come from memory once for all of them and fewer partial outputs are merged.  Items
//           of 4 are cache_tree_kernel's, one workgroup each, longest first.  Where the cache's (row, KV head) stripes
//           times the block's tiles of 32 rows are at most n_slots, each tile is an item instead (8B heads, 960
//           positions, 4 / 2 / 1 row groups: 64 stripes, 64-node trees 30 / 22 / 21 us; 128 stripes, 32 nodes
//           29 / 22 / 21, 64 nodes 32 / 34 / 37; 256 stripes, 16 nodes - / 29 / 26, 32 nodes 31 / 34 / 37, 64 nodes
//           46 / 60 / 69).
// The number of row groups follows from the block's rows and the cache alone, so it never makes a row's result depend
// on the batch.  Items go longest first to the least-loaded of n_slots persistent workgroups, as in lsk_attn_schedule.
static int cache_plan(const char* what, const int32_t* blocks, int nb, int group, int split, int max_batch,
                      int n_kv_heads, int head_dim, int kv8, int tree, int row_groups, int n_slots, int32_t* meta,
                      long meta_cap, long* counts) {
  LSK_REQUIRE(counts && (blocks || nb == 0), LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(nb >= 0 && group > 0 && split >= ATTN_TILE && split % ATTN_TILE == 0 && n_kv_heads > 0 &&
                  n_kv_heads < (1 << 19) && max_batch > 0 && n_slots > 0 && n_slots <= (1 << 16) &&
                  (row_groups == 0 || row_groups == 1 || row_groups == 2 || row_groups == 4),
              LSK_ESHAPE, "%s: bad arguments (split a multiple of %d, row_groups 0, 1, 2 or 4)", what, ATTN_TILE);
  LSK_REQUIRE(head_dim == 64 || head_dim == 128, LSK_EUNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", what,
              head_dim);
  const int step = kv8 ? 64 : 32;
  long most = 0, n_tokens = 0;
  for (int b = 0; b < nb; ++b) {
    const int32_t* bm = blocks + (long)b * 4;
    const long q_start = bm[0], pos0 = bm[1], T = bm[2];
    LSK_REQUIRE(T >= 0 && pos0 >= 0 && pos0 + T <= 0x7fffffffL - split && T * group < (1L << 31), LSK_ESHAPE,
                "%s: block %d has T=%ld pos0=%ld", what, b, T, pos0);
    LSK_REQUIRE(T == 0 || (q_start >= 0 && q_start + T <= 0x7fffffffL && bm[3] >= 0 && bm[3] < max_batch), LSK_ESHAPE,
                "%s: block %d starts at token %ld and is in row %d of %d", what, b, q_start, bm[3], max_batch);
    LSK_REQUIRE((pos0 + T + split - 1) / split <= ATTN_MAX_SPLITS, LSK_ESHAPE,
                "%s: block %d needs more than %d splits of %d positions", what, b, ATTN_MAX_SPLITS, split);
    most = T * group > most ? T * group : most;
    n_tokens += T;
  }
  const int tiles = most <= 16 ? 1 : most <= 32 || tree || head_dim == 128 ? 2 : 3;
  struct It { int32_t rec[8]; int cost; };
  thread_local std::vector<It> items, shared;
  thread_local std::vector<int32_t> groups;
  items.clear();
  shared.clear();
  groups.clear();
  long np = 0;
  int part_rows = 16 * tiles, used = 1;
  for (int b = 0; b < nb; ++b) {
    const int32_t* bm = blocks + (long)b * 4;
    const int pos0 = bm[1];
    const long rows = (long)bm[2] * group;
    int lr = 0;
    const bool few = (long)max_batch * n_kv_heads * ((rows + 31) / 32) <= n_slots;
    const int most_groups = row_groups ? row_groups : few ? 1 : 4;
    while (tree && (1 << lr) < most_groups && rows > (32L << lr)) ++lr;
    used = (1 << lr) > used ? 1 << lr : used;
    const int cap = (16 * tiles) << lr;
    for (long row0 = 0; row0 < rows; row0 += cap) {
      const int nrows = (int)(rows - row0 < cap ? rows - row0 : cap);
      const int end = (int)(pos0 + (row0 + nrows - 1) / group + 1);
      const int ns = (end + split - 1) / split;
      if (ns > 1) {
        const int32_t g[8] = {bm[0], (int32_t)row0, nrows, (int32_t)np, ns, pos0, 0, 0};
        groups.insert(groups.end(), g, g + 8);
        part_rows = cap > part_rows ? cap : part_rows;
      }
      LSK_REQUIRE((long)(items.size() + shared.size()) + (long)ns * n_kv_heads < (1L << 24), LSK_ESHAPE,
                  "%s: too many work items", what);
      for (int sp = 0; sp < ns; ++sp) {
        const int lo = sp * split, hi = lo + split < end ? lo + split : end;
        // in tenths of a one-tile step: a wave's steps, 1.5 times as long per further tile, and the item's own cost
        const int share = step * (CACHE_WAVES >> lr), steps = (hi - lo + share - 1) / share;
        const int cost = steps * (10 + 5 * (tiles - 1)) + 20 + 6 * (tiles - 1);
        for (int h = 0; h < n_kv_heads; ++h)
          (lr < 2 ? items : shared).push_back({{bm[0], (int32_t)row0, nrows | (lr << 10) | (h << 12), lo, hi,
                            ns > 1 ? (int32_t)(np + sp) : -1, pos0, bm[3]}, cost});
      }
      if (ns > 1) np += ns;
    }
  }
  const auto longer = [](const It& a, const It& b) { return a.cost > b.cost; };
  std::stable_sort(items.begin(), items.end(), longer);
  std::stable_sort(shared.begin(), shared.end(), longer);
  thread_local std::vector<std::pair<long, int>> heap;
  thread_local std::vector<int> slot_of, rank, count;
  heap.clear();
  for (int sl = 0; sl < n_slots; ++sl) heap.push_back({0, sl});
  const auto later = [](const std::pair<long, int>& a, const std::pair<long, int>& b) { return a > b; };
  slot_of.resize(items.size());
  rank.resize(items.size());
  count.assign(n_slots, 0);
  int rounds = 0;
  for (size_t i = 0; i < items.size(); ++i) {
    std::pop_heap(heap.begin(), heap.end(), later);
    auto& top = heap.back();
    slot_of[i] = top.second;
    rank[i] = count[top.second]++;
    rounds = count[top.second] > rounds ? count[top.second] : rounds;
    top.first += items[i].cost;
    std::push_heap(heap.begin(), heap.end(), later);
  }
  const long len = (long)groups.size() + 8L * n_slots * rounds + 8L * (long)shared.size();
  counts[0] = n_tokens; counts[1] = (long)groups.size() / 8; counts[2] = np; counts[3] = rounds; counts[4] = tiles;
  counts[5] = part_rows; counts[6] = len; counts[7] = used; counts[8] = (long)shared.size();
  if (meta == nullptr) return 0;
  LSK_REQUIRE(len <= meta_cap, LSK_EWORKSPACE, "%s: %ld metadata words > %ld", what, len, meta_cap);
  std::copy(groups.begin(), groups.end(), meta);
  int32_t* recs = meta + groups.size();
  std::fill(recs, recs + 8L * n_slots * rounds, 0);
  for (size_t i = 0; i < items.size(); ++i)
    std::copy(items[i].rec, items[i].rec + 8, recs + ((long)slot_of[i] * rounds + rank[i]) * 8);
  for (size_t i = 0; i < shared.size(); ++i)
    std::copy(shared[i].rec, shared[i].rec + 8, recs + ((long)n_slots * rounds + (long)i) * 8);
  return 0;
}

extern "C" int lsk_cache_attn_plan(const int32_t* blocks, int nb, int group, int split, int max_batch, int n_kv_heads,
                                   int head_dim, int kv8, int tree, int row_groups, int n_slots, int32_t* meta,
                                   long meta_cap, long* counts) {
  const char* what = "lsk_cache_attn_plan";
  try {
    return cache_plan(what, blocks, nb, group, split, max_batch, n_kv_heads, head_dim, kv8, tree, row_groups, n_slots,
                      meta, meta_cap, counts);
  } catch (const std::exception&) {
    LSK_REQUIRE(false, LSK_EWORKSPACE, "%s: out of host memory", what);
  }
}

extern "C" size_t lsk_cache_attn_workspace_bytes(int n_parts, int n_kv_heads, int part_rows, int head_dim) {
  const size_t rows = (size_t)n_parts * n_kv_heads * part_rows;
  return lsk_align_up(rows * head_dim * sizeof(float), 256) + lsk_align_up(rows * 2 * sizeof(float), 256);
}

// ----------------------------------------------------------------------------- entry points

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Checks and launches shared by the two entry points; kv8: the cache is 8-bit.
static int cache_attn(const char* what, bool kv8, CacheAttnArgs a, const int32_t* groups, int n_groups, int n_parts,
                      int n_slots, int n_shared, int tiles, int row_groups, int head_dim, float scale, void* workspace,
                      size_t ws_bytes, hipStream_t s) {
  LSK_REQUIRE(head_dim == 64 || head_dim == 128, LSK_EUNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", what,
              head_dim);
  LSK_REQUIRE(tiles == 1 || tiles == 2 || (tiles == 3 && head_dim == 64 && a.mask == nullptr), LSK_EARG,
              "%s: a plan of %d tiles", what, tiles);
  LSK_REQUIRE((row_groups == 1 && n_shared == 0) || a.mask != nullptr, LSK_EARG,
              "%s: a tree's plan (%d row groups) without a mask", what, row_groups);
  LSK_REQUIRE(n_slots > 0 && n_groups >= 0 && n_parts >= 0 && (n_groups > 0) == (n_parts > 0), LSK_EARG,
              "%s: a plan of %d slots, %d groups and %d partial slots", what, n_slots, n_groups, n_parts);
  LSK_REQUIRE(a.S % ATTN_TILE == 0 && (long)a.S * head_dim * 2 <= 0x7fffffffL, LSK_ESHAPE,
              "%s: max_seq %d (a multiple of %d, stripes below 2 GiB)", what, a.S, ATTN_TILE);
  LSK_REQUIRE(aligned16(a.kc) && aligned16(a.vc) && (!kv8 || (aligned16(a.ks) && aligned16(a.vs))), LSK_EARG,
              "%s: the cache tensors start at multiples of 16 bytes", what);
  if (n_parts > 0) {
    LSK_REQUIRE(a.part_rows >= 16 * tiles && a.part_rows <= 64 * tiles, LSK_EARG, "%s: a plan of %d rows per partial",
                what, a.part_rows);
    const size_t need = lsk_cache_attn_workspace_bytes(n_parts, a.Hkv, a.part_rows, head_dim);
    LSK_REQUIRE(workspace != nullptr && aligned16(workspace) && ws_bytes >= need && groups != nullptr, LSK_EWORKSPACE,
                "%s: an aligned workspace of %zu bytes needed, %zu given", what, need, ws_bytes);
    a.o_part = (float*)workspace;
    a.ml_part = (float*)((char*)workspace +
                         lsk_align_up((size_t)n_parts * a.Hkv * a.part_rows * head_dim * sizeof(float), 256));
  }
  LSK_REQUIRE(scale >= 0.f && scale <= 1e30f, LSK_EARG, "%s: scale %g (not negative)", what, (double)scale);
  a.scale_log2 = scale * 1.4426950408889634f;
  int rc = 0;
#define LSK_CACHE_ATTN(DD, QT, K8, TR) cache_attn_kernel<DD, QT, K8, TR><<<n_slots, 64 * CACHE_WAVES, 0, s>>>(a)
#define LSK_CACHE_ATTN_D(K8, TR)                                            \
  do {                                                                      \
    if (head_dim == 128 && tiles == 1) LSK_CACHE_ATTN(128, 1, K8, TR);      \
    else if (head_dim == 128) LSK_CACHE_ATTN(128, 2, K8, TR);               \
    else if (tiles == 1) LSK_CACHE_ATTN(64, 1, K8, TR);                     \
    else if (tiles == 2) LSK_CACHE_ATTN(64, 2, K8, TR);                     \
  } while (0)
  if (a.n_rounds == 0) ;
  else if (!kv8) LSK_CACHE_ATTN_D(false, true);
  else if (a.mask != nullptr) LSK_CACHE_ATTN_D(true, true);
  else if (tiles == 3) LSK_CACHE_ATTN(64, 3, true, false);
  else LSK_CACHE_ATTN_D(true, false);
#undef LSK_CACHE_ATTN_D
#undef LSK_CACHE_ATTN
  if (a.n_rounds > 0 && (rc = lsk_check_launch(what))) return rc;
  if (n_shared > 0) {
    const int32_t* items = a.recs + 8L * n_slots * a.n_rounds;
    if (head_dim == 128 && kv8) cache_tree_kernel<128, true><<<n_shared, 64 * TREE_WAVES, 0, s>>>(a, items);
    else if (head_dim == 128) cache_tree_kernel<128, false><<<n_shared, 64 * TREE_WAVES, 0, s>>>(a, items);
    else if (kv8) cache_tree_kernel<64, true><<<n_shared, 64 * TREE_WAVES, 0, s>>>(a, items);
    else cache_tree_kernel<64, false><<<n_shared, 64 * TREE_WAVES, 0, s>>>(a, items);
    if ((rc = lsk_check_launch(what))) return rc;
  }
  if (n_groups == 0) return 0;
  const dim3 cg(n_groups, a.Hkv, (a.part_rows + COMBINE_ROWS - 1) / COMBINE_ROWS);
  if (head_dim == 128)
    cache_combine_kernel<128><<<cg, 256, 0, s>>>(groups, a.o_part, a.ml_part, a.mask, a.W, a.out, a.G, a.Hkv,
                                                 a.part_rows);
  else
    cache_combine_kernel<64><<<cg, 256, 0, s>>>(groups, a.o_part, a.ml_part, a.mask, a.W, a.out, a.G, a.Hkv,
                                                a.part_rows);
  return lsk_check_launch(what);
}

static int shape_args(const char* what, const void* q, const void* kc, const void* vc, const void* out, int n_heads,
                      int n_kv_heads, int head_dim, int max_seq, long q_st, long q_sh) {
  LSK_REQUIRE(q && kc && vc && out, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_kv_heads <= 65535 && n_heads % n_kv_heads == 0 && head_dim > 0 &&
                  max_seq > 0 && q_st >= 0 && q_sh >= 0,
              LSK_ESHAPE, "%s: bad shape", what);
  return 0;
}

extern "C" int lsk_kv8_attn(const void* q, long q_stride_t, long q_stride_h, const void* k8, const void* v8,
                            const void* k_exp, const void* v_exp, const uint32_t* mask, int mask_words,
                            const int32_t* groups, int n_groups, int n_parts, const int32_t* recs, int n_rounds,
                            int n_slots, int n_shared, int tiles, int row_groups, int part_rows, void* out, int n_heads,
                            int n_kv_heads, int head_dim, int max_seq, float scale, void* workspace, size_t ws_bytes,
                            void* stream) {
  const char* what = "lsk_kv8_attn";
  if (int rc = shape_args(what, q, k8, v8, out, n_heads, n_kv_heads, head_dim, max_seq, q_stride_t, q_stride_h))
    return rc;
  LSK_REQUIRE(k_exp && v_exp && (mask == nullptr || mask_words > 0), LSK_EARG, "%s: null scales or an empty mask",
              what);
  LSK_REQUIRE(n_rounds >= 0 && n_shared >= 0, LSK_EARG, "%s: a plan of %d rounds and %d shared items", what, n_rounds,
              n_shared);
  if (n_rounds == 0 && n_shared == 0) return 0;
  LSK_REQUIRE(recs != nullptr, LSK_EARG, "%s: null pointer", what);
  const CacheAttnArgs a = {(const uint16_t*)q, q_stride_t, q_stride_h, k8, v8, (const uint8_t*)k_exp,
                           (const uint8_t*)v_exp, mask, mask_words, recs, n_rounds, (uint16_t*)out, nullptr, nullptr,
                           part_rows, n_heads / n_kv_heads, n_kv_heads, max_seq, 0.f};
  return cache_attn(what, true, a, groups, n_groups, n_parts, n_slots, n_shared, tiles, row_groups, head_dim, scale,
                    workspace, ws_bytes, (hipStream_t)stream);
}

extern "C" int lsk_tree_attn(int dtype, const void* q, long q_stride_t, long q_stride_h, const void* kcache,
                             const void* vcache, const uint32_t* mask, int mask_words, const int32_t* works,
                             int n_works, int rows_cap, const int32_t* groups, int n_groups, int n_parts,
                             const int32_t* recs, int n_rounds, int n_slots, int n_shared, int tiles, int row_groups,
                             int part_rows, void* out, int n_heads, int n_kv_heads, int head_dim, int max_seq,
                             float scale, void* workspace, size_t ws_bytes, void* stream) {
  const char* what = "lsk_tree_attn";
  if (int rc = shape_args(what, q, kcache, vcache, out, n_heads, n_kv_heads, head_dim, max_seq, q_stride_t,
                          q_stride_h)) return rc;
  LSK_REQUIRE(mask && mask_words > 0, LSK_EARG, "%s: no mask", what);
  LSK_REQUIRE(dtype == LSK_DTYPE_BF16 || dtype == LSK_DTYPE_F32, LSK_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  hipStream_t s = (hipStream_t)stream;
  const int G = n_heads / n_kv_heads;
  if (dtype == LSK_DTYPE_BF16) {
    LSK_REQUIRE(n_rounds >= 0 && n_shared >= 0, LSK_EARG, "%s: a plan of %d rounds and %d shared items", what, n_rounds,
                n_shared);
    if (n_rounds == 0 && n_shared == 0) return 0;
    LSK_REQUIRE(recs != nullptr, LSK_EARG, "%s: null pointer", what);
    const CacheAttnArgs a = {(const uint16_t*)q, q_stride_t, q_stride_h, kcache, vcache, nullptr, nullptr, mask,
                             mask_words, recs, n_rounds, (uint16_t*)out, nullptr, nullptr, part_rows, G, n_kv_heads,
                             max_seq, 0.f};
    return cache_attn(what, false, a, groups, n_groups, n_parts, n_slots, n_shared, tiles, row_groups, head_dim, scale,
                      workspace, ws_bytes, s);
  }
  LSK_REQUIRE(n_works >= 0 && rows_cap > 0 && rows_cap % 16 == 0 && rows_cap <= ATTN_ROWS, LSK_EARG,
              "%s: a plan of %d works of up to %d rows (16, 32 or %d)", what, n_works, rows_cap, ATTN_ROWS);
  if (n_works == 0) return 0;
  LSK_REQUIRE(works != nullptr, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(max_seq % 32 == 0, LSK_ESHAPE, "%s: max_seq %d", what, max_seq);
  const dim3 grid(n_works, n_kv_heads, rows_cap / F32_ROWS);
#define LSK_TREE_F32(DD)                                                                                           \
  tree_attn_f32_kernel<DD><<<grid, 64 * F32_ROWS, 0, s>>>((const float*)q, q_stride_t, q_stride_h,                 \
                                                          (const float*)kcache, (const float*)vcache, mask,        \
                                                          mask_words, works, (float*)out, G, n_kv_heads, max_seq,  \
                                                          scale)
  switch (head_dim) {
    case 16: LSK_TREE_F32(16); break;
    case 32: LSK_TREE_F32(32); break;
    case 64: LSK_TREE_F32(64); break;
    case 128: LSK_TREE_F32(128); break;
    default: LSK_REQUIRE(false, LSK_EUNSUPPORTED, "%s: fp32 head_dim %d", what, head_dim);
  }
#undef LSK_TREE_F32
  return lsk_check_launch(what);
}
