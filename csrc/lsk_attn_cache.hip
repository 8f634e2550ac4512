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
// Work items, records, splits and their merge are those of the ragged attention (lsk_attn_plan, lsk_attn_schedule): a
// mask only takes away from the causal rule, so the same plan serves both.
//
// Both cache formats are read as 1 KiB fragments in lane order, 64 D bytes per block of STEP positions:
//   bf16   STEP = 32: K fragment (a, f), lane 16 lg + l16: position 8 (l16 / 4) + 4 a + l16 % 4, d = 32 f + 8 lg .. + 7;
//          V^T: row d, positions 8 lg .. + 7.
//   8-bit  STEP = 64: e4m3 codes; K fragment (a, j): position 16 (l16 / 4) + 4 a + l16 % 4, d = 64 j + 16 lg .. + 15
//          (two MFMA operands of 8 d each); V^T: row d, positions 16 lg .. + 15 (two operands of 8 positions each).
//          A position's K and V are its codes times 2^(ks - 127) and 2^(vs - 127).
// Per step of a wave (v_mfma_f32_16x16x32_bf16): S^T[pos][q] = K Q^T, whose rows are mapped to positions so that lane
// group lg ends up with the consecutive positions its V^T load needs; online softmax with fp32 statistics;
// O^T[d][q] += V^T P^T.  e4m3 values times a power of two are bf16 values, so the conversions in registers are exact and
// K's scale costs nothing (the conversion takes one); V's scale, which differs per position, multiplies the weights.
// The weights are rounded to bf16 for the second product (relative 2^-9 each, independent of one another: it adds about
// as much error as the rounding of the bf16 output); the sum of the weights is taken before that rounding.
//
// The 8 waves of a workgroup take the STEP-position steps of an item round robin and are merged in wave order through
// LDS.  Which wave takes a step and every order of additions depend on absolute positions only: a row's result never
// depends on what else is in the launch, and a chain over a bf16 cache gives the ragged attention's bits.
#include <type_traits>

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
  float* o_part;
  float* ml_part;
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

#define ORDER() __builtin_amdgcn_sched_barrier(0)

template <int D, int QT, bool KV8, bool TREE>
__global__ __launch_bounds__(64 * ATTN_WAVES, 1) void cache_attn_kernel(const CacheAttnArgs A) {
  constexpr int STEP = KV8 ? 64 : 32;                // positions per step of a wave
  constexpr int HV = STEP / 32;                      // 32-position halves of a step; a lane group has 8 slots of each
  constexpr int KF = D / 32;                         // K operands per 16-position tile
  constexpr int CT = D / 16;                         // 16-byte loads per lane of a step, for K and for V
  constexpr int NW = ATTN_WAVES;
  constexpr int ROWS = 16 * QT;
  constexpr bool QREG = QT == 1;                     // one tile: Q fragments in registers
  constexpr int MT = QT < ATTN_MERGE_TILES ? QT : ATTN_MERGE_TILES;
  constexpr int MR = 16 * MT;
  constexpr int QLD = D + 8;                         // 16 rows' 16-byte reads hit distinct banks
  constexpr int QCH = D / 8;
  constexpr int QPT = (ROWS * QCH + 64 * NW - 1) / (64 * NW);
  __shared__ float s_ml[NW][2][ROWS];
  __shared__ __attribute__((aligned(16))) float s_o[NW][MR][D + 4];
  __shared__ __attribute__((aligned(16))) uint16_t s_q[QREG ? 1 : ROWS][QLD];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int G = A.G, Hkv = A.Hkv, S = A.S, Hq = Hkv * G;
  const int32_t* my_recs = A.recs + (long)blockIdx.x * A.n_rounds * 8;

  struct Item {
    int q_start, row0, nrows, kv_lo, kv_hi, part, pos0, crow, kvh;
  };
  auto fetch = [&](int r) {
    Item it;
    if (r >= A.n_rounds) {
      it.nrows = 0;
      return it;
    }
    const int32_t* wk = my_recs + (long)r * 8;
    it.q_start = wk[0]; it.row0 = wk[1]; it.nrows = wk[2] & 255; it.kvh = wk[2] >> 8; it.kv_lo = wk[3];
    it.kv_hi = wk[4]; it.part = wk[5]; it.pos0 = wk[6]; it.crow = wk[7];
    return it;
  };
  // Q: row rl of an item -> 8 elements from d; operand f's k index 8 lg + e stands for d = q_dim(f) + e
  auto q_dim = [&](int f) { return KV8 ? 64 * (f >> 1) + 16 * lg + 8 * (f & 1) : 32 * f + 8 * lg; };
  auto q_ptr = [&](const Item& it, int rl) {
    const int r = it.row0 + rl, t = r / G, g = r - t * G;
    return A.q + (long)(it.q_start + t) * A.q_st + (long)(it.kvh * G + g) * A.q_sh;
  };
  auto ldq = [&](const uint16_t* p) { return __builtin_bit_cast(lsk_bf16x8, *(const lsk_u32x4_u*)p); };
  lsk_bf16x8 qst[QPT];
  lsk_bf16x8 qreg[KF];
  auto q_load = [&](const Item& it) {
    if constexpr (QREG) {
      const bool valid = l16 < it.nrows;
      const uint16_t* p = q_ptr(it, valid ? l16 : 0);
#pragma unroll
      for (int f = 0; f < KF; ++f) qreg[f] = valid ? ldq(p + q_dim(f)) : (lsk_bf16x8){};
    } else {
#pragma unroll
      for (int i = 0; i < QPT; ++i) {
        const int c = tid + i * 64 * NW, r = c / QCH, c8 = c - r * QCH;
        qst[i] = r < it.nrows ? ldq(q_ptr(it, r) + 8 * c8) : (lsk_bf16x8){};
      }
    }
  };
  auto q_store = [&]() {
    if constexpr (!QREG) {
#pragma unroll
      for (int i = 0; i < QPT; ++i) {
        const int c = tid + i * 64 * NW, r = c / QCH, c8 = c - r * QCH;
        if (r < ROWS) *(lsk_bf16x8*)(&s_q[r][8 * c8]) = qst[i];
      }
    }
  };
  // K / V through buffer loads over the item's (row, KV head) stripe, whose range ends with the block that holds the
  // item's last position: loads past it give zeros without touching memory, so the next step's are unconditional
  // (under a branch the compiler would wait for them early).  Non-temporal: read once per launch.
  struct Stripe {
    __amdgpu_buffer_rsrc_t k, v, ks, vs;
  };
  auto stripe = [&](const Item& it) {
    const long st = (long)it.crow * Hkv + it.kvh;
    const long bytes = (long)(S / STEP) * 64 * D;    // of a whole stripe
    const int end = min(S, (it.kv_hi + STEP - 1) / STEP * STEP);
    Stripe s;
    s.k = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)A.kc + st * bytes), (short)0, end / STEP * 64 * D,
                                            LSK_BUFFER_RSRC_WORD3);
    s.v = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)A.vc + st * bytes), (short)0, end / STEP * 64 * D,
                                            LSK_BUFFER_RSRC_WORD3);
    if constexpr (KV8) {
      s.ks = __builtin_amdgcn_make_buffer_rsrc((void*)(A.ks + st * S), (short)0, end, LSK_BUFFER_RSRC_WORD3);
      s.vs = __builtin_amdgcn_make_buffer_rsrc((void*)(A.vs + st * S), (short)0, end, LSK_BUFFER_RSRC_WORD3);
    }
    return s;
  };
  auto ld = [&](__amdgpu_buffer_rsrc_t rs, int vo, int so) -> lsk_i32x4 {
    return __builtin_bit_cast(lsk_i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vo, so, 2));
  };
  const int k_vo = 16 * lane, v_vo = 64 * l16 + 16 * lg;
  constexpr int STRIDE = STEP * NW;
  lsk_i32x4 kr[CT], vr[CT], ksr, vsr;                // this step's K and V as loaded
  auto load_k = [&](const Stripe& s, int sb) {
#pragma unroll
    for (int i = 0; i < CT; ++i) kr[i] = ld(s.k, k_vo, sb / STEP * 64 * D + i * 1024);
    if constexpr (KV8) ksr = ld(s.ks, 16 * (l16 >> 2), sb);
  };
  auto load_v = [&](const Stripe& s, int sb) {
#pragma unroll
    for (int c = 0; c < CT; ++c) vr[c] = ld(s.v, v_vo, sb / STEP * 64 * D + c * 1024);
    if constexpr (KV8) vsr = ld(s.vs, 16 * lg, sb);
  };
  auto first_step = [&](const Item& it) { return it.kv_lo + STEP * wave; };
  auto issue_first = [&](const Item& it) {
    q_load(it);
    const Stripe s = stripe(it);
    load_k(s, first_step(it));
    load_v(s, first_step(it));
  };

  Item cur = fetch(0);
  if (cur.nrows == 0) return;
  issue_first(cur);
  Item nxt = fetch(1);
  if constexpr (!QREG) {
    q_store();
    __syncthreads();
  }
  for (int r = 0; cur.nrows > 0; ++r) {
    const int nq = (cur.nrows + 15) >> 4;
    const int kv_hi = cur.kv_hi;
    const Stripe sr = stripe(cur);
    int qpos[QT];                                    // the row's own slot; -1: no such row
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int rl = 16 * qt + l16;
      qpos[qt] = rl < cur.nrows ? cur.pos0 + (cur.row0 + rl) / G : -1;
    }
    // slots that every row of the item reads
    const int full_lim = min(kv_hi - 1, TREE ? cur.pos0 - 1 : cur.pos0 + cur.row0 / G);
    lsk_f32x4 oacc[QT][CT];
    float m_run[QT], l_run[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      m_run[qt] = -INFINITY;
      l_run[qt] = 0.f;
#pragma unroll
      for (int c = 0; c < CT; ++c) oacc[qt][c] = (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
    }
    // bit e: row l16 of tile qt reads slot s0 + e
    auto allow = [&](int qt, int s0) {
      const int n = min(kv_hi - 1, qpos[qt]) - s0 + 1;
      uint32_t bits = n >= 8 ? 0xffu : n <= 0 ? 0u : (1u << n) - 1u;
      if constexpr (TREE) {
        const int t = max(qpos[qt] - cur.pos0, 0);
        bits &= mask_window(A.mask + (long)(cur.q_start + t) * A.W, A.W, s0 - cur.pos0);
      }
      return bits;
    };
    // One step: 32 slots (8 per lane group) at a time.  FULL: every row reads all of them.  All QT tiles are computed,
    // also those without rows (copies of the loop for fewer tiles cost more in registers than they save).
    auto step = [&](auto full_, int sb) {
      constexpr bool FULL = decltype(full_)::value;
      // In a step that some row does not read whole, a slot whose V holds an infinity or NaN must not reach the rows
      // that do not read it (0 x NaN): the values past the item and the non-finite ones are cleared here, and the rows
      // that do read such a value get it after the products (below).
      bool odd = false;
      if constexpr (!FULL) {
        constexpr int PER = 2 * HV;                  // slots of a dword
        const int nk = kv_hi - (sb + 8 * HV * lg);   // slots of this lane that the item covers
        uint32_t any = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int m = nk - PER * w;
          const uint32_t keep = m >= PER ? 0xffffffffu : m <= 0 ? 0u : (1u << (32 / PER * m)) - 1u;
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            const uint32_t x = (uint32_t)vr[c][w] & keep;
            const uint32_t nf = KV8 ? ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u
                                    : ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;  // the top bits of its slots
            vr[c][w] = (int)(x & ~((nf - (nf >> (KV8 ? 7 : 15))) | nf));
            any |= nf;
          }
        }
        odd = __builtin_amdgcn_ballot_w64(any != 0u) != 0ull;
      }
#pragma unroll
      for (int hv = 0; hv < HV; ++hv) {
        const int s0 = sb + 8 * HV * lg + 8 * hv;    // this lane group's 8 slots
        ORDER();
        lsk_bf16x8 kf[2][KF];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          if constexpr (KV8) {
            const float sc = exp_bits(((uint32_t)ksr[2 * hv + a] >> (8 * (l16 & 3))) & 255u);
#pragma unroll
            for (int f = 0; f < KF; ++f) {
              const lsk_i32x4 x = kr[(2 * hv + a) * (KF / 2) + (f >> 1)];
              kf[a][f] = codes_to_bf16(x[2 * (f & 1)], x[2 * (f & 1) + 1], sc);
            }
          } else {
#pragma unroll
            for (int f = 0; f < KF; ++f) kf[a][f] = __builtin_bit_cast(lsk_bf16x8, kr[a * KF + f]);
          }
        }
        lsk_bf16x8 pb[QT];
        float alpha[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          ORDER();
          // S^T = K Q^T: sacc[a][e] <-> slot s0 + 4 a + e
          lsk_f32x4 sacc[2];
          lsk_bf16x8 qf[KF];
#pragma unroll
          for (int f = 0; f < KF; ++f)
            qf[f] = QREG ? qreg[f] : *(const lsk_bf16x8*)(&s_q[16 * qt + l16][q_dim(f)]);
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            sacc[a] = (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < KF; ++f)
              sacc[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[a][f], qf[f], sacc[a], 0, 0, 0);
          }
          uint32_t reads = 0xffu;
          if constexpr (!FULL) reads = allow(qt, s0);
          // the online softmax of the tile's 16 query columns
          float sv[8];
          float mt = -INFINITY;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float sc = sacc[i >> 2][i & 3] * A.scale_log2;
            if constexpr (!FULL) sc = (reads >> i) & 1u ? sc : -INFINITY;
            sv[i] = sc;
            mt = fmaxf(mt, sc);
          }
          mt = rows_max(mt);
          const float m_new = fmaxf(m_run[qt], mt);
          alpha[qt] = (m_new == m_run[qt]) ? 1.f : fast_exp2(m_run[qt] - m_new);
          float rs = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float pe = (sv[i] == -INFINITY) ? 0.f : fast_exp2(sv[i] - m_new);
            rs += pe;
            float pv = pe;
            if constexpr (KV8) {
              pv = pe * exp_bits(((uint32_t)vsr[2 * hv + (i >> 2)] >> (8 * (i & 3))) & 255u);
              if constexpr (!FULL) pv = (reads >> i) & 1u ? pv : 0.f;  // (a slot never written: any exponent)
            }
            pb[qt][i] = static_cast<__bf16>(pv);
          }
          rs = rows_sum(rs);
          l_run[qt] = l_run[qt] * alpha[qt] + rs;
          m_run[qt] = m_new;
        }
        ORDER();
        if (hv == HV - 1) load_k(sr, sb + STRIDE);   // the next step's K streams in during this step's P V
        // O^T = alpha O^T + V^T P^T
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          if (c % 2 == 0) ORDER();
          lsk_bf16x8 vf;
          if constexpr (KV8) vf = codes_to_bf16(vr[c][2 * hv], vr[c][2 * hv + 1], 1.f);
          else vf = __builtin_bit_cast(lsk_bf16x8, vr[c]);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) oacc[qt][c][i] *= alpha[qt];
            oacc[qt][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pb[qt], oacc[qt][c], 0, 0, 0);
          }
        }
      }
      if constexpr (!FULL) {
        if (odd) {
          // V again, as a count of its non-finite values (cnt) and their kind (sgn: +-1 for +-inf, 2^20 for NaN): of
          // those that a row reads, one kind of infinity gives that infinity, anything else NaN.
#pragma unroll 1
          for (int hv = 0; hv < HV; ++hv)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              const uint32_t reads = allow(qt, sb + 8 * HV * lg + 8 * hv);
              lsk_bf16x8 rd;
#pragma unroll
              for (int e = 0; e < 8; ++e) rd[e] = static_cast<__bf16>((float)((reads >> e) & 1u));
#pragma unroll
              for (int c = 0; c < CT; ++c) {
                ORDER();
                const lsk_i32x4 x = ld(sr.v, v_vo, sb / STEP * 64 * D + c * 1024);
                lsk_bf16x8 cnt, sgn;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  bool nf, nan, neg;
                  if constexpr (KV8) {
                    const uint32_t u = (uint32_t)(hv ? x[2 + e / 4] : x[e / 4]) >> (8 * (e & 3));
                    nf = nan = (u & 0x7fu) == 0x7fu;
                    neg = false;
                  } else {
                    const uint32_t u = (uint32_t)x[e / 2] >> (16 * (e & 1));
                    nf = (u & 0x7f80u) == 0x7f80u;
                    nan = nf && (u & 0x7fu) != 0u;
                    neg = (u & 0x8000u) != 0u;
                  }
                  cnt[e] = static_cast<__bf16>(nf ? 1.f : 0.f);
                  sgn[e] = static_cast<__bf16>(!nf ? 0.f : nan ? 1048576.f : neg ? -1.f : 1.f);
                }
                const lsk_f32x4 z = (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
                const lsk_f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cnt, rd, z, 0, 0, 0);
                const lsk_f32x4 s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sgn, rd, z, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float add = s[i] == n[i] ? INFINITY : s[i] == -n[i] ? -INFINITY : __builtin_nanf("");
                  oacc[qt][c][i] = n[i] > 0.f ? oacc[qt][c][i] + add : oacc[qt][c][i];
                }
              }
            }
        }
      }
      load_v(sr, sb + STRIDE);
    };
    int sb = first_step(cur);
    for (; sb + STEP - 1 <= full_lim; sb += STRIDE) step(std::true_type{}, sb);
    for (; sb < kv_hi; sb += STRIDE) step(std::false_type{}, sb);
    // the next item's Q and first K / V loads fly while this item is merged
    const Item done = cur;
    cur = nxt;
    if (cur.nrows > 0) {
      issue_first(cur);
      nxt = fetch(r + 2);
    }
    // merge the waves in order: M = max m_w, e_w = exp2(m_w - M), L = sum e_w l_w, O = sum e_w O_w
#pragma unroll
    for (int p0 = 0; p0 < QT; p0 += MT) {
      if (p0 >= nq) break;
#pragma unroll
      for (int qt = p0; qt < p0 + MT && qt < QT; ++qt) {
        if (qt < nq) {
          if (lg == 0) {
            s_ml[wave][0][16 * qt + l16] = m_run[qt];
            s_ml[wave][1][16 * qt + l16] = l_run[qt];
          }
#pragma unroll
          for (int c = 0; c < CT; ++c)
            *(float4*)(&s_o[wave][16 * (qt - p0) + l16][16 * c + 4 * lg]) =
                make_float4(oacc[qt][c][0], oacc[qt][c][1], oacc[qt][c][2], oacc[qt][c][3]);
        }
      }
      __syncthreads();
      const int pr = min(done.nrows - 16 * p0, MR);
      for (int e = tid; e < pr * (D / 4); e += 64 * NW) {
        const int ql = e / (D / 4), d = 4 * (e - ql * (D / 4));
        const int qr = 16 * p0 + ql;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, s_ml[w][0][qr]);
        float L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float mw = s_ml[w][0][qr];
          const float ew = (mw == -INFINITY) ? 0.f : ((mw == M) ? 1.f : fast_exp2(mw - M));
          L = L + ew * s_ml[w][1][qr];
          const float4 ow = *(const float4*)(&s_o[w][ql][d]);
          O.x = O.x + ew * ow.x;
          O.y = O.y + ew * ow.y;
          O.z = O.z + ew * ow.z;
          O.w = O.w + ew * ow.w;
        }
        const int rr = done.row0 + qr;
        const int tt = rr / G, gg = rr - tt * G;
        if (done.part < 0) {
          if (TREE && L == 0.f) L = 1.f;             // nothing read: O is 0
          lsk_u32x2_u pk;
          pk[0] = (uint32_t)f2bf(O.x / L) | ((uint32_t)f2bf(O.y / L) << 16);
          pk[1] = (uint32_t)f2bf(O.z / L) | ((uint32_t)f2bf(O.w / L) << 16);
          *(lsk_u32x2_u*)(A.out + ((long)(done.q_start + tt) * Hq + done.kvh * G + gg) * D + d) = pk;
        } else {
          const long slot = ((long)done.part * Hkv + done.kvh) * ATTN_ROWS + qr;
          *(float4*)(A.o_part + slot * D + d) = O;
          if (d == 0) {
            A.ml_part[slot * 2 + 0] = M;
            A.ml_part[slot * 2 + 1] = L;
          }
        }
      }
      if (p0 == 0 && cur.nrows > 0) q_store();
      __syncthreads();
    }
  }
}

// Merge the splits of one query group in split order: M = max_s m_s, w_s = exp2(m_s - M), out = sum w_s O_s / sum w_s l_s
// (zeros where no split read anything).
template <int D>
__global__ __launch_bounds__(256) void cache_combine_kernel(const int32_t* __restrict__ blocks,
                                                            const int32_t* __restrict__ groups,
                                                            const float* __restrict__ o_part,
                                                            const float* __restrict__ ml_part,
                                                            uint16_t* __restrict__ out, int G, int Hkv) {
  __shared__ float s_w[ATTN_ROWS][ATTN_MAX_SPLITS];
  __shared__ float s_L[ATTN_ROWS];
  const int32_t* gp = groups + (long)blockIdx.x * 8;
  const int blk = gp[0], row0 = gp[1], nrows = gp[2], pf = gp[3], ns = gp[4];
  const int kvh = blockIdx.y;
  const int q_start = blocks[(long)blk * 4 + 0];
  const int tid = threadIdx.x;
  if (tid < nrows) {
    float M = -INFINITY;
    for (int s = 0; s < ns; ++s) M = fmaxf(M, ml_part[(((long)(pf + s) * Hkv + kvh) * ATTN_ROWS + tid) * 2]);
    float L = 0.f;
    for (int s = 0; s < ns; ++s) {
      const long slot = ((long)(pf + s) * Hkv + kvh) * ATTN_ROWS + tid;
      const float ms = ml_part[slot * 2], ls = ml_part[slot * 2 + 1];
      const float w = (ms == -INFINITY) ? 0.f : ((ms == M) ? 1.f : fast_exp2(ms - M));
      s_w[tid][s] = w;
      L = L + w * ls;
    }
    s_L[tid] = L == 0.f ? 1.f : L;
  }
  __syncthreads();
  for (int e = tid; e < nrows * (D / 4); e += 256) {
    const int rl = e / (D / 4), d = 4 * (e - rl * (D / 4));
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < ns; ++s) {
      const float w = s_w[rl][s];
      const float4 v = *(const float4*)(o_part + (((long)(pf + s) * Hkv + kvh) * ATTN_ROWS + rl) * D + d);
      O.x = O.x + w * v.x;
      O.y = O.y + w * v.y;
      O.z = O.z + w * v.z;
      O.w = O.w + w * v.w;
    }
    const float L = s_L[rl];
    const int r = row0 + rl, t = r / G, g = r - t * G;
    lsk_u32x2_u pk;
    pk[0] = (uint32_t)f2bf(O.x / L) | ((uint32_t)f2bf(O.y / L) << 16);
    pk[1] = (uint32_t)f2bf(O.z / L) | ((uint32_t)f2bf(O.w / L) << 16);
    *(lsk_u32x2_u*)(out + ((long)(q_start + t) * G * Hkv + kvh * G + g) * D + d) = pk;
  }
}

// ----------------------------------------------------------------------------- fp32 trees
// The token-identity model's kernel: a wave per query row walks the row's slots in 64-position chunks (lane = slot), in
// the ragged attention's order of additions (a chain gives its bits), skipping the slots the row does not read.
// Bound by the chain of a row, as that kernel is.
template <int D>
__global__ __launch_bounds__(256) void tree_attn_f32_kernel(const float* __restrict__ q, long q_st, long q_sh,
                                                            const float* __restrict__ kc, const float* __restrict__ vc,
                                                            const uint32_t* __restrict__ mask, int W,
                                                            const int32_t* __restrict__ works, float* __restrict__ out,
                                                            int G, int Hkv, int S, float scale) {
  constexpr int DPL = (D + 63) / 64;
  constexpr int KB = D < 64 ? D : 64;
  __shared__ __attribute__((aligned(16))) float sp[4][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int kvh = blockIdx.y;
  const int32_t* wk = works + (long)blockIdx.x * 8;
  const int q_start = wk[0], row0 = wk[1], nrows = wk[2], pos0 = wk[6], crow = wk[7];
  const long head_base = ((long)crow * Hkv + kvh) * (long)S * D;
  for (int rl = blockIdx.z * 4 + wave; rl < nrows; rl += 4 * gridDim.z) {
    const int r = row0 + rl, t = r / G, g = r - t * G;
    const int qpos = pos0 + t;
    const float* qv = q + (long)(q_start + t) * q_st + (long)(kvh * G + g) * q_sh;
    const uint32_t* words = mask + (long)(q_start + t) * W;
    float m_run = -INFINITY, l_run = 0.f;
    float o[DPL];
#pragma unroll
    for (int i = 0; i < DPL; ++i) o[i] = 0.f;
    for (int base = 0; base <= qpos; base += 64) {
      const int kp = base + lane, rel = kp - pos0;
      bool reads = kp <= qpos;
      if (rel >= 0) reads = reads && (rel >> 5) < W && ((words[rel >> 5] >> (rel & 31)) & 1u);
      const int nvalid = min(64, qpos + 1 - base);
      const float* vb = vc + head_base + (long)base * D;
      lsk_f32x4 v0[16];
      auto load_v = [&](int d) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          v0[j] = d < D && 32 * (j / 8) < nvalid
                      ? *(const lsk_f32x4_u*)(vb + (long)(j / 8) * 32 * D + d * 32 + 4 * (j % 8))
                      : (lsk_f32x4){0.f, 0.f, 0.f, 0.f};
      };
      load_v(lane);
      float s = -INFINITY;
      if (reads) {
        const float* kr = kc + head_base + (long)kp * D;
        float acc = 0.f;
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += KB) {
          lsk_f32x4 k4[KB / 4];
#pragma unroll
          for (int i = 0; i < KB / 4; ++i) k4[i] = *(const lsk_f32x4_u*)(kr + d0 + 4 * i);
#pragma unroll
          for (int i = 0; i < KB / 4; ++i) {
            acc += qv[d0 + 4 * i] * k4[i][0];
            acc += qv[d0 + 4 * i + 1] * k4[i][1];
            acc += qv[d0 + 4 * i + 2] * k4[i][2];
            acc += qv[d0 + 4 * i + 3] * k4[i][3];
          }
        }
        s = acc * scale;
      }
      float mt = s;
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) mt = fmaxf(mt, __shfl_xor(mt, off, 64));
      const float m_new = fmaxf(m_run, mt);
      const float alpha = (m_new == m_run) ? 1.f : lsk_exp(m_run - m_new);
      const float p = (s == -INFINITY) ? 0.f : lsk_exp(s - m_new);
      float rs = p;
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) rs += __shfl_xor(rs, off, 64);
      l_run = l_run * alpha + rs;
      m_run = m_new;
      sp[wave][lane] = reads ? p : -1.f;             // (weights are never negative: -1 marks a slot not read)
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        if (i > 0) load_v(lane + 64 * i);
        float acc = o[i] * alpha;
        auto step = [&](float pj, float vj) { acc = pj < 0.f ? acc : acc + pj * vj; };
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float4 p4 = *(const float4*)(&sp[wave][4 * j]);
          step(p4.x, v0[j][0]);
          step(p4.y, v0[j][1]);
          step(p4.z, v0[j][2]);
          step(p4.w, v0[j][3]);
        }
        o[i] = acc;
      }
      __builtin_amdgcn_wave_barrier();
    }
    if (l_run == 0.f) l_run = 1.f;
    float* orow = out + ((long)(q_start + t) * Hkv * G + kvh * G + g) * D;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      const int d = lane + 64 * i;
      if (d < D) orow[d] = o[i] / l_run;
    }
  }
}

// ----------------------------------------------------------------------------- entry points

#define ATTN_CACHE_ALIGN 16

static bool aligned16(const void* p) { return ((uintptr_t)p & (ATTN_CACHE_ALIGN - 1)) == 0; }

// Checks and launches shared by the two entry points; kv8 = the cache is 8-bit.
static int cache_attn(const char* what, bool kv8, CacheAttnArgs a, const int32_t* blocks, int n_works,
                      const int32_t* groups, int n_groups, int n_parts, int n_slots, int rows_cap, int n_heads,
                      int head_dim, float scale, void* workspace, size_t ws_bytes, hipStream_t s) {
  LSK_REQUIRE(head_dim == 64 || head_dim == 128, LSK_EUNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", what,
              head_dim);
  LSK_REQUIRE(a.S % ATTN_TILE == 0 && (long)a.S * head_dim * 2 <= 0x7fffffffL, LSK_ESHAPE,
              "%s: max_seq %d (a multiple of %d, stripes below 2 GiB)", what, a.S, ATTN_TILE);
  LSK_REQUIRE(aligned16(a.kc) && aligned16(a.vc) && (!kv8 || (aligned16(a.ks) && aligned16(a.vs))), LSK_EARG,
              "%s: the cache tensors start at multiples of 16 bytes", what);
  LSK_REQUIRE(head_dim == 64 || rows_cap <= 32, LSK_EUNSUPPORTED, "%s: rows_cap %d (head_dim 128: 16 or 32)", what,
              rows_cap);
  if (n_parts > 0) {
    const size_t need = lsk_attn_workspace_bytes(n_parts, a.Hkv, head_dim);
    LSK_REQUIRE(workspace != nullptr && aligned16(workspace) && ws_bytes >= need && groups != nullptr && blocks != nullptr,
                LSK_EWORKSPACE, "%s: an aligned workspace of %zu bytes needed, %zu given", what, need, ws_bytes);
    a.o_part = (float*)workspace;
    a.ml_part = (float*)((char*)workspace +
                         lsk_align_up((size_t)n_parts * a.Hkv * ATTN_ROWS * head_dim * sizeof(float), 256));
  }
  a.scale_log2 = scale * 1.4426950408889634f;
#define LSK_CACHE_ATTN(DD, QT, K8, TR) \
  cache_attn_kernel<DD, QT, K8, TR><<<n_slots, 64 * ATTN_WAVES, 0, s>>>(a)
#define LSK_CACHE_ATTN_D(K8, TR)                                                            \
  do {                                                                                      \
    if (head_dim == 128 && rows_cap == 16) LSK_CACHE_ATTN(128, 1, K8, TR);                  \
    else if (head_dim == 128) LSK_CACHE_ATTN(128, 2, K8, TR);                               \
    else if (rows_cap == 16) LSK_CACHE_ATTN(64, 1, K8, TR);                                 \
    else LSK_CACHE_ATTN(64, ATTN_QT, K8, TR);                                               \
  } while (0)
  if (!kv8) LSK_CACHE_ATTN_D(false, true);
  else if (a.mask != nullptr) LSK_CACHE_ATTN_D(true, true);
  else LSK_CACHE_ATTN_D(true, false);
#undef LSK_CACHE_ATTN_D
#undef LSK_CACHE_ATTN
  int rc = lsk_check_launch(what);
  if (rc || n_groups == 0) return rc;
  const dim3 cg(n_groups, a.Hkv);
  if (head_dim == 128)
    cache_combine_kernel<128><<<cg, 256, 0, s>>>(blocks, groups, a.o_part, a.ml_part, a.out, a.G, a.Hkv);
  else
    cache_combine_kernel<64><<<cg, 256, 0, s>>>(blocks, groups, a.o_part, a.ml_part, a.out, a.G, a.Hkv);
  return lsk_check_launch(what);
}

static int plan_args(const char* what, const void* q, const void* kc, const void* vc, const void* out, int n_works,
                     int n_groups, int n_parts, int rows_cap, int n_heads, int n_kv_heads, int head_dim, int max_seq,
                     long q_st, long q_sh) {
  LSK_REQUIRE(q && kc && vc && out, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(rows_cap > 0 && rows_cap % 16 == 0 && rows_cap <= ATTN_ROWS, LSK_EARG,
              "%s: rows_cap %d (the plan's rows per item: 16, 32 or %d)", what, rows_cap, ATTN_ROWS);
  LSK_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && head_dim > 0 && max_seq > 0 &&
                  n_works >= 0 && n_groups >= 0 && n_parts >= 0 && q_st >= 0 && q_sh >= 0,
              LSK_ESHAPE, "%s: bad shape", what);
  return 0;
}

extern "C" int lsk_kv8_attn(const void* q, long q_stride_t, long q_stride_h, const void* k8, const void* v8,
                            const void* k_exp, const void* v_exp, const uint32_t* mask, int mask_words,
                            const int32_t* blocks, int n_works, const int32_t* groups, int n_groups, int n_parts,
                            const int32_t* recs, int n_rounds, int n_slots, int rows_cap, void* out, int n_heads,
                            int n_kv_heads, int head_dim, int max_seq, float scale, void* workspace, size_t ws_bytes,
                            void* stream) {
  const char* what = "lsk_kv8_attn";
  if (int rc = plan_args(what, q, k8, v8, out, n_works, n_groups, n_parts, rows_cap, n_heads, n_kv_heads, head_dim,
                         max_seq, q_stride_t, q_stride_h)) return rc;
  LSK_REQUIRE(k_exp && v_exp && (mask == nullptr || mask_words > 0), LSK_EARG, "%s: null scales or an empty mask", what);
  if (n_works == 0) return 0;
  LSK_REQUIRE(recs && n_rounds > 0 && n_slots > 0, LSK_EARG, "%s: a schedule is needed (lsk_attn_schedule)", what);
  CacheAttnArgs a = {(const uint16_t*)q, q_stride_t, q_stride_h, k8, v8, (const uint8_t*)k_exp, (const uint8_t*)v_exp,
                     mask, mask_words, recs, n_rounds, (uint16_t*)out, nullptr, nullptr, n_heads / n_kv_heads, n_kv_heads,
                     max_seq, 0.f};
  return cache_attn(what, true, a, blocks, n_works, groups, n_groups, n_parts, n_slots, rows_cap, n_heads, head_dim,
                    scale, workspace, ws_bytes, (hipStream_t)stream);
}

extern "C" int lsk_tree_attn(int dtype, const void* q, long q_stride_t, long q_stride_h, const void* kcache,
                             const void* vcache, const uint32_t* mask, int mask_words, const int32_t* blocks,
                             const int32_t* works, int n_works, const int32_t* groups, int n_groups, int n_parts,
                             const int32_t* recs, int n_rounds, int n_slots, int rows_cap, void* out, int n_heads,
                             int n_kv_heads, int head_dim, int max_seq, float scale, void* workspace, size_t ws_bytes,
                             void* stream) {
  const char* what = "lsk_tree_attn";
  if (int rc = plan_args(what, q, kcache, vcache, out, n_works, n_groups, n_parts, rows_cap, n_heads, n_kv_heads,
                         head_dim, max_seq, q_stride_t, q_stride_h)) return rc;
  LSK_REQUIRE(mask && mask_words > 0, LSK_EARG, "%s: no mask", what);
  LSK_REQUIRE(dtype == LSK_DTYPE_BF16 || dtype == LSK_DTYPE_F32, LSK_EUNSUPPORTED, "%s: dtype %d", what, dtype);
  if (n_works == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  const int G = n_heads / n_kv_heads;
  if (dtype == LSK_DTYPE_BF16) {
    LSK_REQUIRE(recs && n_rounds > 0 && n_slots > 0, LSK_EARG, "%s: a schedule is needed (lsk_attn_schedule)", what);
    CacheAttnArgs a = {(const uint16_t*)q, q_stride_t, q_stride_h, kcache, vcache, nullptr, nullptr, mask, mask_words,
                       recs, n_rounds, (uint16_t*)out, nullptr, nullptr, G, n_kv_heads, max_seq, 0.f};
    return cache_attn(what, false, a, blocks, n_works, groups, n_groups, n_parts, n_slots, rows_cap, n_heads, head_dim,
                      scale, workspace, ws_bytes, s);
  }
  LSK_REQUIRE(works != nullptr, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(n_parts == 0, LSK_EARG, "%s: the fp32 path takes unsplit plans", what);
  LSK_REQUIRE(max_seq % 32 == 0, LSK_ESHAPE, "%s: max_seq %d", what, max_seq);
  const dim3 grid(n_works, n_kv_heads, rows_cap / 4);
#define LSK_TREE_F32(DD)                                                                                           \
  tree_attn_f32_kernel<DD><<<grid, 256, 0, s>>>((const float*)q, q_stride_t, q_stride_h, (const float*)kcache,     \
                                                (const float*)vcache, mask, mask_words, works, (float*)out, G,     \
                                                n_kv_heads, max_seq, scale)
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
