// Trees of drafted tokens: ancestor masks, greedy acceptance, and the move of the accepted path's K / V.
//
// A block's T nodes are its tokens 0 .. T - 1; node 0 is the root (the last committed token) and parents[i] < i is the
// index of node i's parent within the block.  Node i's K / V sit in slot pos0 + i of its cache row, whatever its depth.
#include "lsk_common.h"
#include "../include/lsk.h"

// Node i's ancestors and i itself as bits, and i's depth.  One thread walks from a node to the root; parents decrease
// along the walk, so the words are finished from the last to the first.  A parent outside [0, i) ends the walk.
__global__ __launch_bounds__(64) void tree_masks_kernel(const int32_t* __restrict__ parents,
                                                        const int32_t* __restrict__ starts,
                                                        const int32_t* __restrict__ lens, int N,
                                                        uint32_t* __restrict__ mask, int W,
                                                        int32_t* __restrict__ depth) {
  const int start = starts[blockIdx.x], T = lens[blockIdx.x];
  if (start < 0 || T < 0 || T > N - start) return;
  for (int i = blockIdx.y * 64 + threadIdx.x; i < T; i += 64 * gridDim.y) {
    uint32_t* out = mask + (long)(start + i) * W;
    int n = i, d = 0, w = W - 1;
    uint32_t bits = 0;
    while (true) {
      for (; w > (n >> 5); --w) {                    // (a node past the words: none of its bits fit)
        out[w] = bits;
        bits = 0;
      }
      if (w == (n >> 5)) bits |= 1u << (n & 31);
      const int up = parents[start + n];
      if (up < 0 || up >= n) break;
      n = up;
      ++d;
    }
    for (; w >= 0; --w) {
      out[w] = bits;
      bits = 0;
    }
    if (depth != nullptr) depth[start + i] = d;
  }
}

extern "C" int lsk_tree_masks(const int32_t* parents, const int32_t* starts, const int32_t* lens, int nb, int n_tokens,
                              int max_nodes, uint32_t* mask, int mask_words, int32_t* depth, void* stream) {
  const char* what = "lsk_tree_masks";
  LSK_REQUIRE(parents && starts && lens && mask, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(nb >= 0 && n_tokens >= 0 && max_nodes >= 0 && mask_words > 0 && (long)mask_words * 32 >= max_nodes,
              LSK_ESHAPE, "%s: %d mask words for trees of up to %d nodes", what, mask_words, max_nodes);
  if (nb == 0 || n_tokens == 0 || max_nodes == 0) return 0;
  const int gy = (max_nodes + 63) / 64;
  tree_masks_kernel<<<dim3(nb, gy < 65535 ? gy : 65535), 64, 0, (hipStream_t)stream>>>(parents, starts, lens, n_tokens,
                                                                                      mask, mask_words, depth);
  return lsk_check_launch(what);
}

// Greedy acceptance of one verified tree per wave: from the root, the next node is the lowest child that carries the
// verifier's greedy token of the current one.  path[b] = the accepted nodes (the root first), out[b] = the verifier's
// tokens of those nodes (the tokens to commit), both -1 past the end; acc[b] = the number of accepted drafts.
// A block outside the tokens or without nodes: acc = -1.  At most max_nodes nodes of a block take part.
// Children come after their parent, so the walk only goes up and ends.  Up to 64 nodes a lane holds one node and a step
// is a ballot and two lane reads; the loads of larger trees come from the caches.
__global__ __launch_bounds__(64) void tree_accept_kernel(const int64_t* __restrict__ Yv,
                                                         const int64_t* __restrict__ tokens,
                                                         const int32_t* __restrict__ parents,
                                                         const int32_t* __restrict__ starts,
                                                         const int32_t* __restrict__ lens, int N, int max_nodes,
                                                         int64_t* __restrict__ acc, int32_t* __restrict__ path,
                                                         int64_t* __restrict__ out) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int start = starts[b];
  int T = lens[b];
  if (start < 0 || T <= 0 || T > N - start) T = 0;
  T = min(T, max_nodes);
  int32_t* prow = path + (long)b * max_nodes;
  int64_t* orow = out + (long)b * max_nodes;
  int n = 0;                                         // nodes on the path
  if (T > 0 && T <= 64) {
    const bool in = lane < T;
    const int par = in ? parents[start + lane] : -1;
    const int64_t tok = in ? tokens[start + lane] : 0, y = in ? Yv[start + lane] : 0;
    int cur = 0, my_node = -1;
    int64_t my_out = -1;
    while (true) {
      const int64_t yc = __shfl(y, cur, 64);
      if (lane == n) {
        my_node = cur;
        my_out = yc;
      }
      ++n;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(in && lane > cur && par == cur && tok == yc);
      if (hit == 0ull) break;
      cur = __builtin_ctzll(hit);
    }
    if (lane < T) {                                  // (T <= max_nodes)
      prow[lane] = my_node;
      orow[lane] = my_out;
    }
    for (int i = T + lane; i < max_nodes; i += 64) {
      prow[i] = -1;
      orow[i] = -1;
    }
  } else {
    int cur = 0;
    while (T > 0) {
      const int64_t yc = Yv[start + cur];
      if (lane == 0) {
        prow[n] = cur;
        orow[n] = yc;
      }
      ++n;
      int next = -1;
      for (int base = cur + 1; base < T && next < 0; base += 64) {
        const int i = base + lane;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(i < T && parents[start + i] == cur && tokens[start + i] == yc);
        if (hit != 0ull) next = base + __builtin_ctzll(hit);
      }
      if (next < 0) break;
      cur = next;
    }
    for (int i = n + lane; i < max_nodes; i += 64) {
      prow[i] = -1;
      orow[i] = -1;
    }
  }
  if (lane == 0) acc[b] = n - 1;
}

extern "C" int lsk_tree_accept(const int64_t* Yv, const int64_t* tokens, const int32_t* parents, const int32_t* starts,
                               const int32_t* lens, int nb, int n_tokens, int max_nodes, int64_t* acc_out,
                               int32_t* path_out, int64_t* tokens_out, void* stream) {
  const char* what = "lsk_tree_accept";
  LSK_REQUIRE(Yv && tokens && parents && starts && lens && acc_out && path_out && tokens_out, LSK_EARG,
              "%s: null pointer", what);
  LSK_REQUIRE(nb >= 0 && n_tokens >= 0 && max_nodes > 0, LSK_ESHAPE, "%s: bad shape", what);
  if (nb == 0) return 0;
  tree_accept_kernel<<<nb, 64, 0, (hipStream_t)stream>>>(Yv, tokens, parents, starts, lens, n_tokens, max_nodes,
                                                         acc_out, path_out, tokens_out);
  return lsk_check_launch(what);
}

// Slot pos0 + j takes what slot pos0 + path[j] holds, for the accepted j = 1 .. acc, in every layer: the accepted
// path's K / V become consecutive and the committed length is pos0 + acc + 1.  Sources lie at or after their
// destinations (path is increasing, path[j] >= j) and later destinations never reach an earlier chunk's sources, so a
// workgroup reads 16 slots of one (layer, block, KV head), waits, and writes them, chunk after chunk.  Slots that stay
// are skipped.
// FMT: 0 fp32 (K [S, D], V in 32-position blocks), 1 bf16 (fragment-major K, V in 32-position blocks), 2 8-bit.
#define COMPACT_CHUNK 16
#define COMPACT_THREADS 256

// f over the 16 lanes of a row, in all of them (f associative, commutative and idempotent)
template <typename U, typename F>
__device__ __forceinline__ U row_reduce(U x, F f) {
#define ROW_ROR(N) x = f(x, (U)__builtin_amdgcn_mov_dpp((int)x, 0x120 + N, 0xf, 0xf, false))
  ROW_ROR(8); ROW_ROR(4); ROW_ROR(2); ROW_ROR(1);
#undef ROW_ROR
  return x;
}

template <int FMT> struct CompactElem;                // element, and a 16-byte piece at any address that aligns one
template <> struct CompactElem<0> { using T = uint32_t; using Piece = lsk_f32x4_u; };
template <> struct CompactElem<1> { using T = uint16_t; using Piece = lsk_u32x4_u; };
template <> struct CompactElem<2> { using T = uint8_t; using Piece = lsk_i32x4; };

// Element offsets in a stripe: K's 16-byte piece `ch` of slot p, and V's dim d of slot p.
template <int FMT>
__device__ __forceinline__ long compact_k(int p, int ch, int D) {
  if constexpr (FMT == 0) return (long)p * D + 4 * ch;
  if constexpr (FMT == 1) return k_cache_offset<uint16_t>(p, 8 * ch, D);
  const int pp = p & 63, a = (pp >> 2) & 3, l16 = ((pp >> 4) << 2) | (pp & 3);
  return (long)(p >> 6) * 64 * D + (long)((a * (D >> 6) + (ch >> 2)) * 64 + (ch & 3) * 16 + l16) * 16;
}

// K moves in 16-byte pieces of a slot.  V^T has a slot's values 64 bytes (fp32: 128) apart, D of them: the chunk's
// blocks are turned in LDS, read and written in 16-byte pieces of eight (four, sixteen) slots, so that the memory sees
// a request per dim and piece and not one per moved value, which bounded it (130 slots of 32 requests, 32 layers of 8
// heads of 128: 42 us against 59 where the last-level cache holds the 106 MB that the launch touches; 64 us where it
// does not).  Bound by the chain of path, blocks, LDS and stores in a workgroup, five of which fit a CU.  Only pieces
// that hold a source or a destination are touched; a piece's other slots are written back as they were.
template <int FMT, int D>
__global__ __launch_bounds__(COMPACT_THREADS) void kv_compact_kernel(
    void* kc_, void* vc_, uint8_t* ks, uint8_t* vs, const int32_t* __restrict__ rows, const int32_t* __restrict__ pos0,
    const int64_t* __restrict__ acc, const int32_t* __restrict__ path, int max_nodes, int max_batch, int Hkv, int S) {
  using T = typename CompactElem<FMT>::T;
  using Piece = typename CompactElem<FMT>::Piece;
  constexpr int KCH = D * (int)sizeof(T) / 16;       // pieces of a slot's K
  constexpr int KPER = (COMPACT_CHUNK * KCH + COMPACT_THREADS - 1) / COMPACT_THREADS;
  constexpr int VPER = COMPACT_CHUNK * D / COMPACT_THREADS;
  constexpr int B = FMT == 2 ? 64 : 32;              // slots of a V block
  constexpr int PS = 16 / (int)sizeof(T), PPR = B / PS;  // slots of a piece, pieces of a dim's row
  constexpr int LD = B * (int)sizeof(T) / 4 + 1;     // dwords of a row in LDS
  constexpr int PROWS = COMPACT_THREADS / PPR, NP = (D + PROWS - 1) / PROWS;
  constexpr int none = 0x7fffffff;
  __shared__ int s_from[COMPACT_CHUNK];              // slot that slot to + j takes its contents from; -1: it stays
  __shared__ uint32_t s_v[3][D * LD];                // the two blocks the destinations may lie in, and one other
  const int b = blockIdx.x, h = blockIdx.y, layer = blockIdx.z;
  const int row = rows[b], p0 = pos0[b];
  const int n = (int)min(max(acc[b], (int64_t)0), (int64_t)(max_nodes - 1));
  if (row < 0 || row >= max_batch || p0 < 0 || p0 >= S) return;
  const long stripe = (((long)layer * max_batch + row) * Hkv + h) * (long)S;
  T* kc = (T*)kc_ + stripe * D;
  T* vc = (T*)vc_ + stripe * D;
  const int tid = threadIdx.x, vd = tid % D, vj = tid / D, pc = tid % PPR, pr = tid / PPR;
  for (int j0 = 1; j0 <= n; j0 += COMPACT_CHUNK) {
    const int to = p0 + j0, db = to / B;
    // Every wave's lanes look at the chunk's 16 slots: which pieces of the two destination blocks hold a source or a
    // destination (bytes 0 and 1), a destination (2 and 3), and which later block is the first with a source.
    const int l16 = tid & 15, j = j0 + l16, node = j <= n ? path[(long)b * max_nodes + j] : -1;
    const bool moves = node > j && node < S - p0;
    const int from = moves ? p0 + node : -1;
    uint32_t bits = 0;
    int other = none;
    if (moves) {
      const int src = from / B - db, dst = (to + l16) / B - db;
      bits = 0x10001u << (8 * dst + (to + l16) % B / PS);
      if (src < 2) bits |= 1u << (8 * src + from % B / PS);
      else other = from / B;
    }
    bits = __builtin_amdgcn_readfirstlane(row_reduce(bits, [](uint32_t x, uint32_t y) { return x | y; }));
    if (bits == 0) continue;                         // nothing moves (as every wave finds)
    auto least = [](int x, int y) { return min(x, y); };
    other = __builtin_amdgcn_readfirstlane(row_reduce(other, least));
    auto pieces_of = [&](int blk) {                  // pieces of a later block that hold a source
      const uint32_t u = from >= 0 && from / B == blk ? 1u << (from % B / PS) : 0u;
      return (uint32_t)__builtin_amdgcn_readfirstlane(row_reduce(u, [](uint32_t x, uint32_t y) { return x | y; }));
    };
    if (tid < COMPACT_CHUNK) s_from[tid] = from;
    __syncthreads();
    Piece kx[KPER];
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      const int e = tid + i * COMPACT_THREADS, j = e / KCH, from = j < COMPACT_CHUNK ? s_from[j] : -1;
      if (from >= 0) kx[i] = *(const Piece*)(kc + compact_k<FMT>(from, e % KCH, D));
    }
    uint8_t ek = 0, ev = 0;
    if (FMT == 2 && tid < COMPACT_CHUNK && moves) {
      ek = ks[stripe + s_from[tid]];
      ev = vs[stripe + s_from[tid]];
    }
    // the pieces `need` of block blk: asked for, and put into LDS
    auto fetch = [&](Piece (&x)[NP], int blk, uint32_t need) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int d = pr + i * PROWS;
        if (d < D && (need >> pc & 1u)) x[i] = *(const Piece*)(vc + (long)blk * B * D + d * B + pc * PS);
      }
    };
    auto put = [&](uint32_t* v, const Piece (&x)[NP], uint32_t need) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int d = pr + i * PROWS;
        if (d < D && (need >> pc & 1u)) {
          const lsk_i32x4 u = __builtin_bit_cast(lsk_i32x4, x[i]);
#pragma unroll
          for (int w = 0; w < 4; ++w) v[d * LD + pc * 4 + w] = (uint32_t)u[w];
        }
      }
    };
    T vx[VPER];
    auto take = [&](int buf, int blk) {              // this thread's values of dim vd whose source is in block blk
#pragma unroll
      for (int i = 0; i < VPER; ++i) {
        const int from = s_from[vj * VPER + i];
        if (from >= 0 && from / B == blk) vx[i] = ((const T*)(s_v[buf] + vd * LD))[from % B];
      }
    };
    Piece x0[NP], x1[NP], x2[NP];
    uint32_t need = pieces_of(other);                // (0: there is none)
    fetch(x0, db, bits & 255u);
    fetch(x1, db + 1, bits >> 8 & 255u);
    fetch(x2, other, need);
    put(s_v[0], x0, bits & 255u);
    put(s_v[1], x1, bits >> 8 & 255u);
    put(s_v[2], x2, need);
    __syncthreads();
    take(0, db);
    take(1, db + 1);
    while (other != none) {
      take(2, other);
      other = __builtin_amdgcn_readfirstlane(row_reduce(from / B > other ? from / B : none, least));
      if (other == none) break;
      need = pieces_of(other);
      fetch(x2, other, need);
      __syncthreads();
      put(s_v[2], x2, need);
      __syncthreads();
    }
    __syncthreads();                                 // (every source is in registers)
#pragma unroll
    for (int i = 0; i < VPER; ++i) {
      const int j = vj * VPER + i;
      if (s_from[j] >= 0) ((T*)(s_v[(to + j) / B - db] + vd * LD))[(to + j) % B] = vx[i];
    }
#pragma unroll
    for (int i = 0; i < KPER; ++i) {
      const int e = tid + i * COMPACT_THREADS, j = e / KCH;
      if (j < COMPACT_CHUNK && s_from[j] >= 0) *(Piece*)(kc + compact_k<FMT>(to + j, e % KCH, D)) = kx[i];
    }
    if (FMT == 2 && tid < COMPACT_CHUNK && moves) {
      ks[stripe + to + tid] = ek;
      vs[stripe + to + tid] = ev;
    }
    __syncthreads();
    for (int d = 0; d < 2; ++d) {
      const uint32_t dirty = bits >> (16 + 8 * d) & 255u;
      if (dirty == 0) continue;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int row_d = pr + i * PROWS;
        if (row_d < D && (dirty >> pc & 1u)) {
          lsk_i32x4 u;
#pragma unroll
          for (int w = 0; w < 4; ++w) u[w] = (int)s_v[d][row_d * LD + pc * 4 + w];
          *(Piece*)(vc + (long)(db + d) * B * D + row_d * B + pc * PS) = __builtin_bit_cast(Piece, u);
        }
      }
    }
    __syncthreads();
  }
}

extern "C" int lsk_kv_compact(int dtype, void* kcache, void* vcache, void* k_exp, void* v_exp, int n_layers,
                              const int32_t* rows, const int32_t* pos0, const int64_t* accepted, const int32_t* path,
                              int nb, int max_nodes, int n_kv_heads, int head_dim, int max_batch, int max_seq,
                              void* stream) {
  const char* what = "lsk_kv_compact";
  LSK_REQUIRE(kcache && vcache && rows && pos0 && accepted && path, LSK_EARG, "%s: null pointer", what);
  LSK_REQUIRE(dtype == LSK_DTYPE_F32 || dtype == LSK_DTYPE_BF16 || dtype == LSK_DTYPE_KV8, LSK_EUNSUPPORTED,
              "%s: dtype %d", what, dtype);
  LSK_REQUIRE(dtype != LSK_DTYPE_KV8 || (k_exp && v_exp), LSK_EARG, "%s: null exponents", what);
  LSK_REQUIRE(n_layers >= 0 && n_layers <= 65535 && nb >= 0 && max_nodes > 0 && n_kv_heads > 0 && n_kv_heads <= 65535 &&
                  max_batch > 0 && max_seq > 0 && max_seq % (dtype == LSK_DTYPE_KV8 ? 64 : 32) == 0,
              LSK_ESHAPE, "%s: bad shape", what);
  LSK_REQUIRE(dtype != LSK_DTYPE_KV8 || (((uintptr_t)kcache | (uintptr_t)vcache) & 15) == 0, LSK_EARG,
              "%s: the cache tensors start at multiples of 16 bytes", what);
  if (nb == 0 || n_layers == 0) return 0;
  const dim3 grid(nb, n_kv_heads, n_layers);
  hipStream_t s = (hipStream_t)stream;
#define LSK_COMPACT(FMT, DD)                                                                                       \
  kv_compact_kernel<FMT, DD><<<grid, COMPACT_THREADS, 0, s>>>(kcache, vcache, (uint8_t*)k_exp, (uint8_t*)v_exp, rows, \
                                                              pos0, accepted, path, max_nodes, max_batch, n_kv_heads, \
                                                              max_seq)
#define LSK_COMPACT_D(FMT)                              \
  do {                                                  \
    if (head_dim == 128) LSK_COMPACT(FMT, 128);         \
    else LSK_COMPACT(FMT, 64);                          \
  } while (0)
  if (dtype == LSK_DTYPE_F32 && (head_dim == 16 || head_dim == 32)) {
    if (head_dim == 16) LSK_COMPACT(0, 16);
    else LSK_COMPACT(0, 32);
  } else {
    LSK_REQUIRE(head_dim == 64 || head_dim == 128, LSK_EUNSUPPORTED, "%s: head_dim %d", what, head_dim);
    if (dtype == LSK_DTYPE_F32) LSK_COMPACT_D(0);
    else if (dtype == LSK_DTYPE_BF16) LSK_COMPACT_D(1);
    else LSK_COMPACT_D(2);
  }
#undef LSK_COMPACT_D
#undef LSK_COMPACT
  return lsk_check_launch(what);
}
