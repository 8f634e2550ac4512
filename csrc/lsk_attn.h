// Shared by the attention kernels: the work items' geometry, and reductions over a wave's four 16-lane rows.
#pragma once

#include "lsk_common.h"

#define ATTN_TILE 64   // work ranges are split at multiples of this (planner granularity)
#define ATTN_STEP 32   // KV positions per step of a wave
#define ATTN_QT 3      // 16-row MFMA column tiles per work item
#define ATTN_ROWS (16 * ATTN_QT)  // query rows per work item: a T <= 12 block of a 4-head group in one item
#define ATTN_MERGE_TILES 2  // column tiles merged per LDS pass of the wave merge
#define ATTN_MAX_SPLITS 128
#define ATTN_WAVES 8   // waves per work item; fixed, because it fixes which wave accumulates which step


__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// max / sum over the four 16-lane rows of a wave, result in every lane (the xor-16 then xor-32 butterfly),
// with gfx950's row swaps: v_permlane16_swap(x, x) yields rows {0,0,2,2} and {1,1,3,3},
// v_permlane32_swap(x, x) the lower and the upper half in every lane.  Plain VALU, no LDS round trip;
// a + b == b + a, so every lane ends with the same bits.
__device__ __forceinline__ float rows_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
