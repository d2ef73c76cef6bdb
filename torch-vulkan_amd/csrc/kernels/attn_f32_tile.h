// fp32 attention tiles on v_mfma_f32_32x32x2_f32, shared by the fused attention kernels: rows of DP floats in LDS, their
// products with stationary rows held in registers, and the transposed products with P or dS.
#pragma once

#include "attn_common.h"

namespace hk {

// XOR on the 16-byte chunk index: 16 consecutive rows at one chunk fall in distinct chunks of a 256-byte bank line
// (rows of 8 or 24 chunks: two rows share a line), and a run of 8 aligned chunks stays such a run.
template <int NCH>
__device__ __forceinline__ int f32_swz(int row) {
  return NCH % 16 == 0 ? row & 15 : (row >> 1) & 7;
}
template <int NCH>
__device__ __forceinline__ int f32_off(int row, int c) {
  return row * (NCH * 16) + ((c ^ f32_swz<NCH>(row)) << 4);
}

// Operand fragments of one stationary row per lane: group g holds d = 8 g + 4 h .. + 3.
template <int DP, bool W16>
__device__ __forceinline__ void load_frags(f32x4 (&f)[DP / 8], const HK_G float* row, bool ok, int D, int h) {
#pragma unroll
  for (int g = 0; g < DP / 8; ++g) {
    const int d = 8 * g + 4 * h;
    f[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (ok) {
      if constexpr (W16) {
        if (d < D) f[g] = *reinterpret_cast<const HK_G f32x4*>(row + d);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) f[g][e] = row[d + e];
      }
    }
  }
}

__device__ __forceinline__ f32x16 mfma2(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

// Rows r0 .. r0 + 31 of the tile (A) times the stationary fragments (B), over d, on top of s.  Chunk 2 g + h of row l32 sits at
// (2 g + h) ^ swz: the lane's base address XOR a constant.
template <int DP>
__device__ __forceinline__ f32x16 rows_times(const HK_L uint8_t* T, int r0, const f32x4 (&f)[DP / 8], int l32, int h, f32x16 s) {
  const int row = (r0 + l32) * DP * 4, x = (h ^ f32_swz<DP / 4>(l32)) << 4;
#pragma unroll
  for (int g = 0; g < DP / 8; ++g) {
    const f32x4 a = *reinterpret_cast<const HK_L f32x4*>(T + row + (x ^ (g << 5)));
#pragma unroll
    for (int e = 0; e < 4; ++e) s = mfma2(a[e], f[g][e], s);
  }
  return s;
}
// acc[n] + (columns 32 n .. + 31 of the tile's rows r0 .. r0 + 31)^T times p: d x stationary row.  The swizzle of row
// 8 j + 4 h + r splits into a lane part (four bases) and constants.
template <int DP>
__device__ __forceinline__ void cols_times(f32x16 (&acc)[DP / 32], const HK_L uint8_t* T, int r0, const f32x16& p, int l32, int h) {
  constexpr bool WIDE = (DP / 4) % 16 == 0;
  const HK_L uint8_t* base[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {  // WIDE: k = r; else k = 2 (j & 1) + r / 2
    const int x = WIDE ? 4 * h + k : 4 * (k >> 1) + 2 * h + (k & 1);
    base[k] = T + (r0 + 4 * h) * DP * 4 + (((l32 >> 2) ^ x) << 4) + (l32 & 3) * 4;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        const int blk = WIDE ? n ^ (j & 1) : n;
        const float a = *reinterpret_cast<const HK_L float*>(base[WIDE ? r : 2 * (j & 1) + (r >> 1)] + (8 * j + r) * DP * 4 + blk * 128);
        acc[n] = mfma2(a, p[4 * j + r], acc[n]);
      }
}

// d block n of one stationary row per lane: elements 4 j + r are d = 32 n + 8 j + 4 h + r
template <bool W16>
__device__ __forceinline__ void store_block(HK_G float* row, const f32x16& v, float mul, int n, int D, int h) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = 32 * n + 8 * j + 4 * h;
    if constexpr (W16) {
      if (d < D) *reinterpret_cast<HK_G f32x4*>(row + d) = f32x4{v[4 * j] * mul, v[4 * j + 1] * mul, v[4 * j + 2] * mul, v[4 * j + 3] * mul};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (d + r < D) row[d + r] = v[4 * j + r] * mul;
    }
  }
}

}  // namespace hk
