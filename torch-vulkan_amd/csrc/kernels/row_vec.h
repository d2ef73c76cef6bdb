// Rows of any length and alignment in 16-byte pieces, and sums and maxima over the lanes that share a row.
//
// gfx950 reads and writes 16 bytes at any address that suits the element type, so rows of odd length need no path of their
// own: only the piece that a row ends in is touched element by element.
#pragma once

#include "mfma_common.h"

namespace hk {

typedef u32x4 __attribute__((aligned(2))) u32x4_any2;
typedef u32x4 __attribute__((aligned(4))) u32x4_any4;

// V values of type T in 16 bytes.
template <typename T>
struct RowVec {
  using S = typename T::storage;
  static constexpr int V = 16 / (int)sizeof(S);
  using Any = typename std::conditional<sizeof(S) == 2, u32x4_any2, u32x4_any4>::type;

  __device__ __forceinline__ static void unpack(u32x4 w, float* v) {
    if constexpr (V == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[2 * e] = lo16<T>(w[e]), v[2 * e + 1] = hi16<T>(w[e]);
    }
  }
  __device__ __forceinline__ static u32x4 pack(const float* v) {
    if constexpr (V == 4) return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    else return pack8<T>(v);
  }
  __device__ __forceinline__ static u32x4 get(const HK_G S* p) { return *reinterpret_cast<const HK_G Any*>(p); }
  __device__ __forceinline__ static void put(HK_G S* p, u32x4 w) { *reinterpret_cast<HK_G Any*>(p) = w; }
  // The first n values (0 < n < V), zeros behind them.
  __device__ __forceinline__ static u32x4 get_some(const HK_G S* p, int n) {
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) {
        if constexpr (V == 4) w[e] = __float_as_uint(p[e]);
        else w[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
      }
    return w;
  }
  __device__ __forceinline__ static void put_some(HK_G S* p, u32x4 w, int n) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) {
        if constexpr (V == 4) p[e] = __uint_as_float(w[e]);
        else p[e] = (S)(w[e >> 1] >> (16 * (e & 1)));
      }
  }
};

// Piece `col` of a row of D values, in two steps; TAIL: rows end inside a piece.  row_load reads V values without a branch, the row's
// last ones for lanes whose piece passes its end, so that every load of a row is in flight before the first is used (with a branch
// around the last piece each was waited for: the norm's gradients of 308 x 1001 fp32 10.8 us, so 6.0).  row_fix (TAIL) moves the
// values of a piece that passes the end down, zeros behind them, and makes one past the end zeros; without TAIL what a piece past
// the end holds is the caller's to drop.
template <typename T, bool TAIL>
__device__ __forceinline__ u32x4 row_load(const HK_G typename T::storage* row, int64_t col, int64_t D) {
  constexpr int V = RowVec<T>::V;
  if constexpr (!TAIL) return RowVec<T>::get(row + (col < D ? col : D - V));
  if (D < V) return col < D ? RowVec<T>::get_some(row + col, (int)(D - col)) : u32x4{0, 0, 0, 0};
  return RowVec<T>::get(row + (col + V <= D ? col : D - V));
}
template <typename T, bool TAIL>
__device__ __forceinline__ u32x4 row_fix(u32x4 w, int64_t col, int64_t D) {
  constexpr int V = RowVec<T>::V, PER = V / 4;  // values of a dword
  if (!TAIL || D < V) return w;
  const int64_t past = col + V - D;
  const int down = past <= 0 ? 0 : past < V ? (int)past : V, dw = down / PER;
  const bool two = dw & 2, one = dw & 1, all = dw & 4;
  w = u32x4{two ? w[2] : w[0], two ? w[3] : w[1], two ? 0u : w[2], two ? 0u : w[3]};
  w = u32x4{one ? w[1] : w[0], one ? w[2] : w[1], one ? w[3] : w[2], one ? 0u : w[3]};
  w = u32x4{all ? 0u : w[0], all ? 0u : w[1], all ? 0u : w[2], all ? 0u : w[3]};
  if constexpr (PER == 2) {
    const uint32_t by = (uint32_t)(down & 1) * 2;
    w = u32x4{__builtin_amdgcn_alignbyte(w[1], w[0], by), __builtin_amdgcn_alignbyte(w[2], w[1], by), __builtin_amdgcn_alignbyte(w[3], w[2], by), w[3] >> (8 * by)};
  }
  return w;
}
// Both at once, where nothing waits behind it.
template <typename T, bool TAIL>
__device__ __forceinline__ u32x4 row_piece(const HK_G typename T::storage* row, int64_t col, int64_t D) {
  return row_fix<T, TAIL>(row_load<T, TAIL>(row, col, D), col, D);
}
template <typename T, bool TAIL>
__device__ __forceinline__ void row_put(HK_G typename T::storage* row, int64_t col, int64_t D, u32x4 w) {
  constexpr int V = RowVec<T>::V;
  if (!TAIL ? col < D : col + V <= D) RowVec<T>::put(row + col, w);
  else if (TAIL && col < D) RowVec<T>::put_some(row + col, w, (int)(D - col));
}

// Sum over the LPR lanes (16 or 64) that share a row, or over a workgroup of 256 or 1024 through `red` (a float for each wavefront,
// not those of the call before); the same bits in every lane.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_u32(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return v > o ? v : o;
}
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v, float* red) {
  static_assert(LPR == 16 || LPR == 64 || LPR == 256 || LPR == 1024, "lanes per row");
  if constexpr (LPR == 16) {
    v = dpp_add<0xB1>(v), v = dpp_add<0x4E>(v), v = dpp_add<0x141>(v), v = dpp_add<0x140>(v);
    return v;
  }
  v = wave_sum_dpp(v);
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int k = 0; k < LPR / 64; k += 4) v += (red[k] + red[k + 1]) + (red[k + 2] + red[k + 3]);
  }
  return v;
}
// Largest magnitude, by the bits without sign: a NaN is larger than an infinity.
template <int LPR>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, uint32_t* red) {
  v = dpp_max_u32<0xB1>(v), v = dpp_max_u32<0x4E>(v), v = dpp_max_u32<0x141>(v), v = dpp_max_u32<0x140>(v);
  if constexpr (LPR >= 64) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = a[0] > a[1] ? a[0] : a[1];
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = b[0] > b[1] ? b[0] : b[1];
  }
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < LPR / 64; ++k) v = red[k] > v ? red[k] : v;
  }
  return v;
}

// ---- 8-bit rows -----------------------------------------------------------------------------------------------------------
// A row's values are code * scale with scale = top / 127, top the row's largest magnitude, and code the whole number nearest to
// 127 v / top (ties to even).  scale is rounded to nearest, but stays where 127 scale is finite.  A row of zeros has scale 0, one with an infinity or NaN scale NaN and codes 0.
struct RowCode {
  float mul, per, scale;  // v * mul is in a range where per = 127 / (top * mul) is an ordinary number
  double per64;           // the same in fp64, for 32-bit values
  __device__ __forceinline__ explicit RowCode(uint32_t bits) {
    const float t = __uint_as_float(bits);
    mul = bits < 0x0d800000u /* 2^-100 */ ? 0x1p64f : bits > 0x71800000u /* 2^100 */ ? 0x1p-64f : 1.f;
    if (bits - 1u >= 0x7f7fffffu) {  // zero, infinity, NaN
      mul = per = 0.f, per64 = 0.0, scale = bits ? __uint_as_float(0x7fc00000u) : 0.f;
    } else {
      per = 127.f / (t * mul), per64 = 127.0 / (double)(t * mul);
      scale = fminf(t / 127.f, 0x1.020406p+121f);  // 127 of the largest step that is taken are finite
    }
  }
};
// A code is the low byte of the sum of its quotient and 1.5 2^23, whose last place is one: the addition rounds, ties to even.
constexpr float kRound32 = 12582912.f;
constexpr double kRound64 = 6755399441055744.0;  // 1.5 2^52
// Codes of fp32 values that are roundings themselves: the quotient as it comes out.
__device__ __forceinline__ uint32_t code_of(float v, const RowCode& r) { return __float_as_uint(v * r.mul * r.per + kRound32); }
// The nearest code exactly.  With v and top of p bits, 254 v against an odd multiple k top of a border are whole numbers (times a power
// of two) that differ by 1 at least where v and top share a binade, by 2 below: relative to its size a quotient that is no tie is at
// least 1 / (254 (2^p - 1)) > 2^-19 away from one (p = 11; 2^-32 for 24 bits).  It comes out within 2^-22 (2^-51 in fp64), and is
// rounded to 20 bits (45), which moves it by at most 2^-20 (2^-45): ties, which have 8 bits, are ties again, and nothing else
// reaches one.
template <typename T>
__device__ __forceinline__ uint32_t nearest_code(float v, const RowCode& r) {
  if constexpr (std::is_same<T, F32>::value) {
    const uint64_t q = (__builtin_bit_cast(uint64_t, (double)(v * r.mul) * r.per64) + 0x80u) & ~(uint64_t)0xff;
    return (uint32_t)__builtin_bit_cast(uint64_t, __builtin_bit_cast(double, q) + kRound64);
  } else {
    const uint32_t q = (__float_as_uint(v * r.mul * r.per) + 8u) & ~15u;
    return __float_as_uint(__uint_as_float(q) + kRound32);
  }
}
// Low bytes of four codes.
__device__ __forceinline__ uint32_t pack_codes4(const uint32_t* q) {
  const uint32_t a = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u), b = __builtin_amdgcn_perm(q[3], q[2], 0x0c0c0400u);
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}

}  // namespace hk
