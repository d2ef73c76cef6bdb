// "mx4_quant_{dt}" and "mx4_dequant_{dt}": rows of values to microscaled 4-bit floating point and back (mx4.h).
//
// Bound: HBM.  Quantising moves the value's size + 17/32 bytes an element, the way back the same.  Four neighbouring lanes
// hold one block, eight values each (16-byte loads of 16-bit values, two of fp32): the block's largest magnitude is a local
// maximum and two quad exchanges, taken on the bits as unsigned integers, so that NaN and infinities win; each lane then
// packs its eight codes with four conversions and writes a dword (256 contiguous bytes a wavefront), the first lane of
// each quad the scale byte.  A thread takes kPer groups, their loads issued together.  Rows that are no whole groups of
// eight, or whose groups do not start on 16 bytes, are loaded and stored by elements.  Measured: bf16 [8192, 2048] there and back
// 14.8 us for 84 MB, 5.7 TB/s (a copy of 1 GiB: 5.1 .. 6.5); fp32 [517, 1000] 9.4 us, two launches.
#include "../hrt/registry.h"
#include "mx4.h"

namespace hk {
namespace {

constexpr int kPer = 2;  // groups of eight per thread

// Largest magnitude of eight values as fp32 bits.
__device__ __forceinline__ uint32_t amax8(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  return m;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return o > v ? o : v;
}

__device__ __forceinline__ uint32_t pack_codes(const float* v, float s) {
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
}

// Group g of a row of gpr groups (four per block, the last block filled up with zeros): row = g / gpr.  VEC: cols % 8 == 0
// and groups on 16 bytes.  Threads past the last group repeat it, so that quads stay whole, and store nothing.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx4_quant(hrt_mx4_args p, uint32_t gpr, int64_t groups) {
  float v[kPer][8];
  int64_t row[kPer];
  uint32_t grp[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    int64_t g = ((int64_t)blockIdx.x * kPer + u) * 256 + threadIdx.x;
    // a multiple of four groups exists, and the grid's threads past them repeat the last quad lane by lane
    if (g >= groups) g = groups - 4 + (threadIdx.x & 3);
    row[u] = (uint64_t)groups <= 0xffffffffull ? (int64_t)((uint32_t)g / gpr) : g / gpr;
    grp[u] = (uint32_t)(g - row[u] * gpr);
    const bool in = (int64_t)grp[u] * 8 < p.cols;
    const HK_G typename T::storage* x = gcptr<typename T::storage>(p.x) + row[u] * p.x_sr + (VEC && !in ? 0 : (int64_t)grp[u] * 8);
    if constexpr (VEC && std::is_same<T, F32>::value) {
      const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const HK_G f32x4*>(x));
      const f32x4 b = __builtin_nontemporal_load(reinterpret_cast<const HK_G f32x4*>(x) + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = in ? a[i] : 0.f, v[u][4 + i] = in ? b[i] : 0.f;
    } else if constexpr (VEC) {
      u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const HK_G u32x4*>(x));
      if (!in) w = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][2 * i] = lo16<T>(w[i]), v[u][2 * i + 1] = hi16<T>(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = (int64_t)grp[u] * 8 + i < p.cols ? T::to_f32(x[i]) : 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    uint32_t m = amax8(v[u]);
    m = dpp_umax<0xB1>(m);  // lane ^ 1
    m = dpp_umax<0x4E>(m);  // lane ^ 2
    const uint32_t s = mx_scale_of(m);
    const uint32_t w = s == 255u ? 0u : pack_codes(v[u], mx_scale(s));
    if (((int64_t)blockIdx.x * kPer + u) * 256 + threadIdx.x >= groups) continue;
    const int64_t nb = gpr / 4, pitch = (p.cols + 1) / 2;
    HK_G uint8_t* out = gptr<uint8_t>(p.codes) + row[u] * pitch + (int64_t)grp[u] * 4;
    if constexpr (VEC) {
      if ((int64_t)grp[u] * 8 < p.cols) *reinterpret_cast<HK_G uint32_t*>(out) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((int64_t)grp[u] * 4 + i < pitch) out[i] = (uint8_t)(w >> (8 * i));
    }
    if ((grp[u] & 3) == 0) gptr<uint8_t>(p.scale)[row[u] * nb + (grp[u] >> 2)] = (uint8_t)s;
  }
}

// The same groups the other way; VEC: cols % 8 == 0 (a group's codes are one aligned dword, its values aligned).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx4_dequant(hrt_mx4_args p, uint32_t gpr, int64_t groups) {
  const int64_t nb = (p.cols + 31) / 32, pitch = (p.cols + 1) / 2;
  uint32_t w[kPer], s[kPer];
  int64_t row[kPer], at[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    int64_t g = ((int64_t)blockIdx.x * kPer + u) * 256 + threadIdx.x;
    if (g >= groups) g = groups - 1;
    row[u] = (uint64_t)groups <= 0xffffffffull ? (int64_t)((uint32_t)g / gpr) : g / gpr;
    at[u] = g - row[u] * gpr;
    const HK_G uint8_t* c = gcptr<uint8_t>(p.codes) + row[u] * pitch + at[u] * 4;
    if constexpr (VEC) {
      w[u] = __builtin_nontemporal_load(reinterpret_cast<const HK_G uint32_t*>(c));
    } else {
      w[u] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at[u] * 4 + i < pitch) w[u] |= (uint32_t)c[i] << (8 * i);
    }
    s[u] = gcptr<uint8_t>(p.scale)[row[u] * nb + (at[u] >> 2)];
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    if (((int64_t)blockIdx.x * kPer + u) * 256 + threadIdx.x >= groups) continue;
    const float f = mx_scale(s[u]);
    HK_G typename T::storage* out = gptr<typename T::storage>(p.x) + row[u] * p.cols + at[u] * 8;
    if constexpr (std::is_same<T, F32>::value) {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 1);
      const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 3);
      const f32x4 lo = {a[0], a[1], b[0], b[1]}, hi = {c[0], c[1], d[0], d[1]};
      if constexpr (VEC) {
        __builtin_nontemporal_store(lo, reinterpret_cast<HK_G f32x4*>(out));
        __builtin_nontemporal_store(hi, reinterpret_cast<HK_G f32x4*>(out) + 1);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (at[u] * 8 + i < p.cols) out[i] = i < 4 ? lo[i & 3] : hi[i & 3];
      }
    } else {
      const u32x4 v = mx4_unpack8<T>(w[u], f);
      if constexpr (VEC) {
        __builtin_nontemporal_store(v, reinterpret_cast<HK_G u32x4*>(out));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (at[u] * 8 + i < p.cols) out[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

template <typename T, bool QUANT>
bool launch_mx4(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_mx4_args*>(pp);
  constexpr uint64_t esz = sizeof(typename T::storage);
  if (a.rows < 0 || a.cols < 0 || a.x_sr < 0) return ctx.fail("negative shape or stride");
  if (a.rows == 0 || a.cols == 0) return true;
  if (a.cols > (int64_t)1 << 32) return ctx.fail("rows of more than 2^32 values");
  const int64_t nb = cdiv(a.cols, kMxBlock), pitch = (a.cols + 1) / 2;
  const int64_t xs[2] = {a.rows, a.cols}, xt[2] = {QUANT ? a.x_sr : a.cols, 1};
  if (!ctx.check(a.x, hrt::span_bytes(2, xs, xt, esz), "x") || !ctx.check(a.codes, (uint64_t)(a.rows * pitch), "codes") ||
      !ctx.check(a.scale, (uint64_t)(a.rows * nb), "scale"))
    return false;
  // quantising walks whole blocks (a quad must be whole), the way back only the groups that hold a column
  const int64_t gpr = QUANT ? nb * 4 : cdiv(a.cols, 8), groups = a.rows * gpr;
  const int64_t grid = cdiv(groups, 256 * kPer);
  if (!hrt::grid_fits(grid, 256)) return ctx.fail("too many values for one launch");
  const bool vec = a.cols % 8 == 0 && a.x % 16 == 0 && (xt[0] * (int64_t)esz) % 16 == 0 && a.codes % 4 == 0;
  if constexpr (QUANT) {
    if (vec) hipLaunchKernelGGL((mx4_quant<T, true>), dim3((uint32_t)grid), dim3(256), 0, ctx.stream, a, (uint32_t)gpr, groups);
    else hipLaunchKernelGGL((mx4_quant<T, false>), dim3((uint32_t)grid), dim3(256), 0, ctx.stream, a, (uint32_t)gpr, groups);
  } else {
    if (vec) hipLaunchKernelGGL((mx4_dequant<T, true>), dim3((uint32_t)grid), dim3(256), 0, ctx.stream, a, (uint32_t)gpr, groups);
    else hipLaunchKernelGGL((mx4_dequant<T, false>), dim3((uint32_t)grid), dim3(256), 0, ctx.stream, a, (uint32_t)gpr, groups);
  }
  return hrt::launch_ok(hipGetLastError(), ctx, QUANT ? "mx4_quant" : "mx4_dequant");
}

HRT_REGISTER("mx4_quant_f32", hrt_mx4_args, (launch_mx4<F32, true>));
HRT_REGISTER("mx4_quant_bf16", hrt_mx4_args, (launch_mx4<BF16, true>));
HRT_REGISTER("mx4_quant_f16", hrt_mx4_args, (launch_mx4<F16, true>));
HRT_REGISTER("mx4_dequant_f32", hrt_mx4_args, (launch_mx4<F32, false>));
HRT_REGISTER("mx4_dequant_bf16", hrt_mx4_args, (launch_mx4<BF16, false>));
HRT_REGISTER("mx4_dequant_f16", hrt_mx4_args, (launch_mx4<F16, false>));

}  // namespace
}  // namespace hk
