// Root-mean-square norm of rows, forward ("rms_fwd_*") and backward ("rms_bwd_*"), and rows into 8 bits ("i8_rows_quant_*").
//
// Bound by memory: a row is read once, held in registers as fp32 and written once.  16, 64, 256 or 1024 lanes share a row (heads,
// model widths, wide rows or few of them), which DPP steps and lane swaps add up without LDS, or through a few floats of it.
// Rows longer than a workgroup's registers take several passes.  Measured, GPU us, bf16 with a residual, replayed on the same operands and, in
// brackets, on operands from HBM (rotated through 600 MB): forward; forward in training, which keeps the sums' rests; dx and dw; dx alone:
// 1 x 2048 3.1 (2.3), 3.3 (2.5), 3.3 (2.6), 3.1 (2.2); 4020 x 2048 11.8 (15.7: 66 MB, 4.2 TB/s), 13.5 (19.2: 74 MB), 18.8 (22.4: 74 MB and
// twice 4 MB of sums), 14.1 (17.9); 65536 x 128 12.7 (15.8), 15.1 (18.9), 17.4 (21.4), 13.5 (17.2); 16384 x 2048 40 (49: 268 MB, 5.5 TB/s),
// 52 (58), 54 (69), 48 (57).  Into 8 bits without the norm: 4020 x 2048 5.6 (7.9), 8192 x 2048 10.1 (12.6).
#include <initializer_list>

#include "../hrt/registry.h"
#include "row_vec.h"

namespace hk {
namespace {

__device__ __forceinline__ int64_t row_at(int64_t row, int64_t n1, int64_t n2, const int64_t* s) {
  if (n1 * n2 == 1) return row * s[0];
  const uint32_t r = (uint32_t)row, t = r / (uint32_t)n2, i0 = t / (uint32_t)n1;  // rows < 2^31
  return (int64_t)i0 * s[0] + (int64_t)(t - i0 * (uint32_t)n1) * s[1] + (int64_t)(r - t * (uint32_t)n2) * s[2];
}

// Threads of a workgroup whose rows are shared by LPR lanes each.
constexpr int threads_of(int lpr) { return lpr > 256 ? lpr : 256; }

enum Mode { kNorm, kNorm8, kQuant };

// What rounding a sum to 16 bits took from it, in whole 256ths of the type's last place, for the backward pass, whose gradients would else be
// those of the rounded sum (the weight's of 4020 x 2048 0.0027 of its norm off for 0.0018 of its own rounding).  Neighbouring fp32
// numbers have neighbouring bit patterns across binades too, so it is the patterns' difference, 2^8 of them a unit for bf16 and 2^5 for
// f16; sums that f16 holds as subnormals, whose rests are larger than a byte, keep what fits.  Half the bytes of a second 16-bit
// tensor, and within 2^-16 (2^-19) of the sum.
template <typename T>
struct Rest {
  static constexpr int SH = std::is_same<T, BF16>::value ? 8 : 5;
  __device__ __forceinline__ static int of(float sum, float h) {
    const uint32_t b = __float_as_uint(h);
    const int units = ((int)(__float_as_uint(sum) - b) + (1 << (SH - 1))) >> SH;
    return (b & 0x7f800000u) == 0x7f800000u ? 0 : units > 127 ? 127 : units < -128 ? -128 : units;
  }
  __device__ __forceinline__ static float sum(float h, int rest) { return __uint_as_float(__float_as_uint(h) + ((uint32_t)rest << SH)); }
  // Rows are filled up to whole pieces of eight.
  __device__ __forceinline__ static int64_t pitch(int64_t D) { return (D + 7) & ~(int64_t)7; }
  // Piece `col` of a row; one past its end: any, for `add` to drop.
  __device__ __forceinline__ static u32x2 load(uint64_t rests, int64_t row, int64_t col, int64_t D) {
    return *reinterpret_cast<const HK_G u32x2*>(gcptr<uint8_t>(rests) + row * pitch(D) + (col < D ? col : 0));
  }
  __device__ __forceinline__ static void add(u32x2 w, bool in, float* h) {
    if (!in) w = u32x2{0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = sum(h[e], (int8_t)(w[e >> 2] >> (8 * (e & 3))));
  }
  __device__ __forceinline__ static void put(uint64_t rests, int64_t row, int64_t col, int64_t D, const float* v, u32x4 packed) {
    float h[8];
    uint32_t q[8];
    RowVec<T>::unpack(packed, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = (uint32_t)of(v[e], h[e]);
    if (col < D) *reinterpret_cast<HK_G u32x2*>(gptr<uint8_t>(rests) + row * pitch(D) + col) = u32x2{pack_codes4(q), pack_codes4(q + 4)};
  }
};
template <typename T>
constexpr bool kRests = sizeof(typename T::storage) == 2;

// kQuant reads rows x (stride xs[0]) and writes codes (pitch q_sr) and scales; its arguments come in the same block, so that one
// kernel serves all three.
template <typename T, int MODE, int LPR, int NV, bool TAIL>
__global__ __launch_bounds__(threads_of(LPR)) void rms_rows(hrt_rms_args p, int64_t q_sr) {
  using R = RowVec<T>;
  using S = typename T::storage;
  constexpr int V = R::V, RPB = threads_of(LPR) / LPR;
  __shared__ float red[threads_of(LPR) / 64];
  __shared__ uint32_t redu[threads_of(LPR) / 64];
  const int lane = threadIdx.x % LPR;
  const int64_t row0 = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  const bool live = row0 < p.rows;
  const int64_t row = live ? row0 : p.rows - 1;  // a row past the end repeats the last one and stores nothing
  const HK_G S* const x = gcptr<S>(p.x) + (MODE == kQuant ? row * p.xs[0] : row_at(row, p.n1, p.n2, p.xs));
  u32x4 a[NV], b[NV], w[NV];
  const bool res = MODE != kQuant && p.r, has_w = MODE != kQuant && p.w;
#pragma unroll
  for (int c = 0; c < NV; ++c) a[c] = row_load<T, TAIL>(x, (int64_t)(c * LPR + lane) * V, p.D);
  if (res) {
    const HK_G S* const r = gcptr<S>(p.r) + row_at(row, p.n1, p.n2, p.rs);
#pragma unroll
    for (int c = 0; c < NV; ++c) b[c] = row_load<T, TAIL>(r, (int64_t)(c * LPR + lane) * V, p.D);
  }
  if (has_w) {
#pragma unroll
    for (int c = 0; c < NV; ++c) w[c] = row_load<T, TAIL>(gcptr<S>(p.w), (int64_t)(c * LPR + lane) * V, p.D);
  }
  float v[NV][V];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int64_t col = (int64_t)(c * LPR + lane) * V;
    R::unpack(row_fix<T, TAIL>(a[c], col, p.D), v[c]);
    if (res) {
      float t[V];
      R::unpack(row_fix<T, TAIL>(b[c], col, p.D), t);
#pragma unroll
      for (int e = 0; e < V; ++e) v[c][e] += t[e];
    }
    if (MODE != kQuant && p.h_out && live) {
      const u32x4 h = R::pack(v[c]);
      row_put<T, TAIL>(gptr<S>(p.h_out) + row * p.D, col, p.D, h);
      if constexpr (MODE == kNorm && kRests<T>)
        if (p.h_rest) Rest<T>::put(p.h_rest, row, col, p.D, v[c], h);
    }
    if (!TAIL && col >= p.D) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[c][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) ss = fmaf(v[c][e], v[c][e], ss);
  }
  if constexpr (MODE != kQuant) {
    const float rstd = 1.f / sqrtf(lanes_sum<LPR>(ss, red) / (float)p.D + p.eps);
    if (p.rstd && live && lane == 0) gptr<float>(p.rstd)[row] = rstd;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float t[V];
      if (has_w) R::unpack(row_fix<T, TAIL>(w[c], (int64_t)(c * LPR + lane) * V, p.D), t);
#pragma unroll
      for (int e = 0; e < V; ++e) v[c][e] = has_w ? v[c][e] * rstd * t[e] : v[c][e] * rstd;
    }
  }
  if constexpr (MODE == kNorm) {
    if (!live) return;
#pragma unroll
    for (int c = 0; c < NV; ++c) row_put<T, TAIL>(gptr<S>(p.y) + row * p.D, (int64_t)(c * LPR + lane) * V, p.D, R::pack(v[c]));
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      // lanes past the row hold zeros, but zero times an infinite rstd or weight is no zero
      const int64_t col = (int64_t)(c * LPR + lane) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t m = __float_as_uint(v[c][e]) & 0x7fffffffu;
        if ((TAIL ? col + e < p.D : col < p.D) && m > top) top = m;
      }
    }
    const RowCode code(lanes_max<LPR>(top, redu));
    if (!live) return;
    if (lane == 0) gptr<float>(p.scale)[row] = code.scale;
    HK_G uint8_t* const q = gptr<uint8_t>(p.q) + row * q_sr;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int64_t col = (int64_t)(c * LPR + lane) * V;
      if (col >= q_sr) continue;
      uint32_t k[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        k[e] = MODE == kQuant ? nearest_code<T>(v[c][e], code) : code_of(v[c][e], code);
        if (TAIL && col + e >= p.D) k[e] = 0;
      }
      if (code.per == 0.f) {  // nothing but zeros, or not finite
#pragma unroll
        for (int e = 0; e < V; ++e) k[e] = 0;
      }
      if (col + V <= q_sr) {
        typedef uint32_t __attribute__((aligned(1))) u32_any;
        typedef u32x2 __attribute__((aligned(1))) u32x2_any;
        if constexpr (V == 8) *reinterpret_cast<HK_G u32x2_any*>(q + col) = u32x2{pack_codes4(k), pack_codes4(k + 4)};
        else *reinterpret_cast<HK_G u32_any*>(q + col) = pack_codes4(k);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (col + e < q_sr) q[col + e] = (uint8_t)k[e];
      }
    }
  }
}

// Rows longer than a workgroup's registers: a workgroup a row, passes over it (the later ones read it from L2).
template <typename T, int MODE>
__global__ __launch_bounds__(256) void rms_long(hrt_rms_args p, int64_t q_sr) {
  using R = RowVec<T>;
  using S = typename T::storage;
  constexpr int V = R::V;
  __shared__ float red[4];
  __shared__ uint32_t redu[4];
  const int64_t row = blockIdx.x;
  const HK_G S* const x = gcptr<S>(p.x) + (MODE == kQuant ? row * p.xs[0] : row_at(row, p.n1, p.n2, p.xs));
  const HK_G S* const r = MODE != kQuant && p.r ? gcptr<S>(p.r) + row_at(row, p.n1, p.n2, p.rs) : nullptr;
  auto load = [&](int64_t col, float* v) {
    R::unpack(row_piece<T, true>(x, col, p.D), v);
    if (r) {
      float t[V];
      R::unpack(row_piece<T, true>(r, col, p.D), t);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += t[e];
    }
  };
  float rstd = 1.f;
  if constexpr (MODE != kQuant) {
    float ss = 0.f;
    for (int64_t col = threadIdx.x * V; col < p.D; col += 256 * V) {
      float v[V];
      load(col, v);
#pragma unroll
      for (int e = 0; e < V; ++e) ss = fmaf(v[e], v[e], ss);
      if (p.h_out) row_put<T, true>(gptr<S>(p.h_out) + row * p.D, col, p.D, R::pack(v));
      if constexpr (MODE == kNorm && kRests<T>)
        if (p.h_rest) Rest<T>::put(p.h_rest, row, col, p.D, v, R::pack(v));
    }
    rstd = 1.f / sqrtf(lanes_sum<256>(ss, red) / (float)p.D + p.eps);
    if (p.rstd && threadIdx.x == 0) gptr<float>(p.rstd)[row] = rstd;
  }
  auto norm = [&](int64_t col, float* v) {
    load(col, v);
    if constexpr (MODE == kQuant) return;
    float t[V];
    if (p.w) R::unpack(row_piece<T, true>(gcptr<S>(p.w), col, p.D), t);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = p.w ? v[e] * rstd * t[e] : v[e] * rstd;
  };
  if constexpr (MODE == kNorm) {
    for (int64_t col = threadIdx.x * V; col < p.D; col += 256 * V) {
      float v[V];
      norm(col, v);
      row_put<T, true>(gptr<S>(p.y) + row * p.D, col, p.D, R::pack(v));
    }
  } else {
    uint32_t top = 0;
    for (int64_t col = threadIdx.x * V; col < p.D; col += 256 * V) {
      float v[V];
      norm(col, v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
        if (col + e < p.D && m > top) top = m;
      }
    }
    const RowCode code(lanes_max<256>(top, redu));
    if (threadIdx.x == 0) gptr<float>(p.scale)[row] = code.scale;
    HK_G uint8_t* const q = gptr<uint8_t>(p.q) + row * q_sr;
    for (int64_t col = threadIdx.x * V; col < q_sr; col += 256 * V) {
      float v[V];
      norm(col, v);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (col + e < q_sr) q[col + e] = col + e < p.D && code.per != 0.f ? (uint8_t)(MODE == kQuant ? nearest_code<T>(v[e], code) : code_of(v[e], code)) : 0;
    }
  }
}

// ---- backward -------------------------------------------------------------------------------------------------------------
// dw where there are few rows: the workgroups behind those that take rows have strips of 128 bytes of columns each, of all rows
// (which the others read too: from L2).
template <typename T, bool TAIL, bool REST, int TPB>
__device__ __forceinline__ void rms_strip(const hrt_rms_bwd_args& p, int strip) {
  using R = RowVec<T>;
  using S = typename T::storage;
  constexpr int V = R::V, G = TPB / 8;  // rows at a time
  __shared__ float red[G][8 * V + 1];
  const int lane = threadIdx.x & 7, group = threadIdx.x >> 3;
  const int64_t col = ((int64_t)strip * 8 + lane) * V;
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  for (int64_t r0 = group; r0 < p.rows; r0 += 4 * G) {
    u32x4 a[4], b[4];
    u32x2 rest[4];
    float rstd[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // four rows' loads in flight; a row past the end repeats the last one
      const int64_t row = r0 + u * G < p.rows ? r0 + u * G : p.rows - 1;
      a[u] = row_load<T, TAIL>(gcptr<S>(p.gy) + row_at(row, p.n1, p.n2, p.gys), col, p.D);
      b[u] = row_load<T, TAIL>(gcptr<S>(p.h) + row_at(row, p.n1, p.n2, p.hs), col, p.D);
      rstd[u] = gcptr<float>(p.rstd)[row];
      if constexpr (REST) rest[u] = Rest<T>::load(p.h_rest, row, col, p.D);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float d[V], n[V];
      R::unpack(row_fix<T, TAIL>(a[u], col, p.D), d);
      R::unpack(row_fix<T, TAIL>(b[u], col, p.D), n);
      if constexpr (REST) Rest<T>::add(rest[u], col < p.D, n);
      if (r0 + u * G < p.rows) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += d[e] * (n[e] * rstd[u]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) red[group][lane * V + e] = acc[e];
  __syncthreads();
  const int64_t at = (int64_t)strip * 8 * V + threadIdx.x;
  if ((int)threadIdx.x >= 8 * V || at >= p.D) return;
  float t = red[0][threadIdx.x];
#pragma unroll 8
  for (int k = 1; k < G; ++k) t += red[k][threadIdx.x];
  gptr<S>(p.dw)[at] = T::from_f32(t);
}

// A workgroup takes `per` consecutive rows, one for every LPR threads at a time.  DW: a lane adds gy n of its columns up over its rows, the
// workgroup's lanes of a column are added in order through LDS, and the sums of all workgroups by rms_dw_sum.
// REST: what rounding took from h is there (kernels of their own: without it 800 x 800 would take 8.1 us, so 7.6).
template <typename T, int LPR, int NV, bool TAIL, bool DW, bool REST>
__global__ __launch_bounds__(threads_of(LPR)) void rms_back(hrt_rms_bwd_args p, int64_t per, int blocks) {
  using R = RowVec<T>;
  using S = typename T::storage;
  constexpr int V = R::V, RPB = threads_of(LPR) / LPR;
  if constexpr (!DW) {
    if ((int)blockIdx.x >= blocks) return rms_strip<T, TAIL, REST, threads_of(LPR)>(p, (int)blockIdx.x - blocks);
  }
  __shared__ float red[2][threads_of(LPR) / 64];
  __shared__ __attribute__((aligned(16))) float part[DW && RPB > 1 ? RPB * LPR * NV * V : 4];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int64_t first = (int64_t)blockIdx.x * per, end = first + per < p.rows ? first + per : p.rows;
  float acc[NV][V];
  u32x4 w[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    w[c] = u32x4{0, 0, 0, 0};
    if (p.w) w[c] = row_piece<T, TAIL>(gcptr<S>(p.w), (int64_t)(c * LPR + lane) * V, p.D);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[c][e] = 0.f;
  }
  int turn = 0;
  for (int64_t base = first; base < end; base += RPB, turn ^= 1) {
    const bool live = base + group < end;
    const int64_t row = live ? base + group : end - 1;
    const HK_G S* const gy = gcptr<S>(p.gy) + row_at(row, p.n1, p.n2, p.gys);
    const HK_G S* const h = gcptr<S>(p.h) + row_at(row, p.n1, p.n2, p.hs);
    u32x4 a[NV], b[NV], g[NV];
    u32x2 rest[NV];
    const float rstd = gcptr<float>(p.rstd)[row];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int64_t col = (int64_t)(c * LPR + lane) * V;
      g[c] = u32x4{0, 0, 0, 0};
      b[c] = row_load<T, TAIL>(h, col, p.D);
      a[c] = row_load<T, TAIL>(gy, col, p.D);
      if constexpr (REST) rest[c] = Rest<T>::load(p.h_rest, row, col, p.D);
    }
    if (p.gh) {
      const HK_G S* const gh = gcptr<S>(p.gh) + row_at(row, p.n1, p.n2, p.ghs);
#pragma unroll
      for (int c = 0; c < NV; ++c) g[c] = row_load<T, TAIL>(gh, (int64_t)(c * LPR + lane) * V, p.D);
    }
    float d[NV][V], n[NV][V];
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int64_t col = (int64_t)(c * LPR + lane) * V;
      a[c] = row_fix<T, TAIL>(a[c], col, p.D), b[c] = row_fix<T, TAIL>(b[c], col, p.D);
      if (!live || (!TAIL && col >= p.D)) a[c] = u32x4{0, 0, 0, 0}, b[c] = u32x4{0, 0, 0, 0};
      float t[V];
      R::unpack(a[c], d[c]);
      R::unpack(b[c], n[c]);
      if constexpr (REST) Rest<T>::add(rest[c], live && col < p.D, n[c]);
      if (p.w) R::unpack(w[c], t);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        n[c][e] *= rstd;
        if constexpr (DW) acc[c][e] += !TAIL || col + e < p.D ? (live && col < p.D ? d[c][e] * n[c][e] : 0.f) : 0.f;
        if (p.w) d[c][e] *= t[e];
        if (TAIL ? col + e < p.D : col < p.D) dot = fmaf(d[c][e], n[c][e], dot);
      }
    }
    dot = lanes_sum<LPR>(dot, red[turn]) / (float)p.D;
    if (!p.dx || !live) continue;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float t[V];
      R::unpack(row_fix<T, TAIL>(g[c], (int64_t)(c * LPR + lane) * V, p.D), t);
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = fmaf(rstd, fmaf(-n[c][e], dot, d[c][e]), t[e]);
      row_put<T, TAIL>(gptr<S>(p.dx) + row * p.D, (int64_t)(c * LPR + lane) * V, p.D, R::pack(t));
    }
  }
  if constexpr (DW) {
    HK_G float* const ws = gptr<float>(p.ws) + (int64_t)blockIdx.x * p.D;
    if constexpr (RPB == 1) {
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if ((int64_t)(c * LPR + lane) * V + e < p.D) ws[(c * LPR + lane) * V + e] = acc[c][e];
    } else {
      constexpr int W = LPR * NV * V;
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < V; e += 4)
          *reinterpret_cast<f32x4*>(part + group * W + (c * LPR + lane) * V + e) = f32x4{acc[c][e], acc[c][e + 1], acc[c][e + 2], acc[c][e + 3]};
      __syncthreads();
      for (int i = threadIdx.x; i < p.D; i += 256) {
        float t = part[i];
#pragma unroll
        for (int k = 1; k < RPB; ++k) t += part[k * W + i];
        ws[i] = t;
      }
    }
  }
}

// Rows longer than a workgroup's registers; ws is added to in place, each column by its own thread.
template <typename T>
__global__ __launch_bounds__(256) void rms_back_long(hrt_rms_bwd_args p, int64_t per) {
  using R = RowVec<T>;
  using S = typename T::storage;
  constexpr int V = R::V;
  __shared__ float red[2][4];
  const int64_t first = (int64_t)blockIdx.x * per, end = first + per < p.rows ? first + per : p.rows;
  HK_G float* const ws = gptr<float>(p.ws) + (int64_t)blockIdx.x * p.D;
  for (int64_t row = first; row < end; ++row) {
    const HK_G S* const gy = gcptr<S>(p.gy) + row_at(row, p.n1, p.n2, p.gys);
    const HK_G S* const h = gcptr<S>(p.h) + row_at(row, p.n1, p.n2, p.hs);
    const HK_G S* const gh = gcptr<S>(p.gh) + (p.gh ? row_at(row, p.n1, p.n2, p.ghs) : 0);
    const float rstd = gcptr<float>(p.rstd)[row];
    auto load = [&](int64_t col, float* d, float* n, float* gyn) {
      float t[V];
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = 1.f;
      R::unpack(row_piece<T, true>(gy, col, p.D), d);
      R::unpack(row_piece<T, true>(h, col, p.D), n);
      if constexpr (kRests<T>)
        if (p.h_rest) Rest<T>::add(Rest<T>::load(p.h_rest, row, col, p.D), true, n);
      if (p.w) R::unpack(row_piece<T, true>(gcptr<S>(p.w), col, p.D), t);
#pragma unroll
      for (int e = 0; e < V; ++e) n[e] *= rstd, gyn[e] = d[e] * n[e], d[e] *= t[e];
    };
    float dot = 0.f;
    for (int64_t col = threadIdx.x * V; col < p.D; col += 256 * V) {
      float d[V], n[V], gyn[V];
      load(col, d, n, gyn);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (col + e < p.D) {
          dot = fmaf(d[e], n[e], dot);
          if (p.dw) ws[col + e] = row == first ? gyn[e] : ws[col + e] + gyn[e];
        }
    }
    dot = lanes_sum<256>(dot, red[row & 1]) / (float)p.D;
    if (!p.dx) continue;
    for (int64_t col = threadIdx.x * V; col < p.D; col += 256 * V) {
      float d[V], n[V], t[V];
      load(col, d, n, t);
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = 0.f;
      if (p.gh) R::unpack(row_piece<T, true>(gh, col, p.D), t);
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = fmaf(rstd, fmaf(-n[e], dot, d[e]), t[e]);
      row_put<T, true>(gptr<S>(p.dx) + row * p.D, col, p.D, R::pack(t));
    }
  }
}

// Without gy: the norm's share is zeros whatever the row, and h, rstd and w, which need not be finite, are not read.  A workgroup a row,
// every 65536th from there on.
template <typename T>
__global__ __launch_bounds__(256) void rms_back_rest(hrt_rms_bwd_args p) {
  using S = typename T::storage;
  constexpr int V = RowVec<T>::V;
  for (int64_t row = blockIdx.x; p.dx && row < p.rows; row += gridDim.x) {
    const HK_G S* const gh = gcptr<S>(p.gh) + (p.gh ? row_at(row, p.n1, p.n2, p.ghs) : 0);
    for (int64_t col = threadIdx.x * V; col < p.D; col += 256 * V)
      row_put<T, true>(gptr<S>(p.dx) + row * p.D, col, p.D, p.gh ? row_piece<T, true>(gh, col, p.D) : u32x4{0, 0, 0, 0});
  }
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; p.dw && i < p.D; i += (int64_t)gridDim.x * 256) gptr<S>(p.dw)[i] = 0;
}

// dw: the workgroups' sums of 32 columns, a thread every 32nd of one column in order (16 loads in flight: one round for 512), then the
// 32 of a column in order.
template <typename T>
__global__ __launch_bounds__(1024) void rms_dw_sum(const float* ws, typename T::storage* dw, int64_t parts, int64_t D) {
  constexpr int U = 16;
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int64_t at = (int64_t)blockIdx.x * 32 + lane, col = at < D ? at : D - 1;
  float s = 0.f;
  for (int64_t c = group; c < parts; c += 32 * U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = ws[(c + u * 32 < parts ? c + u * 32 : parts - 1) * D + col];
#pragma unroll
    for (int u = 0; u < U; ++u) s += c + u * 32 < parts ? v[u] : 0.f;
  }
  red[group][lane] = s;
  __syncthreads();
  if (group > 0 || at >= D) return;
  float o = red[0][lane];
#pragma unroll
  for (int i = 1; i < 32; ++i) o += red[i][lane];
  dw[at] = T::from_f32(o);
}

// ---- plan and launch --------------------------------------------------------------------------------------------------------
// Lanes per row and pieces per lane; 0: the passes.  Few rows of model width are shared by a workgroup: its four wavefronts'
// loads are all in flight at once (D 2048 in bf16, us with a wavefront and with a workgroup a row: 64 rows 3.5, 3.1; 308 3.7, 3.3; 1024
// 4.1, 4.3; 2048 5.0, 5.9; 8192 12.0, 15.7).
struct Share {
  int lpr, nv;
};
Share share_of(int64_t rows, int64_t D, int V) {
  const int64_t n = cdiv(D, V);
  if (n <= 16) return {16, 1};
  if (n <= 32) return {16, 2};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return rows >= 1024 ? Share{64, 4} : Share{256, 1};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {256, 4};
  if (n <= 2048) return {1024, 2};
  return {0, 0};
}

template <typename F>
void with_share(Share s, F f) {
#define HK_SHARE(L, N) \
  if (s.lpr == L && s.nv == N) return f(std::integral_constant<int, L>(), std::integral_constant<int, N>())
  HK_SHARE(16, 1);
  HK_SHARE(16, 2);
  HK_SHARE(64, 1);
  HK_SHARE(64, 2);
  HK_SHARE(64, 4);
  HK_SHARE(256, 1);
  HK_SHARE(256, 2);
  HK_SHARE(256, 4);
  HK_SHARE(1024, 2);
#undef HK_SHARE
}

template <typename T, int MODE>
bool queue_rows(const hrt_rms_args& a, int64_t q_sr, hrt::LaunchCtx& ctx) {
  constexpr int V = RowVec<T>::V;
  const Share s = share_of(a.rows, a.D, V);
  if (s.lpr == 0) {
    if (!hrt::grid_fits(a.rows, 256)) return ctx.fail("grid too large");
    hipLaunchKernelGGL((rms_long<T, MODE>), dim3((uint32_t)a.rows), dim3(256), 0, ctx.stream, a, q_sr);
    return true;
  }
  const int64_t blocks = cdiv(a.rows, threads_of(s.lpr) / s.lpr);
  if (!hrt::grid_fits(blocks, threads_of(s.lpr))) return ctx.fail("grid too large");
  with_share(s, [&](auto lc, auto nc) {
    constexpr int L = decltype(lc)::value, N = decltype(nc)::value;
    if (a.D % V == 0) hipLaunchKernelGGL((rms_rows<T, MODE, L, N, false>), dim3((uint32_t)blocks), dim3(threads_of(L)), 0, ctx.stream, a, q_sr);
    else hipLaunchKernelGGL((rms_rows<T, MODE, L, N, true>), dim3((uint32_t)blocks), dim3(threads_of(L)), 0, ctx.stream, a, q_sr);
  });
  return true;
}

// Byte extent of rows reached through three outer dimensions.
uint64_t rows_span(int64_t rows, int64_t n1, int64_t n2, int64_t D, const int64_t* s, uint64_t elem) {
  const int64_t n0 = cdiv(rows, n1 * n2);
  return uint64_t((n0 - 1) * s[0] + (n1 - 1) * s[1] + (n2 - 1) * s[2] + D) * elem;
}
bool rows_ok(int64_t rows, int64_t D, int64_t n1, int64_t n2, std::initializer_list<const int64_t*> strides, uint64_t elem,
             std::initializer_list<uint64_t> addrs, hrt::LaunchCtx& ctx) {
  constexpr int64_t lim = int64_t(1) << 31;
  if (rows <= 0 || D <= 0 || n1 <= 0 || n2 <= 0 || rows >= lim || D >= lim || n1 > rows || n2 > rows || rows % (n1 * n2) != 0)
    return ctx.fail("bad shape");
  for (const int64_t* s : strides)
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0) return ctx.fail("negative stride");
  for (const uint64_t p : addrs)
    if (p % elem != 0) return ctx.fail("operands must be aligned to their elements");
  return true;
}

template <typename T>
bool launch_rms_fwd(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_rms_args*>(pp);
  using S = typename T::storage;
  constexpr uint64_t E = sizeof(S);
  if (!rows_ok(a.rows, a.D, a.n1, a.n2, {a.xs, a.rs}, E, {a.x, a.r, a.w, a.y, a.h_out}, ctx)) return false;
  if (a.scale % 4 != 0 || a.rstd % 4 != 0) return ctx.fail("scale and rstd must be 4-byte aligned");
  if (a.h_rest && (E != 2 || !a.r || !a.y || !a.h_out || a.h_rest % 8 != 0)) return ctx.fail("h_rest: beside a 16-bit h and y of a sum, 8-byte aligned");
  if ((a.q != 0) != (a.scale != 0) || (a.q != 0) == (a.y != 0)) return ctx.fail("either y, or q and scale");
  const uint64_t n = (uint64_t)a.rows * a.D;
  if (!ctx.check(a.x, rows_span(a.rows, a.n1, a.n2, a.D, a.xs, E), "x") ||
      (a.r && !ctx.check(a.r, rows_span(a.rows, a.n1, a.n2, a.D, a.rs, E), "r")) || (a.w && !ctx.check(a.w, a.D * E, "w")) ||
      (a.y && !ctx.check(a.y, n * E, "y")) || (a.h_out && !ctx.check(a.h_out, n * E, "h_out")) || (a.q && !ctx.check(a.q, n, "q")) ||
      (a.h_rest && !ctx.check(a.h_rest, a.rows * (cdiv(a.D, 8) * 8), "h_rest")) ||
      (a.scale && !ctx.check(a.scale, a.rows * 4, "scale")) || (a.rstd && !ctx.check(a.rstd, a.rows * 4, "rstd")))
    return false;
  if (!(a.q ? queue_rows<T, kNorm8>(a, a.D, ctx) : queue_rows<T, kNorm>(a, a.D, ctx))) return false;
  return hrt::launch_ok(hipGetLastError(), ctx, "rms_fwd");
}

template <typename T>
bool launch_quant(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_i8_rows_args*>(pp);
  constexpr uint64_t E = sizeof(typename T::storage);
  const int64_t s[3] = {a.x_sr, 0, 0};
  if (!rows_ok(a.rows, a.cols, 1, 1, {s}, E, {a.x}, ctx)) return false;
  // the lanes of a row cover a multiple of 16 columns: those that follow the row become 0 without a pass of their own
  if (a.q_sr < a.cols || a.q_sr > cdiv(a.cols, 16) * 16 || a.scale % 4 != 0) return ctx.fail("bad pitch of q or alignment of scale");
  const int64_t qt[2] = {a.q_sr, 1}, sz[2] = {a.rows, a.q_sr};
  if (!ctx.check(a.x, rows_span(a.rows, 1, 1, a.cols, s, E), "x") || !ctx.check(a.q, hrt::span_bytes(2, sz, qt, 1), "q") ||
      !ctx.check(a.scale, a.rows * 4, "scale"))
    return false;
  hrt_rms_args r{};
  r.x = a.x, r.q = a.q, r.scale = a.scale, r.rows = a.rows, r.D = a.cols, r.n1 = r.n2 = 1, r.xs[0] = a.x_sr;
  if (!queue_rows<T, kQuant>(r, a.q_sr, ctx)) return false;
  return hrt::launch_ok(hipGetLastError(), ctx, "i8_rows_quant");
}

// Whether dw is summed by strips of columns in the same launch: the GPU's time then meets that of the two launches at 800 x 800 and
// 1024 x 2048 (7.6, 9.5 us both ways; 308 x 1000 fp32 4.5 against 7.5, 512 x 8192 bf16 8.8 against 25), the host's is 5 us less.
bool strips(const hrt_rms_bwd_args& a, Share s) { return a.dw && s.lpr && a.rows <= 1024; }
// Rows per workgroup of the backward: with sums of dw as many as leave 512 workgroups, or 256 of 1024 threads (4096 x 8192 bf16 47 us
// with 512 workgroups, 52 with 256; 2000 x 5001 fp32 36 and 32).
int64_t back_rows(const hrt_rms_bwd_args& a, Share s) {
  const int64_t rpb = s.lpr ? threads_of(s.lpr) / s.lpr : 1;
  return a.dw && !strips(a, s) ? cdiv(cdiv(a.rows, s.lpr > 256 ? 256 : 512), rpb) * rpb : rpb;
}
template <typename T>
int64_t back_blocks(const hrt_rms_bwd_args& a) {
  return cdiv(a.rows, back_rows(a, share_of(a.rows, a.D, RowVec<T>::V)));
}

template <typename T>
bool launch_rms_bwd(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_rms_bwd_args*>(pp);
  using S = typename T::storage;
  constexpr uint64_t E = sizeof(S);
  constexpr int V = RowVec<T>::V;
  if (!rows_ok(a.rows, a.D, a.n1, a.n2, {a.gys, a.ghs, a.hs}, E, {a.gy, a.gh, a.h, a.w, a.dx, a.dw}, ctx)) return false;
  if (a.rstd % 4 != 0 || a.ws % 4 != 0) return ctx.fail("rstd and ws must be 4-byte aligned");
  if (a.h_rest && (E != 2 || a.h_rest % 8 != 0)) return ctx.fail("h_rest: of 16-bit values, 8-byte aligned");
  if (!a.dx && !a.dw) return true;
  const uint64_t n = (uint64_t)a.rows * a.D;
  const int64_t blocks = back_blocks<T>(a);
  if ((a.gy && !ctx.check(a.gy, rows_span(a.rows, a.n1, a.n2, a.D, a.gys, E), "gy")) ||
      (a.gh && !ctx.check(a.gh, rows_span(a.rows, a.n1, a.n2, a.D, a.ghs, E), "gh")) ||
      (a.gy && (!ctx.check(a.h, rows_span(a.rows, a.n1, a.n2, a.D, a.hs, E), "h") || !ctx.check(a.rstd, a.rows * 4, "rstd"))) ||
      (a.gy && a.h_rest && !ctx.check(a.h_rest, a.rows * (cdiv(a.D, 8) * 8), "h_rest")) || (a.gy && a.w && !ctx.check(a.w, a.D * E, "w")) || (a.dx && !ctx.check(a.dx, n * E, "dx")) ||
      (a.dw && !ctx.check(a.dw, a.D * E, "dw")))
    return false;
  if (!a.gy) {
    hipLaunchKernelGGL(rms_back_rest<T>, dim3(a.rows < 65536 ? (uint32_t)a.rows : 65536u), dim3(256), 0, ctx.stream, a);
    return hrt::launch_ok(hipGetLastError(), ctx, "rms_bwd");
  }
  const Share s = share_of(a.rows, a.D, V);
  const bool sums = a.dw && !strips(a, s);
  if (sums && !ctx.check(a.ws, (uint64_t)(blocks * a.D) * 4, "ws")) return false;
  const int64_t per = back_rows(a, s), all = blocks + (a.dw && !sums ? cdiv(a.D, 8 * V) : 0);
  if (!hrt::grid_fits(all, threads_of(s.lpr))) return ctx.fail("grid too large");
  const dim3 grid((uint32_t)all);
  if (s.lpr == 0) {
    hipLaunchKernelGGL(rms_back_long<T>, grid, dim3(256), 0, ctx.stream, a, per);
  } else {
    with_share(s, [&](auto lc, auto nc) {
      constexpr int L = decltype(lc)::value, N = decltype(nc)::value;
      const auto go = [&](auto tail, auto dw, auto rest) {
        hipLaunchKernelGGL((rms_back<T, L, N, decltype(tail)::value, decltype(dw)::value, decltype(rest)::value>), grid, dim3(threads_of(L)), 0, ctx.stream, a,
                           per, (int)blocks);
      };
      using Y = std::true_type;
      using No = std::false_type;
      const auto both = [&](auto rest) {
        if (a.D % V == 0) sums ? go(No(), Y(), rest) : go(No(), No(), rest);
        else sums ? go(Y(), Y(), rest) : go(Y(), No(), rest);
      };
      if constexpr (kRests<T>) a.h_rest ? both(Y()) : both(No());
      else both(No());
    });
  }
  if (sums)
    hipLaunchKernelGGL(rms_dw_sum<T>, dim3((uint32_t)cdiv(a.D, 32)), dim3(1024), 0, ctx.stream, (const float*)a.ws, (S*)a.dw, blocks, a.D);
  return hrt::launch_ok(hipGetLastError(), ctx, "rms_bwd");
}

#define HK_ROWS(SUFFIX, T)                                              \
  HRT_REGISTER("rms_fwd_" SUFFIX, hrt_rms_args, launch_rms_fwd<T>);     \
  HRT_REGISTER("rms_bwd_" SUFFIX, hrt_rms_bwd_args, launch_rms_bwd<T>); \
  HRT_REGISTER("i8_rows_quant_" SUFFIX, hrt_i8_rows_args, launch_quant<T>)
HK_ROWS("f32", F32);
HK_ROWS("bf16", BF16);
HK_ROWS("f16", F16);

}  // namespace
}  // namespace hk

extern "C" int64_t hrt_rms_workspace(const hrt_rms_bwd_args* a, int32_t dtype) {
  using namespace hk;
  if (!a || a->rows <= 0 || a->D <= 0 || !a->dw || !a->gy) return 0;
  if (strips(*a, share_of(a->rows, a->D, dtype == HRT_F32 ? 4 : 8))) return 0;
  return (dtype == HRT_F32 ? back_blocks<F32>(*a) : back_blocks<BF16>(*a)) * a->D;
}
