// 8-bit rows back to values ("i8_rows_dequant_*"), alone and beside the sums of a gradient's columns ("i8_linear_back_*"): what the
// gradients of the 8-bit linear layer take beside a product, in one launch.
//
// The values are rounded to 16 bits because the matrix cores take them so: their scales differ along the axis that the product sums over,
// and moved to the gradient they would round that instead, by as much.  It puts the input's gradient 0.0024 of its norm off in bf16, of
// which its own rounding is 0.0017.
//
// Both are bound by memory.  The sums' workgroups come first: each has 128 bytes of columns (a cache line) of all rows, eight loads of
// a lane in flight, so that no second launch has to join partial sums.  Measured, GPU us (values, sums, both): W 8192 x 2048 under 4096 rows
// 10.4, 14.2, 21.1 (117 MB: 5.5 TB/s); W 2048 x 2048 under 308 rows 4.8, 3.3, 5.0.
#include "../hrt/registry.h"
#include "row_vec.h"

namespace hk {
namespace {

constexpr int kThreads = 512;

// 16 codes a lane, lpr lanes a row; a workgroup takes whole rows, several where they are short.  A row's last piece is its last 16
// codes, some of them its neighbour's too, which writes the same values (one by one the last codes cost a load's latency each).
template <typename T>
__device__ __forceinline__ void dequant_rows(const hrt_i8_rows_args& p, int64_t block, int lpr) {
  using R = RowVec<T>;
  using S = typename T::storage;
  constexpr int V = R::V;
  const int per = kThreads / lpr;
  const int64_t row = block * per + threadIdx.x / lpr;
  if ((int)threadIdx.x >= per * lpr || row >= p.rows) return;
  const float s = gcptr<float>(p.scale)[row];
  const HK_G uint8_t* const q = gcptr<uint8_t>(p.q) + row * p.q_sr;
  HK_G S* const x = gptr<S>(p.x) + row * p.x_sr;
  for (int64_t piece = (int64_t)(threadIdx.x % lpr) * 16; piece < p.cols; piece += (int64_t)lpr * 16) {
    const int64_t col = piece + 16 <= p.cols ? piece : p.cols - 16;
    if (col >= 0) {
      typedef u32x4 __attribute__((aligned(1))) any1;
      const u32x4 c = *reinterpret_cast<const HK_G any1*>(q + col);
#pragma unroll
      for (int i = 0; i < 16; i += V) {
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)(int8_t)(c[(i + e) >> 2] >> (8 * (e & 3))) * s;
        R::put(x + col + i, R::pack(v));
      }
    } else {
      for (int64_t e = 0; e < p.cols; ++e) x[e] = T::from_f32((float)(int8_t)q[e] * s);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void i8_dequant(hrt_i8_rows_args p, int lpr) {
  dequant_rows<T>(p, blockIdx.x, lpr);
}

// TAIL: N is no multiple of 8.
template <typename T, bool TAIL>
__global__ __launch_bounds__(kThreads) void i8_linear_back(hrt_i8_linear_back_args p, int sums, int lpr) {
  using R = RowVec<T>;
  constexpr int V = R::V, G = kThreads / 8, U = 8;  // rows at a time, of them in flight
  if ((int)blockIdx.x >= sums) {
    dequant_rows<T>({p.v, p.w, p.w_scale, p.N, p.K, p.K, p.w_sn}, blockIdx.x - sums, lpr);
    return;
  }
  __shared__ float red[G][8 * V + 1];
  const int lane = threadIdx.x & 7, group = threadIdx.x >> 3;
  const int64_t col = ((int64_t)blockIdx.x * 8 + lane) * V;
  const HK_G uint16_t* const g = gcptr<uint16_t>(p.g);
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  for (int64_t r0 = group; r0 < p.M; r0 += U * G) {
    u32x4 a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = row_load<T, TAIL>(g + (r0 + u * G < p.M ? r0 + u * G : p.M - 1) * p.g_sm, col, p.N);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[V];
      R::unpack(row_fix<T, TAIL>(a[u], col, p.N), v);
      if (r0 + u * G < p.M) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += v[e];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) red[group][lane * V + e] = acc[e];
  __syncthreads();
  // eight of the 64 sums of a column to a thread, then the eight, in a fixed order
  const int c = threadIdx.x & 63, k = threadIdx.x >> 6;
  float t = red[8 * k][c];
#pragma unroll
  for (int i = 1; i < 8; ++i) t += red[8 * k + i][c];
  __syncthreads();
  red[k][c] = t;
  __syncthreads();
  const int64_t at = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x >= 64 || at >= p.N) return;
  float o = red[0][threadIdx.x];
#pragma unroll
  for (int i = 1; i < 8; ++i) o += red[i][threadIdx.x];
  gptr<uint16_t>(p.db)[at] = T::from_f32(o);
}

// Lanes of a row of codes, and the workgroups that all rows take.
int lanes_of(int64_t cols) { return cdiv(cols, 16) < kThreads ? (int)cdiv(cols, 16) : kThreads; }
int64_t blocks_of(int64_t rows, int64_t cols) { return cdiv(rows, kThreads / lanes_of(cols)); }

bool check_rows(const hrt_i8_rows_args& a, uint64_t elem, hrt::LaunchCtx& ctx) {
  const int64_t lim = (int64_t)1 << 31;
  if (a.rows <= 0 || a.cols <= 0 || a.rows >= lim || a.cols >= lim) return ctx.fail("bad shape");
  if (a.x_sr < a.cols || a.q_sr < 0) return ctx.fail("overlapping rows of x, or a negative stride");
  if (a.x % elem != 0 || a.scale % 4 != 0) return ctx.fail("operands must be aligned to their elements");
  const int64_t sz[2] = {a.rows, a.cols}, xs[2] = {a.x_sr, 1}, qs[2] = {a.q_sr, 1};
  if (!ctx.check(a.x, hrt::span_bytes(2, sz, xs, elem), "x") || !ctx.check(a.q, hrt::span_bytes(2, sz, qs, 1), "q") ||
      !ctx.check(a.scale, (uint64_t)a.rows * 4, "scale"))
    return false;
  return true;
}

template <typename T>
bool launch_dequant(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_i8_rows_args*>(pp);
  if (!check_rows(a, sizeof(typename T::storage), ctx)) return false;
  const int64_t blocks = blocks_of(a.rows, a.cols);
  if (!hrt::grid_fits(blocks, kThreads)) return ctx.fail("grid too large");
  hipLaunchKernelGGL(i8_dequant<T>, dim3((uint32_t)blocks), dim3(kThreads), 0, ctx.stream, a, lanes_of(a.cols));
  return hrt::launch_ok(hipGetLastError(), ctx, "i8_rows_dequant");
}

template <typename T>
bool launch_back(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_i8_linear_back_args*>(pp);
  const int64_t lim = (int64_t)1 << 31;
  if (a.N <= 0 || a.N >= lim) return ctx.fail("bad shape");
  if (!a.v && !a.db) return true;
  if (a.v && !check_rows({a.v, a.w, a.w_scale, a.N, a.K, a.K, a.w_sn}, 2, ctx)) return false;
  if (a.db) {
    if (a.M <= 0 || a.M >= lim || a.g_sm < 0 || a.g % 2 != 0 || a.db % 2 != 0) return ctx.fail("bad rows of g");
    const int64_t sz[2] = {a.M, a.N}, gs[2] = {a.g_sm, 1};
    if (!ctx.check(a.g, hrt::span_bytes(2, sz, gs, 2), "g") || !ctx.check(a.db, (uint64_t)a.N * 2, "db")) return false;
  }
  const int64_t sums = a.db ? cdiv(a.N, 64) : 0, blocks = sums + (a.v ? blocks_of(a.N, a.K) : 0);
  if (!hrt::grid_fits(blocks, kThreads)) return ctx.fail("grid too large");
  const int lpr = a.v ? lanes_of(a.K) : 1;
  if (a.N % 8 == 0) hipLaunchKernelGGL((i8_linear_back<T, false>), dim3((uint32_t)blocks), dim3(kThreads), 0, ctx.stream, a, (int)sums, lpr);
  else hipLaunchKernelGGL((i8_linear_back<T, true>), dim3((uint32_t)blocks), dim3(kThreads), 0, ctx.stream, a, (int)sums, lpr);
  return hrt::launch_ok(hipGetLastError(), ctx, "i8_linear_back");
}

HRT_REGISTER("i8_rows_dequant_f32", hrt_i8_rows_args, launch_dequant<F32>);
HRT_REGISTER("i8_rows_dequant_bf16", hrt_i8_rows_args, launch_dequant<BF16>);
HRT_REGISTER("i8_rows_dequant_f16", hrt_i8_rows_args, launch_dequant<F16>);
HRT_REGISTER("i8_linear_back_bf16", hrt_i8_linear_back_args, launch_back<BF16>);
HRT_REGISTER("i8_linear_back_f16", hrt_i8_linear_back_args, launch_back<F16>);

}  // namespace
}  // namespace hk
