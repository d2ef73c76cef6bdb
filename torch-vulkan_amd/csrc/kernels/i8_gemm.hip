// "i8_mm_{bf16,f16}": y = (X W^T) * x_scale * w_scale + bias on 8-bit rows, whole sums in 32 bits (exact), one rounding at the end.
//
// Two kernels:
//   * i8_rows for few rows: bound by the weights' bytes, in practice by one memory latency.  A wavefront takes 16 columns of y and
//     every NWVth 128-wide piece of K, its loads all in flight at once; no LDS but for the wavefronts' sums.
//   * i8_tile for the rest: bound by the matrix cores and by L2 -> LDS.  Both operands are copied global -> LDS directly, in rows
//     of 128 bytes (whole cache lines), XOR-swizzled by 16-byte chunks (tile_swz<8>).
// Lane layout of the 8-bit products (checked on the device), l = lane: 32x32x32: operand row l % 32, bytes 16 (l / 32) .. + 15 of K;
// 16x16x64: row l % 16, bytes 16 (l / 16) .. + 15; accumulators as for the 16-bit products of the same shape.
// W is the first operand, so an accumulator holds four consecutive columns n of one row m of y.
// Measured, M x N x K, us, replayed on the same operands (in brackets on operands from HBM, rotated through 600 MB): 1 x 8192 x 2048 5.8 (5.5),
// 16 x 8192 x 2048 7.1 (7.4), 308 x 2048 x 2048 6.2 (9.9), 308 x 8192 x 2048 11.6 (17.9), 2048 cubed 15 (18.6), 1024 x 2048 x 8192 26 (34),
// 4096 x 8192 x 2048 69 to 72 by box (74 to 78; 1.9 to 2.0 POP/s), 4096 x 2048 x 8192 63 to 66 (73; 2.1 to 2.2), 8192 cubed 422 to 452 (2.4 to
// 2.6 POP/s; a library's 8-bit product of that size: 526).
// The largest tiles' step has 2048 cycles of products, 2048 of LDS (192 KiB of fragments, 64 KiB of copies) and 2200 of L2 -> LDS; it takes
// 2900 on half of the CUs and 4000 on all of them (matrix cores busy 55%).
#include <utility>

#include "../hrt/registry.h"
#include "lds_stage.h"
#include "row_vec.h"

namespace hk {
namespace {

// Lambdas of a kernel with many copies of its step: the compiler would make them functions.
#define HK_INLINE __attribute__((always_inline))

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ i32x4 mac16(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ i32x16 mac32(u32x4 a, u32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Values n .. n + 3 of row m from whole sums: sum * x_scale is taken first (the product of two small scales may underflow), or
// sum * w_scale where x_scale is so large that the sum times it might overflow under a small w_scale: a sum is at most 2^31.
constexpr float kFarScale = 0x1p64f;
template <typename T>
__device__ __forceinline__ void store4(const hrt_i8_mm_args& p, int64_t m, int64_t n, const int* v, float sx, bool vec) {
  if (m >= p.M || n >= p.N) return;
  const HK_G float* sw = gcptr<float>(p.w_scale) + n;
  HK_G uint16_t* y = gptr<uint16_t>(p.y) + m * p.N + n;
  const HK_G uint16_t* b = gcptr<uint16_t>(p.bias) + n;
  float o[4];
  const bool far = sx > kFarScale;
  auto value = [&](int sum, float s, float add) HK_INLINE { return (float)sum * (far ? s : sx) * (far ? sx : s) + add; };
  if (vec) {
    u32x2 w = {0, 0};
    if (p.bias) w = *reinterpret_cast<const HK_G u32x2*>(b);
    const f32x4 s = *reinterpret_cast<const HK_G f32x4*>(sw);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = value(v[e], s[e], e & 1 ? hi16<T>(w[e >> 1]) : lo16<T>(w[e >> 1]));
    *reinterpret_cast<HK_G u32x2*>(y) = pack4<T>(o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) y[e] = T::from_f32(value(v[e], sw[e], p.bias ? T::to_f32(b[e]) : 0.f));
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------
// 16 MB rows (MB 1 or 2), NWV wavefronts.  A wavefront's pieces of 128 bytes of K come in batches of UB whose loads are all issued
// before the first product: one memory latency a batch.
// PX > 0 (hrt_i8_mm_quantises): X is one to eight rows in 16 bits, and every workgroup quantises them for itself while its first
// weights are on the way: each row by its share of the wavefronts, PX 16-byte pieces a lane, into LDS.  GPU time against a
// launch of its own, M x N x K: 1 x 2048 x 512 3.0 us against 4.8, 1 x 8192 x 2048 4.3 against 6.6, 8 x 8192 x 2048 5.6 against 7.4,
// 1 x 8192 x 16384 26 against 36.
template <typename T, int MB, int NWV, int UB, int PX>
__global__ __launch_bounds__(64 * NWV) void i8_rows(hrt_i8_mm_args p, bool vec) {
  constexpr bool Q = PX > 0;
  static_assert(!Q || MB == 1, "few rows");
  constexpr int kCodes = Q ? 512 * PX * NWV : 16;
  __shared__ int part[NWV - 1][MB][64][4];
  __shared__ __attribute__((aligned(16))) uint8_t xq[kCodes];
  __shared__ uint32_t tops[NWV];
  __shared__ float scales[NWV];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + r16 < p.N ? n0 + r16 : p.N - 1;  // columns past N repeat the last one and are not stored
  const int64_t chunks = p.K / 16, steps = cdiv(p.K, 128);
  const HK_G uint8_t* const w = gcptr<uint8_t>(p.w) + n * p.w_sn;
  // this lane's chunk t of piece k; chunks past the end of K: any, and zeros for W
  auto place = [&](int64_t k, int t) HK_INLINE { return (k * 8 + 4 * t + g < chunks ? k * 8 + 4 * t + g : 0) * 16; };
  u32x4 wf[UB][2];
  auto load_w = [&](int64_t st) HK_INLINE {
#pragma unroll
    for (int u = 0; u < UB; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t) wf[u][t] = __builtin_nontemporal_load(reinterpret_cast<const HK_G u32x4*>(w + place(st + u * NWV, t)));
  };
  if constexpr (Q) {
    const int rows = p.M == 1 ? 1 : p.M == 2 ? 2 : p.M <= 4 ? 4 : 8, wpr = NWV / rows, row = wave / wpr;  // wavefronts per row
    const int m = row < p.M ? row : (int)p.M - 1, first = (wave % wpr * 64 + lane) * 8, stride = wpr * 512;
    const HK_G uint16_t* const x = gcptr<uint16_t>(p.x) + m * p.x_sm;
    u32x4 raw[PX];
#pragma unroll
    for (int i = 0; i < PX; ++i) raw[i] = first + i * stride < p.K ? RowVec<T>::get(x + first + i * stride) : u32x4{0, 0, 0, 0};
    issue_order_fence();
    load_w(wave);
    float v[PX][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < PX; ++i) {
      RowVec<T>::unpack(raw[i], v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(v[i][e]) & 0x7fffffffu;
        top = b > top ? b : top;
      }
    }
    top = lanes_max<64>(top, nullptr);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    for (int k = 0; k < wpr; ++k) top = tops[row * wpr + k] > top ? tops[row * wpr + k] : top;
    const RowCode code(top);
    if (lane == 0) scales[row] = code.scale;
#pragma unroll
    for (int i = 0; i < PX; ++i) {
      uint32_t k[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = nearest_code<T>(v[i][e], code);
      const u32x2 q = code.per == 0.f ? u32x2{0, 0} : u32x2{pack_codes4(k), pack_codes4(k + 4)};
      if (row < p.M && first + i * stride < p.K) *reinterpret_cast<u32x2*>(xq + m * p.K + first + i * stride) = q;
    }
    __syncthreads();
  }
  const HK_G uint8_t* x[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) x[b] = gcptr<uint8_t>(p.x) + (b * 16 + r16 < p.M ? b * 16 + r16 : p.M - 1) * p.x_sm;  // rows past M: not stored
  const HK_L uint8_t* const xl = (const HK_L uint8_t*)xq + (Q ? (r16 < p.M ? r16 : (int)p.M - 1) * (int)p.K : 0);
  i32x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = i32x4{0, 0, 0, 0};
  for (int64_t st = wave; st < steps; st += NWV * UB) {
    u32x4 xf[UB][2][MB];
    if (!Q || st != wave) load_w(st);
#pragma unroll
    for (int u = 0; u < UB; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int64_t at = place(st + u * NWV, t);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          if constexpr (Q) xf[u][t][b] = *reinterpret_cast<const HK_L u32x4*>(xl + at);
          else xf[u][t][b] = *reinterpret_cast<const HK_G u32x4*>(x[b] + at);
        }
      }
#pragma unroll
    for (int u = 0; u < UB; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if ((st + u * NWV) * 8 + 4 * t + g >= chunks) wf[u][t] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[b] = mac16(wf[u][t], xf[u][t][b], acc[b]);
      }
  }
  if (wave > 0) {
#pragma unroll
    for (int b = 0; b < MB; ++b) *reinterpret_cast<i32x4*>(part[wave - 1][b][lane]) = acc[b];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int b = 0; b < MB; ++b) {
#pragma unroll
    for (int w2 = 0; w2 < NWV - 1; ++w2) acc[b] += *reinterpret_cast<const i32x4*>(part[w2][b][lane]);
    const int v[4] = {acc[b][0], acc[b][1], acc[b][2], acc[b][3]};
    const int64_t m = b * 16 + r16;
    store4<T>(p, m, n0 + 4 * g, v, Q ? scales[m < p.M ? m : 0] : gcptr<float>(p.x_scale)[m < p.M ? m : 0], vec);
  }
}

// ---- tiles ---------------------------------------------------------------------------------------------------------------
constexpr int kLine = 128;  // bytes and values of K in a row of a stage

// A workgroup's wavefronts are KG groups along K times a grid of WM x WN sub-tiles; a step takes a line per group.  KG > 1 gives
// small grids the wavefronts that hide a copy's latency without a second launch; the groups' sums are added at the end (whole
// numbers: the order is free).  X has a ring of XR stages, W of WR: X may be a step further ahead, which the largest tiles' 160 KiB
// just hold (4096 x 2048 x 8192 on 128 CUs 84 us, so 78; 8192 cubed 430, so 422).  A step's copies are issued between the products
// of its first SP slices, W's first (0: all at its start, where every wavefront of the workgroup then waits at issue for the
// others' to be taken: 8192 cubed on 256 x 256 tiles 454 us, so 436, on 128 x 256 ones 504, so 485; smaller tiles do not gain).
template <int BM, int BN, int WM, int WN, int KG, int XR, int WR>
struct TileShape {
  static constexpr int NWT = (BM / WM) * (BN / WN), NW = NWT * KG;    // wavefronts per group, in all
  static constexpr int XT = KG * BM * kLine, WT = KG * BN * kLine;    // bytes of a stage
  static constexpr int IPX = XT / 1024 / NW, IPW = WT / 1024 / NW;    // copies per wavefront
  static constexpr int FM = WM / 32, FN = WN / 32;
  static constexpr int U = XR == WR ? XR : XR * WR;                   // steps after which the buffers repeat
  static_assert(XT % (1024 * NW) == 0 && WT % (1024 * NW) == 0, "copy split");
};

template <typename T, int BM, int BN, int WM, int WN, int KG, int XR, int WR, int SP>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN) * KG) void i8_tile(hrt_i8_mm_args p, int tiles_n, int nk, bool lines) {
  using S = TileShape<BM, BN, WM, WN, KG, XR, WR>;
  constexpr int NWT = S::NWT, IPX = S::IPX, IPW = S::IPW, FM = S::FM, FN = S::FN;
  // One LDS object per stage, so that the compiler can tell the reads of one from the copies into another.
  __shared__ __attribute__((aligned(1024))) uint8_t x0[S::XT], x1[S::XT], x2[XR > 2 ? S::XT : 16];
  __shared__ __attribute__((aligned(1024))) uint8_t w0[S::WT], w1[S::WT], w2[WR > 2 ? S::WT : 16];
  auto xbuf = [&](auto ic) HK_INLINE { constexpr int I = decltype(ic)::value; return (HK_L uint8_t*)(I == 0 ? x0 : I == 1 ? x1 : x2); };
  auto wbuf = [&](auto ic) HK_INLINE { constexpr int I = decltype(ic)::value; return (HK_L uint8_t*)(I == 0 ? w0 : I == 1 ? w1 : w2); };

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / NWT, wt = wave % NWT, wm = wt % (BM / WM), wn = wt / (BM / WM), l32 = lane & 31, h = lane >> 5;
  // n-fastest tile numbers, in scalar registers, and with them every buffer resource
  const uint32_t tm = __builtin_amdgcn_readfirstlane(blockIdx.x / (uint32_t)tiles_n);
  const uint32_t tn = __builtin_amdgcn_readfirstlane(blockIdx.x % (uint32_t)tiles_n);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int ml = p.M - m0 < BM ? (int)(p.M - m0) : BM, nl = p.N - n0 < BN ? (int)(p.N - n0) : BN;

  // copy sources; lane offsets inside a stage, kNoRow where the row does not exist (the buffer's range check gives zeros)
  const uint32_t xss = (uint32_t)p.x_sm, wss = (uint32_t)p.w_sn;
  const HK_G uint8_t* Xb = gcptr<uint8_t>(p.x) + m0 * p.x_sm;
  const HK_G uint8_t* Wb = gcptr<uint8_t>(p.w) + n0 * p.w_sn;
  // copy j of a stage: this lane's row, and its byte of K in the step
  auto row_of = [&](int j, int rows) HK_INLINE { return (j * 8 + (lane >> 3)) % rows; };
  auto byte_of = [&](int j, int rows) HK_INLINE { return ((lane & 7) ^ tile_swz<8>(row_of(j, rows))) * 16 + j / (rows / 8) * kLine; };
  uint32_t xo[IPX], wo[IPW];
#pragma unroll
  for (int i = 0; i < IPX; ++i) {
    const int j = wave * IPX + i, row = row_of(j, BM);
    xo[i] = row < ml ? (uint32_t)row * xss + (uint32_t)byte_of(j, BM) : kNoRow;
  }
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const int j = wave * IPW + i, row = row_of(j, BN);
    wo[i] = row < nl ? (uint32_t)row * wss + (uint32_t)byte_of(j, BN) : kNoRow;
  }
  // The last stage may hold fewer values: chunks past K are zeros (a select, not a branch: the compiler counts the copies in
  // flight along every path).
  auto left_of = [&](int ks) HK_INLINE {
    const int64_t left = p.K - (int64_t)ks * (KG * kLine);
    return left >= KG * kLine ? KG * kLine : (int)left;
  };
  auto copy_x = [&](auto ic, int ks, int i) HK_INLINE {
    edge_copy(edge_rsrc(Xb + (int64_t)ks * (KG * kLine)), xbuf(ic), wave * IPX + i, byte_of(wave * IPX + i, BM) < left_of(ks) ? xo[i] : kNoRow);
  };
  auto copy_w = [&](auto ic, int ks, int i) HK_INLINE {
    edge_copy(edge_rsrc(Wb + (int64_t)ks * (KG * kLine)), wbuf(ic), wave * IPW + i, byte_of(wave * IPW + i, BN) < left_of(ks) ? wo[i] : kNoRow);
  };
  auto stage_x = [&](auto ic, int ks) HK_INLINE {
#pragma unroll
    for (int i = 0; i < IPX; ++i) copy_x(ic, ks, i);
  };
  auto stage_w = [&](auto ic, int ks) HK_INLINE {
#pragma unroll
    for (int i = 0; i < IPW; ++i) copy_w(ic, ks, i);
  };
  // This lane's rows: the sub-tile's other 32-row blocks lie a constant further (the swizzle repeats every 16 rows).
  const int xrow = wm * WM + l32, wrow = wn * WN + l32;

  i32x16 acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0;

  constexpr int KEEP = (XR - WR) * IPX + (WR - 2) * (IPX + IPW);
  static_assert(XR == WR || XR == WR + 1, "copies in flight past a step's W");
  // Step ks, number I of the unrolled ones.  GUARD: near the end, where no copy is left to be made; it waits for all of them.
  auto step = [&](auto ic, auto guard, int ks) HK_INLINE {
    constexpr int I = decltype(ic)::value;
    constexpr bool GUARD = decltype(guard)::value;
    using IX = std::integral_constant<int, (I + XR - 1) % XR>;
    using IW = std::integral_constant<int, (I + WR - 1) % WR>;
    const HK_L uint8_t* const xs = xbuf(std::integral_constant<int, I % XR>()) + kg * BM * kLine;
    const HK_L uint8_t* const ws = wbuf(std::integral_constant<int, I % WR>()) + kg * BN * kLine;
    u32x4 wf[2][FN], xf[2][FM];
    // a line is four slices; the fragments of the next one are read while this one's products run (two register sets, fenced)
    auto read = [&](int s) HK_INLINE {
#pragma unroll
      for (int j = 0; j < FN; ++j) wf[s & 1][j] = *reinterpret_cast<const HK_L u32x4*>(ws + tile_off<8>(wrow, 2 * s + h) + j * 32 * kLine);
#pragma unroll
      for (int i = 0; i < FM; ++i) xf[s & 1][i] = *reinterpret_cast<const HK_L u32x4*>(xs + tile_off<8>(xrow, 2 * s + h) + i * 32 * kLine);
    };
    read(0);
    const bool more_w = !GUARD || ks + WR - 1 < nk, more_x = !GUARD || ks + XR - 1 < nk;
    if (SP == 0) {
      if (more_w) stage_w(IW(), ks + WR - 1);
      issue_order_fence();  // the barrier counts on X being issued last
      if (more_x) stage_x(IX(), ks + XR - 1);
    }
    auto slice = [&](auto sc) HK_INLINE {
      constexpr int SL = decltype(sc)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (SL < 3) read(SL + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          acc[j][i] = mac32(wf[SL & 1][j], xf[SL & 1][i], acc[j][i]);
          if constexpr (SL < SP) {  // PER copies a slice, one behind every EV products
            constexpr int SLICES = SP > 0 ? SP : 1, PER = (IPX + IPW + SLICES - 1) / SLICES, EV = FM * FN / PER;
            static_assert(SP == 0 || EV >= 1, "a product for each copy");
            const int q = j * FM + i, c = SL * PER + q / EV;
            if (q % EV == EV - 1 && q / EV < PER && c < IPX + IPW) {
              __builtin_amdgcn_sched_barrier(0);
              if (c == IPW) issue_order_fence();  // as above: X behind W
              if (c < IPW) {
                if (more_w) copy_w(IW(), ks + WR - 1, c < IPW ? c : 0);
              } else {
                if (more_x) copy_x(IX(), ks + XR - 1, c < IPW ? 0 : c - IPW);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
    };
    slice(std::integral_constant<int, 0>()), slice(std::integral_constant<int, 1>());
    slice(std::integral_constant<int, 2>()), slice(std::integral_constant<int, 3>());
    // The products are pure, and the compiler puts them off to the end of the loop body unless their results are used here.
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) asm volatile("" : "+v"(acc[j][i]));
    // The next step's stages have landed everywhere; what was issued after its W may stay in flight.
    if (!GUARD || more_x) barrier_keep_vm_lds<KEEP>();
    else barrier_keep_vm_lds<0>();
  };
  using Whole = std::integral_constant<bool, false>;
  using Guard = std::integral_constant<bool, true>;
  auto steps = [&](auto guard, int ks) HK_INLINE {
    auto one = [&](auto ic) HK_INLINE {
      if (!decltype(guard)::value || ks + decltype(ic)::value < nk) step(ic, guard, ks + decltype(ic)::value);
    };
    one(std::integral_constant<int, 0>()), one(std::integral_constant<int, 1>());
    if constexpr (S::U > 2) one(std::integral_constant<int, 2>());
    if constexpr (S::U > 3) one(std::integral_constant<int, 3>()), one(std::integral_constant<int, 4>()), one(std::integral_constant<int, 5>());
  };
  stage_x(std::integral_constant<int, 0>(), 0);
  stage_w(std::integral_constant<int, 0>(), 0);
  // stages of the steps before the first one's own copies (past the end of K: zeros that nobody reads)
  issue_order_fence();  // the first barrier counts on them being the last ones issued
  if constexpr (WR > 2) stage_w(std::integral_constant<int, 1>(), 1);
  if constexpr (XR > 2) stage_x(std::integral_constant<int, 1>(), 1);
  barrier_keep_vm<KEEP>();
  int ks = 0;
  for (; ks + S::U + XR - 1 <= nk; ks += S::U) steps(Whole(), ks);
  for (; ks < nk; ks += S::U) steps(Guard(), ks);

  if constexpr (KG > 1) {  // the groups' sums, through the stages' memory (every copy has landed)
    constexpr int NB = FN * FM, PER = S::XT / 4096;  // accumulators of a wavefront; how many an X stage holds
    static_assert((KG - 1) * NWT * NB <= 2 * PER && PER % NB == 0, "merge areas");
    auto area = [&](int k, int b) {
      const int q = ((k - 1) * NWT + wt) * NB;
      return (int*)(q < PER ? x0 + q * 4096 : x1 + (q - PER) * 4096) + b * 1024 + lane;
    };
    if (kg > 0) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        int* const mine = area(kg, b);
#pragma unroll
        for (int e = 0; e < 16; ++e) mine[e * 64] = acc[b / FM][b % FM][e];
      }
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int k = 1; k < KG; ++k)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int* const part = area(k, b);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b / FM][b % FM][e] += part[e * 64];
      }
  }
  float sxs[FM];
  bool far = false;  // rows that store4 takes the other way round, which the lines below do not
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = m0 + wm * WM + i * 32 + l32;
    sxs[i] = gcptr<float>(p.x_scale)[m < p.M ? m : p.M - 1];
    far |= sxs[i] > kFarScale;
  }
  if (!lines || __any(far)) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int64_t m = m0 + wm * WM + i * 32 + l32;
      const float sx = sxs[i];
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int v[4] = {acc[j][i][4 * e], acc[j][i][4 * e + 1], acc[j][i][4 * e + 2], acc[j][i][4 * e + 3]};
          store4<T>(p, m, n0 + wn * WN + j * 32 + 8 * e + 4 * h, v, sx, false);
        }
    }
    return;
  }
  // Whole lines of y: 32 rows at a time go through the wavefront's own LDS area, so that a store writes 16 bytes a lane along a row.
  constexpr int RB = WN * 2 + 16;  // bytes of a row in the area, its pad off the banks of the next
  // KG > 1: in the merge area of group 1's wavefront, which this one has read; else in the stages
  constexpr int AREA = 32 * RB, MERGED = FN * FM * 4096, PX = S::XT / AREA, PW = S::WT / AREA;
  static_assert(KG > 1 ? AREA <= MERGED : 2 * PX + 2 * PW >= NWT, "epilogue areas");
  HK_L uint8_t* const area = KG > 1           ? (HK_L uint8_t*)(wt * MERGED < S::XT ? x0 + wt * MERGED : x1 + (wt * MERGED - S::XT))
                             : wt < PW        ? (HK_L uint8_t*)w0 + wt * AREA
                             : wt < 2 * PW    ? (HK_L uint8_t*)w1 + (wt - PW) * AREA
                             : wt < 2 * PW + PX ? (HK_L uint8_t*)x0 + (wt - 2 * PW) * AREA
                                              : (HK_L uint8_t*)x1 + (wt - 2 * PW - PX) * AREA;
  const int64_t nw = n0 + wn * WN;
  u32x2 bias[FN][4];
  f32x4 sw[FN][4];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t n = nw + j * 32 + 8 * e + 4 * h, at = n < p.N ? n : 0;
      bias[j][e] = u32x2{0, 0};
      if (p.bias) bias[j][e] = *reinterpret_cast<const HK_G u32x2*>(gcptr<uint16_t>(p.bias) + at);
      sw[j][e] = *reinterpret_cast<const HK_G f32x4*>(gcptr<float>(p.w_scale) + at);
    }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const float sx = sxs[i];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o[r] = (float)acc[j][i][4 * e + r] * sx * sw[j][e][r] + (r & 1 ? hi16<T>(bias[j][e][r >> 1]) : lo16<T>(bias[j][e][r >> 1]));
        *reinterpret_cast<HK_L u32x2*>(area + l32 * RB + (j * 32 + 8 * e + 4 * h) * 2) = pack4<T>(o);
      }
    constexpr int CPR = WN / 8;  // 16-byte chunks per row
#pragma unroll
    for (int u = 0; u < 32 * CPR / 64; ++u) {
      const int ch = u * 64 + lane, row = ch / CPR, c = ch % CPR;
      const u32x4 v = *reinterpret_cast<const HK_L u32x4*>(area + row * RB + c * 16);
      const int64_t m = m0 + wm * WM + i * 32 + row, n = nw + c * 8;
      if (m < p.M && n < p.N) *reinterpret_cast<HK_G u32x4*>(gptr<uint16_t>(p.y) + m * p.N + n) = v;
    }
  }
}

// ---- plan and launch -----------------------------------------------------------------------------------------------------
// Tiles, and what a grid of them takes in us, fitted to full rounds of K 2048 and 8192: once, for every 256 workgroups, and for those
// per 128 values of K.  One workgroup of the first two fits a CU, two of the others, whose copies then cover each other's
// barriers.  A grid that leaves CUs idle runs up to a fifth faster.  Measured, us (tiles in this order): 4096 x 8192 x 2048 71, 84, 79, 99,
// 130; 4096 x 2048 x 8192 79, 65, 72, 86, 104; 2048 cubed 27, 17, 15.6, 15.8, 19; 1024 x 2048 x 8192 73, 41, 34, 26, 29; 308 x 8192 x 2048
// 25, 15.5, 11.4, 13.5, 15; 308 x 2048 x 2048 25, 14.5, 10, 7.7, 6.2 (before: 128 x 128 in two groups along K and 64 x 64 in four, one to a
// CU, 11.6 and 7.5).
struct Tile {
  int bm, bn, wm, wn, kg, xr, wr, sp;  // as i8_tile has them
  float once, per256, per128;
};
constexpr int kNumTiles = HRT_I8_MM_TILES;
constexpr Tile kTiles[kNumTiles] = {{256, 256, 128, 64, 1, 3, 2, 3, 0.f, 11.f, 1.48f},
                                    {128, 256, 64, 64, 1, 3, 3, 3, 0.f, 9.f, 0.82f},
                                    {128, 128, 32, 64, 1, 3, 2, 0, 6.5f, 1.2f, 0.49f},
                                    {128, 64, 32, 32, 1, 3, 3, 0, 4.f, 1.35f, 0.29f},
                                    {64, 64, 32, 32, 2, 3, 2, 0, 3.2f, 0.97f, 0.183f}};

int64_t tiles_of(const hrt_i8_mm_args& a, int t) { return cdiv(a.M, kTiles[t].bm) * cdiv(a.N, kTiles[t].bn); }
// Index of the tile, -1: i8_rows (up to 16 rows, or 32 where K is short).  us of i8_rows and of the tile chosen otherwise, at 16, 17 and 32
// rows, N x K: 2048 x 1024 3.7, 4.0, 4.3 against 4.9, 4.9, 5.0; 2048 x 2048 4.5, 5.0, 5.5 against 5.9, 5.9, 6.0; 8192 x 1024 4.8, 5.3, 5.9
// against 5.1; 8192 x 2048 6.9, 7.4, 8.5 against 6.1; 2048 x 8192 11.4, 11.7, 14.2 against 11.8.  The rule is on M and K alone: it is up
// to 0.8 us off the better one on either side.
int plan_of(const hrt_i8_mm_args& a) {
  if (a.x_scale == 0 || a.M <= 16 || (a.M <= 32 && a.K <= 1024)) return -1;
  int best = 0;
  float us = 0.f;
  for (int t = 0; t < kNumTiles; ++t) {
    const float n = (float)tiles_of(a, t) / 256.f, rounds = (float)cdiv(tiles_of(a, t), 256);
    const float e = (kTiles[t].once + rounds * (kTiles[t].per256 + kTiles[t].per128 * (float)a.K / 128.f)) * (n >= 1.f ? 1.f : n > 0.5f ? 0.56f + 0.44f * n : 0.78f);
    if (t == 0 || e < us) best = t, us = e;
  }
  return best;
}

// Steps of a product, and how many rounds of them i8_tile takes without a guard.
int64_t steps_of(const hrt_i8_mm_args& a, const Tile& t) { return cdiv(a.K, kLine * t.kg); }
int64_t whole_rounds(const hrt_i8_mm_args& a, const Tile& t) {
  const int64_t left = steps_of(a, t) - (t.xr - 1);
  return left > 0 ? left / (t.xr == t.wr ? t.xr : t.xr * t.wr) : 0;
}

template <typename T, int I>
void queue_tile(const hrt_i8_mm_args& a, hipStream_t s, bool lines) {
  constexpr Tile t = kTiles[I];
  const int64_t tm = cdiv(a.M, t.bm), tn = cdiv(a.N, t.bn);
  hipLaunchKernelGGL((i8_tile<T, t.bm, t.bn, t.wm, t.wn, t.kg, t.xr, t.wr, t.sp>), dim3((uint32_t)(tm * tn)),
                     dim3(64 * TileShape<t.bm, t.bn, t.wm, t.wn, t.kg, t.xr, t.wr>::NW), 0, s, a, (int)tn, (int)steps_of(a, t), lines);
}

template <typename T>
void queue_mm(const hrt_i8_mm_args& a, int tile, hipStream_t s) {
  const bool vec = a.N % 4 == 0 && a.y % 8 == 0 && a.bias % 8 == 0 && a.w_scale % 16 == 0, lines = vec && a.N % 8 == 0 && a.y % 16 == 0;
  switch (tile) {
    case 0: return queue_tile<T, 0>(a, s, lines);
    case 1: return queue_tile<T, 1>(a, s, lines);
    case 2: return queue_tile<T, 2>(a, s, lines);
    case 3: return queue_tile<T, 3>(a, s, lines);
    case 4: return queue_tile<T, 4>(a, s, lines);
  }
  // wavefronts and batches that cover K once where they can
  const dim3 grid((uint32_t)cdiv(a.N, 16));
  const int64_t pieces = cdiv(a.K, 128);
  const auto go = [&](auto px) {
    constexpr int Q = decltype(px)::value;
    if (pieces <= 8) hipLaunchKernelGGL((i8_rows<T, 1, 4, 2, Q>), grid, dim3(256), 0, s, a, vec);
    else if (pieces <= 16) hipLaunchKernelGGL((i8_rows<T, 1, 8, 2, Q>), grid, dim3(512), 0, s, a, vec);
    else hipLaunchKernelGGL((i8_rows<T, 1, 8, 4, Q>), grid, dim3(512), 0, s, a, vec);
  };
  if (a.M > 16) hipLaunchKernelGGL((i8_rows<T, 2, 4, 2, 0>), grid, dim3(256), 0, s, a, vec);
  else if (a.x_scale != 0) go(std::integral_constant<int, 0>());
  else if (hrt_i8_mm_row_slots(a.M) * a.K <= (pieces <= 8 ? 4096 : 8192)) go(std::integral_constant<int, 2>());
  else go(std::integral_constant<int, 4>());
}

template <typename T>
bool launch_i8_mm(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_i8_mm_args*>(pp);
  if (a.M <= 0 || a.N <= 0 || a.K <= 0) return ctx.fail("empty product");
  if (a.K % 16 != 0 || a.K > 131056) return ctx.fail("K must be a multiple of 16 and at most 131056");
  const bool q = a.x_scale == 0;
  if (q && !hrt_i8_mm_quantises(a.M, a.K)) return ctx.fail("too many values to quantise on the way");
  if (a.x_sm < 0 || (!q && a.x_sm % 16 != 0) || a.w_sn < 0 || a.w_sn % 16 != 0) return ctx.fail("row strides must be non-negative multiples of 16");
  if (a.x % (q ? 2 : 16) != 0 || a.w % 16 != 0 || a.x_scale % 4 != 0 || a.w_scale % 4 != 0 || a.y % 2 != 0 || a.bias % 2 != 0)
    return ctx.fail("x and w must be 16-byte aligned, scales 4-byte aligned");
  const int64_t xs[2] = {a.M, a.K}, xt[2] = {a.x_sm, 1}, wz[2] = {a.N, a.K}, wt[2] = {a.w_sn, 1};
  if (!ctx.check(a.x, hrt::span_bytes(2, xs, xt, q ? 2 : 1), "x") || !ctx.check(a.w, hrt::span_bytes(2, wz, wt, 1), "w") ||
      (!q && !ctx.check(a.x_scale, (uint64_t)a.M * 4, "x_scale")) || !ctx.check(a.w_scale, (uint64_t)a.N * 4, "w_scale") ||
      !ctx.check(a.y, (uint64_t)(a.M * a.N) * 2, "y") || (a.bias && !ctx.check(a.bias, (uint64_t)a.N * 2, "bias")))
    return false;
  const int tile = plan_of(a);
  const int64_t lim = (int64_t)1 << 31;  // offsets of a tile's rows are 31-bit
  if (tile >= 0 && (a.x_sm * 257 >= lim || a.w_sn * 257 >= lim)) return ctx.fail("operand rows too long for one launch");
  if (!hrt::grid_fits(tile < 0 ? cdiv(a.N, 16) : tiles_of(a, tile), 512)) return ctx.fail("grid too large");
  queue_mm<T>(a, tile, ctx.stream);
  return hrt::launch_ok(hipGetLastError(), ctx, "i8_mm");
}

HRT_REGISTER("i8_mm_bf16", hrt_i8_mm_args, launch_i8_mm<BF16>);
HRT_REGISTER("i8_mm_f16", hrt_i8_mm_args, launch_i8_mm<F16>);

}  // namespace
}  // namespace hk

extern "C" int32_t hrt_i8_mm_plan(const hrt_i8_mm_args* a, int64_t* rounds) {
  using namespace hk;
  const int tile = a && a->M > 0 && a->N > 0 && a->K > 0 ? plan_of(*a) : -1;
  if (rounds) *rounds = tile < 0 ? 0 : whole_rounds(*a, kTiles[tile]);
  return tile;
}
