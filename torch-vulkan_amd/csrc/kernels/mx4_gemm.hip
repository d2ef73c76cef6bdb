// "mx4_mm_{bf16,f16}": y = X W^T + bias with W in microscaled 4-bit floating point (mx4.h) and X in 16 bits or in 4.
//
// Two kernels, each in both forms:
//   * mx4_rows for few rows: bound by the weights' bytes, in practice by one memory latency.  A wavefront takes 16 columns of
//     y and every NWVth 128-wide piece of K, its loads all in flight at once; no LDS but for the wavefronts' sums.
//   * mx4_tile for the rest: bound by the matrix cores and by L2 -> LDS.  Both operands are copied global -> LDS directly,
//     the weights as codes, which a lane's own registers turn into fragments.
// 16-bit X: a lane's 16 bytes of codes are one scale block of one column; dword t of them becomes the 32x32x16 fragment of
// eight K values by four conversions, and X is read with the same K order (chunk 4 h + t of a 64-wide step), so the weights
// never exist in LDS or memory as 16-bit values.
// 4-bit X: v_mfma_scale_f32_32x32x64_f8f6f4 takes a lane's 16 bytes of codes as they are, with the block's scale byte.
// Lane layout of the scaled products (checked on the device), l = lane: 32x32x64: operand row l % 32, K block l / 32;
// 16x16x128: row l % 16, K block l / 16; the scale operand's byte `opsel` belongs to the lane's own block.
// W is the first operand in both kernels, so an accumulator holds four consecutive columns n of one row m of y.
// Measured, M x N x K, 16-bit X / 4-bit X: 1 x 8192 x 2048 5.4 / 4.7 us, 16 x 8192 x 2048 8.2 / 6.2, 308 x 2048 x 2048 10.3 / 6.7,
// 1024 x 8192 x 2048 36 / 17, 4096 x 8192 x 2048 114 / 51 (1.20, 2.71 PFLOP/s), 4096 x 2048 x 8192 124 / 50, 8192 cubed 822 / 285 us
// (1.34, 3.86 PFLOP/s; a library's bf16 product of that size takes 911).
#include <utility>

#include "../hrt/registry.h"
#include "mx4.h"

namespace hk {
namespace {

// Lambdas of a kernel with many copies of its step: the compiler would make them functions.
#define HK_INLINE __attribute__((always_inline))

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
// The eight-dword operand type's upper half is not read for 4-bit values.
__device__ __forceinline__ i32x8 fp4_operand(u32x4 c) {
  const i32x4 v = __builtin_bit_cast(i32x4, c);
  return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}

// y[m, n .. n + 3].  Columns past N are not stored; vec: whole groups of four columns, aligned.
template <typename T>
__device__ __forceinline__ void store4(const hrt_mx4_mm_args& p, int64_t m, int64_t n, const float* v, bool vec) {
  if (m >= p.M || n >= p.N) return;
  HK_G uint16_t* y = gptr<uint16_t>(p.y) + m * p.N + n;
  const HK_G uint16_t* b = gcptr<uint16_t>(p.bias) + n;
  float o[4];
  if (vec) {
    u32x2 w = {0, 0};
    if (p.bias) w = *reinterpret_cast<const HK_G u32x2*>(b);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = v[e] + (e & 1 ? hi16<T>(w[e >> 1]) : lo16<T>(w[e >> 1]));
    *reinterpret_cast<HK_G u32x2*>(y) = pack4<T>(o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) y[e] = T::from_f32(v[e] + (p.bias ? T::to_f32(b[e]) : 0.f));
  }
}

template <typename F>
__device__ __forceinline__ void both(F f) {
  f(std::integral_constant<int, 0>()), f(std::integral_constant<int, 1>());
}

// ---- few rows ------------------------------------------------------------------------------------------------------------
// dword t of lane group g (16 lanes) becomes dword g of group t's: [block g][dword t] -> [block t][dword g].
__device__ __forceinline__ u32x4 transpose_groups(u32x4 c) {
  const auto a = __builtin_amdgcn_permlane32_swap(c[0], c[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(c[1], c[3], false, false);
  const auto lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{(uint32_t)lo[0], (uint32_t)lo[1], (uint32_t)hi[0], (uint32_t)hi[1]};
}

// 16 MB rows (MB 1 or 2), NWV wavefronts.  A wavefront's pieces of 128 values of K come in batches of UB whose loads are all
// issued before the first product: one memory latency a batch.  16-bit rows are read 64 bytes at a time (fragment t: values
// 32 t + 8 g of a piece; 16 bytes out of each block of a row, as the codes lie in their lanes, touched four times the lines), so
// the lane groups exchange their codes.
template <typename T, bool A4, int MB, int NWV, int UB>
__global__ __launch_bounds__(64 * NWV) void mx4_rows(hrt_mx4_mm_args p, bool vec) {
  constexpr int XF = A4 ? 1 : 4;  // 16-byte pieces of X per row and piece of K
  __shared__ float part[NWV - 1][MB][64][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + r16 < p.N ? n0 + r16 : p.N - 1;  // columns past N repeat the last one and are not stored
  const int64_t nb = p.K / 32, steps = cdiv(p.K, 128);
  const int gb = g < nb ? g : 0;  // a row of fewer than four blocks: the other lane groups stay inside it
  const HK_G uint8_t* wc = gcptr<uint8_t>(p.w) + n * (p.K / 2) + 16 * gb;
  const HK_G uint8_t* ws = gcptr<uint8_t>(p.w_scale) + n * nb + gb;
  f32x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const HK_G uint8_t* xr[MB];
  const HK_G uint8_t* xs[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {  // rows past M repeat the last one and are not stored
    const int64_t m = b * 16 + r16 < p.M ? b * 16 + r16 : p.M - 1;
    xr[b] = A4 ? gcptr<uint8_t>(p.x) + m * (p.K / 2) + 16 * gb : gcptr<uint8_t>(p.x) + m * p.x_sm * 2 + 16 * g;
    xs[b] = gcptr<uint8_t>(p.x_scale) + m * nb + gb;
  }
  for (int64_t st = wave; st < steps; st += NWV * UB) {
    u32x4 c[UB], x[UB][MB][XF];
    uint32_t s[UB], sx[UB][MB];
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      // a block past the end of K (the last piece may have fewer than four) counts as zeros with scale 0 (2^-127)
      const int64_t k = st + u * NWV, at = k * 4 + g < nb ? k : 0;
      c[u] = __builtin_nontemporal_load(reinterpret_cast<const HK_G u32x4*>(wc + at * 64));
      s[u] = ws[at * 4];
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        if constexpr (A4) {
          sx[u][b] = xs[b][at * 4];
          x[u][b][0] = *reinterpret_cast<const HK_G u32x4*>(xr[b] + at * 64);
        } else {
#pragma unroll
          for (int t = 0; t < XF; ++t) x[u][b][t] = *reinterpret_cast<const HK_G u32x4*>(xr[b] + (k * 4 + t < nb ? k * 256 + 64 * t : 0));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const int64_t k = (st + u * NWV) * 4;
      if (k + g >= nb) c[u] = u32x4{0, 0, 0, 0}, s[u] = 0;
      if constexpr (A4) {
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          if (k + g >= nb) x[u][b][0] = u32x4{0, 0, 0, 0}, sx[u][b] = 0;
          acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(c[u]), fp4_operand(x[u][b][0]), acc[b], 4, 4, 0, (int)s[u], 0,
                                                                    (int)sx[u][b]);
        }
      } else {
        const u32x4 w = transpose_groups(c[u]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const u32x4 wf = mx4_unpack8<T>(w[t], mx_scale(__shfl(s[u], r16 + 16 * t, 64)));
#pragma unroll
          for (int b = 0; b < MB; ++b) acc[b] = Mfma<T>::mac(wf, k + t < nb ? x[u][b][t] : u32x4{0, 0, 0, 0}, acc[b]);
        }
      }
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int b = 0; b < MB; ++b) *reinterpret_cast<f32x4*>(part[wave - 1][b][lane]) = acc[b];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int b = 0; b < MB; ++b) {
#pragma unroll
    for (int w = 0; w < NWV - 1; ++w) acc[b] += *reinterpret_cast<const f32x4*>(part[w][b][lane]);
    const float v[4] = {acc[b][0], acc[b][1], acc[b][2], acc[b][3]};
    store4<T>(p, b * 16 + r16, n0 + 4 * g, v, vec);
  }
}

// ---- tiles ---------------------------------------------------------------------------------------------------------------
// Everything in LDS is rows of 128 bytes, whole cache lines of both operands: 64 16-bit values or 256 codes.  (Rows of 32 or 64
// bytes of codes, one step's worth, fetched each line four or two times over, since X streams through the L1 in between; that
// traffic from L2 bounded the kernel: 4096 x 2048 x 8192 bf16 157 us, so 132.)  A row's 16-byte chunks are XOR-swizzled
// (tile_swz<8>).
constexpr int kLine = 128;
__device__ __forceinline__ int line_off(int row, int c) { return tile_off<8>(row, c); }

// A workgroup's wavefronts are KG groups along K times a grid of WM x WN sub-tiles.  A step takes KG pieces of K, one per group:
// a piece is a line of X (KX values of K: 64, or 256 codes).  A stage of W holds whole lines of 256 values: 4-bit X uses
// one per piece, 16-bit X one in four pieces, so that a W stage serves SPW steps.  KG > 1 gives small grids (few rows) the
// wavefronts that hide a copy's latency without a second launch; the groups' sums are added in order at the end.
// X has a ring of XR stages, W and the scales two.
template <bool A4, int BM, int BN, int WM, int WN, int KG, int XR>
struct TileShape {
  static constexpr int KX = A4 ? 256 : 64, PPL = A4 ? 1 : 4;          // K values per piece, pieces per line of W
  static constexpr int SPW = PPL > KG ? PPL / KG : 1, WL = KG > PPL ? KG / PPL : 1;  // steps per W stage, its lines per row
  static constexpr int NWT = (BM / WM) * (BN / WN), NW = NWT * KG;    // wavefronts per group, in all
  static constexpr int XT = KG * BM * kLine, WT = WL * BN * kLine;    // bytes of a stage
  static constexpr int IPX = XT / 1024 / NW, IPW = WT / 1024 / NW;    // copies per wavefront
  static constexpr int FM = WM / 32, FN = WN / 32;
  static constexpr int U = XR % (2 * SPW) == 0 ? XR : 2 * SPW;        // steps after which the buffers repeat
  static_assert(XT % (1024 * NW) == 0 && WT % (1024 * NW) == 0 && U % XR == 0, "copy split, ring");
};

// Scale bytes are staged apart, 32 of a row (1024 values of K) at a time: a lane that fetches one step's few bytes of its row
// still occupies a cache line's turn, and 512 such lanes a step cost as much as the step's products.
// STR: rows of scales do not start on dwords (K / 32 not a multiple of 4): fetched from the dword before, shifted when used.
template <typename T, bool A4, int BM, int BN, int WM, int WN, int KG, int XR, bool STR>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN) * KG) void mx4_tile(hrt_mx4_mm_args p, int tiles_n, int nk, bool lines) {
  using S = TileShape<A4, BM, BN, WM, WN, KG, XR>;
  constexpr int NW = S::NW, NWT = S::NWT, IPX = S::IPX, IPW = S::IPW, FM = S::FM, FN = S::FN, KX = S::KX, SPW = S::SPW, U = S::U;
  constexpr int SB = KX / 32;                                    // scale bytes per row and piece
  constexpr int SR = BN + (A4 ? BM : 0), SRB = STR ? 48 : 32;    // rows with scales (W's first), bytes of one in LDS
  constexpr int SPB = 1024 / (KG * KX);                          // steps per block of scales
  constexpr int SI = SR * SRB / 1024, IPS = (SI + NW - 1) / NW;  // copies per block, per wavefront (the last ones repeat a copy)
  static_assert(SR * SRB % 1024 == 0 && BN * SRB % 1024 == 0 && SPB >= 1, "whole scale copies");
  // One LDS object per stage, so that the compiler can tell the reads of one from the copies into another.
  __shared__ __attribute__((aligned(1024))) uint8_t x0[S::XT], x1[S::XT], x2[XR > 2 ? S::XT : 16], x3[XR > 2 ? S::XT : 16];
  __shared__ __attribute__((aligned(1024))) uint8_t w0[S::WT], w1[S::WT], sc[2 * SR * SRB];
  auto xbuf = [&](auto ic) HK_INLINE { constexpr int I = decltype(ic)::value; return (HK_L uint8_t*)(I == 0 ? x0 : I == 1 ? x1 : I == 2 ? x2 : x3); };
  auto wbuf = [&](auto ic) HK_INLINE { return (HK_L uint8_t*)(decltype(ic)::value ? w1 : w0); };

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / NWT, wt = wave % NWT, wm = wt % (BM / WM), wn = wt / (BM / WM), l32 = lane & 31, h = lane >> 5;
  // n-fastest tile numbers, in scalar registers, and with them every buffer resource
  const uint32_t tm = __builtin_amdgcn_readfirstlane(blockIdx.x / (uint32_t)tiles_n);
  const uint32_t tn = __builtin_amdgcn_readfirstlane(blockIdx.x % (uint32_t)tiles_n);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int64_t nb = p.K / 32;
  const int ml = p.M - m0 < BM ? (int)(p.M - m0) : BM, nl = p.N - n0 < BN ? (int)(p.N - n0) : BN;

  // copy sources; lane offsets inside a stage, kNoRow where the row does not exist (the buffer's range check gives zeros)
  const uint32_t xss = (uint32_t)(A4 ? p.K / 2 : p.x_sm * 2), wss = (uint32_t)(p.K / 2);
  const HK_G uint8_t* Xb = gcptr<uint8_t>(p.x) + m0 * xss;
  const HK_G uint8_t* Wb = gcptr<uint8_t>(p.w) + n0 * wss;
  // copy j of a stage: its line (piece of X, line of W), and this lane's row and chunk in it
  auto row_of = [&](int j, int rows) HK_INLINE { return (j * 8 + (lane >> 3)) % rows; };
  auto chunk_of = [&](int j, int rows) HK_INLINE { return (lane & 7) ^ tile_swz<8>(row_of(j, rows)); };
  uint32_t xo[IPX], wo[IPW];
#pragma unroll
  for (int i = 0; i < IPX; ++i) {
    const int j = wave * IPX + i, row = row_of(j, BM);
    xo[i] = row < ml ? (uint32_t)row * xss + (uint32_t)(chunk_of(j, BM) * 16 + j / (BM / 8) * kLine) : kNoRow;
  }
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const int j = wave * IPW + i, row = row_of(j, BN);
    wo[i] = row < nl ? (uint32_t)row * wss + (uint32_t)(chunk_of(j, BN) * 16 + j / (BN / 8) * kLine) : kNoRow;
  }
  // The last stage may hold fewer values: chunks past K are zeros (a select, not a branch: the compiler counts the copies in
  // flight along every path).
  auto copy_x = [&](int ks, HK_L uint8_t* to) HK_INLINE {
    const __amdgpu_buffer_rsrc_t rs = edge_rsrc(Xb + (int64_t)ks * (KG * kLine));
    const int64_t left = p.K - (int64_t)ks * (KG * KX);
    const int l = left >= KG * KX ? KG * KX : (int)left;
#pragma unroll
    for (int i = 0; i < IPX; ++i) {
      const int j = wave * IPX + i;
      edge_copy(rs, to, j, chunk_of(j, BM) * (A4 ? 32 : 8) + j / (BM / 8) * KX < l ? xo[i] : kNoRow);
    }
  };
  auto copy_w = [&](int ws, HK_L uint8_t* to) HK_INLINE {
    const __amdgpu_buffer_rsrc_t rs = edge_rsrc(Wb + (int64_t)ws * (S::WL * kLine));
    const int64_t left = p.K - (int64_t)ws * (S::WL * 256);
    const int l = left >= S::WL * 256 ? S::WL * 256 : (int)left;
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int j = wave * IPW + i;
      edge_copy(rs, to, j, chunk_of(j, BN) * 32 + j / (BN / 8) * 256 < l ? wo[i] : kNoRow);
    }
  };
  const __amdgpu_buffer_rsrc_t wsr = __builtin_amdgcn_make_buffer_rsrc((void*)p.w_scale, (short)0, (int)((p.N * nb + 3) & ~3), 0x00020000);
  const __amdgpu_buffer_rsrc_t xsr =
      __builtin_amdgcn_make_buffer_rsrc((void*)(A4 ? p.x_scale : p.w_scale), (short)0, (int)(((A4 ? p.M : p.N) * nb + 3) & ~3), 0x00020000);
  // scales of block blk (bytes past a row's end belong to the next one and are masked out where they are used)
  auto copy_scales = [&](int blk) HK_INLINE {
    HK_L uint8_t* const to = (HK_L uint8_t*)sc + (blk & 1) * (SR * SRB);
#pragma unroll
    for (int i = 0; i < IPS; ++i) {
      const int j = (wave * IPS + i) % SI;  // wavefronts past the last copy repeat an earlier one: the same bytes again
      const bool isx = j * 1024 / SRB >= BN;
      const int ch = j * 64 + lane, r = ch / (SRB / 16) - (isx ? BN : 0), c = ch % (SRB / 16);
      const uint32_t o = ((uint32_t)(((isx ? m0 : n0) + r) * nb) & ~3u) + (uint32_t)(blk * 32 + c * 16);
      edge_copy(isx ? xsr : wsr, to, j, r < (isx ? ml : nl) ? o : kNoRow);
    }
  };

  // This lane's rows: the sub-tile's other 32-row blocks lie a constant further (the swizzle repeats every 16 rows).
  const int xrow = wm * WM + l32, wrow = wn * WN + l32;
  auto xat = [&](int i, int c) HK_INLINE { return kg * BM * kLine + line_off(xrow, c) + i * 32 * kLine; };
  auto wat = [&](int j, int c) HK_INLINE { return (S::WL > 1 ? kg * BN * kLine : 0) + line_off(wrow, c) + j * 32 * kLine; };
  // byte of a row's first scale modulo 4 (STR)
  uint32_t wsh[FN], xsh[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) xsh[i] = (uint32_t)((m0 + xrow + 32 * i) * nb) & 3u;
#pragma unroll
  for (int j = 0; j < FN; ++j) wsh[j] = (uint32_t)((n0 + wrow + 32 * j) * nb) & 3u;
  // four scale bytes of one row from byte h + 4 d of this wavefront's piece on, those past the end of K zero
  auto scales = [&](const HK_L uint8_t* cs, int row, uint32_t sh, int ks, int d) HK_INLINE {
    const int64_t have = nb - ((int64_t)ks * KG + kg) * SB - 4 * d;
    const uint32_t keep = have >= 4 ? ~0u : have <= 0 ? 0u : (1u << (8 * (int)have)) - 1u;
    const uint32_t pos = ((uint32_t)((ks * KG + kg) * SB) & 31u) + 4 * d;
    const HK_L uint8_t* const at = cs + row * SRB;
    uint32_t v;
    if constexpr (STR) {
      const HK_L uint32_t* const q = reinterpret_cast<const HK_L uint32_t*>(at + ((pos + sh) & ~3u));
      v = __builtin_amdgcn_alignbyte(q[1], q[0], (pos + sh) & 3u);
    } else {
      v = *reinterpret_cast<const HK_L uint32_t*>(at + (pos & ~3u)) >> (8 * (pos & 3u));
    }
    return (v & keep) >> (8 * h);
  };

  f32x16 acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = zero16();

  // Step ks, number i of the unrolled U.  GUARD: near the end, where not every copy exists; it waits for all of them.
  auto step = [&](auto ic, auto guard, int ks) HK_INLINE {
    constexpr int I = decltype(ic)::value, WI = I % SPW;
    constexpr bool GUARD = decltype(guard)::value;
    const HK_L uint8_t* const xs = xbuf(std::integral_constant<int, I % XR>());
    const HK_L uint8_t* const ws = wbuf(std::integral_constant<int, I / SPW % 2>());
    const HK_L uint8_t* const cs = (const HK_L uint8_t*)sc + (ks / SPB & 1) * (SR * SRB);
    u32x4 wf[2][FN], xf[2][FM];  // 16-bit X: wf[0] the piece's codes; 4-bit X: fragments of two slices
    uint32_t sw[2][FN], sx[2][FM];
    // a piece is four slices; the fragments of the next one are read while this one's products run (two register sets, fenced:
    // in the compiler's own order every slice waited for its reads)
    auto read_w = [&](int s) HK_INLINE {
      // 16-bit X: piece WI KG + kg of the line
#pragma unroll
      for (int j = 0; j < FN; ++j)
        wf[s & 1][j] = *reinterpret_cast<const HK_L u32x4*>(ws + wat(j, A4 ? 2 * s + h : S::WL > 1 || KG == 1 ? 2 * WI + h : 2 * (WI * KG + kg) + h));
    };
    auto read_x = [&](int s) HK_INLINE {
#pragma unroll
      for (int i = 0; i < FM; ++i) xf[s & 1][i] = *reinterpret_cast<const HK_L u32x4*>(xs + xat(i, A4 ? 2 * s + h : 4 * h + s));
    };
#pragma unroll
    for (int d = 0; d < (A4 ? 2 : 1); ++d) {
#pragma unroll
      for (int j = 0; j < FN; ++j) sw[d][j] = scales(cs, wrow + 32 * j, wsh[j], ks, d);
      if constexpr (A4)
#pragma unroll
        for (int i = 0; i < FM; ++i) sx[d][i] = scales(cs, BN + xrow + 32 * i, xsh[i], ks, d);
    }
    read_w(0);
    read_x(0);
    // copies: the next block of scales, the next stage of W, X of XR - 1 steps on
    if (ks % SPB == 0 && (ks / SPB + 1) * SPB < nk) copy_scales(ks / SPB + 1);
    if (WI == 0 && (!GUARD || ks + SPW < nk)) copy_w(ks / SPW + 1, wbuf(std::integral_constant<int, 1 - I / SPW % 2>()));
    if (!GUARD || ks + XR - 1 < nk) copy_x(ks + XR - 1, xbuf(std::integral_constant<int, (I + XR - 1) % XR>()));
    auto slice = [&](auto sc) HK_INLINE {
      constexpr int SL = decltype(sc)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (SL < 3) {
        if constexpr (A4) read_w(SL + 1);
        read_x(SL + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if constexpr (A4) {
#pragma unroll
          for (int i = 0; i < FM; ++i)
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(wf[SL & 1][j]), fp4_operand(xf[SL & 1][i]), acc[j][i], 4, 4,
                                                                        2 * (SL & 1), (int)sw[SL >> 1][j], 2 * (SL & 1), (int)sx[SL >> 1][i]);
        } else {
          const u32x4 f = mx4_unpack8<T>(wf[0][j][SL], mx_scale(sw[0][j] & 255u));
#pragma unroll
          for (int i = 0; i < FM; ++i) acc[j][i] = Mfma32<T>::mac(f, xf[SL & 1][i], acc[j][i]);
        }
      }
    };
    slice(std::integral_constant<int, 0>()), slice(std::integral_constant<int, 1>());
    slice(std::integral_constant<int, 2>()), slice(std::integral_constant<int, 3>());
    // The products are pure, and the compiler puts them off to the end of the loop body, the steps' fragments held in registers
    // until then, unless their results are used here.
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) asm volatile("" : "+v"(acc[j][i]));
    // The next step's X has landed everywhere, and W and scales if it begins a stage of theirs; later X may stay in flight, and
    // with it W copied in this step or the one before (XR 4: its stage begins two steps on or later).
    constexpr int KEEP = GUARD || XR == 2 ? 0 : (XR - 2) * IPX + (SPW > 2 && WI < 2 ? IPW : 0);
    barrier_keep_vm_lds<KEEP>();
  };
  using Whole = std::integral_constant<bool, false>;
  using Guard = std::integral_constant<bool, true>;
  auto steps = [&](auto guard, int ks) HK_INLINE {
    auto one = [&](auto ic) HK_INLINE {
      if (!decltype(guard)::value || ks + decltype(ic)::value < nk) step(ic, guard, ks + decltype(ic)::value);
    };
    one(std::integral_constant<int, 0>()), one(std::integral_constant<int, 1>());
    if constexpr (U > 2) one(std::integral_constant<int, 2>()), one(std::integral_constant<int, 3>());
    if constexpr (U > 4)
      one(std::integral_constant<int, 4>()), one(std::integral_constant<int, 5>()), one(std::integral_constant<int, 6>()), one(std::integral_constant<int, 7>());
  };
  static_assert(U == 2 || U == 4 || U == 8, "unrolled steps");
  copy_scales(0);
  copy_w(0, wbuf(std::integral_constant<int, 0>()));
  copy_x(0, xbuf(std::integral_constant<int, 0>()));
  if constexpr (XR > 2) {  // X of the steps before the first one's own copies (past the end: zeros that nobody reads)
    issue_order_fence();     // the first barrier counts on them being the last ones issued
    copy_x(1, xbuf(std::integral_constant<int, 1>()));
    copy_x(2, xbuf(std::integral_constant<int, 2>()));
  }
  barrier_keep_vm<(XR - 2) * IPX>();
  int ks = 0;
  for (; ks + U + (XR - 1 > SPW ? XR - 1 : SPW) <= nk; ks += U) steps(Whole(), ks);
  for (; ks < nk; ks += U) steps(Guard(), ks);

  if constexpr (KG > 1) {  // the groups' sums, in order, through the stages' memory (every copy has landed)
    constexpr int NB = FN * FM, PER = S::XT / 4096;  // accumulators of a wavefront; how many an X stage holds
    static_assert((KG - 1) * NWT * NB <= 2 * PER && PER % NB == 0, "merge areas");
    auto area = [&](int k, int b) {
      const int q = ((k - 1) * NWT + wt) * NB;
      return (float*)(q < PER ? x0 + q * 4096 : x1 + (q - PER) * 4096) + b * 1024 + lane;
    };
    if (kg > 0) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float* const mine = area(kg, b);
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
        const float* const part = area(k, b);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b / FM][b % FM][e] += part[e * 64];
      }
  }
  if (!lines) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v[4] = {acc[j][i][4 * e], acc[j][i][4 * e + 1], acc[j][i][4 * e + 2], acc[j][i][4 * e + 3]};
          store4<T>(p, m0 + wm * WM + i * 32 + l32, n0 + wn * WN + j * 32 + 8 * e + 4 * h, v, false);
        }
    return;
  }
  // Whole lines of y: 32 rows at a time go through the wavefront's own LDS area, so that a store writes 16 bytes a lane along
  // a row (8-byte stores straight from the accumulators touch 32 rows each: 4096 x 8192 x 2048 130 us, so 121).
  constexpr int RB = WN * 2 + 16;  // bytes of a row in the area, its pad off the banks of the next
  // KG > 1: in the merge area of group 1's wavefront, which this one has read; else in the stages of W
  constexpr int HALF = (NWT + 1) / 2, AREA = 32 * RB, MERGED = FN * FM * 4096;
  static_assert(KG > 1 ? AREA <= MERGED : HALF * AREA <= S::WT, "epilogue areas");
  HK_L uint8_t* const area = KG > 1      ? (HK_L uint8_t*)(wt * MERGED < S::XT ? x0 + wt * MERGED : x1 + (wt * MERGED - S::XT))
                             : wt < HALF ? (HK_L uint8_t*)w0 + wt * AREA
                                         : (HK_L uint8_t*)w1 + (wt - HALF) * AREA;
  const int64_t nw = n0 + wn * WN;
  u32x2 bias[FN][4];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bias[j][e] = u32x2{0, 0};
      const int64_t n = nw + j * 32 + 8 * e + 4 * h;
      if (p.bias && n < p.N) bias[j][e] = *reinterpret_cast<const HK_G u32x2*>(gcptr<uint16_t>(p.bias) + n);
    }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = acc[j][i][4 * e + r] + (r & 1 ? hi16<T>(bias[j][e][r >> 1]) : lo16<T>(bias[j][e][r >> 1]));
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
struct Tile2 {
  int bm, bn;
};
constexpr Tile2 kTiles[] = {{256, 256}, {128, 256}, {128, 128}, {64, 64}};

int64_t tiles_of(const hrt_mx4_mm_args& a, int t) { return cdiv(a.M, kTiles[t].bm) * cdiv(a.N, kTiles[t].bn); }
// Index of the tile, -1: mx4_rows.
// Few rows: up to 16, or 32 where K is short (32 rows, 16 bits: 1024 x 1024 5.2 us against 6.4 on 64 x 64 tiles, 8192 x 2048 12.0
// against 9.7).
// Tiles: one workgroup fits a CU, so a grid runs in rounds of 256, each a fixed cost (first copies, epilogue) and a time per
// 256 values of K, both fitted to 512 .. 8192 rows and columns, K 1024 .. 8192 (16-bit rows: 1024 x 8192 x 2048 128 x 256 tiles
// 37 us, 128 x 128 41, 256 x 256 48; 4096 x 8192 x 2048 134, 158, 119; 640 x 4096 x 4096 51, 31, 83).
int plan_of(const hrt_mx4_mm_args& a) {
  if (a.M <= 16 || (a.M <= 32 && a.K <= 1024)) return -1;
  const bool a4 = a.x_scale != 0;
  static constexpr struct { float fixed, per256; } kCost[2][4] = {{{8.5f, 6.3f}, {6.2f, 3.9f}, {6.1f, 2.1f}, {4.f, 0.75f}},
                                                                  {{11.f, 1.9f}, {7.4f, 1.4f}, {5.4f, 0.74f}, {4.2f, 0.25f}}};
  int best = 3;
  float us = 0.f;
  for (int t = 3; t >= 0; --t) {
    // 256 x 256 tiles of 4-bit rows leave no LDS for scale rows that do not start on dwords
    if (t == 0 && a4 && (a.K / 32) % 4 != 0) continue;
    const float e = (float)cdiv(tiles_of(a, t), 256) * (kCost[a4][t].fixed + kCost[a4][t].per256 * (float)a.K / 256.f);
    if (t == 3 || e < us) best = t, us = e;
  }
  return best;
}

template <typename T, bool A4, int BM, int BN, int WM, int WN, int KG, int XR, bool ODD = true>
void queue_tile(const hrt_mx4_mm_args& a, hipStream_t s, bool lines) {
  using S = TileShape<A4, BM, BN, WM, WN, KG, XR>;
  const int64_t tm = cdiv(a.M, BM), tn = cdiv(a.N, BN), nk = cdiv(a.K, S::KX * KG);
  const dim3 grid((uint32_t)(tm * tn)), block(64 * S::NW);
  if constexpr (ODD)
    if ((a.K / 32) % 4 != 0) {
      hipLaunchKernelGGL((mx4_tile<T, A4, BM, BN, WM, WN, KG, XR, true>), grid, block, 0, s, a, (int)tn, (int)nk, lines);
      return;
    }
  hipLaunchKernelGGL((mx4_tile<T, A4, BM, BN, WM, WN, KG, XR, false>), grid, block, 0, s, a, (int)tn, (int)nk, lines);
}

template <typename T, bool A4>
void queue_mm(const hrt_mx4_mm_args& a, int tile, hipStream_t s) {
  const bool vec = a.N % 4 == 0 && a.y % 8 == 0 && a.bias % 8 == 0, lines = vec && a.N % 8 == 0 && a.y % 16 == 0;
  switch (tile) {
    case 0: return queue_tile<T, A4, 256, 256, 128, 64, 1, 2, !A4>(a, s, lines);
    case 1: return queue_tile<T, A4, 128, 256, 64, 64, 1, A4 ? 2 : 4>(a, s, lines);
    case 2: return queue_tile<T, A4, 128, 128, 64, 64, 2, 2>(a, s, lines);
    case 3: return queue_tile<T, A4, 64, 64, 32, 64, 4, 2>(a, s, lines);
  }
  // wavefronts and batches that cover K once where they can
  const dim3 grid((uint32_t)cdiv(a.N, 16));
  const int64_t pieces = cdiv(a.K, 128);
  if (a.M > 16) hipLaunchKernelGGL((mx4_rows<T, A4, 2, 4, 2>), grid, dim3(256), 0, s, a, vec);
  else if (pieces <= 8) hipLaunchKernelGGL((mx4_rows<T, A4, 1, 4, 2>), grid, dim3(256), 0, s, a, vec);
  else if (pieces <= 16) hipLaunchKernelGGL((mx4_rows<T, A4, 1, 8, 2>), grid, dim3(512), 0, s, a, vec);
  else hipLaunchKernelGGL((mx4_rows<T, A4, 1, 8, 4>), grid, dim3(512), 0, s, a, vec);
}

template <typename T>
bool launch_mx4_mm(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_mx4_mm_args*>(pp);
  if (a.M <= 0 || a.N <= 0 || a.K <= 0) return ctx.fail("empty product");
  if (a.K % kMxBlock != 0) return ctx.fail("K must be a multiple of 32");
  const bool a4 = a.x_scale != 0;
  if (!a4 && (a.x_sm < 0 || a.x_sm % 8 != 0)) return ctx.fail("x's row stride must be a non-negative multiple of 8");
  if (a.x % 16 != 0 || a.w % 16 != 0 || a.w_scale % 4 != 0 || a.x_scale % 4 != 0 || a.y % 2 != 0 || a.bias % 2 != 0)
    return ctx.fail("x and w must be 16-byte aligned, scales 4-byte aligned");
  const int64_t nb = a.K / kMxBlock, xs[2] = {a.M, a.K}, xt[2] = {a.x_sm, 1};
  if (!(a4 ? ctx.check(a.x, (uint64_t)(a.M * (a.K / 2)), "x") && ctx.check(a.x_scale, (uint64_t)(a.M * nb), "x_scale")
           : ctx.check(a.x, hrt::span_bytes(2, xs, xt, 2), "x")) ||
      !ctx.check(a.w, (uint64_t)(a.N * (a.K / 2)), "w") || !ctx.check(a.w_scale, (uint64_t)(a.N * nb), "w_scale") ||
      !ctx.check(a.y, (uint64_t)(a.M * a.N) * 2, "y") || (a.bias && !ctx.check(a.bias, (uint64_t)a.N * 2, "bias")))
    return false;
  // offsets of a tile's rows and of a scale byte are 32-bit
  const int64_t lim = (int64_t)1 << 31;
  if ((a4 ? a.K / 2 : a.x_sm * 2) * 257 >= lim || a.K / 2 * 257 >= lim || a.N * nb + 8 >= lim || (a4 && a.M * nb + 8 >= lim))
    return ctx.fail("operand rows too long for one launch");
  const int tile = plan_of(a);
  if (!hrt::grid_fits(tile < 0 ? cdiv(a.N, 16) : tiles_of(a, tile), 512)) return ctx.fail("grid too large");
  if (a4) queue_mm<T, true>(a, tile, ctx.stream);
  else queue_mm<T, false>(a, tile, ctx.stream);
  return hrt::launch_ok(hipGetLastError(), ctx, "mx4_mm");
}

HRT_REGISTER("mx4_mm_bf16", hrt_mx4_mm_args, launch_mx4_mm<BF16>);
HRT_REGISTER("mx4_mm_f16", hrt_mx4_mm_args, launch_mx4_mm<F16>);

}  // namespace
}  // namespace hk
