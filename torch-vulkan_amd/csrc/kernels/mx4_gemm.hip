// "mx4_mm_{bf16,f16}": y = X W^T + bias with W in microscaled 4-bit floating point (mx4.h) and X in 16 bits or in 4.
//
// Two kernels, each in both forms:
//   * mx4_rows for few rows (M <= 64): bound by the weights' bytes.  A wavefront takes 16 columns of y and every fourth
//     128-wide piece of K; lane (n, g) loads the 32 codes of its column's block g straight into registers.
//   * mx4_tile for the rest: bound by the matrix cores and by L2 -> LDS.  Both operands are copied global -> LDS directly
//     through a ring of three stages (the scheme of gemm_dma_kernel.h), the weights as codes.
// 16-bit X: a lane's 16 bytes of codes are one scale block of one column; dword t of them becomes the 32x32x16 fragment of
// eight K values by four conversions, and X is read with the same K order (chunk 4 h + t of a 64-wide step), so the weights
// never exist in LDS or memory as 16-bit values and no lane exchange is needed.
// 4-bit X: v_mfma_scale_f32_32x32x64_f8f6f4 takes a lane's 16 bytes of codes as they are, with the block's scale byte.
// Lane layout of the scaled products (checked on the device), l = lane: 32x32x64: operand row l % 32, K block l / 32;
// 16x16x128: row l % 16, K block l / 16; the scale operand's byte `opsel` belongs to the lane's own block.
// W is the first operand in both kernels, so an accumulator holds four consecutive columns n of one row m of y.
#include <utility>

#include "../hrt/registry.h"
#include "mx4.h"

namespace hk {
namespace {

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
constexpr int kRowsWaves = 4;

template <typename T, bool A4, int MB>
__global__ __launch_bounds__(64 * kRowsWaves) void mx4_rows(hrt_mx4_mm_args p, bool vec) {
  __shared__ float part[kRowsWaves - 1][MB][64][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + r16 < p.N ? n0 + r16 : p.N - 1;  // columns past N repeat the last one and are not stored
  const int64_t nb = p.K / 32, steps = cdiv(p.K, 128);
  const HK_G uint8_t* wc = gcptr<uint8_t>(p.w) + n * (p.K / 2) + 16 * g;
  const HK_G uint8_t* ws = gcptr<uint8_t>(p.w_scale) + n * nb + g;
  f32x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const HK_G uint8_t* xr[MB];
  const HK_G uint8_t* xs[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {  // rows past M repeat the last one and are not stored
    const int64_t m = b * 16 + r16 < p.M ? b * 16 + r16 : p.M - 1;
    xr[b] = A4 ? gcptr<uint8_t>(p.x) + m * (p.K / 2) + 16 * g : gcptr<uint8_t>(p.x) + m * p.x_sm * 2 + 64 * g;
    xs[b] = gcptr<uint8_t>(p.x_scale) + m * nb + g;
  }
  for (int64_t st = wave; st < steps; st += kRowsWaves) {
    // a block past the end of K (the last step may have fewer than four) contributes zeros with scale 0 (2^-127)
    const bool in = st * 4 + g < nb;
    const int64_t at = in ? st : 0;
    u32x4 c = __builtin_nontemporal_load(reinterpret_cast<const HK_G u32x4*>(wc + at * 64));
    const uint32_t s = in ? ws[at * 4] : 0u;
    if (!in) c = u32x4{0, 0, 0, 0};
    if constexpr (A4) {
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        u32x4 x = *reinterpret_cast<const HK_G u32x4*>(xr[b] + at * 64);
        const uint32_t xv = in ? xs[b][at * 4] : 0u;
        if (!in) x = u32x4{0, 0, 0, 0};
        acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(c), fp4_operand(x), acc[b], 4, 4, 0, (int)s, 0, (int)xv);
      }
    } else {
      const float f = mx_scale(s);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const u32x4 wf = mx4_unpack8<T>(c[t], f);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          u32x4 x = *reinterpret_cast<const HK_G u32x4*>(xr[b] + at * 256 + 16 * t);
          if (!in) x = u32x4{0, 0, 0, 0};
          acc[b] = Mfma<T>::mac(wf, x, acc[b]);
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
    for (int w = 0; w < kRowsWaves - 1; ++w) acc[b] += *reinterpret_cast<const f32x4*>(part[w][b][lane]);
    const float v[4] = {acc[b][0], acc[b][1], acc[b][2], acc[b][3]};
    store4<T>(p, b * 16 + r16, n0 + 4 * g, v, vec);
  }
}

// ---- tiles ---------------------------------------------------------------------------------------------------------------
// Rows of RB bytes in LDS: 32 (64 codes), 64 (128 codes) or 128 (64 16-bit values); a row's 16-byte chunks are XOR-swizzled
// so that 16 consecutive rows read at one chunk hit distinct banks of a 256-byte line.
template <int RB>
__device__ __forceinline__ int row_swz(int row) {
  if constexpr (RB == 128) return tile_swz<8>(row);
  else if constexpr (RB == 64) return (row >> 2) & 3;
  else return (row >> 3) & 1;
}
template <int RB>
__device__ __forceinline__ int row_off(int row, int c) {
  return row * RB + ((c ^ row_swz<RB>(row)) << 4);
}

// A workgroup's wavefronts are KG groups along K times a grid of WM x WN sub-tiles: a step covers KG pieces of KS values of K,
// one per group, and the groups' sums are added in order at the end.  KG > 1 gives small grids (few rows) the wavefronts that
// hide a copy's latency without a second launch.
template <bool A4, int BM, int BN, int WM, int WN, int KG>
struct TileShape {
  static constexpr int KS = A4 ? 128 : 64;                // K values per piece
  static constexpr int NWT = (BM / WM) * (BN / WN);       // wavefronts per group
  static constexpr int NW = NWT * KG;
  static constexpr int XB = A4 ? 64 : 128, WB = KS / 2;   // bytes of an LDS row of X and of W
  static constexpr int XT = BM * XB, WT = BN * WB;        // bytes of a piece
  static constexpr int IPX = KG * XT / 1024 / NW, IPW = KG * WT / 1024 / NW;  // copies per wavefront and step
  static constexpr int FM = WM / 32, FN = WN / 32;
  static_assert(KG * XT % (1024 * NW) == 0 && KG * WT % (1024 * NW) == 0 && IPX >= 1 && IPW >= 1, "copy split");
};

// STR: a row's scale bytes of one piece may straddle two dwords (K / 32 not a multiple of the bytes per piece).
template <typename T, bool A4, int BM, int BN, int WM, int WN, int KG, bool STR>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN) * KG) void mx4_tile(hrt_mx4_mm_args p, int tiles_n, int nk, bool lines) {
  using S = TileShape<A4, BM, BN, WM, WN, KG>;
  constexpr int NW = S::NW, NWT = S::NWT, XB = S::XB, WB = S::WB, IPX = S::IPX, IPW = S::IPW, FM = S::FM, FN = S::FN, KS = S::KS;
  constexpr int SD = STR ? 2 : 1;                                  // scale dwords per row and piece
  constexpr int SR = BN + (A4 ? BM : 0), SI = KG * SR * SD / 64;   // rows with scales; copies of 64 dwords
  constexpr int IPS = (SI + NW - 1) / NW;                          // per wavefront (the last ones repeat a copy)
  constexpr int SB = KS / 32;                                      // scale bytes per row and piece
  static_assert(SR * SD % 64 == 0 && BN * SD % 64 == 0, "whole scale copies");
  // One LDS object per stage, so that the compiler can tell the reads of one from the copies into another (it tracks only
  // a few objects: with X, W and the scales apart it waited for every copy at the loop's head).
  constexpr int STAGE = KG * (S::XT + S::WT) + SI * 256;
  __shared__ __attribute__((aligned(1024))) uint8_t st0[STAGE], st1[STAGE], st2[STAGE];
  auto buf = [&](auto ic) { constexpr int I = decltype(ic)::value; return (HK_L uint8_t*)(I == 0 ? st0 : I == 1 ? st1 : st2); };

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / NWT, wt = wave % NWT, wm = wt % (BM / WM), wn = wt / (BM / WM), l32 = lane & 31, h = lane >> 5;
  // n-fastest tile numbers, in scalar registers, and with them every buffer resource
  const uint32_t tm = __builtin_amdgcn_readfirstlane(blockIdx.x / (uint32_t)tiles_n);
  const uint32_t tn = __builtin_amdgcn_readfirstlane(blockIdx.x % (uint32_t)tiles_n);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int64_t nb = p.K / 32;
  const int ml = p.M - m0 < BM ? (int)(p.M - m0) : BM, nl = p.N - n0 < BN ? (int)(p.N - n0) : BN;

  // copy sources; lane offsets inside a step, kNoRow where the row does not exist (the buffer's range check gives zeros)
  const uint32_t xss = (uint32_t)(A4 ? p.K / 2 : p.x_sm * 2), wss = (uint32_t)(p.K / 2);
  const HK_G uint8_t* Xb = gcptr<uint8_t>(p.x) + m0 * xss;
  const HK_G uint8_t* Wb = gcptr<uint8_t>(p.w) + n0 * wss;
  uint32_t xo[IPX], wo[IPW];
  auto xchunk = [&](int i) {  // copy i's chunk within the piece: row and column
    const int ch = ((wave * IPX + i) * 64 + lane) % (S::XT / 16), row = ch / (XB / 16);
    return std::pair<int, int>{row, (ch % (XB / 16)) ^ row_swz<XB>(row)};
  };
  auto wchunk = [&](int i) {
    const int ch = ((wave * IPW + i) * 64 + lane) % (S::WT / 16), row = ch / (WB / 16);
    return std::pair<int, int>{row, (ch % (WB / 16)) ^ row_swz<WB>(row)};
  };
  auto xpiece = [&](int i) { return (wave * IPX + i) / (S::XT / 1024); };
  auto wpiece = [&](int i) { return (wave * IPW + i) / (S::WT / 1024); };
#pragma unroll
  for (int i = 0; i < IPX; ++i) {
    const auto [row, c] = xchunk(i);
    xo[i] = row < ml ? (uint32_t)row * xss + (uint32_t)(c * 16 + xpiece(i) * XB) : kNoRow;
  }
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const auto [row, c] = wchunk(i);
    wo[i] = row < nl ? (uint32_t)row * wss + (uint32_t)(c * 16 + wpiece(i) * WB) : kNoRow;
  }
  // scales: dword d of row r (W rows first, then X rows) of piece k is LDS dword (k * SR + r) * SD + d.  Dwords are aligned
  // down; what a row does not own is shifted or masked out where it is used.
  const __amdgpu_buffer_rsrc_t wsr = edge_rsrc(gcptr<uint8_t>(p.w_scale)), xsr = edge_rsrc(gcptr<uint8_t>(A4 ? p.x_scale : p.w_scale));
  uint32_t so[IPS];
  bool sx[IPS];
#pragma unroll
  for (int i = 0; i < IPS; ++i) {
    const int j = (wave * IPS + i) % SI;  // wavefronts past the last copy repeat an earlier one: the same bytes again
    const int d = (j * 64 + lane) % (SR * SD), row = d / SD, piece = j * 64 / (SR * SD);
    sx[i] = A4 && j * 64 % (SR * SD) / SD >= BN;  // uniform: BN * SD is a multiple of 64
    const int r = sx[i] ? row - BN : row;
    const int64_t o = ((sx[i] ? m0 : n0) + r) * nb + piece * SB;  // byte of the row's first scale in this piece
    // (4 (d % SD): the second dword)
    so[i] = r < (sx[i] ? ml : nl) ? (uint32_t)(o + 4 * (d % SD)) : kNoRow;
  }

  auto copy = [&](int ks, HK_L uint8_t* xt) {
    HK_L uint8_t* const wt = xt + KG * S::XT;
    HK_L uint8_t* const st = wt + KG * S::WT;
    const __amdgpu_buffer_rsrc_t xr = edge_rsrc(Xb + (int64_t)ks * (KG * XB)), wr = edge_rsrc(Wb + (int64_t)ks * (KG * WB));
    // the last step may hold fewer values: chunks past K are zeros (a select, not a branch: the compiler counts the copies
    // in flight along every path)
    const int64_t left = p.K - (int64_t)ks * (KG * KS);
    const int l = left >= KG * KS ? KG * KS : (int)left;
#pragma unroll
    for (int i = 0; i < IPX; ++i)
      edge_copy(xr, xt, wave * IPX + i, xchunk(i).second * (A4 ? 32 : 8) + xpiece(i) * KS < l ? xo[i] : kNoRow);
#pragma unroll
    for (int i = 0; i < IPW; ++i) edge_copy(wr, wt, wave * IPW + i, wchunk(i).second * 32 + wpiece(i) * KS < l ? wo[i] : kNoRow);
#pragma unroll
    for (int i = 0; i < IPS; ++i) {
      const int j = (wave * IPS + i) % SI;
      const uint32_t o = so[i] == kNoRow ? kNoRow : (so[i] + (uint32_t)(ks * KG * SB)) & ~3u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(sx[i] ? xsr : wsr, st + j * 256, 4, (int)o, 0, 0, 0);
    }
  };

  // This lane's rows: the sub-tile's other 32-row blocks lie a constant further (the swizzle repeats every 16 rows).
  const int xrow = wm * WM + l32, wrow = wn * WN + l32;
  const int xbase = kg * S::XT, wbase = KG * S::XT + kg * S::WT, sbase = KG * (S::XT + S::WT) + kg * SR * SD * 4;
  auto xat = [&](int i, int c) { return xbase + row_off<XB>(xrow, c) + i * 32 * XB; };
  auto wat = [&](int j, int c) { return wbase + row_off<WB>(wrow, c) + j * 32 * WB; };
  uint32_t wsh[FN], xsh[FM];  // byte of the row's first scale, modulo 4
#pragma unroll
  for (int i = 0; i < FM; ++i) xsh[i] = (uint32_t)((m0 + xrow + 32 * i) * nb) & 3u;
#pragma unroll
  for (int j = 0; j < FN; ++j) wsh[j] = (uint32_t)((n0 + wrow + 32 * j) * nb) & 3u;

  f32x16 acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = zero16();

  // the scale bytes of one row in this wavefront's piece, the first in byte 0, those past the end of K zero
  auto scales = [&](const HK_L uint8_t* st, int row, uint32_t sh, int ks) {
    const int64_t first = ((int64_t)ks * KG + kg) * SB, have = nb - first;
    const uint32_t keep = have >= 4 ? ~0u : have <= 0 ? 0u : (1u << (8 * (int)have)) - 1u;
    const uint32_t by = (sh + (uint32_t)first) & 3u;
    const HK_L uint8_t* const at = st + sbase + row * SD * 4;
    uint32_t v;
    if constexpr (STR) {
      const u32x2 d = *reinterpret_cast<const HK_L u32x2*>(at);
      v = __builtin_amdgcn_alignbyte(d.y, d.x, by);
    } else {
      v = *reinterpret_cast<const HK_L uint32_t*>(at) >> (8 * by);
    }
    return v & keep;
  };

  constexpr int PER = IPX + IPW + IPS;  // copies per wavefront and step
  auto step = [&](auto bc, int ks, bool more) {
    constexpr int BUF = decltype(bc)::value, NXT = (BUF + 2) % 3;
    const HK_L uint8_t* const st = buf(bc);
    using N = std::integral_constant<int, NXT>;
    // fragments of the next slice are read while this one's products run (two register sets, fenced: in the compiler's own
    // order every slice waited for its reads)
    if constexpr (A4) {
      uint32_t sw[FN], sxv[FM];
      u32x4 wf[2][FN], xf[2][FM];
      auto read = [&](int s) {
#pragma unroll
        for (int j = 0; j < FN; ++j) wf[s][j] = *reinterpret_cast<const HK_L u32x4*>(st + wat(j, 2 * s + h));
#pragma unroll
        for (int i = 0; i < FM; ++i) xf[s][i] = *reinterpret_cast<const HK_L u32x4*>(st + xat(i, 2 * s + h));
      };
#pragma unroll
      for (int j = 0; j < FN; ++j) sw[j] = scales(st, wrow + 32 * j, wsh[j], ks) >> (8 * h);
#pragma unroll
      for (int i = 0; i < FM; ++i) sxv[i] = scales(st, BN + xrow + 32 * i, xsh[i], ks) >> (8 * h);
      read(0);
      if (more) copy(ks + 2, buf(N()));
      both([&](auto sc) {
        constexpr int K64 = decltype(sc)::value;
        __builtin_amdgcn_sched_barrier(0);
        if (K64 == 0) read(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int i = 0; i < FM; ++i)
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(wf[K64][j]), fp4_operand(xf[K64][i]), acc[j][i], 4, 4,
                                                                        2 * K64, (int)sw[j], 2 * K64, (int)sxv[i]);
      });
    } else {
      u32x4 wc[FN], xf[2][FM];
      float f[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        wc[j] = *reinterpret_cast<const HK_L u32x4*>(st + wat(j, h));
        f[j] = mx_scale((scales(st, wrow + 32 * j, wsh[j], ks) >> (8 * h)) & 255u);
      }
      auto read = [&](int t) {
#pragma unroll
        for (int i = 0; i < FM; ++i) xf[t & 1][i] = *reinterpret_cast<const HK_L u32x4*>(st + xat(i, 4 * h + t));
      };
      read(0);
      if (more) copy(ks + 2, buf(N()));
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        if (t < 3) read(t + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const u32x4 wf = mx4_unpack8<T>(wc[j][t], f[j]);
#pragma unroll
          for (int i = 0; i < FM; ++i) acc[j][i] = Mfma32<T>::mac(wf, xf[t & 1][i], acc[j][i]);
        }
      }
    }
    // The products are pure, and the compiler puts them off to the end of the loop body, all three steps' fragments held
    // in registers until then, unless their results are used here.
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) asm volatile("" : "+v"(acc[j][i]));
    // the next step's copies (issued a step ago) have landed everywhere; this step's stay in flight
    if (more) barrier_keep_vm_lds<PER>();
    else barrier_keep_vm_lds<0>();
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  copy(0, buf(I0()));
  issue_order_fence();
  copy(nk > 1 ? 1 : 0, buf(I1()));  // a single step: a copy that nobody reads, on every path alike
  barrier_keep_vm<PER>();
  int ks = 0;
  for (; ks + 5 <= nk; ks += 3) {  // every step of the body copies: no branch around the copies
    step(I0(), ks, true);
    step(I1(), ks + 1, true);
    step(I2(), ks + 2, true);
  }
  // the last one to four
  step(I0(), ks, ks + 2 < nk);
  if (ks + 1 < nk) step(I1(), ks + 1, ks + 3 < nk);
  if (ks + 2 < nk) step(I2(), ks + 2, false);
  if (ks + 3 < nk) step(I0(), ks + 3, false);

  if constexpr (KG > 1) {  // the groups' sums, in order, through the stages' memory (every copy has landed)
    constexpr int NB = FN * FM, PB = KG == 2 ? NB / 2 : NB;  // accumulators, and how many of a wavefront's share a stage
    static_assert((KG == 4 || (KG == 2 && NB % 2 == 0)) && NWT * PB * 4096 <= STAGE, "merge areas");
    // accumulator b of group k: KG 4: the groups 1, 2, 3 have a stage each; KG 2: group 1 has two
    auto area = [&](int k, int b) {
      const int o = KG == 4 ? k - 1 : b / PB;
      return (float*)(o == 0 ? st0 : o == 1 ? st1 : st2) + (wt * PB + b % PB) * 1024 + lane;
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
  // KG > 1: in the merge area of group 1's wavefront, which this one has read; else half of the areas in each of two stages
  constexpr int HALF = (NWT + 1) / 2, MERGED = KG > 1 ? FN * FM / (KG == 2 ? 2 : 1) * 4096 : 0;
  static_assert(KG > 1 ? 32 * RB <= MERGED : HALF * 32 * RB <= STAGE, "epilogue areas");
  HK_L uint8_t* const area = KG > 1      ? (HK_L uint8_t*)st0 + wt * MERGED
                             : wt < HALF ? (HK_L uint8_t*)st0 + wt * (32 * RB)
                                         : (HK_L uint8_t*)st1 + (wt - HALF) * (32 * RB);
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
int plan_of(const hrt_mx4_mm_args& a) {
  if (a.M <= 64) return -1;
  return tiles_of(a, 0) >= 256 ? 0 : tiles_of(a, 1) >= 192 ? 1 : tiles_of(a, 2) >= 192 ? 2 : 3;
}

template <typename T, bool A4, int BM, int BN, int WM, int WN, int KG>
void queue_tile(const hrt_mx4_mm_args& a, hipStream_t s, bool lines) {
  using S = TileShape<A4, BM, BN, WM, WN, KG>;
  const int64_t tm = cdiv(a.M, BM), tn = cdiv(a.N, BN), nk = cdiv(a.K, S::KS * KG);
  const dim3 grid((uint32_t)(tm * tn)), block(64 * S::NW);
  if ((a.K / 32) % (S::KS / 32) != 0) hipLaunchKernelGGL((mx4_tile<T, A4, BM, BN, WM, WN, KG, true>), grid, block, 0, s, a, (int)tn, (int)nk, lines);
  else hipLaunchKernelGGL((mx4_tile<T, A4, BM, BN, WM, WN, KG, false>), grid, block, 0, s, a, (int)tn, (int)nk, lines);
}

template <typename T, bool A4>
void queue_mm(const hrt_mx4_mm_args& a, int tile, hipStream_t s) {
  const bool vec = a.N % 4 == 0 && a.y % 8 == 0 && a.bias % 8 == 0, lines = vec && a.N % 8 == 0 && a.y % 16 == 0;
  switch (tile) {
    case 0: return queue_tile<T, A4, 256, 256, 128, 64, 1>(a, s, lines);
    case 1: return queue_tile<T, A4, 128, 256, 64, 64, 1>(a, s, lines);
    case 2: return queue_tile<T, A4, 128, 128, 64, 64, 2>(a, s, lines);
    case 3: return queue_tile<T, A4, 64, 64, 32, 64, 4>(a, s, lines);
  }
  const dim3 grid((uint32_t)cdiv(a.N, 16)), block(64 * kRowsWaves);
  switch (cdiv(a.M, 16)) {
    case 1: hipLaunchKernelGGL((mx4_rows<T, A4, 1>), grid, block, 0, s, a, vec); return;
    case 2: hipLaunchKernelGGL((mx4_rows<T, A4, 2>), grid, block, 0, s, a, vec); return;
    case 3: hipLaunchKernelGGL((mx4_rows<T, A4, 3>), grid, block, 0, s, a, vec); return;
    default: hipLaunchKernelGGL((mx4_rows<T, A4, 4>), grid, block, 0, s, a, vec); return;
  }
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
