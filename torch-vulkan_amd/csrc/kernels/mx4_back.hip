// "mx4_mm_back_{bf16,f16}": y = G W, the input gradient of the product y' = X W^T (mx4_gemm.hip), with W [N, K] in microscaled
// 4-bit floating point (mx4.h) and G [M, N], y [M, K] in 16 bits.
//
// The sum runs over W's rows, while a block's scale and a byte's two codes run along them, so the codes have to be turned
// over on their way into the matrix cores.  W's rows lie in LDS as codes; a lane owns four consecutive columns k of y and
// reads its two bytes from each of eight rows n, converts them with the scale of (n, k's block) - four conversions
// give two columns of two rows - and two byte permutations make (n, n + 1) pairs of each column of them.  Eight rows give one
// 32x32x16 operand fragment for each of the lane's columns: fragment i holds the columns 4 r + i of the wavefront's 128, which
// costs nothing, as the columns of a product may be taken in any order; an accumulator's rows come out 4 r + i too, so
// the four accumulators of a lane hold 16 neighbouring values of a row of y.  Nothing of W is stored in 16 bits.
// Bound: the matrix cores and the 32 vector instructions that a slice of 16 rows takes beside its 4 FM products of 36 cycles; half a
// slice's conversions are issued between the other half's products.  Measured, bf16, M x N x K (in brackets a dequantised copy
// and its product, which also takes 2 N K bytes of scratch): 16 x 2048 x 2048 13 us (15), 308 x 2048 x 2048 13 (24),
// 308 x 8192 x 2048 35 (40), 512 x 4096 x 4096 37 (50), 1024 x 2048 x 8192 43 (51), 4096 x 8192 x 2048 140 us, 983 TFLOP/s (149),
// 4096 x 2048 x 8192 142 (146).
#include "../hrt/registry.h"
#include "mx4.h"

namespace hk {
namespace {

#define HK_INLINE __attribute__((always_inline))

constexpr int kSlice = 64, kLine = 2 * kSlice;  // rows of W in a stage, bytes of a row of G in it

// A workgroup's wavefronts are KG groups along N times a grid of WM x 128 sub-tiles; a step takes kSlice rows of W per group.
// G, W and the scales have rings of R stages: three where one workgroup of four wavefronts has a CU to itself.
template <int BM, int BK, int WM, int KG>
struct BackShape {
  static constexpr int NWT = (BM / WM) * (BK / 128), NW = NWT * KG, FM = WM / 32;
  static constexpr int RB = BK / 2, KB = BK / 32;                          // bytes of codes, scales of a row
  static constexpr int XT = KG * BM * kLine, WT = KG * kSlice * RB;        // bytes of a stage
  static constexpr int IPX = XT / 1024 / NW, IPW = WT / 1024 / NW;         // copies per wavefront
  static constexpr int SPT = KG * kSlice * KB / (64 * NW), SP = kSlice + 8;  // scales per thread; LDS pitch, off the next one's banks
  static_assert(XT % (1024 * NW) == 0 && WT % (1024 * NW) == 0 && SPT * 64 * NW == KG * kSlice * KB, "copy split");
  static_assert(KG == 1 || (KG - 1) * NWT * FM * 4096 <= XT, "merge area");
};

// The place of row n of a slice in LDS: rows n and n + 8 of sixteen, which the two half-waves read together, next to each other.
__device__ __forceinline__ int row_at(int place) { return (place & ~15) | ((place & 1) << 3) | ((place & 15) >> 1); }

template <typename T, int BM, int BK, int WM, int KG, int R>
__global__ __launch_bounds__(64 * (BM / WM) * (BK / 128) * KG, R > 2 ? 1 : 2) void mx4_back(hrt_mx4_mm_args p, int tiles_k, int steps) {
  using S = BackShape<BM, BK, WM, KG>;
  constexpr int NW = S::NW, NWT = S::NWT, FM = S::FM, RB = S::RB, KB = S::KB, IPX = S::IPX, IPW = S::IPW, SPT = S::SPT, SP = S::SP;
  // One LDS object per stage, so that the compiler can tell the reads of one from the copies into another.
  __shared__ __attribute__((aligned(1024))) uint8_t x0[S::XT], x1[S::XT], x2[R > 2 ? S::XT : 16], w0[S::WT], w1[S::WT], w2[R > 2 ? S::WT : 16];
  __shared__ __attribute__((aligned(16))) float sc[R][KG * KB * SP];
  auto xbuf = [&](auto ic) HK_INLINE { constexpr int I = decltype(ic)::value; return (HK_L uint8_t*)(I == 0 ? x0 : I == 1 ? x1 : x2); };
  auto wbuf = [&](auto ic) HK_INLINE { constexpr int I = decltype(ic)::value; return (HK_L uint8_t*)(I == 0 ? w0 : I == 1 ? w1 : w2); };

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave / NWT, wt = wave % NWT, wm = wt % (BM / WM), wk = wt / (BM / WM), l32 = lane & 31, h = lane >> 5;
  // every XCD takes a run of neighbouring tiles, whose rows of G its L2 then holds (4096 x 8192 x 2048: 154 us without, so 143)
  const uint32_t id = gridDim.x % 8 == 0 ? blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
  const uint32_t tm = __builtin_amdgcn_readfirstlane(id / (uint32_t)tiles_k);
  const uint32_t tk = __builtin_amdgcn_readfirstlane(id % (uint32_t)tiles_k);
  const int64_t m0 = (int64_t)tm * BM, k0 = (int64_t)tk * BK, nb = p.K / 32;
  const int ml = p.M - m0 < BM ? (int)(p.M - m0) : BM, kl = p.K - k0 < BK ? (int)(p.K - k0) : BK;
  const uint32_t xss = (uint32_t)(p.x_sm * 2), wss = (uint32_t)(p.K / 2);
  const HK_G uint8_t* Xb = gcptr<uint8_t>(p.x) + m0 * xss;
  const HK_G uint8_t* Wb = gcptr<uint8_t>(p.w) + k0 / 2;
  const HK_G uint8_t* Sb = gcptr<uint8_t>(p.w_scale) + k0 / 32;

  // copy sources: lane offsets inside a stage, kNoRow where the row or column does not exist (zeros)
  uint32_t xo[IPX], wo[IPW];
  int xn[IPX], wn[IPW];  // first value of N of the lane's chunk, its row of W
#pragma unroll
  for (int i = 0; i < IPX; ++i) {
    const int j = wave * IPX + i, row = (j * 8 + (lane >> 3)) % BM, c = (lane & 7) ^ tile_swz<8>(row);
    xn[i] = j / (BM / 8) * kSlice + c * 8;
    xo[i] = row < ml ? (uint32_t)row * xss + (uint32_t)xn[i] * 2 : kNoRow;
  }
#pragma unroll
  for (int i = 0; i < IPW; ++i) {
    const int ch = (wave * IPW + i) * 64 + lane, place = ch / (RB / 16), c = ch % (RB / 16);
    wn[i] = row_at(place);
    wo[i] = c * 32 < kl ? (uint32_t)wn[i] * wss + (uint32_t)c * 16 : kNoRow;
  }
  auto copy = [&](auto ic, int st) HK_INLINE {
    const int64_t n0 = (int64_t)st * (KG * kSlice);
    const int left = p.N - n0 >= KG * kSlice ? KG * kSlice : (int)(p.N - n0);  // none past the last step: nothing is fetched
    const __amdgpu_buffer_rsrc_t xr = edge_rsrc(Xb + n0 * 2), wr = edge_rsrc(Wb + n0 * wss);
#pragma unroll
    for (int i = 0; i < IPX; ++i) edge_copy(xr, xbuf(ic), wave * IPX + i, xn[i] < left ? xo[i] : kNoRow);
#pragma unroll
    for (int i = 0; i < IPW; ++i) edge_copy(wr, wbuf(ic), wave * IPW + i, wn[i] < left ? wo[i] : kNoRow);
  };
  // Scales go through registers, as they are turned over: [block of K][row of W], in fp32 (a byte shifted once, not in every lane).
  // Those past the end are 1.  Range-checked loads, so that every step issues the same number: a branch around a load of no
  // lane would let the barrier's count pass a copy that is still in flight.
  uint32_t sb[SPT];
  auto load_scales = [&](int st) HK_INLINE {
    const int64_t n0 = (int64_t)st * (KG * kSlice);
    const __amdgpu_buffer_rsrc_t rs = edge_rsrc(Sb + n0 * nb);
#pragma unroll
    for (int u = 0; u < SPT; ++u) {
      const int e = u * 64 * NW + tid, n = e / KB, kb = e % KB;
      const bool ok = n0 + n < p.N && kb * 32 < kl;
      const uint32_t s = __builtin_amdgcn_raw_buffer_load_b8(rs, ok ? n * (int)nb + kb : (int)kNoRow, 0, 0);
      sb[u] = ok ? s : 127u;
    }
  };
  auto store_scales = [&](int at) HK_INLINE {
#pragma unroll
    for (int u = 0; u < SPT; ++u) {
      const int e = u * 64 * NW + tid, n = e / KB, kb = e % KB;
      sc[at][(n / kSlice * KB + kb) * SP + (n & (kSlice - 13)) + ((n & 4) << 1) + ((n & 8) >> 1)] = mx_scale(sb[u]);
    }
  };

  // this lane's addresses in a stage: fragment row l32 of sub-tile wm, two bytes of sub-tile wk's columns
  const int xrow = wm * WM + l32, wcol = wk * 64 + 2 * l32;
  const int sat = (kg * KB + wk * 4 + (l32 >> 3)) * SP + 4 * h;

  f32x16 acc[4][FM];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int f = 0; f < FM; ++f) acc[i][f] = zero16();

  constexpr int KEEP = R > 2 ? IPX + IPW + SPT : 0;  // R 3: the copies and scales of the step after the next may stay in flight
  auto step = [&](auto ic, int st) HK_INLINE {
    constexpr int I = decltype(ic)::value;
    const HK_L uint8_t* const xs = xbuf(ic) + kg * BM * kLine;
    const HK_L uint8_t* const ws = wbuf(ic) + kg * kSlice * RB;
    const float* const ss = &sc[I][sat];
    if (R == 2) load_scales(st + 1);
    copy(std::integral_constant<int, (I + R - 1) % R>(), st + R - 1);
    uint32_t cw[2][8];
    f32x4 cs[2][2];
    u32x4 xf[2][FM];
    auto read = [&](int s) HK_INLINE {
#pragma unroll
      for (int j = 0; j < 8; ++j) cw[s & 1][j] = *reinterpret_cast<const HK_L uint16_t*>(ws + (s * 16 + 2 * j + h) * RB + wcol);
#pragma unroll
      for (int j = 0; j < 2; ++j) cs[s & 1][j] = *reinterpret_cast<const f32x4*>(ss + s * 16 + 8 * j);
#pragma unroll
      for (int f = 0; f < FM; ++f) xf[s & 1][f] = *reinterpret_cast<const HK_L u32x4*>(xs + tile_off<8>(xrow, 2 * s + h) + f * 32 * kLine);
    };
    // two columns' fragments, of byte B of slice SL's rows
    u32x4 wf[2][2];
    auto turn = [&](auto tc) HK_INLINE {
      constexpr int B = decltype(tc)::value & 1, SL = decltype(tc)::value >> 1;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t a = mx4_pair<T, B>(cw[SL & 1][2 * t], cs[SL & 1][t >> 1][2 * (t & 1)]);
        const uint32_t b = mx4_pair<T, B>(cw[SL & 1][2 * t + 1], cs[SL & 1][t >> 1][2 * (t & 1) + 1]);
        wf[B][0][t] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        wf[B][1][t] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      }
    };
    read(0);
    turn(std::integral_constant<int, 0>());
    // half a slice: its products, with the next half's conversions between them
    auto half = [&](auto tc) HK_INLINE {
      constexpr int I = decltype(tc)::value, B = I & 1, SL = I >> 1;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (B == 0 && SL < 3) read(SL + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int m = 0; m < FM; ++m) acc[2 * B + e][m] = Mfma32<T>::mac(wf[B][e], xf[SL & 1][m], acc[2 * B + e][m]);
      if constexpr (I < 7) {
        turn(std::integral_constant<int, I + 1>());
#pragma unroll
        for (int q = 0; q < 2 * FM; ++q) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);         // a product
          __builtin_amdgcn_sched_group_barrier(0x002, 8 / FM, 0);    // its share of the vector instructions
        }
      }
    };
    auto slice = [&](auto sc_) HK_INLINE {
      constexpr int SL = decltype(sc_)::value;
      half(std::integral_constant<int, 2 * SL>()), half(std::integral_constant<int, 2 * SL + 1>());
    };
    slice(std::integral_constant<int, 0>()), slice(std::integral_constant<int, 1>());
    if (R > 2) store_scales((I + 1) % R), load_scales(st + 2);
    slice(std::integral_constant<int, 2>()), slice(std::integral_constant<int, 3>());
    // The products' results are used here, else the compiler puts them off past the barrier.  One wavefront on a SIMD has
    // them in accumulator registers: ordinary ones would be copied every step.
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int f = 0; f < FM; ++f) {
        if constexpr (R > 2) asm volatile("" : "+a"(acc[i][f]));
        else asm volatile("" : "+v"(acc[i][f]));
      }
    if (R == 2) store_scales(1 - I);
    barrier_keep_vm_lds<KEEP>();
  };
  load_scales(0);
  copy(std::integral_constant<int, 0>(), 0);
  if (R > 2) {
    issue_order_fence();  // the first barrier counts on stage 1's copies and scales being the last ones issued
    copy(std::integral_constant<int, 1>(), 1);
  }
  store_scales(0);
  if (R > 2) load_scales(1);
  barrier_keep_vm_lds<KEEP>();
  int st = 0;
  for (; st + R <= steps; st += R) {
    step(std::integral_constant<int, 0>(), st);
    step(std::integral_constant<int, 1>(), st + 1);
    if constexpr (R > 2) step(std::integral_constant<int, 2>(), st + 2);
  }
  if (st < steps) step(std::integral_constant<int, 0>(), st);
  if constexpr (R > 2)
    if (st + 1 < steps) step(std::integral_constant<int, 1>(), st + 1);
  if constexpr (KG > 1) barrier_keep_vm_lds<0>();

  if constexpr (KG > 1) {  // the groups' sums, in order, a column of accumulators at a time through the two stages of G in turn
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* const area = (float*)(i & 1 ? x1 : x0);
      if (kg > 0) {
#pragma unroll
        for (int f = 0; f < FM; ++f)
#pragma unroll
          for (int e = 0; e < 16; ++e) area[(((kg - 1) * NWT + wt) * FM + f) * 1024 + e * 64 + lane] = acc[i][f][e];
      }
      __syncthreads();
      if (kg == 0) {
#pragma unroll
        for (int k = 1; k < KG; ++k)
#pragma unroll
          for (int f = 0; f < FM; ++f)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][f][e] += area[(((k - 1) * NWT + wt) * FM + f) * 1024 + e * 64 + lane];
      }
    }
    if (kg > 0) return;
  }
  // element 4 j + e of accumulator i: column 4 (8 j + 4 h + e) + i
#pragma unroll
  for (int f = 0; f < FM; ++f) {
    const int64_t m = m0 + wm * WM + f * 32 + l32;
    if (m >= p.M) continue;
    HK_G uint16_t* const y = gptr<uint16_t>(p.y) + m * p.K;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int64_t k = k0 + wk * 128 + 4 * (8 * j + 4 * h) + 8 * q;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[e & 3][f][4 * j + 2 * q + (e >> 2)];
        const u32x2 lo = pack4<T>(v), hi = pack4<T>(v + 4);
        if (k < p.K) *reinterpret_cast<HK_G u32x4*>(y + k) = u32x4{lo.x, lo.y, hi.x, hi.y};
      }
  }
}

// Tiles, and what a grid of them takes in us, fitted to 16 .. 4096 rows and 2048 .. 8192 rows and columns of W: once, per round of 256
// workgroups, and per 256 rows of W for each round, `alone` at least (where two workgroups share a CU, a lone one does not
// fill it).  308 x 2048 x 2048: tiles in this order 50, 34, 19, 23 and 13 us; 512 x 4096 x 4096 94, 60, 33, 42, 36;
// 2048 x 2048 x 2048 51, 36, 39, 30, 38; 1024 x 2048 x 8192 56, 46, 81, 58, 77; 4096 x 2048 x 8192 142, 171, 313, 228, 286.
struct BackTile {
  int bm, bk;
  float once, round, alone, per256;
};
constexpr BackTile kTiles[] = {{256, 256, 0.f, 5.f, 8.4f, 8.4f}, {128, 256, 0.f, 7.f, 4.7f, 4.7f}, {64, 128, 0.f, 7.f, 1.6f, 1.6f},
                               {64, 128, 6.f, 0.f, 2.1f, 1.55f}, {32, 128, 5.5f, 0.f, 0.92f, 0.92f}};
int64_t tiles_of(const hrt_mx4_mm_args& a, int t) { return cdiv(a.M, kTiles[t].bm) * cdiv(a.K, kTiles[t].bk); }

int plan_of(const hrt_mx4_mm_args& a) {
  int best = 4;
  float us = 0.f;
  for (int t = 4; t >= 0; --t) {
    const BackTile& k = kTiles[t];
    const float rounds = (float)cdiv(tiles_of(a, t), 256), per = k.per256 * rounds > k.alone ? k.per256 * rounds : k.alone;
    const float e = k.once + rounds * k.round + per * (float)a.N / 256.f;
    if (t == 4 || e < us) best = t, us = e;
  }
  return best;
}

template <typename T, int BM, int BK, int WM, int KG, int R>
void queue_back(const hrt_mx4_mm_args& a, hipStream_t s) {
  const int64_t tm = cdiv(a.M, BM), tk = cdiv(a.K, BK);
  hipLaunchKernelGGL((mx4_back<T, BM, BK, WM, KG, R>), dim3((uint32_t)(tm * tk)), dim3(64 * BackShape<BM, BK, WM, KG>::NW), 0, s, a, (int)tk,
                     (int)cdiv(a.N, KG * kSlice));
}

template <typename T>
bool launch_mx4_back(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_mx4_mm_args*>(pp);
  if (a.M <= 0 || a.N <= 0 || a.K <= 0) return ctx.fail("empty product");
  if (a.K % kMxBlock != 0 || a.N % 8 != 0) return ctx.fail("K must be a multiple of 32 and N of 8");
  if (a.x_scale != 0 || a.bias != 0) return ctx.fail("takes 16-bit rows and no bias");
  if (a.x_sm < 0 || a.x_sm % 8 != 0) return ctx.fail("x's row stride must be a non-negative multiple of 8");
  if (a.x % 16 != 0 || a.w % 16 != 0 || a.y % 16 != 0) return ctx.fail("x, w and y must be 16-byte aligned");
  const int64_t nb = a.K / kMxBlock, xs[2] = {a.M, a.N}, xt[2] = {a.x_sm, 1};
  if (!ctx.check(a.x, hrt::span_bytes(2, xs, xt, 2), "x") || !ctx.check(a.w, (uint64_t)(a.N * (a.K / 2)), "w") ||
      !ctx.check(a.w_scale, (uint64_t)(a.N * nb), "w_scale") || !ctx.check(a.y, (uint64_t)(a.M * a.K) * 2, "y"))
    return false;
  // offsets of a stage's rows are 31-bit
  const int64_t lim = (int64_t)1 << 31;
  if (a.x_sm * 2 * 257 >= lim || a.K / 2 * 257 >= lim) return ctx.fail("operand rows too long for one launch");
  const int tile = plan_of(a);
  if (!hrt::grid_fits(tiles_of(a, tile), 512)) return ctx.fail("grid too large");
  switch (tile) {
    case 0: queue_back<T, 256, 256, 64, 1, 2>(a, ctx.stream); break;
    case 1: queue_back<T, 128, 256, 64, 2, 2>(a, ctx.stream); break;
    case 2: queue_back<T, 64, 128, 64, 4, 3>(a, ctx.stream); break;
    case 3: queue_back<T, 64, 128, 64, 2, 3>(a, ctx.stream); break;
    case 4: queue_back<T, 32, 128, 32, 4, 2>(a, ctx.stream); break;
  }
  return hrt::launch_ok(hipGetLastError(), ctx, "mx4_mm_back");
}

HRT_REGISTER("mx4_mm_back_bf16", hrt_mx4_mm_args, launch_mx4_back<BF16>);
HRT_REGISTER("mx4_mm_back_f16", hrt_mx4_mm_args, launch_mx4_back<F16>);

}  // namespace
}  // namespace hk
