// Fused attention with a learned relative position bias on gfx950 matrix cores: the kernel behind "attn_rel_{fwd,dq,dkdv}_{dt}",
// forward, dQ with the bias table's gradient, and dK/dV, for bf16, f16 and fp32 (one instance file each).
//
//   s = scale q k^T + table[bucket(j - i - off), h],  P = softmax over the keys that are not masked,  o = P v
//   dS = P (dO v^T - rowsum(o dO)),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T dO,
//   dtable[b, h] = sum of dS over the batch and over all pairs (i, j) in bucket b
//
// The bias depends on r = j - i - off alone and is constant from |r| = R on (R: where the last bucket of a direction begins),
// so nothing of size Sq x Sk exists anywhere:
//   * a workgroup spreads its head's table over an LDS array `band` of the distances -R - 63 .. R + 63.  A 32 x 32 tile whose
//     distances all lie beyond R on one side takes its bias as one scalar, folded into the softmax's subtraction; any other
//     tile reads the 16 values of each lane from the band (consecutive lanes, consecutive addresses) and hands them to its
//     first matrix instruction as the accumulator's start, so the bias costs no arithmetic.
//   * the table's gradient is the sum of dS along diagonals.  Tiles beyond R add their 16 values to one register per lane and
//     side.  Other tiles go through a 32 x 33 LDS patch: written by rows, read back along wrapped diagonals (lane t of a
//     half-wave meets diagonals t and t - 32), so that 16 writes and 16 reads per lane sum 63 diagonals, which are added to a
//     band array of the wavefront's own.  Every sum has a fixed order: no atomics, the same bits every run.
// Bound: in 16 bits the matrix cores and the softmax arithmetic between the two products, in fp32 the matrix cores and how the
// workgroups fall on the CUs.  Measured, forward / dQ and table / dK and dV:
// bf16, 128 heads of 2048 x 2048 x 64 215 / 309 / 326 us (638, 667, 844 TFLOP/s), 48 heads of 512 x 512 x 64 14 / 26 / 20;
// 128 heads of 2048 x 2048 x 128 360 / 574 / 934 us; f16, 8 heads of 4020 x 4020 x 128 causal 88 / 125 / 135; fp32, 16 heads of
// 1040 x 1040 x 64 73 / 144 / 168 (61, 46, 53 TFLOP/s of about 150).  128-wide dK/dV holds 224 accumulators and
// operands a lane, so one wavefront runs on a SIMD; 128-wide dQ of 16 bits fits two with one buffer a stage (729 us with two buffers
// and one workgroup on a CU, so 574; 8 heads of 4020 the same either way).
// Tiling: a workgroup's four wavefronts are G groups of 32 stationary rows (queries; keys for dK/dV) times KH = 4 / G, which
// share out the 32-row tiles of each streamed stage.  Stages are copied global -> LDS directly, double-buffered; rows that do
// not exist or whose key is masked are copied as zeros without reading memory (a masked infinity or NaN meets no product),
// stages and tiles without a single key to see are skipped.  The first product leaves a stationary row per lane, so that the
// softmax statistics are per lane and P and dS feed the second product from registers (attn_common.h, attn_f32_tile.h).
// 16-bit P and dS are rounded to the input type before the second product, as in the other fused kernels; sums, statistics
// and the table's gradient are fp32.  delta = rowsum(o dO) is one error for a whole row of dS, so o comes with what its rounding
// left (o_lo, a training forward's): f16, one head of 512 x 512 x 128 causal, these roundings alone put dk and dq off by 0.00029 of
// their norm, 0.00032 without o_lo (the gradients' own rounding 0.00021).  It costs 2 % of forward and backward.
#pragma once

#include <cmath>
#include <type_traits>

#include "../hrt/registry.h"
#include "attn_f32_tile.h"
#include "attn_rel_plan.h"

namespace hk {

template <typename T, int DP, int ST>
struct RelTile;

// 16-bit tiles: rows of DP / 8 swizzled chunks (lds_stage.h).
template <typename T, int DP, int ST>
struct RelTile16 {
  using frag = u32x4;
  static constexpr int ESZ = 2, NF = DP / 16, NCH = DP / 8, BYTES = ST * NCH * 16, DCH = DP / 32;
  __device__ __forceinline__ static void load(frag (&f)[NF], const HK_G uint8_t* row, bool ok, int D, int h) {
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const int d = 16 * i + 8 * h;
      f[i] = ok && d < D ? *reinterpret_cast<const HK_G u32x4*>(row + 2 * d) : u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ static float dot(const frag (&a)[NF], const frag (&b)[NF]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(hi16<T>(a[i][e]), hi16<T>(b[i][e]), fmaf(lo16<T>(a[i][e]), lo16<T>(b[i][e]), s));
    return s;
  }
  // rows r0 .. r0 + 31 times the stationary fragments, on top of `s`
  __device__ __forceinline__ static f32x16 rows(const HK_L uint8_t* t, int r0, const frag (&f)[NF], f32x16 s, int l32, int h) {
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const u32x4 a = *reinterpret_cast<const HK_L u32x4*>(t + r0 * NCH * 16 + tile_off<NCH>(l32, 2 * i + h));
      s = Mfma32<T>::mac(a, f[i], s);
    }
    return s;
  }
  __device__ __forceinline__ static void cols(f32x16 (&acc)[DCH], const HK_L uint8_t* t, int r0, const f32x16& p, int lane) {
    const u32x4 b[2] = {pack_slots<T>(p, 0, 1), pack_slots<T>(p, 2, 3)};
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), c = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    const HK_L uint8_t* const base = t + r0 * NCH * 16 + (lane & 1) * 8;
#pragma unroll
    for (int n = 0; n < DCH; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const u32x2 lo = lds_tr4(base + tile_off<NCH>(row, 4 * n + c) + k * 16 * NCH * 16);
        const u32x2 hi = lds_tr4(base + tile_off<NCH>(row + 8, 4 * n + c) + k * 16 * NCH * 16);
        acc[n] = Mfma32<T>::mac(u32x4{lo.x, lo.y, hi.x, hi.y}, b[k], acc[n]);
      }
  }
  // stage rows whose bit in w is set
  __device__ __forceinline__ static void copy(const HK_G uint8_t* base, uint32_t ss, int D, const uint64_t (&w)[2], HK_L uint8_t* t, int wave, int lane) {
    constexpr int IPW = BYTES / 1024 / 4, RPI = 64 / NCH;
    const __amdgpu_buffer_rsrc_t rs = edge_rsrc(base);
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int j = wave * IPW + i, row = j * RPI + lane / NCH, c = (lane % NCH) ^ tile_swz<NCH>(row);
      const bool ok = (((ST > 64 && row >= 64 ? w[1] : w[0]) >> (row & 63)) & 1) && c * 8 < D;
      edge_copy(rs, t, j, ok ? (uint32_t)row * ss + (uint32_t)c * 16 : kNoRow);
    }
  }
  __device__ __forceinline__ static void store(HK_G uint8_t* row, const f32x16& v, float mul, int n, int D, int h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = 32 * n + 8 * j + 4 * h;
      const float o[4] = {v[4 * j] * mul, v[4 * j + 1] * mul, v[4 * j + 2] * mul, v[4 * j + 3] * mul};
      if (d < D) *reinterpret_cast<HK_G u32x2*>(row + 2 * d) = pack4<T>(o);
    }
  }
  // what `store` of the same values leaves, a row like its own
  __device__ __forceinline__ static void store_left(HK_G uint8_t* row, const f32x16& v, float mul, int n, int D, int h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = 32 * n + 8 * j + 4 * h;
      float o[4], left[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = v[4 * j + e] * mul;
      const u32x2 w = pack4<T>(o);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float r = e & 1 ? hi16<T>(w[e >> 1]) : lo16<T>(w[e >> 1]);
        left[e] = fabsf(r) < INFINITY ? o[e] - r : 0.f;
      }
      if (d < D) *reinterpret_cast<HK_G u32x2*>(row + 2 * d) = pack4<T>(left);
    }
  }
};
template <int DP, int ST>
struct RelTile<BF16, DP, ST> : RelTile16<BF16, DP, ST> {};
template <int DP, int ST>
struct RelTile<F16, DP, ST> : RelTile16<F16, DP, ST> {};

template <int DP, int ST>
struct RelTile<F32, DP, ST> {
  using frag = f32x4;
  static constexpr int ESZ = 4, NF = DP / 8, NCH = DP / 4, BYTES = ST * DP * 4, DCH = DP / 32;
  __device__ __forceinline__ static void load(frag (&f)[NF], const HK_G uint8_t* row, bool ok, int D, int h) {
    load_frags<DP, true>(f, reinterpret_cast<const HK_G float*>(row), ok, D, h);
  }
  __device__ __forceinline__ static float dot(const frag (&a)[NF], const frag (&b)[NF]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(a[i][e], b[i][e], s);
    return s;
  }
  __device__ __forceinline__ static f32x16 rows(const HK_L uint8_t* t, int r0, const frag (&f)[NF], f32x16 s, int l32, int h) {
    return rows_times<DP>(t, r0, f, l32, h, s);
  }
  __device__ __forceinline__ static void cols(f32x16 (&acc)[DCH], const HK_L uint8_t* t, int r0, const f32x16& p, int lane) {
    cols_times<DP>(acc, t, r0, p, lane & 31, lane >> 5);
  }
  __device__ __forceinline__ static void copy(const HK_G uint8_t* base, uint32_t ss, int D, const uint64_t (&w)[2], HK_L uint8_t* t, int wave, int lane) {
    constexpr int IPW = BYTES / 1024 / 4;
    const __amdgpu_buffer_rsrc_t rs = edge_rsrc(base);
    asm volatile("" : "+v"(lane));  // keeps the lane offsets out of registers between stages
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int j = wave * IPW + i, ch = j * 64 + lane, row = ch / NCH, c = (ch % NCH) ^ f32_swz<NCH>(row);
      const bool ok = (((ST > 64 && row >= 64 ? w[1] : w[0]) >> (row & 63)) & 1) && c * 4 < D;
      edge_copy(rs, t, j, ok ? (uint32_t)row * ss + (uint32_t)c * 16 : kNoRow);
    }
  }
  __device__ __forceinline__ static void store(HK_G uint8_t* row, const f32x16& v, float mul, int n, int D, int h) {
    store_block<true>(reinterpret_cast<HK_G float*>(row), v, mul, n, D, h);
  }
};

// WHICH: 0 forward, 1 dK/dV, 2 dQ and the table's gradient
template <typename T, int WHICH, int DP, int G>
struct RelShape {
  static constexpr int KH = 4 / G;
  static constexpr int ST = rel_stage(std::is_same<T, F32>::value, DP, G);  // streamed rows per stage
  static constexpr int TPW = ST / 32 / KH;          // tiles of a stage per wavefront
  static constexpr int DCH = DP / 32, NACC = WHICH == 1 ? 2 * DCH : DCH;
  using Tile = RelTile<T, DP, ST>;
  static constexpr int TB = Tile::BYTES;
// one buffer a stage where it lets two workgroups share a CU: 128 fp32 rows, 128-wide dQ
  static constexpr int NBUF = (std::is_same<T, F32>::value ? G == 1 : WHICH == 2 && DP == 128 && G > 1) ? 1 : 2;
  // registers for two workgroups on a CU
  static constexpr bool TWO = DP == 64 || (G > 1 && (WHICH == 0 || (WHICH == 2 && !std::is_same<T, F32>::value)));
  static int lds(int R) { return rel_lds(WHICH, R); }
};

__device__ __forceinline__ uint64_t low_bits(int64_t n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

template <typename T, int WHICH, int DP, int G>
__global__ __launch_bounds__(256, (RelShape<T, WHICH, DP, G>::TWO ? 2 : 1)) void attn_rel_k(hrt_attn_rel_args p, RelBuckets bk, RelPlan pl) {
  using S = RelShape<T, WHICH, DP, G>;
  using Tile = typename S::Tile;
  using frag = typename Tile::frag;
  constexpr int KH = S::KH, ST = S::ST, NBUF = S::NBUF, TPW = S::TPW, DCH = S::DCH, NACC = S::NACC, TB = S::TB, ESZ = Tile::ESZ, NF = Tile::NF;
  // one LDS object per buffer: the compiler then knows that reads of one do not wait for the copies into the other
  __shared__ __attribute__((aligned(1024))) uint8_t a0_raw[TB], a1_raw[NBUF > 1 ? TB : 16], b0_raw[TB], b1_raw[NBUF > 1 ? TB : 16];
  __shared__ float stat[2][2][WHICH == 1 ? ST : 1];  // dK/dV: lse (log2 units) and delta of the streamed rows, per buffer
  __shared__ float ml[3][64][2];                     // the merge's maxima and sums; dQ: sums beyond R
  __shared__ int border[WHICH == 2 ? 256 : 1];       // dQ: the buckets' borders
  extern __shared__ float dyn[];
  auto abuf = [&](auto ic) { return (HK_L uint8_t*)(decltype(ic)::value ? a1_raw : a0_raw); };
  auto bbuf = [&](auto ic) { return (HK_L uint8_t*)(decltype(ic)::value ? b1_raw : b0_raw); };

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = wave % G, kh = wave / G, l32 = lane & 31, h = lane >> 5;
  uint32_t bh, blk, total = (uint32_t)pl.nblk * p.B * p.H, id = blockIdx.x, split = 0;
  if constexpr (WHICH == 1) {
    if (id < (uint32_t)pl.table) {
      rel_table<T>(p, pl.parts, (int64_t)id * 4 + wave, lane);
      return;
    }
    id -= (uint32_t)pl.table;
  }
  if (WHICH == 0 && pl.splits > 1) split = id / total, id -= split * total;
  // causal, and all workgroups resident two to a CU: the second ones in the other order, long beside short (2 x 12 heads of 1000 x
  // 1000 x 64: 86 us forward and backward, so 80)
  if (S::TWO && p.causal && pl.splits <= 1 && total % 8 == 0 && total > 256 && total <= 512 && id >= 256)
    id = id % 8 + (total - 8) - (id - 256) / 8 * 8;
  xcd_map32(id, total, pl.nblk, bh, blk);
  if (WHICH != 1 && p.causal) blk = pl.nblk - 1 - blk;  // the longest rows first
  bh = __builtin_amdgcn_readfirstlane(bh), blk = __builtin_amdgcn_readfirstlane(blk), split = __builtin_amdgcn_readfirstlane(split);
  const int64_t b = bh / (uint32_t)p.H, hh = bh % (uint32_t)p.H;
  const int D = p.D, R = bk.R;
  const int64_t Sq = p.Sq, Sk = p.Sk, off = p.q_off;
  // streamed rows: all queries; the keys, where causal up to the last one that any query sees (one past it would meet a P of zero in a
  // product, and zero times an infinity or NaN of a cache that nothing was written to is no zero)
  const int64_t seen = p.causal && off < Sk - Sq ? (Sq + off > 0 ? Sq + off : 0) : Sk;
  const int64_t own_n = WHICH == 1 ? Sk : Sq, str_n = WHICH == 1 ? Sq : seen;
  const int64_t own0 = (int64_t)blk * (32 * G), grp0 = own0 + 32 * g, own = grp0 + l32;  // this lane's stationary row
  const HK_G uint8_t* Q = gcptr<uint8_t>(p.q) + (b * p.q_sb + hh * p.q_sh) * ESZ;
  const HK_G uint8_t* K = gcptr<uint8_t>(p.k) + (b * p.k_sb + hh * p.k_sh) * ESZ;
  const HK_G uint8_t* V = gcptr<uint8_t>(p.v) + (b * p.v_sb + hh * p.v_sh) * ESZ;
  const HK_G uint8_t* dO = gcptr<uint8_t>(p.dout) + (b * p.do_sb + hh * p.do_sh) * ESZ;
  const HK_G uint8_t* mask = gcptr<uint8_t>(p.mask) + b * p.mask_sb;
  const HK_G typename T::storage* table = gcptr<typename T::storage>(p.table) + hh;
  const HK_G uint8_t* T0 = WHICH == 1 ? Q : K;  // streamed: K and V, or Q and dO
  const HK_G uint8_t* T1 = WHICH == 1 ? dO : V;
  const uint32_t s0 = (uint32_t)((WHICH == 1 ? p.q_ss : p.k_ss) * ESZ), s1 = (uint32_t)((WHICH == 1 ? p.do_ss : p.v_ss) * ESZ);
  const float sl2 = p.scale * kLog2e;

  // the range of stages that can hold an allowed pair, then this split's share of it
  int64_t st0 = 0, st1 = (str_n + ST - 1) / ST;
  if (p.causal) {  // key <= query + off
    if (WHICH == 1) {
      const int64_t first = own0 - off;
      st0 = first > 0 ? first / ST : 0;
    } else {
      const int64_t last = (own0 + 32 * G < Sq ? own0 + 32 * G : Sq) - 1 + off;
      const int64_t n = last < 0 ? 0 : last / ST + 1;
      st1 = n < st1 ? n : st1;
    }
  }
  if (WHICH == 0 && pl.splits > 1) {
    st0 = (int64_t)split * pl.per;
    st1 = st0 + pl.per < st1 ? st0 + pl.per : st1;
  }

  // a stage's rows: bit set where the row exists and (a key) is not masked, (a query) has a key by causal
  constexpr bool KEYS = WHICH != 1;
  const bool masked = p.mask != 0;
  uint8_t mb0 = 0, mb1 = 0;
  auto mask_load = [&](int64_t st) {
    if (KEYS && masked) {
      const int64_t k0 = st * ST + lane, k1 = k0 + 64;
      mb0 = k0 < str_n ? mask[k0] : 0;
      if (ST > 64) mb1 = k1 < str_n ? mask[k1] : 0;
    }
  };
  auto stage_rows = [&](int64_t st, uint64_t (&w)[2]) {
    if (KEYS && masked) {
      w[0] = __ballot(mb0 != 0), w[1] = ST > 64 ? __ballot(mb1 != 0) : 0;
    } else {
      w[0] = low_bits(str_n - st * ST), w[1] = ST > 64 ? low_bits(str_n - st * ST - 64) : 0;
      if (!KEYS && p.causal) {  // what stands in Q and dO before the first key may be no number either
        w[0] &= ~low_bits(-off - st * ST);
        if (ST > 64) w[1] &= ~low_bits(-off - st * ST - 64);
      }
    }
  };
  auto copy = [&](auto ic, int64_t st, const uint64_t (&w)[2]) {
    if ((w[0] | w[1]) == 0) return;
    Tile::copy(T0 + st * ST * (int64_t)s0, s0, D, w, abuf(ic), wave, lane);
    Tile::copy(T1 + st * ST * (int64_t)s1, s1, D, w, bbuf(ic), wave, lane);
    if constexpr (WHICH == 1) {
      if (tid < ST) {  // rows without a key (lse -inf) and rows past the end: P = exp2(-inf) = 0
        const int64_t q = st * ST + tid;
        float l = q < Sq ? gcptr<float>(p.lse)[(int64_t)bh * Sq + q] * kLog2e : INFINITY;
        stat[decltype(ic)::value][0][tid] = l == -INFINITY ? INFINITY : l;
        stat[decltype(ic)::value][1][tid] = q < Sq ? gcptr<float>(p.delta)[(int64_t)bh * Sq + q] : 0.f;
      }
    }
  };

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  uint64_t w[2] = {0, 0}, wn[2] = {0, 0};
  if (st0 < st1) {
    mask_load(st0);
    stage_rows(st0, w);
    copy(I0(), st0, w);
    mask_load(st0 + 1);
  }

  // the stationary rows
  bool own_ok = own < own_n;
  if (WHICH == 1 && masked) own_ok = own_ok && mask[own < Sk ? own : Sk - 1] != 0;
  frag f0[NF], f1[WHICH == 0 ? 1 : NF];  // Q; Q, dO; K, V
  Tile::load(f0, WHICH == 1 ? K + own * p.k_ss * ESZ : Q + own * p.q_ss * ESZ, own_ok, D, h);
  if constexpr (WHICH != 0) Tile::load(f1, WHICH == 1 ? V + own * p.v_ss * ESZ : dO + own * p.do_ss * ESZ, own_ok, D, h);
  float lse2 = 0.f, dlt = 0.f;
  if constexpr (WHICH == 2) {
    frag o[NF];  // delta = rowsum(o dO), from the stored o and what its rounding left
    const int64_t at = ((b * Sq + own) * p.H + hh) * D * ESZ;
    Tile::load(o, gcptr<uint8_t>(p.o) + at, own_ok, D, h);
    dlt = Tile::dot(o, f1);
    if (ESZ == 2 && p.o_lo) {
      Tile::load(o, gcptr<uint8_t>(p.o_lo) + at, own_ok, D, h);
      dlt += Tile::dot(o, f1);
    }
    dlt = halfswap_sum(dlt);
    lse2 = own_ok ? gcptr<float>(p.lse)[(int64_t)bh * Sq + own] * kLog2e : INFINITY;
    if (lse2 == -INFINITY) lse2 = INFINITY;
    if (own_ok && kh == 0 && h == 0) gptr<float>(p.delta)[(int64_t)bh * Sq + own] = dlt;
  }

  // the head's bias by distance, divided by the scale (it starts the logits' accumulator)
  float* const band = dyn;
  const int NB = 2 * R + 1 + 2 * kRelMargin, mid = R + kRelMargin;
  float* const sums = dyn + NB * (1 + wave);                      // dQ: this wavefront's sums by distance
  float* const patch = dyn + NB * 5 + wave * (32 * 33);           // dQ: its patch
  const float inv_scale = 1.f / p.scale;
  for (int t = tid; t < NB; t += 256) {
    const int r = t - mid, n = r < 0 ? -r : r;
    const int k = rel_bucket(bk, n);
    // one direction: positive distances are masked, and their values not used
    band[t] = r > 0 && bk.sides == 1 ? 0.f : T::to_f32(table[(int64_t)(r > 0 ? bk.nb + k : k) * p.H]) * inv_scale;
  }
  if constexpr (WHICH == 2) {
    if (p.dtable) {
      for (int t = lane; t < NB; t += 64) sums[t] = 0.f;
      int from = 0;
      for (int i = 0; i < bk.nb; i += 16)
#pragma unroll
        for (int j = 0; j < 16; ++j) from = tid == i + j ? bk.start[i + j] : from;
      border[tid] = from;
    }
  }
  const float far_lo = T::to_f32(table[(int64_t)(bk.nb - 1) * p.H]) * kLog2e;
  const float far_hi = bk.sides == 2 ? T::to_f32(table[(int64_t)(bk.total - 1) * p.H]) * kLog2e : 0.f;

  f32x16 acc[NACC > DCH ? 2 : 1][DCH];
#pragma unroll
  for (auto& a : acc)
#pragma unroll
    for (int n = 0; n < DCH; ++n) a[n] = zero16();
  float m = -INFINITY, l = 0.f;              // forward: running max in log2 units, sum
  float beyond_lo = 0.f, beyond_hi = 0.f;    // dQ: dS of tiles beyond R

  // tile r0 .. r0 + 31 of stage st; bits: its rows that exist and are not masked
  auto tile = [&](auto ic, int64_t st, int r0, uint32_t bits) {
    const int64_t str0 = st * ST + r0;
    const int64_t rb = WHICH == 1 ? grp0 - str0 - off : str0 - grp0 - off;  // distance at (row 0, lane 0)
    if (p.causal && rb - 31 > 0) return;                                    // every pair in the future
    const bool beyond = rb - 31 >= R || rb + 31 <= -R, all = !(p.causal && rb + 31 > 0) && bits == ~0u;
    const float c2 = beyond ? (rb > 0 ? far_hi : far_lo) : 0.f;
    f32x16 s;
    if (beyond) {
      s = zero16();
    } else {
      const int at = (int)rb + mid + (WHICH == 1 ? l32 - 4 * h : 4 * h - l32);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = band[WHICH == 1 ? at - (8 * (e >> 2) + (e & 3)) : at + 8 * (e >> 2) + (e & 3)];
    }
    const HK_L uint8_t* const t0 = abuf(ic);
    const HK_L uint8_t* const t1 = bbuf(ic);
    s = Tile::rows(t0, r0, f0, s, l32, h);
    // element e is an allowed pair: its row's bit, and key <= query + off
    const uint32_t mybits = bits >> (4 * h);
    const int lim = WHICH == 1 ? (rb + 31 < 0 ? 0 : (int)rb + l32 - 4 * h)             // row >= lim
                               : (rb + 31 < 0 ? 31 : l32 - (int)rb - 4 * h);           // row <= lim
    auto allowed = [&](int e) {
      const int row = 8 * (e >> 2) + (e & 3);
      return ((mybits >> row) & 1u) != 0 && !(p.causal && (WHICH == 1 ? row < lim : row > lim));
    };
    if constexpr (WHICH == 0) {
      if (!all) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = allowed(e) ? s[e] : -INFINITY;
      }
      float mx = fmaxf(s[0], s[1]);
#pragma unroll
      for (int e = 2; e < 16; ++e) mx = fmaxf(mx, s[e]);
      const float cand = fmaf(halfswap_max(mx), sl2, c2);  // scale > 0: max commutes with the scaling
      // the running max moves only when a row exceeds it by 2^8: P stays below 2^8, far inside every type's range
      const bool up = cand > m + 8.f;
      if (__any(up)) {
        const float mn = up ? cand : m, alpha = up ? __builtin_amdgcn_exp2f(m - mn) : 1.f;  // m = -inf: 0, and l, o are 0
        l *= alpha;
#pragma unroll
        for (int n = 0; n < DCH; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[0][n][e] *= alpha;
        m = mn;
      }
      const float nm = m == -INFINITY ? c2 : c2 - m;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], sl2, nm));
        l += s[e];
      }
      Tile::cols(acc[0], t1, r0, s, lane);
    } else {
      f32x16 dp;
      if constexpr (WHICH == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(&stat[decltype(ic)::value][1][r0 + 8 * j + 4 * h]);
#pragma unroll
          for (int r = 0; r < 4; ++r) dp[4 * j + r] = -d4[r];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = -dlt;
      }
      dp = Tile::rows(t1, r0, f1, dp, l32, h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 ls;
        if constexpr (WHICH == 1) ls = *reinterpret_cast<const f32x4*>(&stat[decltype(ic)::value][0][r0 + 8 * j + 4 * h]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 4 * j + r;
          s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], sl2, c2 - (WHICH == 1 ? ls[r] : lse2)));
        }
      }
      if (!all) {  // selected, not multiplied: what stands at a masked pair may be no number
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = allowed(e) ? s[e] : 0.f, dp[e] = allowed(e) ? dp[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] *= s[e];
      if constexpr (WHICH == 1) {
        Tile::cols(acc[0], t0, r0, dp, lane);                        // dK^T += Q^T dS
        Tile::cols(acc[NACC > DCH ? 1 : 0], t1, r0, s, lane);        // dV^T += dO^T P
      } else {
        if (p.dtable) {
          if (beyond) {
            float t = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) t += dp[e];
            (rb > 0 ? beyond_hi : beyond_lo) += t;
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) patch[(8 * (e >> 2) + 4 * h + (e & 3)) * 33 + l32] = dp[e];
            // half-wave h takes columns 16 h .. + 15 of wrapped diagonal l32: row (l32 + column) mod 32, which is diagonal
            // l32 (row - column) before the wrap and l32 - 32 after it
            float over = 0.f, under = 0.f;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const int col = 16 * h + c, row = (l32 + col) & 31;
              const float x = patch[row * 33 + col];
              if (l32 + col < 32) over += x;
              else under += x;
            }
            over = halfswap_sum(over), under = halfswap_sum(under);
            const int at = (int)rb + mid;  // distance of diagonal 0
            if (h == 0) sums[at + l32] += over;
            else if (l32 > 0) sums[at + l32 - 32] += under;
          }
        }
        Tile::cols(acc[0], t0, r0, dp, lane);  // dQ^T += K^T dS^T
      }
    }
  };

  auto stage = [&](auto ic, int64_t st) {
    // stage st's copies are complete everywhere (and its mask, and the table's band); the other buffer is free
    barrier_keep_vm_lds<0>();
    auto following = [&](auto other) {
      if (st + 1 < st1) {
        stage_rows(st + 1, wn);
        copy(other, st + 1, wn);
        mask_load(st + 2);
      }
    };
    if constexpr (NBUF > 1) following(std::integral_constant<int, 1 - decltype(ic)::value>());
#pragma unroll
    for (int u = 0; u < TPW; ++u) {
      const int r0 = 32 * (kh + u * KH);
      const uint32_t bits = (uint32_t)((r0 >= 64 ? w[1] : w[0]) >> (r0 & 63));
      if (bits) tile(ic, st, r0, bits);
    }
    if constexpr (NBUF == 1) {
      if (st + 1 < st1) barrier_keep_vm_lds<0>();  // every wavefront is done with the stage
      following(ic);
    }
    w[0] = wn[0], w[1] = wn[1];
  };
  int64_t st = st0;
  if constexpr (NBUF > 1) {
    for (; st + 2 <= st1; st += 2) {
      stage(I0(), st);
      stage(I1(), st + 1);
    }
    if (st < st1) stage(I0(), st);
  } else {
    for (; st < st1; ++st) stage(I0(), st);
  }

  // ---- merge the KH partial results of each group into the wavefront kh = 0, in order, through the tiles' memory
  __syncthreads();
  if constexpr (WHICH == 0) {
    float mt = m;
    if constexpr (KH > 1) {
      const int slot = g * (KH - 1) + kh - 1;
      if (kh > 0) ml[slot][lane][0] = m, ml[slot][lane][1] = l;
      __syncthreads();
      if (kh == 0) {
#pragma unroll
        for (int k = 0; k < KH - 1; ++k) mt = fmaxf(mt, ml[g * (KH - 1) + k][lane][0]);
      }
    }
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mt);  // kh > 0: 1
    if (kh == 0) {
      l *= a;
#pragma unroll
      for (int n = 0; n < DCH; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[0][n][e] *= a;
      m = mt;
    }
  }
  if constexpr (KH > 1) {
    constexpr int CH = TB / 4096 < NACC ? TB / 4096 : NACC;  // accumulators per round: 4 KiB each
    static_assert(CH >= 1 && NACC % CH == 0 && (NBUF > 1 || KH == 2 || 2 * NACC * 4096 <= TB), "merge rounds");
    auto piece = [&](int s) { return (float*)(s == 0 ? a0_raw : s == 2 ? b0_raw : NBUF > 1 ? a1_raw : KH == 2 ? b0_raw : a0_raw + NACC * 4096); };
#pragma unroll
    for (int r = 0; r < NACC; r += CH) {
      if (r > 0) __syncthreads();
      if (kh > 0) {
        float* const mine = piece(g * (KH - 1) + kh - 1);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) mine[(c * 16 + e) * 64 + lane] = acc[(r + c) / DCH][(r + c) % DCH][e];
      }
      __syncthreads();
      if (kh == 0) {
#pragma unroll
        for (int k = 0; k < KH - 1; ++k) {
          const float* const part = piece(g * (KH - 1) + k);
          float f = 1.f;
          if constexpr (WHICH == 0) {
            const float mk = ml[g * (KH - 1) + k][lane][0];
            f = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - m);
            if (r == 0) l += f * ml[g * (KH - 1) + k][lane][1];
          }
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[(r + c) / DCH][(r + c) % DCH][e] = fmaf(f, part[(c * 16 + e) * 64 + lane], acc[(r + c) / DCH][(r + c) % DCH][e]);
        }
      }
    }
  }

  if constexpr (WHICH == 2) {  // this workgroup's sums by bucket
    if (p.dtable) {
      const float lo = wave_sum(beyond_lo), hi = wave_sum(beyond_hi);
      __syncthreads();
      if (lane == 0) ml[0][wave][0] = lo, ml[0][wave][1] = hi;
      for (int t = tid; t < NB; t += 256) band[t] = (dyn[NB + t] + dyn[2 * NB + t]) + (dyn[3 * NB + t] + dyn[4 * NB + t]);
      __syncthreads();
      // partial sums [H][B][nblk][buckets]; eight lanes a bucket
      HK_G float* const out = gptr<float>(p.ws) + ((hh * p.B + b) * pl.nblk + blk) * (int64_t)bk.total;
      for (int k = tid >> 3; k < bk.total; k += 32) {
        const bool pos = k >= bk.nb;
        const int j = pos ? k - bk.nb : k;
        const int from = border[j], to = j + 1 < bk.nb ? border[j + 1] : mid + 1;
        float t = 0.f;
        for (int n = from + (tid & 7); n < to; n += 8)
          if (!(pos && n == 0)) t += band[pos ? mid + n : mid - n];
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) t += __shfl_xor(t, x, 64);
        if (j + 1 == bk.nb) t += (ml[0][0][pos] + ml[0][1][pos]) + (ml[0][2][pos] + ml[0][3][pos]);
        if ((tid & 7) == 0) out[k] = t;
      }
    }
  }

  if (kh > 0 || own >= own_n) return;
  if constexpr (WHICH == 0) {
    const float lrow = halfswap_sum(l);
    const int64_t row = (int64_t)bh * Sq + own;
    if (pl.splits > 1) {  // partial sums of this key range: [split][row][D], then [split][row][max, sum]
      const int64_t rows = (int64_t)p.B * p.H * Sq;
      HK_G float* const o = gptr<float>(p.ws) + (split * rows + row) * D;
      HK_G float* const s = gptr<float>(p.ws) + pl.splits * rows * D + (split * rows + row) * 2;
#pragma unroll
      for (int n = 0; n < DCH; ++n) store_block<true>(o, acc[0][n], 1.f, n, D, h);
      if (h == 0) s[0] = m, s[1] = lrow;
      return;
    }
    const float inv = lrow > 0.f ? 1.f / lrow : 0.f;  // no key: zeros
    if (h == 0) gptr<float>(p.lse)[row] = lrow > 0.f ? (m + log2f(lrow)) * kLn2 : -INFINITY;
    const int64_t at = ((b * Sq + own) * p.H + hh) * D * ESZ;
#pragma unroll
    for (int n = 0; n < DCH; ++n) Tile::store(gptr<uint8_t>(p.o) + at, acc[0][n], inv, n, D, h);
    if constexpr (ESZ == 2) {
      if (p.o_lo) {
#pragma unroll
        for (int n = 0; n < DCH; ++n) Tile::store_left(gptr<uint8_t>(p.o_lo) + at, acc[0][n], inv, n, D, h);
      }
    }
  } else {
    const bool like = (p.flags & HRT_ATTN_GRAD_LIKE_INPUT) != 0;
    auto row_of = [&](uint64_t base, int64_t sb, int64_t sh, int64_t ss, int64_t n) {
      return gptr<uint8_t>(base) + (like ? b * sb + hh * sh + own * ss : ((b * n + own) * p.H + hh) * D) * ESZ;
    };
    if constexpr (WHICH == 1) {
      HK_G uint8_t* const dk = row_of(p.dk, p.k_sb, p.k_sh, p.k_ss, Sk);
      HK_G uint8_t* const dv = row_of(p.dv, p.v_sb, p.v_sh, p.v_ss, Sk);
#pragma unroll
      for (int n = 0; n < DCH; ++n) {
        f32x16 a = acc[0][n], c = acc[NACC > DCH ? 1 : 0][n];
        if (!own_ok) a = zero16(), c = zero16();  // a masked key: its lane saw a row of zeros, and P of any size
        Tile::store(dk, a, p.scale, n, D, h);
        Tile::store(dv, c, 1.f, n, D, h);
      }
    } else {
      if (!p.dq) return;
      HK_G uint8_t* const dq = row_of(p.dq, p.q_sb, p.q_sh, p.q_ss, Sq);
#pragma unroll
      for (int n = 0; n < DCH; ++n) Tile::store(dq, acc[0][n], p.scale, n, D, h);
    }
  }
}

template <typename T, int WHICH, int DP, int G>
void attn_rel_go(const hrt_attn_rel_args& a, const RelBuckets& bk, const RelPlan& pl, hipStream_t s) {
  const uint32_t grid = (uint32_t)((int64_t)pl.nblk * a.B * a.H * pl.splits + pl.table);
  hipLaunchKernelGGL((attn_rel_k<T, WHICH, DP, G>), dim3(grid), dim3(256), (RelShape<T, WHICH, DP, G>::lds(bk.R)), s, a, bk, pl);
}

template <typename T, int WHICH, int DP>
void attn_rel_g(const hrt_attn_rel_args& a, const RelBuckets& bk, const RelPlan& pl, hipStream_t s) {
  if (pl.g == 4) attn_rel_go<T, WHICH, DP, 4>(a, bk, pl, s);
  if constexpr (!std::is_same<T, F32>::value || DP == 64)
    if (pl.g == 2) attn_rel_go<T, WHICH, DP, 2>(a, bk, pl, s);
  if constexpr (!std::is_same<T, F32>::value || DP == 64)
    if (pl.g == 1) attn_rel_go<T, WHICH, DP, 1>(a, bk, pl, s);
}

// Instantiated once per type.
template <typename T>
void attn_rel_queue(const hrt_attn_rel_args& a, int which, const RelBuckets& bk, const RelPlan& pl, hipStream_t s) {
  if (a.D <= 64) {
    if (which == 0) attn_rel_g<T, 0, 64>(a, bk, pl, s);
    else if (which == 1) attn_rel_g<T, 1, 64>(a, bk, pl, s);
    else attn_rel_g<T, 2, 64>(a, bk, pl, s);
  } else {
    if (which == 0) attn_rel_g<T, 0, 128>(a, bk, pl, s);
    else if (which == 1) attn_rel_g<T, 1, 128>(a, bk, pl, s);
    else attn_rel_g<T, 2, 128>(a, bk, pl, s);
  }
}

}  // namespace hk
