// "rotary_{f32,bf16,f16}": queries and keys turned by positions of several axes.
//
// Bound by memory: every value is read once and written once.  The sines and cosines depend on the token and the pair alone, so a
// workgroup takes all heads of a few tokens, computes each of them once into LDS and its lanes keep theirs in registers over
// the heads.  Far positions: the angle is reduced to an eighth of a turn in fp64 (position times frequency in 53 bits) before its
// sine and cosine are taken in fp32, which leaves them within 2^-22 + |angle| 2^-51: up to 2^29 radians the fp32 steps are the larger part.  Measured, bf16, 16 + 16 heads of 128: 2 x 4096 tokens 25 us
// by the kernel trace (26.6 with four tokens to a workgroup), 22.4 replayed on the same operands, 26.5 on operands from HBM (134 MB, 5.1 TB/s); 8 tokens
// 3.7 us.  Few heads leave threads idle: 16384 tokens of 4 + 4 heads of 64, 32 threads of 256, 15.6 us (18.3 from HBM, 1.8 TB/s), of 8 + 4 heads
// of 128 21.9 (27.8, 3.6 TB/s).
#include "../hrt/registry.h"
#include "row_vec.h"

namespace hk {
namespace {

// cos and sin of `turns` full turns.
__device__ __forceinline__ void turn_of(double turns, float& c, float& s) {
  const double quarter = rint(turns * 4.0);
  const float rest = (float)((turns - quarter * 0.25) * 2.0);  // in half turns, |rest| <= 1/4
  float cr, sr;
  sincospif(rest, &sr, &cr);
  const int k = (int)(quarter - 4.0 * floor(quarter * 0.25));
  c = k == 0 ? cr : k == 1 ? -sr : k == 2 ? -cr : sr;
  s = k == 0 ? sr : k == 1 ? cr : k == 2 ? -sr : -cr;
}

// W values at a time: 16 bytes or 8, or one where the pairs do not fill such pieces.
template <typename T, int W>
struct Piece {
  using S = typename T::storage;
  __device__ __forceinline__ static void get(const HK_G S* p, float* v) {
    if constexpr (W == RowVec<T>::V) {
      RowVec<T>::unpack(RowVec<T>::get(p), v);
    } else if constexpr (W == 4) {
      typedef u32x2 __attribute__((aligned(2))) any;
      const u32x2 w = *reinterpret_cast<const HK_G any*>(p);
      v[0] = lo16<T>(w.x), v[1] = hi16<T>(w.x), v[2] = lo16<T>(w.y), v[3] = hi16<T>(w.y);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = T::to_f32(p[e]);
    }
  }
  __device__ __forceinline__ static void put(HK_G S* p, const float* v) {
    if constexpr (W == RowVec<T>::V) {
      RowVec<T>::put(p, RowVec<T>::pack(v));
    } else if constexpr (W == 4) {
      typedef u32x2 __attribute__((aligned(2))) any;
      *reinterpret_cast<HK_G any*>(p) = pack4<T>(v);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) p[e] = T::from_f32(v[e]);
    }
  }
};

// A head has `turned` pieces of W pairs, two stretches of W values each (W and W apart by P, or 2 W neighbours), and behind them
// `plain` pieces of W values that are copied.  Thread i of a workgroup has piece i % m of head i / m, m = turned + plain, and of every
// `step`th head from there on; step * m of the 256 work.  m > 256: pieces in rounds.
template <typename T, int W, bool IL>
__global__ __launch_bounds__(256) void rotary(hrt_rotary_args p, int tokens, int m, int step) {
  using S = typename T::storage;
  extern __shared__ float cs[];  // [tokens][2][P]
  const uint32_t t0 = blockIdx.x * (uint32_t)tokens, all = (uint32_t)(p.B * p.S);  // B S < 2^31
  const int n = all - t0 < (uint32_t)tokens ? (int)(all - t0) : tokens;
  for (int i = threadIdx.x; i < n * p.P; i += 256) {
    const int t = i / p.P, j = i - t * p.P;
    const uint32_t b = (t0 + t) / (uint32_t)p.S, s = t0 + t - b * (uint32_t)p.S;
    int a = 0;
#pragma unroll
    for (int i = 0; i + 1 < HRT_ROTARY_AXES; ++i)
      if (i + 1 < p.axes && j >= p.ends[i]) a = i + 1;
    const int64_t at = (int64_t)b * p.p_sb + (int64_t)s * p.p_ss + a * p.p_sa;
    const double pos = p.pos_type == 0 ? (double)gcptr<int32_t>(p.pos)[at] : p.pos_type == 1 ? (double)gcptr<int64_t>(p.pos)[at] : (double)gcptr<float>(p.pos)[at];
    float c, sn;
    turn_of(pos * (gcptr<double>(p.freqs)[j] * 0.15915494309189533577), c, sn);
    cs[t * 2 * p.P + j] = c;
    cs[t * 2 * p.P + p.P + j] = p.back ? -sn : sn;
  }
  __syncthreads();
  const int heads = p.Hq + p.Hk, pairs = p.P / W;
  for (int piece = m <= 256 ? threadIdx.x % m : threadIdx.x; piece < m; piece += m <= 256 ? m : 256) {
    const int h0 = m <= 256 ? threadIdx.x / m : 0;
    if (h0 >= step) return;
    const bool turned = piece < pairs;
    const int one = turned ? (IL ? 2 * W * piece : W * piece) : 2 * p.P + W * (piece - pairs), two = IL ? one + W : one + p.P;
    for (int t = 0; t < n; ++t) {
      const uint32_t b = (t0 + t) / (uint32_t)p.S, s = t0 + t - b * (uint32_t)p.S;
      float c[W], sn[W];
      if (turned) {
#pragma unroll
        for (int e = 0; e < W; ++e) c[e] = cs[t * 2 * p.P + W * piece + e], sn[e] = cs[t * 2 * p.P + p.P + W * piece + e];
      }
      for (int h = h0; h < heads; h += step) {
        const bool isq = h < p.Hq;
        const int hh = isq ? h : h - p.Hq;
        const HK_G S* const x = gcptr<S>(isq ? p.q : p.k) + b * (isq ? p.qs[0] : p.ks[0]) + hh * (isq ? p.qs[1] : p.ks[1]) + s * (isq ? p.qs[2] : p.ks[2]);
        HK_G S* const y = gptr<S>(isq ? p.q_out : p.k_out) + ((int64_t)(t0 + t) * (isq ? p.Hq : p.Hk) + hh) * p.D;
        float u[W], v[W], ou[W], ov[W];
        Piece<T, W>::get(x + one, u);
        if (!turned) {
          Piece<T, W>::put(y + one, u);
          continue;
        }
        Piece<T, W>::get(x + two, v);
        if constexpr (IL) {
#pragma unroll
          for (int e = 0; e < W; ++e) {  // pair e of 2 W neighbours
            const float a = 2 * e < W ? u[2 * e % W] : v[2 * e % W], bb = 2 * e + 1 < W ? u[(2 * e + 1) % W] : v[(2 * e + 1) % W];
            const float ta = a * c[e] - bb * sn[e], tb = bb * c[e] + a * sn[e];
            if (2 * e < W) ou[2 * e % W] = ta;
            else ov[2 * e % W] = ta;
            if (2 * e + 1 < W) ou[(2 * e + 1) % W] = tb;
            else ov[(2 * e + 1) % W] = tb;
          }
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e) ou[e] = u[e] * c[e] - v[e] * sn[e], ov[e] = v[e] * c[e] + u[e] * sn[e];
        }
        Piece<T, W>::put(y + one, ou);
        Piece<T, W>::put(y + two, ov);
      }
    }
  }
}

template <typename T, int W>
void queue_rotary(const hrt_rotary_args& a, int tokens, hipStream_t s) {
  const int m = a.P / W + (a.D - 2 * a.P) / W, step = m <= 256 ? 256 / m : 1;
  const dim3 grid((uint32_t)cdiv(a.B * a.S, tokens));
  const size_t lds = (size_t)tokens * 2 * a.P * 4;
  if (a.interleaved) hipLaunchKernelGGL((rotary<T, W, true>), grid, dim3(256), lds, s, a, tokens, m, step);
  else hipLaunchKernelGGL((rotary<T, W, false>), grid, dim3(256), lds, s, a, tokens, m, step);
}

template <typename T>
bool launch_rotary(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_rotary_args*>(pp);
  using S = typename T::storage;
  constexpr uint64_t E = sizeof(S);
  constexpr int V = RowVec<T>::V;
  if (a.B <= 0 || a.S <= 0 || a.Hq <= 0 || a.Hk < 0 || (a.Hk > 0) != (a.k != 0) || a.Hq > 65536 || a.Hk > 65536) return ctx.fail("bad shape");
  if (a.D <= 0 || a.D > 1024 || a.P <= 0 || 2 * a.P > a.D) return ctx.fail("D must be 1..1024 and pairs must fit it");
  if (a.axes < 1 || a.axes > HRT_ROTARY_AXES || a.ends[a.axes - 1] != a.P) return ctx.fail("bad axes");
  for (int i = 0; i < a.axes; ++i)
    if (a.ends[i] < (i ? a.ends[i - 1] : 0)) return ctx.fail("bad axes");
  if (a.pos_type < 0 || a.pos_type > 2) return ctx.fail("bad type of positions");
  const uint64_t pe = a.pos_type == 1 ? 8 : 4;
  if (a.q % E || a.k % E || a.q_out % E || a.k_out % E || a.pos % pe || a.freqs % 8) return ctx.fail("operands must be aligned to their elements");
  for (int i = 0; i < 3; ++i)
    if (a.qs[i] < 0 || a.ks[i] < 0) return ctx.fail("negative stride");
  if (a.p_sb < 0 || a.p_ss < 0 || a.p_sa < 0) return ctx.fail("negative stride");
  const int64_t qz[4] = {a.B, a.Hq, a.S, a.D}, kz[4] = {a.B, a.Hk, a.S, a.D}, qt[4] = {a.qs[0], a.qs[1], a.qs[2], 1}, kt[4] = {a.ks[0], a.ks[1], a.ks[2], 1};
  const int64_t pz[3] = {a.B, a.S, a.axes}, pt[3] = {a.p_sb, a.p_ss, a.p_sa};
  const uint64_t row = (uint64_t)a.B * a.S * a.D * E;
  if (!ctx.check(a.q, hrt::span_bytes(4, qz, qt, E), "q") || !ctx.check(a.q_out, row * a.Hq, "q_out") ||
      !ctx.check(a.k, hrt::span_bytes(4, kz, kt, E), "k") || !ctx.check(a.k_out, row * a.Hk, "k_out") ||
      !ctx.check(a.pos, hrt::span_bytes(3, pz, pt, pe), "pos") || !ctx.check(a.freqs, (uint64_t)a.P * 8, "freqs"))
    return false;
  // A workgroup for every token until the chip is full, then one for two; other shapes of heads were not measured for it.  bf16, 16 + 16 heads of 128, replayed on the same operands, us
  // with 1, 2, 4 tokens each: 2048 tokens 7.6, 7.7, 8.4; 4096 13.5, 12.8, 13.6; 8192 23.7, 22.5, 23.6; 16384 46.5, 44.0, 46.6.
  const int64_t all = a.B * a.S;
  const int tokens = all >= 4096 ? 2 : 1;
  if (all >= (int64_t(1) << 31) || !hrt::grid_fits(cdiv(all, tokens), 256)) return ctx.fail("grid too large");
  // whole pieces: pairs by W, and what is copied by W
  const auto fits = [&](int w) { return a.P % w == 0 && (a.D - 2 * a.P) % w == 0; };
  if (fits(V)) queue_rotary<T, V>(a, tokens, ctx.stream);
  else if (V == 8 && fits(4)) queue_rotary<T, 4>(a, tokens, ctx.stream);
  else queue_rotary<T, 1>(a, tokens, ctx.stream);
  return hrt::launch_ok(hipGetLastError(), ctx, "rotary");
}

HRT_REGISTER("rotary_f32", hrt_rotary_args, launch_rotary<F32>);
HRT_REGISTER("rotary_bf16", hrt_rotary_args, launch_rotary<BF16>);
HRT_REGISTER("rotary_f16", hrt_rotary_args, launch_rotary<F16>);

}  // namespace
}  // namespace hk
