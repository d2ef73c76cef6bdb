// Attention with a relative position bias: argument checks, the buckets' borders, the plan, and the two small kernels that
// join partial results.  The attention kernel itself is attn_rel.h.
#include <cmath>
#include <cstring>
#include <vector>

#include "../hrt/registry.h"
#include "attn_rel_plan.h"
#include "lds_stage.h"

namespace hk {

namespace {

// ---- buckets ---------------------------------------------------------------------------------------------------------------
// a^x b^y as little-endian 32-bit digits.
std::vector<uint32_t> power_product(uint32_t a, int x, uint32_t b, int y) {
  std::vector<uint32_t> v{1};
  for (int i = 0; i < x + y; ++i) {
    uint64_t carry = 0;
    for (uint32_t& d : v) carry += (uint64_t)d * (i < x ? a : b), d = (uint32_t)carry, carry >>= 32;
    if (carry) v.push_back((uint32_t)carry);
  }
  return v;
}

// (n / e)^L >= (m / e)^t, exactly: by logarithms where they differ clearly, else n^L e^t >= m^t e^L in whole numbers.
bool reaches(int n, int e, int L, int m, int t) {
  const double a = L * std::log((double)n / e), b = t * std::log((double)m / e);
  if (std::fabs(a - b) > 1e-9 * (1.0 + std::fabs(b))) return a > b;
  const std::vector<uint32_t> x = power_product(n, L, e, t), y = power_product(m, t, e, L);
  if (x.size() != y.size()) return x.size() > y.size();
  for (size_t i = x.size(); i-- > 0;)
    if (x[i] != y[i]) return x[i] > y[i];
  return true;
}

bool make_buckets(int buckets, int m, int causal, RelBuckets* out) {
  const int nb = causal ? buckets : buckets / 2, e = nb / 2;
  if ((!causal && buckets % 2 != 0) || nb < 2 || nb > 256 || m <= e || m > 1024) return false;
  out->nb = nb, out->sides = causal ? 1 : 2, out->total = buckets;
  for (int k = 0; k <= e; ++k) out->start[k] = k;
  const int L = nb - e;
  for (int t = 1, n = e; t < L; ++t) {
    while (!reaches(n, e, L, m, t)) ++n;  // borders rise with t: m distances in all
    out->start[e + t] = n;
  }
  out->R = out->start[nb - 1];
  for (int k = nb; k < 256; ++k) out->start[k] = INT32_MAX;
  return true;
}

// The last one is kept: a model has one kind of bias, and every launch needs it.
const RelBuckets* buckets_of(const hrt_attn_rel_args& a) {
  thread_local int key[3] = {-1, -1, -1};
  thread_local RelBuckets kept;
  const int want[3] = {a.buckets, a.max_distance, a.causal != 0};
  if (memcmp(key, want, sizeof(key)) != 0) {
    key[0] = -1;
    if (!make_buckets(want[0], want[1], want[2], &kept)) return nullptr;
    memcpy(key, want, sizeof(key));
  }
  return &kept;
}

// ---- plan ------------------------------------------------------------------------------------------------------------------
// Queries that the forward takes one at a time: their keys are then read once per query, by L2 from the second one on.
constexpr int kOneMost = 4;

RelPlan plan_of(const hrt_attn_rel_args& a, int which, bool f32, bool ws, int R) {
  const int64_t n = which == 1 ? a.Sk : a.Sq, bh = (int64_t)a.B * a.H;
  auto blocks = [&](int g) { return cdiv(n, 32 * g); };
  const int dp = a.D <= 64 ? 64 : 128;
  RelPlan p{};
  p.splits = 1;
  if (which == 0 && n <= kOneMost) {  // g 0: one query at a time
    const int64_t wgs = n * bh, want = cdiv(1024, wgs), most = cdiv(a.Sk, 256);
    p.nblk = 1;
    if (ws && want > 1 && most > 1) p.splits = (int)(want < most ? want : most);
    if (p.splits > 64) p.splits = 64;
    // a range's offsets are 31-bit; longer ones of rows far apart take the stages below
    if (cdiv(a.Sk, p.splits) * (a.k_ss > a.v_ss ? a.k_ss : a.v_ss) * (f32 ? 4 : 2) < ((int64_t)1 << 31) - 65536) return p;
    p.splits = 1;
  }
  // groups a workgroup: more share a stage, fewer give more workgroups.  bf16, forward and backward, by one / two / four groups:
  // 48 heads of 512 x 512 x 64 (768 / 384 / 192 workgroups) 90 / 60 / 86 us, 128 heads of 2048 x 2048 x 64 (8192 / 4096 / 2048)
  // 1641 / 963 / 850 us
  p.g = blocks(4) * bh >= 512 ? 4 : blocks(2) * bh >= 256 ? 2 : 1;
  if (f32) {
    // fp32 is bound by the matrix cores, so by the CU with the most workgroups: a workgroup of one / two / four groups takes
    // 50 / 80 / 150 us against 1024 keys.  16 heads of 1040 x 1040 x 64 (528 / 272 / 144): 394 / 411 / 385 us, 12 heads of
    // 512 x 512 (192 / 96 / 48): 87 / 119 / 187 us
    const int cost[5] = {0, 10, 16, 0, 30};
    int64_t least = 0;
    for (int g : {4, 2, 1}) {
      const int64_t t = cdiv(blocks(g) * bh, 256) * cost[g];
      if (g == 4 || t < least) p.g = g, least = t;
    }
  }
  // fp32 rows of 128 have a form for four groups only (two or one would need stages of 64 or 128 rows, which fit LDS with one buffer),
  // so that few heads leave CUs idle: forward and backward, 8 heads of 1000 x 1000 x 128 (64 workgroups) 573 us, elementary operations
  // 816; one of 4000 x 4000 x 128 (32) 2003, elementary operations 1540
  if (f32 && dp == 128) p.g = 4;
  // four buffers of 128 rows leave 29 KiB for the bands of far-reaching tables
  if (p.g == 1 && dp == 128 && rel_lds(which, R) > 29 * 1024) p.g = 2;
  p.nblk = (int)blocks(p.g);
  const int64_t stages = cdiv(a.Sk, rel_stage(f32, dp, p.g)), wgs = p.nblk * bh;
  p.per = (int)stages;
  if (which == 0 && ws && wgs < 256 && stages >= 4) {
    int64_t want = cdiv(512, wgs), most = stages / 2;
    if (most > 64) most = 64;  // attn_rel_join
    p.per = (int)cdiv(stages, want < most ? want : most);
    p.splits = (int)cdiv(stages, p.per);
  }
  return p;
}

// ---- one query at a time ---------------------------------------------------------------------------------------------------
// Few queries (decoding): bound by the bytes of K and V, which tiles through LDS fetch too few of at a time.  A workgroup takes
// one query of one head and one range of its keys; LPK lanes hold a key's 16-byte pieces, so a wavefront loads 64 / LPK keys
// with one instruction, UB such instructions of K and of V in flight before the first is used.  Each lane group keeps its own
// running maximum, sum and output piece over its keys; the groups are joined at the end, the wavefronts through LDS, the
// ranges by attn_rel_join, always in one order.  Keys past the range's end or masked get an offset beyond the buffer and
// are not fetched.  As many ranges as give 1024 workgroups (2048: 1 % slower; batches of eight keys, and loads past the
// caches, were slower too).  Measured: bf16, 128 heads of one query and 4096 x 64 keys, 134 MB of K and V in 25 us and 5 us of
// join, 4.5 TB/s over both; fp32, 268 MB in 44 us with the join, 6.0 TB/s.
template <typename T>
struct Piece {  // 16 bytes of a row
  static constexpr int N = 16 / sizeof(typename T::storage);
  __device__ __forceinline__ static void unpack(u32x4 w, float* v) {
    if constexpr (N == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = lo16<T>(w[i]), v[2 * i + 1] = hi16<T>(w[i]);
    }
  }
};

// The same in every lane of an aligned group of LPK.
template <int LPK>
__device__ __forceinline__ float group_sum(float v) {
  v = dpp_add<0xB1>(v), v = dpp_add<0x4E>(v), v = dpp_add<0x141>(v);  // quads, then their mirror in the half row
  if constexpr (LPK > 8) v = dpp_add<0x140>(v);
  if constexpr (LPK > 16) v += __shfl_xor(v, 16, 64);
  return v;
}

// One value of o, and what its rounding left (none of a value that became no number).
template <typename T>
__device__ __forceinline__ void put_o(const hrt_attn_rel_args& p, int64_t at, float v) {
  const typename T::storage o = T::from_f32(v);
  gptr<typename T::storage>(p.o)[at] = o;
  if constexpr (!std::is_same<T, F32>::value) {
    const float r = T::to_f32(o);
    if (p.o_lo) gptr<typename T::storage>(p.o_lo)[at] = T::from_f32(fabsf(r) < INFINITY ? v - r : 0.f);
  }
}

template <typename T, int LPK>
__global__ __launch_bounds__(256) void attn_rel_one(hrt_attn_rel_args p, RelBuckets bk, int64_t rows, int splits, int64_t range) {
  constexpr int N = Piece<T>::N, KPW = 64 / LPK, UB = 4, ESZ = sizeof(typename T::storage);
  __shared__ float band[2 * 1024 + 1];
  __shared__ float part[3][LPK * N + 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), piece = lane % LPK, sub = lane / LPK;
  const uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x % (uint32_t)rows), split = __builtin_amdgcn_readfirstlane(blockIdx.x / (uint32_t)rows);
  const int64_t q = row % (uint32_t)p.Sq, bh = row / (uint32_t)p.Sq, b = bh / p.H, hh = bh % p.H;
  const int64_t at = q + p.q_off, R = bk.R;  // the query's position among the keys
  int64_t k0 = split * range, k1 = k0 + range < p.Sk ? k0 + range : p.Sk;
  if (p.causal && k1 > at + 1) k1 = at + 1 > 0 ? at + 1 : 0;
  const uint32_t kss = (uint32_t)(p.k_ss * ESZ), vss = (uint32_t)(p.v_ss * ESZ);
  const __amdgpu_buffer_rsrc_t kr = edge_rsrc(gcptr<uint8_t>(p.k) + (b * p.k_sb + hh * p.k_sh + k0 * p.k_ss) * ESZ);
  const __amdgpu_buffer_rsrc_t vr = edge_rsrc(gcptr<uint8_t>(p.v) + (b * p.v_sb + hh * p.v_sh + k0 * p.v_ss) * ESZ);
  const HK_G uint8_t* mask = gcptr<uint8_t>(p.mask) + b * p.mask_sb;
  const int len = (int)(k1 > k0 ? k1 - k0 : 0);
  const bool has = piece * N < p.D;
  // the wavefronts take batches of UB KPW keys in turn; the next batch's mask is read under this one's arithmetic
  constexpr int STEP = UB * KPW;
  bool ok[UB], next[UB];
  u32x4 kw[UB], vw[UB];
  auto look = [&](int first, bool (&f)[UB]) {
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const int k = first + u * KPW + sub;
      f[u] = k < len;
      if (p.mask) f[u] = f[u] && mask[k0 + (f[u] ? k : 0)] != 0;
    }
  };
  auto load = [&](int first) {
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const uint32_t k = first + u * KPW + sub;
      kw[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, ok[u] && has ? (int)(k * kss + piece * 16) : (int)kNoRow, 0, 0));
    }
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const uint32_t k = first + u * KPW + sub;
      vw[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, ok[u] && has ? (int)(k * vss + piece * 16) : (int)kNoRow, 0, 0));
    }
  };
  int first = wave * STEP;
  look(first, ok);
  load(first);
  float qv[N], o[N], m = -INFINITY, l = 0.f;
  {
    u32x4 w = {0, 0, 0, 0};
    if (has) w = *reinterpret_cast<const HK_G u32x4*>(gcptr<uint8_t>(p.q) + (b * p.q_sb + hh * p.q_sh + q * p.q_ss) * ESZ + piece * 16);
    Piece<T>::unpack(w, qv);
#pragma unroll
    for (int i = 0; i < N; ++i) qv[i] *= p.scale * 1.4426950408889634f, o[i] = 0.f;
  }
  // this query's bias by distance, in log2 units
  const HK_G typename T::storage* table = gcptr<typename T::storage>(p.table) + hh;
  for (int t = tid; t <= 2 * R; t += 256) {
    const int r = t - (int)R, n = r < 0 ? -r : r;
    const int k = rel_bucket(bk, n);
    band[t] = r > 0 && bk.sides == 1 ? 0.f : T::to_f32(table[(int64_t)(r > 0 ? bk.nb + k : k) * p.H]) * 1.4426950408889634f;
  }
  __syncthreads();
  for (; first < len; first += 4 * STEP) {
    const bool more = first + 4 * STEP < len;
    if (more) look(first + 4 * STEP, next);
    bool any = false;
#pragma unroll
    for (int u = 0; u < UB; ++u) any = any || ok[u];
    if (__any(any)) {
      float s[UB], mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < UB; ++u) {
        float kv[N], d = 0.f;
        Piece<T>::unpack(kw[u], kv);
#pragma unroll
        for (int i = 0; i < N; ++i) d = fmaf(qv[i], kv[i], d);
        const int64_t r = k0 + first + u * KPW + sub - at;
        s[u] = group_sum<LPK>(d) + band[(r < -R ? -R : r > R ? R : r) + R];
        if (!ok[u]) s[u] = -INFINITY;
        mx = fmaxf(mx, s[u]);
      }
      const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - base);  // m = -inf: 0
      m = mn;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] *= alpha;
#pragma unroll
      for (int u = 0; u < UB; ++u) {
        float vv[N];
        const float e = __builtin_amdgcn_exp2f(s[u] - base);
        Piece<T>::unpack(vw[u], vv);
        l += e;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(e, vv[i], o[i]);
      }
    }
    if (more) {
#pragma unroll
      for (int u = 0; u < UB; ++u) ok[u] = next[u];
      load(first + 4 * STEP);
    }
  }
  // the lane groups of a wavefront, then the wavefronts
#pragma unroll
  for (int x = LPK; x < 64; x <<= 1) {
    const float m2 = __shfl_xor(m, x, 64), mt = fmaxf(m, m2), base = mt == -INFINITY ? 0.f : mt;
    const float a = __builtin_amdgcn_exp2f(m - base), c = __builtin_amdgcn_exp2f(m2 - base);
    l = a * l + c * __shfl_xor(l, x, 64);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = a * o[i] + c * __shfl_xor(o[i], x, 64);
    m = mt;
  }
  if (wave > 0 && sub == 0) {
    float* const mine = part[wave - 1];
#pragma unroll
    for (int i = 0; i < N; ++i) mine[piece * N + i] = o[i];
    if (piece == 0) mine[LPK * N] = m, mine[LPK * N + 1] = l;
  }
  __syncthreads();
  if (wave > 0 || sub > 0) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    const float m2 = part[w][LPK * N], mt = fmaxf(m, m2), base = mt == -INFINITY ? 0.f : mt;
    const float a = __builtin_amdgcn_exp2f(m - base), c = __builtin_amdgcn_exp2f(m2 - base);
    l = a * l + c * part[w][LPK * N + 1];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = a * o[i] + c * part[w][piece * N + i];
    m = mt;
  }
  if (splits > 1) {  // as the tile kernel leaves them
    HK_G float* const to = gptr<float>(p.ws) + ((int64_t)split * rows + row) * p.D + piece * N;
    if (has)
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<HK_G f32x4*>(to + i) = f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]};
    HK_G float* const st = gptr<float>(p.ws) + splits * rows * p.D + ((int64_t)split * rows + row) * 2;
    if (piece == 0) st[0] = m, st[1] = l;
    return;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (piece == 0) gptr<float>(p.lse)[row] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  if (has) {
    const int64_t out = ((b * p.Sq + q) * p.H + hh) * p.D + piece * N;
#pragma unroll
    for (int i = 0; i < N; ++i) put_o<T>(p, out + i, o[i] * inv);
  }
}

// ---- joins -----------------------------------------------------------------------------------------------------------------
// Forward partial sums of the key ranges, added in order: a wavefront per row.  The ranges' maxima and sums come in one load
// per 64 ranges, the outputs four ranges at a time.
template <typename T>
__global__ __launch_bounds__(256) void attn_rel_join(hrt_attn_rel_args p, int splits, int64_t rows) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= rows) return;
  const HK_G float* o = gcptr<float>(p.ws);
  const HK_G float* ms = o + splits * rows * p.D;
  float mine = -INFINITY, sum = 0.f;  // of range `lane`, splits <= 64
  if (lane < splits) mine = ms[(lane * rows + row) * 2], sum = ms[(lane * rows + row) * 2 + 1];
  const float m = wave_max(mine);
  const float f = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - m);
  const float l = wave_sum(f * sum);
  float acc[2] = {0.f, 0.f};
  for (int s = 0; s < splits; s += 4) {
    float v[4][2];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t r = s + x < splits ? s + x : 0;
        v[x][u] = lane + 64 * u < p.D ? o[(r * rows + row) * p.D + lane + 64 * u] : 0.f;
      }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float w = s + x < splits ? __shfl(f, s + x, 64) : 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) acc[u] = fmaf(w, v[x][u], acc[u]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int64_t q = row % p.Sq, bh = row / p.Sq, b = bh / p.H, h = bh % p.H;
  if (lane == 0) gptr<float>(p.lse)[row] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  const int64_t out = ((b * p.Sq + q) * p.H + h) * p.D + lane;
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 64 * u < p.D) put_o<T>(p, out + 64 * u, acc[u] * inv);
}

template <typename T>
__global__ __launch_bounds__(256) void attn_rel_table(hrt_attn_rel_args p, int64_t n) {
  rel_table<T>(p, n, (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), threadIdx.x & 63);
}

template <typename T>
void queue_one(const hrt_attn_rel_args& a, const RelBuckets& bk, const RelPlan& pl, hipStream_t s) {
  const int64_t rows = (int64_t)a.B * a.H * a.Sq, range = cdiv(a.Sk, pl.splits);
  const dim3 grid((uint32_t)(rows * pl.splits)), block(256);
  const int pieces = (int)cdiv(a.D, Piece<T>::N);
  if (pieces <= 8) hipLaunchKernelGGL((attn_rel_one<T, 8>), grid, block, 0, s, a, bk, rows, pl.splits, range);
  else if (pieces <= 16) hipLaunchKernelGGL((attn_rel_one<T, 16>), grid, block, 0, s, a, bk, rows, pl.splits, range);
  else hipLaunchKernelGGL((attn_rel_one<T, 32>), grid, block, 0, s, a, bk, rows, pl.splits, range);
}

// ---- launch ----------------------------------------------------------------------------------------------------------------
bool check(const hrt_attn_rel_args& a, int which, int esz, hrt::LaunchCtx& ctx) {
  if (a.B < 1 || a.H < 1 || a.Sq < 1 || a.Sk < 1 || a.D < 1 || a.D > 128) return ctx.fail("attention needs B, H, Sq, Sk >= 1 and 1 <= D <= 128");
  const int per16 = 16 / esz;
  if (a.D % per16 != 0) return ctx.fail("D must fill 16-byte pieces");
  if (!(a.scale >= 1e-20f && a.scale <= 1e20f)) return ctx.fail("scale must lie in 1e-20 .. 1e20");
  if (a.q_off < -((int64_t)1 << 40) || a.q_off > ((int64_t)1 << 40)) return ctx.fail("query offset out of range");
  const int64_t strides[] = {a.q_sb, a.q_sh, a.q_ss, a.k_sb, a.k_sh, a.k_ss, a.v_sb, a.v_sh, a.v_ss, a.do_sb, a.do_sh, a.do_ss};
  const int nstr = which == 0 ? 9 : 12;
  for (int i = 0; i < nstr; ++i)
    if (strides[i] < 0 || strides[i] % per16 != 0) return ctx.fail("strides must be non-negative and keep rows on 16 bytes");
  if (a.mask && a.mask_sb < 0) return ctx.fail("negative mask stride");
  const int64_t lim = ((int64_t)1 << 31) / (130 * esz);  // a stage's row offsets are 31-bit
  for (int i : {2, 5, 8, 11})
    if (i < nstr && strides[i] >= lim) return ctx.fail("rows too far apart");
  auto view = [&](uint64_t at, int i, int64_t S, const char* what) {
    const int64_t sz[4] = {a.B, a.H, S, a.D}, st[4] = {strides[i], strides[i + 1], strides[i + 2], 1};
    if (at % 16 != 0) return ctx.fail(std::string(what) + " must be 16-byte aligned");
    return ctx.check(at, hrt::span_bytes(4, sz, st, (uint64_t)esz), what);
  };
  const uint64_t bh = (uint64_t)a.B * a.H, rows = bh * (uint64_t)a.Sq;
  if (!view(a.q, 0, a.Sq, "q") || !view(a.k, 3, a.Sk, "k") || !view(a.v, 6, a.Sk, "v") ||
      !ctx.check(a.table, (uint64_t)a.buckets * a.H * esz, "table") || !ctx.check(a.lse, rows * 4, "lse"))
    return false;
  if (a.mask && !ctx.check(a.mask, (uint64_t)((a.B - 1) * a.mask_sb + a.Sk), "mask")) return false;
  if (which != 1 && a.o % 16 != 0) return ctx.fail("o must be 16-byte aligned");
  if (which != 1 && !ctx.check(a.o, rows * a.D * esz, "o")) return false;
  if (which != 1 && esz == 2 && a.o_lo && (a.o_lo % 16 != 0 || !ctx.check(a.o_lo, rows * a.D * esz, "o_lo")))
    return a.o_lo % 16 != 0 ? ctx.fail("o_lo must be 16-byte aligned") : false;
  if (which != 0 && (!view(a.dout, 9, a.Sq, "dout") || !ctx.check(a.delta, rows * 4, "delta"))) return false;
  // gradients: contiguous, or spread like their inputs
  auto grad = [&](uint64_t at, int i, int64_t S, const char* what) {
    if (a.flags & HRT_ATTN_GRAD_LIKE_INPUT) return view(at, i, S, what);
    if (at % 16 != 0) return ctx.fail(std::string(what) + " must be 16-byte aligned");
    return ctx.check(at, bh * (uint64_t)S * a.D * esz, what);
  };
  if (which == 1 && (!grad(a.dk, 3, a.Sk, "dk") || !grad(a.dv, 6, a.Sk, "dv"))) return false;
  if (which == 2 && a.dq && !grad(a.dq, 0, a.Sq, "dq")) return false;
  return true;
}

int64_t fwd_floats(const hrt_attn_rel_args& a, const RelPlan& p) { return p.splits > 1 ? (int64_t)p.splits * a.B * a.H * a.Sq * (a.D + 2) : 0; }
int64_t table_floats(const hrt_attn_rel_args& a, const RelPlan& p) { return (int64_t)a.B * a.H * p.nblk * a.buckets; }

template <typename T, int WHICH>
bool launch_rel(const void* pp, const uint32_t*, hrt::LaunchCtx& ctx) {
  const auto& a = *static_cast<const hrt_attn_rel_args*>(pp);
  constexpr int esz = sizeof(typename T::storage);
  const RelBuckets* bk = buckets_of(a);
  if (bk == nullptr) return ctx.fail("buckets: causal 2..256, else even and 4..512, with max_distance above half of one direction's and at most 1024");
  if (!check(a, WHICH, esz, ctx)) return false;
  RelPlan pl = plan_of(a, WHICH, esz == 4, a.ws != 0, bk->R);
  if (WHICH == 0 && pl.splits > 1) {
    const int64_t need = fwd_floats(a, pl);
    if (a.ws % 16 != 0 || a.ws_floats < need) pl = plan_of(a, WHICH, esz == 4, false, bk->R);
    else if (!ctx.check(a.ws, (uint64_t)need * 4, "ws")) return false;
  }
  const bool later = (a.flags & HRT_ATTN_REL_TABLE_LATER) != 0;
  if (a.dtable && (WHICH == 2 || (WHICH == 1 && later))) {
    const RelPlan dq = plan_of(a, 2, esz == 4, false, bk->R);
    const int64_t need = table_floats(a, dq);
    if (a.ws_floats < need || a.ws % 4 != 0) return ctx.fail("the table's gradient needs a workspace of hrt_attn_rel_workspace floats");
    if (!ctx.check(a.ws, (uint64_t)need * 4, "ws") || !ctx.check(a.dtable, (uint64_t)a.buckets * a.H * esz, "dtable")) return false;
    if (WHICH == 1) pl.table = (int)(cdiv((int64_t)a.buckets * a.H, 32) * 8), pl.parts = (int64_t)a.B * dq.nblk;
  }
  if (!hrt::grid_fits((int64_t)(pl.g == 0 ? a.Sq : pl.nblk) * a.B * a.H * pl.splits + pl.table, 256) || !hrt::grid_fits(cdiv((int64_t)a.B * a.H * a.Sq, 4), 256))
    return ctx.fail("too many rows for one launch");
  if (pl.g == 0) {
    queue_one<T>(a, *bk, pl, ctx.stream);
  } else {
    attn_rel_queue<T>(a, WHICH, *bk, pl, ctx.stream);
  }
  if (!hrt::launch_ok(hipGetLastError(), ctx, "attn_rel")) return false;
  if (WHICH == 0 && pl.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.H * a.Sq;
    hipLaunchKernelGGL(attn_rel_join<T>, dim3((uint32_t)cdiv(rows, 4)), dim3(256), 0, ctx.stream, a, pl.splits, rows);
    return hrt::launch_ok(hipGetLastError(), ctx, "attn_rel_join");
  }
  if (WHICH == 2 && a.dtable && !later) {
    hipLaunchKernelGGL(attn_rel_table<T>, dim3((uint32_t)cdiv((int64_t)a.buckets * a.H, 4)), dim3(256), 0, ctx.stream, a, (int64_t)a.B * pl.nblk);
    return hrt::launch_ok(hipGetLastError(), ctx, "attn_rel_table");
  }
  return true;
}

HRT_REGISTER("attn_rel_fwd_f32", hrt_attn_rel_args, (launch_rel<F32, 0>));
HRT_REGISTER("attn_rel_fwd_bf16", hrt_attn_rel_args, (launch_rel<BF16, 0>));
HRT_REGISTER("attn_rel_fwd_f16", hrt_attn_rel_args, (launch_rel<F16, 0>));
HRT_REGISTER("attn_rel_dkdv_f32", hrt_attn_rel_args, (launch_rel<F32, 1>));
HRT_REGISTER("attn_rel_dkdv_bf16", hrt_attn_rel_args, (launch_rel<BF16, 1>));
HRT_REGISTER("attn_rel_dkdv_f16", hrt_attn_rel_args, (launch_rel<F16, 1>));
HRT_REGISTER("attn_rel_dq_f32", hrt_attn_rel_args, (launch_rel<F32, 2>));
HRT_REGISTER("attn_rel_dq_bf16", hrt_attn_rel_args, (launch_rel<BF16, 2>));
HRT_REGISTER("attn_rel_dq_f16", hrt_attn_rel_args, (launch_rel<F16, 2>));

}  // namespace
}  // namespace hk

extern "C" int64_t hrt_attn_rel_workspace(const hrt_attn_rel_args* a, int32_t dtype, int32_t backward) {
  if (a == nullptr || a->B < 1 || a->H < 1 || a->Sq < 1 || a->Sk < 1) return 0;
  const hk::RelBuckets* bk = hk::buckets_of(*a);
  if (bk == nullptr) return 0;
  const bool f32 = dtype == HRT_F32;
  return backward ? hk::table_floats(*a, hk::plan_of(*a, 2, f32, false, bk->R)) : hk::fwd_floats(*a, hk::plan_of(*a, 0, f32, true, bk->R));
}

extern "C" int hrt_attn_rel_buckets(int32_t buckets, int32_t max_distance, int32_t causal, uint16_t start[256]) {
  hk::RelBuckets b;
  if (start == nullptr || !hk::make_buckets(buckets, max_distance, causal != 0, &b)) return -1;
  for (int k = 0; k < b.nb; ++k) start[k] = (uint16_t)b.start[k];
  return b.nb;
}
