// Verification of drafted tokens against the target's probabilities (speculative decoding).
//
// Sequence b has K + 1 rows of target logits (row i: after i drafted tokens) and n_b <= K drafts
// d_0 .. d_{n-1}.  Per row, on l = sf(logits) (NaN -> 0, +-inf -> +-FLT_MAX):
//   x_j   = exp((l_j - max l) / temperature)
//   tau   = the largest l value v with #{l >= v} >= top_k or mass{l >= v} >= top_p sum x
//   kept  = x_j (l_j > tau), comp x_j (l_j == tau), 0 (l_j < tau), comp = clamp(min((top_k -
//           #{l > tau}) / #{l == tau}, (top_p sum x - mass{l > tau}) / mass{l == tau}), 0, 1)
//   p     = kept / Z, Z = sum kept
// the filter of the token sampler, with ties by logit.  Draft i is accepted while
// u_i q_i(d_i) < p_i(d_i), q the drafter's probabilities (1 at the draft where none are given).  At
// the first rejected draft the new token is drawn from w = max(p_i - q_i, 0) (p_i without the draft),
// or from p_i where that is empty; with all accepted from p_n: the first j with
// sum_{j' <= j} w > u_K sum w, in vocabulary order.
//
// Numbers are whole-token decisions next to borders of sums over the vocabulary, so they are held in
// 64 bits: weights by a polynomial of relative error 1.1e-12, masses as integers in units of 2^-43
// (sums of up to 2^20 weights <= 1 do not overflow, and integer sums do not depend on their order),
// the draw's prefix sums in fp64.  A token differs from that of exact arithmetic only where a
// uniform lies within ~1e-11 of a border (6e-8 where 2^20 equal weights round the same way).
//
// Launches:
//   sums   every row in groups of 2048 entries, a wave each: the group's largest logit, its mass relative
//          to that (without a filter also that of its 8 segments of 256), and for a small top_k or a
//          nucleus a list of its largest entries
//   rows   (with a filter) one workgroup per row: tau, comp, Z and the test of the row's draft; from the
//          lists, where they reach down to tau, also the token if the sequence stops at this row;
//          otherwise from the whole row (of a nucleus, in a launch of its own)
//   parts  (with a drafter's distribution, and where lists may not do) the segments' sums of w for the row
//          that each sequence stops at, by several workgroups
//   draw   one workgroup per sequence: the segment that the uniform falls on, and the entry

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

constexpr int kListThreads = 256;  // rows' kernel: rows searched in lists (320 rows of 1220:
                                    // a call of 19.2 us, 21.0 with 512)
constexpr int kMaxWaves = 1024 / 64;
constexpr int kVerBins = 2048;   // histogram of (max - l) for the threshold
constexpr int kVerCand = 512;    // entries of one bin that are ranked directly
constexpr int kVerList = 4 * kListThreads;  // listed entries of a row: four per lane
constexpr int kVerDraw = 256;    // kept entries that the rows' kernel draws from directly
constexpr int kVerMaxV = 1 << 20;
constexpr int kSeg = 256;        // consecutive entries whose weights are added up for the draw (one wave's 64 x 4)
constexpr int kMaxSegs = kVerMaxV / kSeg;
constexpr int kGroupSegs = 8;    // segments per wave of the sums' kernel
constexpr double kMassUnit = 1.0 / 8796093022208.0;  // 2^-43

struct RowStat {
  double z, comp;
  float max, tau;
  int ok, mode;
  int token;    // the new token if the sequence stops here; -1: not known yet
  int verdict;  // where a second launch searches what the lists leave open
};
static_assert(sizeof(RowStat) == 40, "row stat size");
// How a row's logits are read so that only finite values and -inf (weight 0) remain:
enum {
  kNanZero = 0, // NaN -> 0
  kInfOnly = 1, // the largest is FLT_MAX, which +inf stands for and beside which every other value weighs
                // nothing (its neighbours are 2e31 apart): FLT_MAX and +inf -> 0, anything else -> -inf
  kAllLow = 2   // nothing above -FLT_MAX, which -inf stands for: all entries tied
};

enum { kOpen = 0, kAccepted = 1, kRejected = 2 };  // kRejected: rows behind a rejection too

struct VerifyArgs {
  int K, V;
  const void* logits;
  const int32_t *drafts, *n_draft;
  const float *q, *u;
  int32_t *tokens, *accepted;
  RowStat* stat;       // [B, K+1] (with a filter)
  double* seg_sum;     // [B, K+1, segs] (without one)
  double* group_sum;   // [B, K+1, groups]
  float *group_max, *group_floor;  // group_floor: all entries of the group from it up are listed
  int32_t* group_count;
  float2* list;        // [B, K+1, groups, cap] logit, index
  double* part_sum;    // [B, segs]
  int segs, groups;
  int cap, rank;       // entries listed per group (0: no lists); maxima that a row of lanes gives
  int again;           // rows that the lists leave open are searched by a launch of their own
  double scale, d_min;  // log2(e) / temperature; -1023 / scale (weight 0)
  double unscale, light;  // 1 / scale; (1 - top_p) / V
  float bin_scale;
  int top_k;
  double top_p;
  int use_mass, truncate;
};

// 2^(d scale) for d <= 0: d scale = n + f with |f| <= 1/2, n from the sum with 1.5 2^52, whose low word
// it is; 2^f by the degree-8 polynomial through 2^f at the Chebyshev points of [-1/2, 1/2] (relative
// error 1.1e-12, exactly 1 at 0); 2^n from its exponent bits.  d_min = -1023 / scale is where those
// are all zero: from there down (masks too) the weight is exactly 0.  16 instructions at the rate of an
// fp32 FMA (ldexp and the conversion of n took four times that each).
__device__ __forceinline__ double exp2_neg(double d, double scale, double d_min) {
  constexpr double kMagic = 6755399441055744.0;
  d = fmax(d, d_min);
  const double t = __builtin_fma(d, scale, kMagic);
  const double f = __builtin_fma(d, scale, kMagic - t);
  double p = 1.3255224884799127e-06;
  p = __builtin_fma(p, f, 1.5310079402383103e-05);
  p = __builtin_fma(p, f, 1.5403455852419016e-04);
  p = __builtin_fma(p, f, 1.3333450568000008e-03);
  p = __builtin_fma(p, f, 9.61812915940262e-03);
  p = __builtin_fma(p, f, 5.550410941205934e-02);
  p = __builtin_fma(p, f, 2.402265069581299e-01);
  p = __builtin_fma(p, f, 6.931471805459335e-01);
  p = __builtin_fma(p, f, 1.0);
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
  return p * __builtin_bit_cast(double, u2{0u, (n << 20) + (1023u << 20)});
}

// A weight in [0, 1] as a whole number of 2^-43: 512 + x has that spacing.
__device__ __forceinline__ uint64_t mass_of(double x) {
  return __builtin_bit_cast(uint64_t, 512.0 + x) - __builtin_bit_cast(uint64_t, 512.0);
}

// ---- wave reductions: DPP inside rows of 16 lanes, readlane across the four rows.  Fixed order; the
// result is wave-uniform.
template <int CTRL, class X>
__device__ __forceinline__ X dpp(X x) {
  static_assert(sizeof(X) == 4 || sizeof(X) == 8, "one or two registers");
  if constexpr (sizeof(X) == 4) {
    return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
  } else {
    typedef int i2 __attribute__((ext_vector_type(2)));
    const i2 v = __builtin_bit_cast(i2, x);
    return __builtin_bit_cast(X, i2{__builtin_amdgcn_update_dpp(0, v[0], CTRL, 0xF, 0xF, true),
                                    __builtin_amdgcn_update_dpp(0, v[1], CTRL, 0xF, 0xF, true)});
  }
}
template <class X>
__device__ __forceinline__ X lane_read(X x, int l) {
  if constexpr (sizeof(X) == 4) {
    return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
  } else {
    typedef int i2 __attribute__((ext_vector_type(2)));
    const i2 v = __builtin_bit_cast(i2, x);
    return __builtin_bit_cast(X, i2{__builtin_amdgcn_readlane(v[0], l), __builtin_amdgcn_readlane(v[1], l)});
  }
}
template <class X>
__device__ __forceinline__ X wave_add(X x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  x += dpp<0x140>(x);
  return (lane_read(x, 0) + lane_read(x, 16)) + (lane_read(x, 32) + lane_read(x, 48));
}
// Sums of four values over the wave, x[l & 3] in lane l: each step on lane bits 0 and 1 halves the number
// of values a lane carries; then the 16 quads.  A third of four separate sums' instructions.
__device__ __forceinline__ double wave_add4(const double* x, int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
  const double p = (b0 ? x[1] : x[0]) + dpp<0xB1>(b0 ? x[0] : x[1]);
  const double q = (b0 ? x[3] : x[2]) + dpp<0xB1>(b0 ? x[2] : x[3]);
  double r = (b1 ? q : p) + dpp<0x4E>(b1 ? p : q);
  r += dpp<0x124>(r);  // rotations by 4 and 8 inside the row
  r += dpp<0x128>(r);
  r += __shfl_xor(r, 16, 64);
  return r + __shfl_xor(r, 32, 64);
}
__device__ __forceinline__ float wave_fmax(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  x = fmaxf(x, dpp<0x140>(x));
  return fmaxf(fmaxf(lane_read(x, 0), lane_read(x, 16)), fmaxf(lane_read(x, 32), lane_read(x, 48)));
}
// Inclusive sum in lane order: row_shr 1, 2, 4, 8 with zero fill, then the rows before.
template <class X>
__device__ __forceinline__ X wave_scan(X x, int lane) {
  x += dpp<0x111>(x);
  x += dpp<0x112>(x);
  x += dpp<0x114>(x);
  x += dpp<0x118>(x);
  const X r0 = lane_read(x, 15), r1 = lane_read(x, 31), r2 = lane_read(x, 47);
  const X r01 = r0 + r1;
  return x + (lane < 16 ? X(0) : lane < 32 ? r0 : lane < 48 ? r01 : r01 + r2);
}

struct StatShared {
  union {
    uint64_t mass[kVerBins];
    struct {  // behind the histogram
      double w[kVerDraw], sorted_w[kVerDraw];
      alignas(16) int at[kVerDraw];
      int sorted_at[kVerDraw];
    } draw;
  };
  uint32_t cnt[kVerBins];
  uint64_t redm[2][kMaxWaves];
  uint32_t redc[2][kMaxWaves], rede[2][kMaxWaves];
  float redf[2][kMaxWaves];
  alignas(16) float cand[kVerCand];
  uint64_t candm[kVerCand];
  int n_cand, bin;
  uint32_t before_c;
  uint64_t before_m;
};

// Sum (maximum) of the values that 8 (16) consecutive lanes hold, in every one of them.
template <class X>
__device__ __forceinline__ X oct_add(X x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  return x + dpp<0x141>(x);
}
__device__ __forceinline__ float oct_fmax(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  return fmaxf(x, dpp<0x141>(x));
}
__device__ __forceinline__ float row_fmax(float x) {
  x = oct_fmax(x);
  return fmaxf(x, dpp<0x140>(x));
}
// ... that W consecutive lanes hold, W = 8 or 16.
template <int W, class X>
__device__ __forceinline__ X lanes_add(X x) {
  static_assert(W == 4 || W == 8 || W == 16, "part of a row of lanes or a row");
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  if constexpr (W >= 8) x += dpp<0x141>(x);
  if constexpr (W == 16) x += dpp<0x140>(x);
  return x;
}
template <int W>
__device__ __forceinline__ float lanes_fmax(float x) {
  if constexpr (W >= 8) return W == 16 ? row_fmax(x) : oct_fmax(x);
  x = fmaxf(x, dpp<0xB1>(x));
  return fmaxf(x, dpp<0x4E>(x));
}

// Block reductions with one barrier: consecutive ones alternate between two buffers (par), so a wave
// overwrites a buffer only behind the barrier that every wave reaches after reading it.  W lanes add the W
// waves' values.
template <int W>
__device__ __forceinline__ float block_max(StatShared& sh, int& par, float a) {
  a = wave_fmax(a);
  if ((threadIdx.x & 63) == 0) sh.redf[par][threadIdx.x >> 6] = a;
  __syncthreads();
  a = lanes_fmax<W>(sh.redf[par][threadIdx.x & (W - 1)]);
  par ^= 1;
  return a;
}
template <int W>
__device__ __forceinline__ void block_add(StatShared& sh, int& par, uint32_t& a, uint32_t& b, uint64_t& m) {
  a = wave_add(a);
  b = wave_add(b);
  m = wave_add(m);
  if ((threadIdx.x & 63) == 0) {
    const int w = threadIdx.x >> 6;
    sh.redc[par][w] = a;
    sh.rede[par][w] = b;
    sh.redm[par][w] = m;
  }
  __syncthreads();
  const int w = threadIdx.x & (W - 1);
  a = lanes_add<W>(sh.redc[par][w]);
  b = lanes_add<W>(sh.rede[par][w]);
  m = lanes_add<W>(sh.redm[par][w]);
  par ^= 1;
}

__device__ __forceinline__ float read_as(float l, int mode) {
  if (mode == kInfOnly) return l >= FLT_MAX ? 0.0f : -INFINITY;
  if (mode == kAllLow) return 0.0f;
  return __builtin_isnan(l) ? 0.0f : l;
}

// The largest logit of a group, with those at the ends of the range as the infinities that they are tied with:
// what tells how a row is read.
__device__ __forceinline__ float saturated(float x) {
  return x >= FLT_MAX ? INFINITY : x <= -FLT_MAX ? -INFINITY : x;
}

// Order-preserving key of a finite float.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 -> +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Four consecutive entries of a row, as stored and as finite fp32 values.
typedef _Float16 hv4 __attribute__((ext_vector_type(4)));
template <bool kHalf>
struct Raw {
  typedef hv4 type;
};
template <>
struct Raw<false> {
  typedef f4 type;
};
template <bool kHalf>
__device__ __forceinline__ typename Raw<kHalf>::type load_raw(const void* row, int i) {
  typedef typename Raw<kHalf>::type R;
  return *reinterpret_cast<const R*>(reinterpret_cast<const char*>(row) + (size_t)i * (kHalf ? 2 : 4));
}
template <class R>
__device__ __forceinline__ f4 to_f4(R x) {
  return f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
template <bool kHalf>
__device__ __forceinline__ const void* row_at(const VerifyArgs& p, int64_t row) {
  return reinterpret_cast<const char*>(p.logits) + row * p.V * (kHalf ? 2 : 4);
}

// The kept weight of logit l in units of its row's largest weight.
__device__ __forceinline__ double kept_of(const VerifyArgs& p, const RowStat& st, float l) {
  const double x = exp2_neg((double)l - (double)st.max, p.scale, p.d_min);
  return l > st.tau ? x : l == st.tau ? x * st.comp : 0.0;
}

// One wave per group of kGroupSegs segments, four groups per workgroup.  fp32: bound by memory (566 rows of
// 65536: 32 us, 4.7 TB/s), or where it looks for nuclei's lists by its vector instructions (38 us, 88 % of the
// SIMDs' cycles).  fp16, 144 rows with lists: 15 us, of which the CUs have waves for 11, their SIMDs busy for 73 %
// of that: 1080 vector instructions a wave, 640 of them the mass's 20 an entry.
template <bool kHalf>
__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs p) {
  const int T = p.K + 1, wgs = (p.groups + 3) / 4;
  const int64_t id = blockIdx.x / wgs;
  const int b = (int)(id / T), i = (int)(id - (int64_t)b * T);
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  if (n < 0 || n > p.K || i > n) return;
  const int lane = threadIdx.x & 63, group = (int)(blockIdx.x - id * wgs) * 4 + (threadIdx.x >> 6);
  if (group >= p.groups) return;
  const void* row = row_at<kHalf>(p, id);
  // The group's entries: 8 consecutive segments; for lists, 64 consecutive entries in every 64 groups' worth,
  // as likely tokens often have neighbouring indices and a list has room for a few of a row's top_k.
  const bool spread = p.cap > 0;
  const int at0 = spread ? (group + p.groups * (lane >> 4)) * 64 + 4 * (lane & 15) : group * (kGroupSegs * kSeg) + 4 * lane;
  const int step = spread ? p.groups * kSeg : kSeg;
  typename Raw<kHalf>::type raw[kGroupSegs];
#pragma unroll
  for (int k = 0; k < kGroupSegs; ++k) raw[k] = load_raw<kHalf>(row, min(at0 + k * step, p.V - 4));
  f4 l[kGroupSegs];
  float lane_max = -INFINITY;
#pragma unroll
  for (int k = 0; k < kGroupSegs; ++k) {
    l[k] = to_f4(raw[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) l[k][e] = __builtin_isnan(l[k][e]) ? 0.0f : l[k][e];
  }
  if ((spread ? p.groups : group + 1) * (kGroupSegs * kSeg) > p.V) {  // padding
#pragma unroll
    for (int k = 0; k < kGroupSegs; ++k)
      if (at0 + k * step >= p.V) l[k] = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  }
#pragma unroll
  for (int k = 0; k < kGroupSegs; ++k)
    lane_max = fmaxf(lane_max, fmaxf(fmaxf(l[k][0], l[k][1]), fmaxf(l[k][2], l[k][3])));
  const float mx = saturated(wave_fmax(lane_max));
  if (lane == 0) p.group_max[id * p.groups + group] = mx;
  bool flat = false;
  if (!p.truncate || p.use_mass) {
    double total = 0.0;
    if (mx > -INFINITY) {
      if (mx == INFINITY) {
        lane_max = read_as(lane_max, kInfOnly);
#pragma unroll
        for (int k = 0; k < kGroupSegs; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) l[k][e] = read_as(l[k][e], kInfOnly);
      }
      const double mxd = mx == INFINITY ? 0.0 : (double)mx;
#pragma unroll
      for (int k0 = 0; k0 < kGroupSegs; k0 += 4) {
        double s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          double w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = exp2_neg((double)l[k0 + u][e] - mxd, p.scale, p.d_min);
          s[u] = (w[0] + w[1]) + (w[2] + w[3]);
        }
        total += (s[0] + s[1]) + (s[2] + s[3]);
        if (!p.truncate) {
          const double w = wave_add4(s, lane);
          const int seg = group * kGroupSegs + k0 + lane;
          if (lane < 4 && seg < p.segs) p.seg_sum[id * p.segs + seg] = w;
        }
      }
      total = wave_add(total);
      // A list holds about what the lanes' maxima are.  Where those are less than half of top_p of the mass,
      // either no entry of the group is kept (its list is empty, from just above its largest up), or more
      // are than lists hold.
      if (p.again) flat = !(wave_add(exp2_neg((double)lane_max - mxd, p.scale, p.d_min)) >= 0.5 * p.top_p * total);
    }
    if (lane == 0) p.group_sum[id * p.groups + group] = total;
  }
  if (flat) {
    if (lane == 0) {
      p.group_floor[id * p.groups + group] = mx == INFINITY ? mx : of_key(key_of(mx) + 1u);
      p.group_count[id * p.groups + group] = 0;
    }
  } else if (p.cap > 0) {
    // The rank-th largest lane maximum of each row of 16 lanes, the smallest of the four: 4 rank entries
    // or more lie at or above it.  More than cap (likely entries side by side): halved from there to the
    // largest, until cap / 2 to cap do.
    float lm = lane_max, at = -INFINITY;
    for (int k = 0; k < p.rank; ++k) {
      at = row_fmax(lm);
      lm = lm == at ? -INFINITY : lm;
    }
    at = fmaxf(fminf(fminf(lane_read(at, 0), lane_read(at, 16)), fminf(lane_read(at, 32), lane_read(at, 48))), -FLT_MAX);
    // A bit per entry of the lane from x up, the first one highest: a compare and m = 2 m + carry each.
    auto from = [&](float x) __attribute__((always_inline)) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < kGroupSegs; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          asm("v_cmp_ge_f32 vcc, %1, %2\n\tv_addc_co_u32 %0, vcc, %0, %0, vcc" : "+v"(m) : "v"(l[k][e]), "v"(x) : "vcc");
      return m;
    };
    uint32_t in = from(at);
    int place = wave_scan(__builtin_popcount(in), lane), count = lane_read(place, 63);
    if (count > p.cap) {
      float lo = at, hi = mx;
      at = INFINITY;
      in = 0;
      count = place = 0;
      for (int k = 0; k < 12 && 2 * count < p.cap; ++k) {
        const float mid = 0.5f * lo + 0.5f * hi;
        const uint32_t some = from(mid);
        const int to = wave_scan(__builtin_popcount(some), lane), c = lane_read(to, 63);
        if (c > p.cap) {
          lo = mid;
        } else {
          hi = at = mid;
          in = some;
          place = to;
          count = c;
        }
      }
    }
    // lane by lane, each lane's listed entries (one or two) read again
    float2* out = p.list + (id * p.groups + group) * p.cap + (place - __builtin_popcount(in));
    while (in != 0) {
      const int e = __builtin_clz(in), i = at0 + (e >> 2) * step + (e & 3);
      in &= ~(0x80000000u >> e);
      const float x = kHalf ? (float)reinterpret_cast<const _Float16*>(row)[i] : reinterpret_cast<const float*>(row)[i];
      *out++ = make_float2(__builtin_isnan(x) ? 0.0f : x, __builtin_bit_cast(float, i));
    }
    if (lane == 0) {
      p.group_floor[id * p.groups + group] = at;
      p.group_count[id * p.groups + group] = count;
    }
  }
}

// What a group's sums, relative to its own largest logit, are in units of the row's largest weight.
__device__ __forceinline__ double group_factor(const VerifyArgs& p, float group_max, float mx) {
  return group_max == mx ? 1.0 : exp2_neg((double)group_max - (double)mx, p.scale, p.d_min);
}

// Largest logit, how to read the row, its mass and its lists' reach, from the groups': one wave.
struct RowSummary {
  float max;  // as read
  int mode;
  double mass;
  float floor;  // top_k entries or more lie at or above it (-inf: not known)
  float reach;  // all entries from it up are listed
};
// The lane's first group (up to 131072 entries: its only one), to be requested early.
struct GroupLoads {
  float max, floor;
  double sum;
  int count;
};
__device__ __forceinline__ GroupLoads load_group(const VerifyArgs& p, int64_t id, int g) {
  GroupLoads x{-INFINITY, -INFINITY, 0.0, 0};
  if (g < p.groups) {
    x.max = p.group_max[id * p.groups + g];
    if (!p.truncate || p.use_mass) x.sum = p.group_sum[id * p.groups + g];
    if (p.cap > 0) {
      x.floor = p.group_floor[id * p.groups + g];
      x.count = p.group_count[id * p.groups + g];
    }
  }
  return x;
}
__device__ __forceinline__ RowSummary summarize(const VerifyArgs& p, int64_t id, int lane, const GroupLoads& first) {
  RowSummary r;
  const bool sums = !p.truncate || p.use_mass;
  float mx = first.max, below = -INFINITY, reach = -INFINITY;
  const int count = first.count;  // lists: at most 64 groups
  if (p.cap > 0 && lane < p.groups) {
    below = -first.floor;
    reach = first.floor;
  }
  for (int g = lane + 64; g < p.groups; g += 64) mx = fmaxf(mx, p.group_max[id * p.groups + g]);
  mx = wave_fmax(mx);
  double m = 0.0;
  if (sums) {
    m = first.sum * group_factor(p, first.max, mx);
    for (int g = lane + 64; g < p.groups; g += 64)
      m += p.group_sum[id * p.groups + g] * group_factor(p, p.group_max[id * p.groups + g], mx);
    m = wave_add(m);
  }
  r.mode = mx == INFINITY ? kInfOnly : mx == -INFINITY ? kAllLow : kNanZero;
  r.mass = r.mode == kAllLow ? (double)p.V : m;
  r.max = r.mode == kNanZero ? mx : 0.0f;
  r.floor = -INFINITY;
  r.reach = INFINITY;
  if (p.cap > 0 && r.mode == kNanZero) {
    r.floor = wave_add(count) >= p.top_k ? -wave_fmax(below) : -INFINITY;
    r.reach = wave_fmax(reach);
  }
  return r;
}

__device__ __forceinline__ RowSummary summarize(const VerifyArgs& p, int64_t id, int lane) {
  return summarize(p, id, lane, load_group(p, id, lane));
}

// Draft k of sequence b: its logit as stored, the drafter's probability and the uniform.
struct Draft {
  bool in;  // in the vocabulary
  float l, q, u;
};
template <bool kHalf>
__device__ __forceinline__ Draft load_draft(const VerifyArgs& p, int b, int k) {
  const int64_t id = (int64_t)b * (p.K + 1) + k, at = (int64_t)b * p.K + k;
  const int d = p.drafts[at];
  Draft r{d >= 0 && d < p.V, 0.0f, 1.0f, p.u[id]};
  if (r.in) {
    const void* row = row_at<kHalf>(p, id);
    r.l = kHalf ? (float)reinterpret_cast<const _Float16*>(row)[d] : reinterpret_cast<const float*>(row)[d];
    if (p.q) r.q = p.q[at * p.V + d];
  }
  return r;
}

// With top_p alone the kept mass is top_p S exactly, so p(d) <= x_d / (top_p S), which rejects many a draft
// without tau; and if tau <= l_d, p(d) >= (x_d - (1 - top_p) S) / (top_p S) (the entries above d hold at most
// S - n x_d if n are tied with it, so d keeps (top_p S - (S - n x_d)) / n or all of x_d), which also says that
// tau <= l_d where it is positive.  Margins of 1e-7 for the rounding of either side: 2^19 units of 2^-43 at most
// (6e-8) where all of a row's masses round the same way; a rejection here and the full test never disagree.
enum { kUnsure, kAccept, kReject };
// A row looks at this many drafts before its own: without an end K drafts were K^2 / 2 tests (262143 drafts of
// one sequence: 34 thousand million).  Rows behind a later rejection are searched for nothing.
constexpr int kQuickRows = 64;
template <bool kHalf>
__device__ __forceinline__ int quick_test(const VerifyArgs& p, int b, int k, int lane) {
  const Draft d = load_draft<kHalf>(p, b, k);
  const RowSummary s = summarize(p, (int64_t)b * (p.K + 1) + k, lane);
  if (!d.in) return kReject;
  const double x = exp2_neg((double)read_as(d.l, s.mode) - (double)s.max, p.scale, p.d_min);
  const double goal = p.top_p * s.mass, uq = (double)d.u * (double)d.q;
  if (!(uq * goal < x * (1.0 + 1.0e-7))) return kReject;
  return uq * goal < (x - (1.0 - p.top_p) * s.mass) - 1.0e-7 * s.mass ? kAccept : kUnsure;
}

// kLists: the groups' lists are searched first.  A row that is searched as a whole is read twice more:
// for the histogram and for the entries of one bin.  (Kept in LDS, 128 KiB left one workgroup per CU, whose
// loads and arithmetic then took turns.)  Bound by one workgroup's chain: lists, 144 rows 8 us; whole rows,
// 640 of which 271 are searched, 65536 fp32 entries, 63 us, of which 23 vector instructions.
template <bool kHalf, bool kLists, int kThreads>
__global__ __launch_bounds__(kThreads, kLists ? 3 : 4) void verify_rows_kernel(VerifyArgs p) {
  static_assert(!kLists || kThreads == kListThreads, "four listed entries per lane");
  constexpr int W = kThreads / 64;
  constexpr int kBins = kLists ? 512 : kVerBins;  // a row's lists: at most 1024 entries
  constexpr int kCand = kLists ? 256 : kVerCand;  // a lane each
  constexpr int kTile = 4 * kThreads;  // consecutive entries read at once
  typedef typename Raw<kHalf>::type R;
  __shared__ StatShared sh;
  const int T = p.K + 1;
  const int b = blockIdx.x / T, i = blockIdx.x - b * T;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = p.V;
  const int64_t id = (int64_t)b * T + i;
  // What does not depend on another load is requested first, needed or not: the chain of loads is a third
  // of the kernel's time where the lists decide.  Four listed entries per lane (in the lists' room if not
  // written).
  const GroupLoads own_group = load_group(p, id, lane);
  float2 listed_at[4] = {};
  int list_group[4] = {}, list_place[4] = {}, list_count[4] = {};
  if (kLists) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = t + u * kThreads;
      list_group[u] = at / p.cap;
      list_place[u] = at - list_group[u] * p.cap;
      if (list_group[u] < p.groups) {
        listed_at[u] = p.list[(id * p.groups + list_group[u]) * p.cap + list_place[u]];
        list_count[u] = p.group_count[id * p.groups + list_group[u]];
      }
    }
  }
  int lookup = -1;  // the draft that a drafter without a distribution gave
  if (kLists && !p.q && i < p.K)  // (an ordinary scalar load is moved to its use, far behind)
    lookup = __hip_atomic_load(p.drafts + (int64_t)b * p.K + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  const float last_u = p.u[(int64_t)b * T + p.K];
  Draft draft{false, 0.0f, 1.0f, 0.0f};
  if (t == 0 && i < p.K) draft = load_draft<kHalf>(p, b, i);
  if (n < 0 || n > p.K || i > n) return;
  if (i == n) draft.in = false;
  const void* row = row_at<kHalf>(p, id);
  const int tiles = (V + kTile - 1) / kTile;
  int par = 0;
  if (kLists == (p.cap > 0) && p.use_mass && p.top_k == V) {
    // Rows that a quick test can do without: those behind a rejection, and accepted ones (no statistics
    // but the verdict are read of them).  Of 128 sequences' 566 rows (4 drafts, nucleus 0.95) 271 are left.
    if (t == 0) sh.bin = sh.n_cand = 0;
    __syncthreads();
    const int before = min(i, kQuickRows);  // of the drafts before row i the first ones; then its own
    for (int k = wv; k <= before; k += W) {
      const int at = k < before ? k : i;
      if (at >= n) continue;
      const int v = quick_test<kHalf>(p, b, at, lane);
      if (lane == 0 && at < i && v == kReject) sh.bin = 1;
      if (lane == 0 && at == i && v == kAccept) sh.n_cand = 1;
    }
    __syncthreads();
    if (sh.bin != 0 || sh.n_cand != 0) {
      if (t == 0) {
        p.stat[id].ok = sh.bin != 0 ? 0 : 1;
        p.stat[id].verdict = sh.bin != 0 ? kRejected : kAccepted;
      }
      return;
    }
    __syncthreads();
  }
  if (!kLists && p.cap > 0) {  // the launch behind the lists': open rows that no known rejection is before
    static_assert(kQuickRows <= 64, "a lane each");
    const int own = p.stat[id].verdict;  // (neither these are written by this launch's others)
    const int v = lane < min(i, kQuickRows) ? p.stat[(int64_t)b * T + lane].verdict : kOpen;
    if (own != kOpen || __ballot(v == kRejected) != 0) return;
  }
  const RowSummary sum = summarize(p, id, lane, own_group);
  const float mx = sum.max;
  const int mode = sum.mode;
  const double mxd = (double)mx, all = sum.mass;
  auto weight = [&](float l) __attribute__((always_inline)) { return exp2_neg((double)l - mxd, p.scale, p.d_min); };
  const double goal = p.top_p * all;  // in units of the largest weight
  auto enough = [&](uint32_t c, uint64_t m) {
    return c >= (uint32_t)p.top_k || (p.use_mass && (double)m * kMassUnit >= goal);
  };
  const bool by_count = p.top_k < V;
  // floor: a value that tau cannot lie below; entries under it are left out of the search.  By count: the
  // smallest of the groups' floors has top_k entries at or above it, listed.  By mass: the entries lighter than
  // (1 - top_p) all / V together hold less than 1 - top_p of it, so the others hold top_p (with room for
  // the roundings of the logarithm and of the sum).  Masked entries have no weight.
  float floor0 = sum.floor;
  if (p.use_mass) {
    const float least = (float)(p.light * all);
    if (least > 1.0e-30f) floor0 = fmaxf(floor0, (float)(mxd + ((double)__log2f(least) - 0.01) * p.unscale));
  }
  floor0 = fmaxf(floor0, -FLT_MAX);

  auto entries = [&](int j, R x) __attribute__((always_inline)) -> f4 {
    f4 l = to_f4(x);
#pragma unroll
    for (int e = 0; e < 4; ++e) l[e] = __builtin_isnan(l[e]) ? 0.0f : l[e];
    if (mode != kNanZero)
      for (int e = 0; e < 4; ++e) l[e] = read_as(l[e], mode);
    if ((j + 1) * kTile > V && j * kTile + 4 * t >= V) l = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    return l;
  };
  // f(four entries) over this lane's part of the row, eight tiles' loads at a time; padding is -inf
  auto each_row = [&](auto&& f) __attribute__((always_inline)) {
    constexpr int kB = kLists ? 4 : 8;  // (lists: no registers for more)
    for (int j = 0; j < tiles; j += kB) {
      R x[kB];
#pragma unroll
      for (int u = 0; u < kB; ++u) x[u] = load_raw<kHalf>(row, min((j + u) * kTile + 4 * t, V - 4));
#pragma unroll
      for (int u = 0; u < kB; ++u) {
        if (j + u >= tiles) break;
        f(entries(j + u, x[u]));
      }
    }
  };

  // The lists: four entries per lane.
  bool listed = kLists && sum.reach <= mx;  // (else none is listed)
  float mine[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  int mine_at[4] = {-1, -1, -1, -1};
  if (listed) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (list_place[u] < list_count[u]) {
        mine[u] = listed_at[u].x;
        mine_at[u] = __builtin_bit_cast(int, listed_at[u].y);
      }
    }
  }
  uint32_t none = 0, none2 = 0;
  if (kLists && !listed && p.again) {
    if (t == 0) p.stat[id].verdict = kOpen;
    return;
  }
  auto each4 = [&](auto&& f) __attribute__((always_inline)) {
    if (kLists && listed) f(f4{mine[0], mine[1], mine[2], mine[3]});
    else each_row(f);
  };
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    each4([&](f4 x) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(x[e]);
    });
  };

  RowStat st;
  st.max = mx;
  st.mode = mode;
  st.ok = 0;
  st.token = -1;
  st.verdict = kOpen;
  for (;;) {
    const float floor = listed ? fmaxf(floor0, sum.reach) : floor0;
    // Histogram of (mx - l) in kBins equal steps: 32 per octave of the weight, or finer where the
    // entries from floor up span less.  Larger l never falls in a later bin.
    const float far = mx - floor, bin_scale = p.bin_scale * ((float)kBins / kVerBins);
    const float s = far > 0.0f ? fminf(fmaxf(bin_scale, (float)(kBins - 1) / far), FLT_MAX) : bin_scale;
    auto bin_at = [&](float l) __attribute__((always_inline)) { return fminf((mx - l) * s, (float)(kBins - 1)); };
    for (int k = t; k < kBins; k += kThreads) {
      sh.cnt[k] = 0;
      sh.mass[k] = 0;
    }
    if (t == 0) {
      sh.n_cand = 0;
      sh.bin = kBins;
    }
    __syncthreads();
    each4([&](f4 x) __attribute__((always_inline)) {
      if (__ballot(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= floor) == 0) return;
      uint64_t m[4];
      if (p.use_mass) {
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = mass_of(weight(x[e]));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (x[e] >= floor) {
          const int k = (int)bin_at(x[e]);
          if (by_count) atomicAdd(&sh.cnt[k], 1u);
          if (p.use_mass) atomicAdd((unsigned long long*)&sh.mass[k], (unsigned long long)m[e]);
        }
      }
    });
    __syncthreads();
    // inclusive prefix over the bins (kPer per lane) and the first bin that reaches the budget
    constexpr int kPer = kBins / kThreads;
    uint32_t c[kPer], ci = 0;
    uint64_t m[kPer], mi = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      ci += c[k] = sh.cnt[kPer * t + k];
      mi += m[k] = sh.mass[kPer * t + k];
    }
    const uint32_t c_own = ci;
    const uint64_t m_own = mi;
    ci = wave_scan(ci, lane);
    mi = wave_scan(mi, lane);
    if (lane == 63) {
      sh.redc[par][wv] = ci;
      sh.redm[par][wv] = mi;
    }
    __syncthreads();
    ci += lanes_add<W>((lane & (W - 1)) < wv ? sh.redc[par][lane & (W - 1)] : 0u);
    mi += lanes_add<W>((lane & (W - 1)) < wv ? sh.redm[par][lane & (W - 1)] : (uint64_t)0);
    par ^= 1;
    if (enough(ci, mi) && !enough(ci - c_own, mi - m_own)) {
      uint32_t cb = ci - c_own;
      uint64_t mb = mi - m_own;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        if (enough(cb + c[k], mb + m[k])) {
          sh.bin = kPer * t + k;
          sh.before_c = cb;
          sh.before_m = mb;
          break;
        }
        cb += c[k];
        mb += m[k];
      }
    }
    __syncthreads();
    const bool found = sh.bin < kBins;
    if (kLists && !found && listed && sum.reach > -FLT_MAX) {  // tau lies below the lists' reach: the whole row
      if (p.again) {
        if (t == 0) p.stat[id].verdict = kOpen;
        return;
      }
      __syncthreads();
      listed = false;
      continue;
    }
    // Not found: fewer entries than top_k have a weight at all (the others are masked); all are kept.
    const int bin = found ? sh.bin : kBins - 1;
    const uint32_t before_c = found ? sh.before_c : 0;
    const uint64_t before_m = found ? sh.before_m : 0;
    if (found) {
      const float bf = (float)bin;
      // the bin's span in logits with room for rounding, so that most groups are passed over quickly
      const float room = 1.0e-5f * (fabsf(mx) + (float)kBins / s);
      const float top = bin == 0 ? mx : mx - bf / s + room;
      const float low = bin == kBins - 1 ? floor : fmaxf(floor, mx - (bf + 1.0f) / s - room);
      each4([&](f4 x) __attribute__((always_inline)) {
        bool in[4], any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) any = any || (x[e] >= low && x[e] <= top);
        if (__ballot(any) == 0) return;
        any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float at = bin_at(x[e]);
          in[e] = at >= bf && at < bf + 1.0f && x[e] >= floor;
          any = any || in[e];
        }
        if (__ballot(any) == 0) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (in[e]) {
            const int at = atomicAdd(&sh.n_cand, 1);  // any order: only sums and a maximum follow
            if (at < kCand) {
              sh.cand[at] = x[e];
              sh.candm[at] = p.use_mass ? mass_of(weight(x[e])) : 0;
            }
          }
        }
      });
    }
    __syncthreads();
    const int in_bin = found ? sh.n_cand : kCand + 1;
    uint32_t ngt = 0, neq = 0;
    uint64_t mgt = 0;
    if (in_bin <= kCand) {
      uint32_t c = before_c;
      uint64_t m = before_m;
      float v = -INFINITY;
      if (t < 4 && in_bin + t < kCand) sh.cand[in_bin + t] = -INFINITY;  // fills the last group of four
      __syncthreads();
      if (t < in_bin) {
        v = sh.cand[t];
        for (int k = 0; k < in_bin; k += 4) {
          const f4 o = *reinterpret_cast<const f4*>(&sh.cand[k]);
          uint64_t om[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) om[e] = sh.candm[k + e];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            c += o[e] >= v ? 1u : 0u;
            m += o[e] >= v ? om[e] : 0;
          }
        }
      }
      st.tau = block_max<W>(sh, par, t < in_bin && enough(c, m) ? v : -INFINITY);
      ngt = t < in_bin && v > st.tau ? 1 : 0;
      neq = t < in_bin && v == st.tau ? 1 : 0;
      mgt = ngt ? sh.candm[t] : 0;
      block_add<W>(sh, par, ngt, neq, mgt);
      ngt += before_c;
      mgt += before_m;
    } else {
      // many entries in one bin (ties, or a spread that outliers stretch): bisection over the keys of
      // every entry, at most 32 rounds, for the largest value with enough entries at or above it
      uint32_t lo = key_of(found ? floor : -FLT_MAX), hi = found ? key_of(mx) : lo;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2u + 1u;
        const float v = of_key(mid);
        uint32_t c = 0;
        uint64_t m = 0;
        each([&](float l) {
          if (l >= v) {
            c += 1;
            m += p.use_mass ? mass_of(weight(l)) : 0;
          }
        });
        block_add<W>(sh, par, c, none, m);
        if (enough(c, m)) lo = mid;
        else hi = mid - 1u;
      }
      // lo may lie below every entry: then tau is the smallest of them
      float least = -INFINITY;
      const float lov = of_key(lo);
      each([&](float l) { least = l >= lov ? fmaxf(least, -l) : least; });
      st.tau = -block_max<W>(sh, par, least);
      each([&](float l) {
        ngt += l > st.tau ? 1 : 0;
        neq += l == st.tau ? 1 : 0;
        mgt += l > st.tau && p.use_mass ? mass_of(weight(l)) : 0;
      });
      block_add<W>(sh, par, ngt, neq, mgt);
    }
    if (!p.use_mass) {  // the mass above tau was not needed so far
      mgt = 0;
      each4([&](f4 x) __attribute__((always_inline)) {
        if (__ballot(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > st.tau) == 0) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) mgt += x[e] > st.tau ? mass_of(weight(x[e])) : 0;
      });
      block_add<W>(sh, par, none, none2, mgt);
    }
    const double x = weight(st.tau);
    double comp = by_count ? (double)((int64_t)p.top_k - (int64_t)ngt) / (double)neq : 1.0;
    if (p.use_mass) comp = fmin(comp, (goal - (double)mgt * kMassUnit) / (x * (double)neq));
    comp = fmax(fmin(comp, 1.0), 0.0);
    // no entry above tau: the kept ones are ties, whose common share does not matter
    st.comp = mgt == 0 ? 1.0 : comp;
    st.z = (double)mgt * kMassUnit + st.comp * x * (double)neq;
    break;
  }

  const double unit = 1.0 / st.z;
  if (t == 0 && draft.in)
    st.ok = (double)draft.u * (double)draft.q < kept_of(p, st, read_as(draft.l, mode)) * unit ? 1 : 0;
  // The token if the sequence stops here: all kept entries are listed.  Sorted by index (places counted,
  // so that the sums' order does not hang on the order of the atomics), then the prefix sums in one wave.
  if (kLists && listed) {
    if (t == 0) {
      sh.n_cand = 0;
      sh.bin = st.ok;
    }
    if (t < kVerDraw) sh.draw.at[t] = INT_MAX;
    const int d = i < n ? lookup : -1;
    double w[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (!(mine[u] >= st.tau && mine[u] > -INFINITY)) continue;
      w[u] = kept_of(p, st, mine[u]) * unit;
      if (i < n && p.q) w[u] = fmax(w[u] - (double)p.q[((int64_t)b * p.K + i) * V + mine_at[u]], 0.0);
      if (mine_at[u] == d) w[u] = 0.0;
    }
    __syncthreads();
    if (sh.bin == 0) {  // not where the draft is accepted
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (mine[u] >= st.tau && mine[u] > -INFINITY) {
          const int at = atomicAdd(&sh.n_cand, 1);
          if (at < kVerDraw) {
            sh.draw.w[at] = w[u];
            sh.draw.at[at] = mine_at[u];
          }
        }
      }
    }
    __syncthreads();
    const int kept = sh.n_cand;
    if (kept > 0 && kept <= kVerDraw) {
      if (t < kept) {
        const int my = sh.draw.at[t];
        int place = 0;
        for (int k = 0; k < kept; k += 16) {
          int4 o[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) o[u] = *reinterpret_cast<const int4*>(&sh.draw.at[k + 4 * u]);
#pragma unroll
          for (int u = 0; u < 4; ++u) place += (o[u].x < my) + (o[u].y < my) + (o[u].z < my) + (o[u].w < my);
        }
        sh.draw.sorted_w[place] = sh.draw.w[t];
        sh.draw.sorted_at[place] = my;
      }
      __syncthreads();
      if (wv == 0) {
        double x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = 4 * lane + e < kept ? sh.draw.sorted_w[4 * lane + e] : 0.0;
        const double s = (x[0] + x[1]) + (x[2] + x[3]);
        const double incl = wave_scan(s, lane);
        const double total = lane_read(incl, 63), target = (double)last_u * total;
        double run = incl - s;
        int pick = -1, end = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          run += x[e];
          if (x[e] > 0.0) {
            end = 4 * lane + e;
            if (pick < 0 && run > target) pick = 4 * lane + e;
          }
        }
        const uint64_t hit = __ballot(pick >= 0), any = __ballot(end >= 0);
        if (hit) st.token = sh.draw.sorted_at[__builtin_amdgcn_readlane(pick, __builtin_ctzll(hit))];
        else if (any) st.token = sh.draw.sorted_at[__builtin_amdgcn_readlane(end, 63 - __builtin_clzll(any))];
      }
    }
  }
  if (t == 0) {
    if (kLists && p.again) st.verdict = st.ok ? kAccepted : kRejected;
    p.stat[id] = st;
  }
}

// What the last two kernels share: the row a sequence stops at and the weights it draws from.  Without a
// filter the workgroup's kWaves waves make the rows' statistics from the groups' sums, a row each.
struct StopShared {
  RowStat stat[64];
};
template <bool kHalf, int kWaves>
struct Stop {
  const VerifyArgs& p;
  int64_t id;      // row b (K + 1) + j
  int j, draft;
  const float* q;  // the drafter's row, where j is a rejected draft's and there is one
  bool beyond;     // draw from what p has beyond q
  RowStat st;
  double unit, unit_tau;  // of a weight above tau, and at it
  const void* row;

  __device__ __forceinline__ Stop(const VerifyArgs& a, StopShared& sh, int b, int n, int lane, int wv) : p(a) {
    const int T = p.K + 1;
    j = -1;
    for (int k0 = 0; j < 0; k0 += 64) {  // 64 rows at a time; row n ends the search
      bool last = k0 + lane >= n;
      if (p.truncate) {
        last = last || !p.stat[(int64_t)b * T + k0 + lane].ok;
      } else {
        if (k0 > 0) __syncthreads();
        for (int k = wv; k < 64 && k0 + k <= n; k += kWaves) {
          const int64_t r = (int64_t)b * T + k0 + k;
          Draft d{false, 0.0f, 1.0f, 0.0f};
          if (k0 + k < n) d = load_draft<kHalf>(p, b, k0 + k);
          const RowSummary sum = summarize(p, r, lane);
          RowStat s{sum.mass, 1.0, sum.max, -INFINITY, 0, sum.mode, -1, 0};
          s.ok = d.in && (double)d.u * (double)d.q < kept_of(p, s, read_as(d.l, sum.mode)) / s.z ? 1 : 0;
          if (lane == 0) sh.stat[k] = s;
        }
        __syncthreads();
        last = last || !sh.stat[lane].ok;
      }
      const uint64_t hit = __ballot(last);
      if (hit) j = k0 + __builtin_ctzll(hit);
    }
    id = (int64_t)b * T + j;
    st = p.truncate ? p.stat[id] : sh.stat[j & 63];
    row = row_at<kHalf>(p, id);
    beyond = j < n;
    q = p.q && beyond ? p.q + ((int64_t)b * p.K + j) * p.V : nullptr;
    draft = beyond && !p.q ? p.drafts[(int64_t)b * p.K + j] : -1;
    unit = 1.0 / st.z;
    unit_tau = unit * st.comp;
  }
  __device__ __forceinline__ f4 load_l(int at) const {
    f4 x = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (at < p.V) {
      x = to_f4(load_raw<kHalf>(row, at));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = read_as(x[e], st.mode);
    }
    return x;
  }
  __device__ __forceinline__ f4 load_q(int at) const {
    return q && beyond && at < p.V ? *reinterpret_cast<const f4*>(q + at) : f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // weights of the four entries at `at`
  __device__ __forceinline__ void weights(f4 l, f4 qv, int at, double* w) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = 0.0;
    if (p.truncate && __ballot(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= st.tau) == 0) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double x = exp2_neg((double)l[e] - (double)st.max, p.scale, p.d_min);
      w[e] = x * (l[e] > st.tau ? unit : l[e] == st.tau ? unit_tau : 0.0);
    }
    if (!beyond) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = p.q ? fmax(w[e] - (double)qv[e], 0.0) : at + e == draft ? 0.0 : w[e];
  }
};

// The segments' sums of w for the row each sequence stops at (not where the sums' kernel left them:
// without a filter, all drafts accepted).  A workgroup takes 8 segments for each of its 4 waves.  128 rows of
// 65536 fp32 entries and as many of the drafter's: 19 us, 3.5 TB/s.
constexpr int kPartSegs = 8;
template <bool kHalf>
__global__ __launch_bounds__(256) void verify_parts_kernel(VerifyArgs p) {
  __shared__ StopShared shared;
  const int parts = (p.segs + 4 * kPartSegs - 1) / (4 * kPartSegs);
  const int b = blockIdx.x / parts, part = blockIdx.x - b * parts, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  if (n < 0 || n > p.K) return;
  const Stop<kHalf, 4> stop(p, shared, b, n, lane, wv);
  if (p.truncate ? stop.st.token >= 0 : !stop.beyond) return;
  const int seg0 = (part * 4 + wv) * kPartSegs;
  f4 l[kPartSegs], qv[kPartSegs];
#pragma unroll
  for (int k = 0; k < kPartSegs; ++k) {
    const int at = (seg0 + k) * kSeg + 4 * lane;
    l[k] = stop.load_l(at);
    qv[k] = stop.load_q(at);
  }
  double* const sums = p.part_sum + (int64_t)b * p.segs + seg0;
#pragma unroll
  for (int k0 = 0; k0 < kPartSegs; k0 += 4) {
    double s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      double w[4];
      stop.weights(l[k0 + u], qv[k0 + u], (seg0 + k0 + u) * kSeg + 4 * lane, w);
      s[u] = (w[0] + w[1]) + (w[2] + w[3]);
    }
    const double w = wave_add4(s, lane);
    if (lane < 4 && seg0 + k0 + lane < p.segs) sums[k0 + lane] = w;
  }
}

constexpr int kDrawThreads = 512;
struct DrawShared {
  StopShared stop;
  double sum[kMaxSegs];
  double red[kDrawThreads / 64];
  int first, last;
};

// One workgroup per sequence: the segment that holds the target, then the entry.  Dependent loads: 6 us,
// or 4 where the rows' kernel left the token.
template <bool kHalf>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs p) {
  __shared__ DrawShared sh;
  const int T = p.K + 1, b = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6, segs = p.segs;
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  const double u = (double)p.u[(int64_t)b * T + p.K];
  int32_t* out = p.tokens + (int64_t)b * T;
  if (n < 0 || n > p.K) {
    for (int k = t; k < T; k += kDrawThreads) out[k] = -1;
    if (t == 0) p.accepted[b] = -1;
    return;
  }
  Stop<kHalf, kDrawThreads / 64> stop(p, sh.stop, b, n, lane, wv);
  const int j = stop.j;
  for (int k = t; k < T; k += kDrawThreads)
    if (k != j) out[k] = k < j ? p.drafts[(int64_t)b * p.K + k] : -1;
  if (t == 0) p.accepted[b] = j;
  if (stop.st.token >= 0) {
    if (t == 0) out[j] = stop.st.token;
    return;
  }
  const bool parts = p.truncate ? p.cap == 0 || p.again : stop.q != nullptr;  // the parts' kernel has run
  // the sum of segment k by one wave (the rows' and parts' kernels' order of additions aside)
  auto segment = [&](int k) {
    double w[4];
    const int at = k * kSeg + 4 * lane;
    stop.weights(stop.load_l(at), stop.load_q(at), at, w);
    return wave_add((w[0] + w[1]) + (w[2] + w[3]));
  };
  const int per = (segs + kDrawThreads - 1) / kDrawThreads;  // segments per lane of the scan: at most 8
  const int k0 = min(t * per, segs), k1 = min(k0 + per, segs);
  double total, run0;
  for (bool again = false;; again = true) {
    if (again || (p.truncate && !parts)) {
      // nothing beyond the drafter's probabilities (then p itself), or lists that did not reach down to tau
      for (int k = wv; k < segs; k += kDrawThreads / 64) {
        const double s = segment(k);
        if (lane == 0) sh.sum[k] = s;
      }
    } else {
      // the sums' kernel's are relative to their group's largest weight, and hold a lookup's rejected draft
      const int own = !parts && stop.draft >= 0 && stop.draft < p.V ? stop.draft / kSeg : -1;
      const double* src = parts ? p.part_sum + (int64_t)b * segs : p.seg_sum + stop.id * segs;
      const float top = stop.st.mode == kInfOnly ? INFINITY : stop.st.max;
      for (int k = t; k < segs; k += kDrawThreads) {
        if (k == own) continue;
        double s;
        if (parts) s = src[k];
        else if (stop.st.mode == kAllLow) s = (double)(min(p.V, (k + 1) * kSeg) - k * kSeg) * stop.unit;
        else {
          const float gm = p.group_max[stop.id * p.groups + k / kGroupSegs];
          s = gm > -INFINITY ? src[k] * group_factor(p, gm, top) : 0.0;
          // (weights end at 2^-1022: a sum of 256 down to 2^-1013 has one that is more than 0, a smaller one
          // may have none, and a uniform of 0 would fall on it)
          s = s >= 0x1p-1013 ? s * stop.unit : 0.0;
        }
        sh.sum[k] = s;
      }
      if (own >= 0 && wv == kDrawThreads / 64 - 1) {  // the wave with the fewest sums to load
        const double s = segment(own);
        if (lane == 0) sh.sum[own] = s;
      }
    }
    if (t == 0) {
      sh.first = segs;
      sh.last = -1;
    }
    __syncthreads();
    double s = 0.0;
    for (int k = k0; k < k1; ++k) s += sh.sum[k];
    const double incl = wave_scan(s, lane);
    if (lane == 63) sh.red[wv] = incl;
    __syncthreads();
    const double of_wave = sh.red[lane & 7];
    total = oct_add(of_wave);
    run0 = oct_add((lane & 7) < wv ? of_wave : 0.0) + incl - s;
    if (total > 0.0 || !stop.beyond) break;
    stop.beyond = false;
    __syncthreads();
  }
  const double target = u * total;
  {
    double run = run0;
    int first = segs, last = -1;
    for (int k = k0; k < k1; ++k) {
      const double s = sh.sum[k];
      if (s > 0.0) {
        last = k;
        if (run + s > target && first == segs) first = k;
      }
      run += s;
    }
    // lanes hold segments in order; an atomic per wave (per lane the compiler puts a loop over the lanes around
    // it, 4 us)
    const uint64_t hit = __ballot(first < segs), any = __ballot(last >= 0);
    if (hit && lane == __builtin_ctzll(hit)) atomicMin(&sh.first, first);
    if (any && lane == 63 - __builtin_clzll(any)) atomicMax(&sh.last, last);
  }
  __syncthreads();
  // the segment that holds the target (rounding short of the end: the last with weight), by one wave
  const int seg = sh.first < segs ? sh.first : sh.last;
  if (wv != 0) return;
  if (seg < 0) {
    if (lane == 0) out[j] = -1;
    return;
  }
  const int at = seg * kSeg + 4 * lane;
  const f4 l = stop.load_l(at), qv = stop.load_q(at);
  double before = 0.0;
  for (int k = lane; k < seg; k += 64) before += sh.sum[k];
  before = wave_add(before);
  double w[4];
  stop.weights(l, qv, at, w);
  const double mine = (w[0] + w[1]) + (w[2] + w[3]);
  double run = before + wave_scan(mine, lane) - mine;
  int pick = -1, end = -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    run += w[e];
    if (w[e] > 0.0) {
      end = at + e;
      if (pick < 0 && run > target) pick = at + e;
    }
  }
  const uint64_t hit = __ballot(pick >= 0), any = __ballot(end >= 0);
  if (hit) {
    if (lane == __builtin_ctzll(hit)) out[j] = pick;
  } else if (any) {
    if (lane == 63 - __builtin_clzll(any)) out[j] = end;
  }
}

template <bool kHalf>
void launch_verify(const VerifyArgs& a, int B, hipStream_t s) {
  const unsigned rows = (unsigned)B * (a.K + 1);
  hipLaunchKernelGGL(verify_sums_kernel<kHalf>, dim3(rows * ((a.groups + 3) / 4)), dim3(256), 0, s, a);
  if (a.truncate) {
    // As a whole: up to a row per CU 16 waves each, more rows 8, two workgroups to a CU (nucleus of 65536
    // entries, 4 drafts: 16 sequences 67 us with 16 waves, 77 with 8; 128 sequences 140 and 128).
    if (a.cap > 0)
      hipLaunchKernelGGL((verify_rows_kernel<kHalf, true, kListThreads>), dim3(rows), dim3(kListThreads), 0, s, a);
    if ((a.cap == 0 || a.again) && rows <= (unsigned)device_cus())
      hipLaunchKernelGGL((verify_rows_kernel<kHalf, false, 1024>), dim3(rows), dim3(1024), 0, s, a);
    else if (a.cap == 0 || a.again)
      hipLaunchKernelGGL((verify_rows_kernel<kHalf, false, 512>), dim3(rows), dim3(512), 0, s, a);
  }
  if (a.truncate ? a.cap == 0 || a.again : a.q != nullptr)
    hipLaunchKernelGGL(verify_parts_kernel<kHalf>, dim3(B * ((a.segs + 4 * kPartSegs - 1) / (4 * kPartSegs))), dim3(256), 0,
                       s, a);
  hipLaunchKernelGGL(verify_draw_kernel<kHalf>, dim3(B), dim3(kDrawThreads), 0, s, a);
}

// Entries listed per group: kVerList per row, at most 128; no lists for rows of more than 64 groups.
int list_cap(int64_t groups) { return groups <= 64 ? (int)std::min<int64_t>(128, kVerList / groups) : 0; }

// Workspace: row statistics, segments', groups' and parts' sums, groups' maxima, floors and lists.
struct VerifySpace {
  int64_t seg_sum, group_sum, part_sum, list, group_max, group_floor, group_count, bytes;
};
VerifySpace verify_space(int64_t B, int64_t K, int64_t V) {
  const int64_t rows = B * (K + 1), segs = (V + kSeg - 1) / kSeg, groups = (segs + kGroupSegs - 1) / kGroupSegs;
  VerifySpace w;
  w.seg_sum = rows * (int64_t)sizeof(RowStat);
  w.group_sum = w.seg_sum + rows * segs * 8;
  w.part_sum = w.group_sum + rows * groups * 8;
  w.list = w.part_sum + B * segs * 8;
  w.group_max = w.list + rows * groups * list_cap(groups) * 8;
  w.group_floor = w.group_max + rows * groups * 4;
  w.group_count = w.group_floor + rows * groups * 4;
  w.bytes = w.group_count + rows * groups * 4;
  return w;
}

// A launch has fewer than 2^32 threads: 256 per 8192 entries of a row, 1024 per row.
bool verify_rows_fit(int64_t B, int64_t K, int64_t V) {
  return B * (K + 1) <= (1 << 22) / std::max<int64_t>(4, (V + 8191) / 8192);
}

// Lists pay where they nearly always reach down to the top_k-th entry.  The r-th largest of 16 lane maxima
// of 32 entries each has about 64 (-ln(1 - r / 16)) of a group's 2048 entries above it; the largest r
// that leaves the list a third of room is taken.  That has to hold a group's share of the top_k: m = top_k
// / groups on average, hardly ever more than m + 5 sqrt(m) + 3 where they are spread at random.  24
// sequences of 5 drafts, 65536 entries, top_k 40: 41 us without lists, 26.5 with, 87 where all 40 are side by
// side in one group, whose list ends above the last of them.
// A nucleus (top_p without a top_k that lists hold) is a few entries or most of the row; rows that the lists
// leave open are searched as a whole by a launch of their own.  128 sequences of 4 drafts, 65536 fp32
// entries: nuclei of 4 entries 70 us (96 without lists), of 85 72 (109), of 32000 149 (130); 4 sequences: 21 (42),
// 23 (49), 69 (63).
void use_lists(VerifyArgs& a) {
  a.cap = a.truncate ? list_cap(a.groups) : 0;
  a.rank = 0;
  const auto above = [](int r) { return -64.0 * std::log1p(-r / 16.0); };
  while (a.rank < 14 && above(a.rank + 1) * 1.33 <= a.cap) ++a.rank;
  const double m = (double)a.top_k / a.groups;
  const bool hold = a.top_k < a.V && above(a.rank) >= (a.groups > 1 ? m + 5.0 * std::sqrt(m) + 3.0 : m);
  a.again = a.cap > 0 && !hold && a.use_mass;
  if (!hold && !a.again) a.cap = a.rank = 0;
}

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int64_t vkwr_sampling_verify_workspace_bytes(int B, int K, int V) {
  if (B <= 0 || K < 0 || V <= 0 || V > kVerMaxV || !verify_rows_fit(B, K, V)) return 0;  // refused
  return verify_space(B, K, V).bytes;
}

extern "C" int vkwr_sampling_verify_drafts(int B, int K, int V, const void* logits, int logits_f16,
                                           const int32_t* drafts, const int32_t* n_draft, const float* draft_probs,
                                           const float* uniforms, int32_t* tokens, int32_t* accepted,
                                           double temperature, int top_k, double top_p, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "vkwr_sampling_verify_drafts";
  VK_REQUIRE(B >= 0 && K >= 0, "%s: negative size (B=%d K=%d)", fn, B, K);
  VK_REQUIRE(V > 0 && V <= kVerMaxV && V % 4 == 0,
             "%s: vocabulary size must be a multiple of 4 and at most 1048576, got %d", fn, V);
  VK_REQUIRE(temperature >= 0.001 && temperature <= 1000, "%s: temperature %g outside [0.001, 1000]", fn,
             temperature);
  VK_REQUIRE(verify_rows_fit(B, K, V), "%s: B*(K+1) too large", fn);
  if (B == 0) return VKWR_OK;
  VK_REQUIRE(logits && uniforms && tokens && accepted && (K == 0 || drafts), "%s: null pointer", fn);
  VK_REQUIRE((uintptr_t)logits % (logits_f16 ? 8 : 16) == 0 && (uintptr_t)draft_probs % 16 == 0,
             "%s: logits must be %d-byte and draft_probs 16-byte aligned", fn, logits_f16 ? 8 : 16);
  const int64_t need = vkwr_sampling_verify_workspace_bytes(B, K, V);
  VK_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0,
             "%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)need);
  if (top_k <= 0 || top_k > V) top_k = V;
  if (!(top_p >= 0 && top_p <= 1)) top_p = 1;
  if (top_p == 0) {
    top_k = 1;
    top_p = 1;
  }
  VerifyArgs a{};
  a.K = K;
  a.V = V;
  a.logits = logits;
  a.drafts = drafts;
  a.n_draft = n_draft;
  a.q = K > 0 ? draft_probs : nullptr;
  a.u = uniforms;
  a.tokens = tokens;
  a.accepted = accepted;
  char* const ws = reinterpret_cast<char*>(workspace);
  const VerifySpace w = verify_space(B, K, V);
  a.stat = reinterpret_cast<RowStat*>(ws);
  a.seg_sum = reinterpret_cast<double*>(ws + w.seg_sum);
  a.group_sum = reinterpret_cast<double*>(ws + w.group_sum);
  a.part_sum = reinterpret_cast<double*>(ws + w.part_sum);
  a.group_max = reinterpret_cast<float*>(ws + w.group_max);
  a.group_floor = reinterpret_cast<float*>(ws + w.group_floor);
  a.group_count = reinterpret_cast<int32_t*>(ws + w.group_count);
  a.list = reinterpret_cast<float2*>(ws + w.list);
  a.segs = (V + kSeg - 1) / kSeg;
  a.groups = (a.segs + kGroupSegs - 1) / kGroupSegs;
  a.scale = 1.4426950408889634 / temperature;
  a.d_min = -1023.0 / a.scale;
  a.unscale = 1.0 / a.scale;
  a.light = (1.0 - top_p) / V;
  a.bin_scale = (float)(32.0 * a.scale);
  a.top_k = top_k;
  a.top_p = top_p;
  a.use_mass = top_p < 1.0;
  a.truncate = top_k < V || a.use_mass;
  use_lists(a);
  if (logits_f16) launch_verify<true>(a, B, (hipStream_t)stream);
  else launch_verify<false>(a, B, (hipStream_t)stream);
  return check_launch(fn);
}
