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
// uniform lies within ~1e-11 of a border.
//
// Launches: one workgroup per row finds max, tau, comp and Z and tests the row's draft; the row that a
// sequence stops at is added up in segments of 256 entries, by several workgroups (without a filter and
// without a drafter's distribution the rows' workgroups have done that already: no launch); one
// workgroup per sequence finds the segment and the entry that the uniform falls on.

#include <cfloat>

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

constexpr int kVerThreads = 1024;
constexpr int kVerWaves = kVerThreads / 64;
constexpr int kVerBins = 2048;   // histogram of (max - l) for the threshold
constexpr int kVerCand = 512;    // entries of one bin that are ranked directly
constexpr int kVerTile = 4 * kVerThreads;  // consecutive entries a workgroup reads at once
constexpr int kVerMaxV = 1 << 20;
constexpr int kSeg = 256;        // consecutive entries whose weights are added up for the draw (one wave's 64 x 4)
constexpr int kMaxSegs = kVerMaxV / kSeg;
constexpr double kMassUnit = 1.0 / 8796093022208.0;  // 2^-43

struct RowStat {
  double z, comp;
  float max, tau;
  int ok, mode;
};
// How a row's logits are read so that only finite values and -inf (weight 0) remain:
enum {
  kPlain = 0,   // as they are: no NaN and no +inf
  kNanZero = 1, // NaN -> 0
  kInfOnly = 2, // +inf present (it stands for the largest float, beside which every finite value
                // weighs nothing): +inf -> 0, anything else -> -inf
  kAllLow = 3   // -inf everywhere: all entries tied
};
static_assert(sizeof(RowStat) == 32, "row stat size");

struct VerifyArgs {
  int K, V;
  const void* logits;
  const int32_t *drafts, *n_draft;
  const float *q, *u;
  int32_t *tokens, *accepted;
  RowStat* stat;   // [B, K+1]
  double* sums;    // [B, K+1, segments] what the segments of a row hold
  int segs;
  double scale, d_min;  // log2(e) / temperature; -1023 / scale (weight 0)
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
  uint64_t mass[kVerBins];
  uint32_t cnt[kVerBins];
  uint64_t redm[2][kVerWaves];
  double redd[2][kVerWaves];
  uint32_t redc[2][kVerWaves], rede[2][kVerWaves];
  float redf[2][kVerWaves], redg[2][kVerWaves];
  alignas(16) float cand[kVerCand];
  uint64_t candm[kVerCand];
  int n_cand, bin;
  uint32_t before_c;
  uint64_t before_m;
};

// Sum (maximum) of the 16 values that the lanes of a row hold, in every lane.
template <class X>
__device__ __forceinline__ X row_add(X x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  return x + dpp<0x140>(x);
}
__device__ __forceinline__ float row_fmax(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  return fmaxf(x, dpp<0x140>(x));
}

// Block reductions with one barrier: consecutive ones alternate between two buffers (par), so a wave
// overwrites a buffer only behind the barrier that every wave reaches after reading it.  Each row of 16
// lanes adds the 16 wave values.
static_assert(kVerWaves == 16, "a row of lanes holds the wave values");
__device__ __forceinline__ void block_max2(StatShared& sh, int& par, float& a, float& b) {
  a = wave_fmax(a);
  b = wave_fmax(b);
  if ((threadIdx.x & 63) == 0) {
    sh.redf[par][threadIdx.x >> 6] = a;
    sh.redg[par][threadIdx.x >> 6] = b;
  }
  __syncthreads();
  a = row_fmax(sh.redf[par][threadIdx.x & 15]);
  b = row_fmax(sh.redg[par][threadIdx.x & 15]);
  par ^= 1;
}
__device__ __forceinline__ float block_max(StatShared& sh, int& par, float a) {
  a = wave_fmax(a);
  if ((threadIdx.x & 63) == 0) sh.redf[par][threadIdx.x >> 6] = a;
  __syncthreads();
  a = row_fmax(sh.redf[par][threadIdx.x & 15]);
  par ^= 1;
  return a;
}
__device__ __forceinline__ double block_sum(StatShared& sh, int& par, double a) {
  a = wave_add(a);
  if ((threadIdx.x & 63) == 0) sh.redd[par][threadIdx.x >> 6] = a;
  __syncthreads();
  a = row_add(sh.redd[par][threadIdx.x & 15]);
  par ^= 1;
  return a;
}
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
  const int w = threadIdx.x & 15;
  a = row_add(sh.redc[par][w]);
  b = row_add(sh.rede[par][w]);
  m = row_add(sh.redm[par][w]);
  par ^= 1;
}

__device__ __forceinline__ float read_as(float l, int mode) {
  if (mode == kInfOnly) return l == INFINITY ? 0.0f : -INFINITY;
  if (mode == kAllLow) return 0.0f;
  return __builtin_isnan(l) ? 0.0f : l;
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
struct Elem {
  typedef _Float16 type;
};
template <>
struct Elem<false> {
  typedef float type;
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

// kTiles > 0: the row (V <= kTiles * kVerTile) stays in LDS as stored; 0: it is re-read from memory in
// every pass.
template <bool kHalf, int kTiles>
__global__ __launch_bounds__(kVerThreads) void verify_rows_kernel(VerifyArgs p) {
  typedef typename Raw<kHalf>::type R;
  __shared__ StatShared sh;
  __shared__ R lrow[kTiles > 0 ? kTiles * kVerThreads : 1];
  const int T = p.K + 1;
  const int b = blockIdx.x / T, i = blockIdx.x - b * T;
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  if (n < 0 || n > p.K || i > n) return;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = p.V;
  const void* row = row_at<kHalf>(p, (int64_t)b * T + i);
  const int tiles = (V + kVerTile - 1) / kVerTile;
  int par = 0, mode = kPlain;
  typedef typename Elem<kHalf>::type E;
  const E kLow = (E)(-INFINITY);
  const R kPad = R{kLow, kLow, kLow, kLow};

  // Largest value, and whether any is NaN or infinite (x * 0 is NaN exactly then); from the first tile
  // the smallest that is not a mask's, a guess at the histogram's range.  Every lane reads back only
  // what it stored.
  float mx = -INFINITY, mn = INFINITY;
  bool odd = false;
  {
    R big = kPad, acc = R{};
    constexpr int kB = 8;  // tiles whose loads are in flight together
    for (int j0 = 0; j0 < tiles; j0 += kB) {
      R x[kB];
#pragma unroll
      for (int u = 0; u < kB; ++u) x[u] = load_raw<kHalf>(row, min((j0 + u) * kVerTile + 4 * t, V - 4));
#pragma unroll
      for (int u = 0; u < kB; ++u) {
        if (j0 + u >= tiles) break;
        acc = __builtin_elementwise_fma(x[u], R{}, acc);  // past the end: the row's last entries again
        if ((j0 + u + 1) * kVerTile > V) x[u] = (j0 + u) * kVerTile + 4 * t < V ? x[u] : kPad;
        big = __builtin_elementwise_max(big, x[u]);
        if (j0 + u == 0)
          for (int e = 0; e < 4; ++e) mn = fminf(mn, (float)x[0][e] > -30000.0f ? (float)x[0][e] : INFINITY);
        if constexpr (kTiles > 0) lrow[(j0 + u) * kVerThreads + t] = x[u];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mx = fmaxf(mx, (float)big[e]);
      odd = odd || __builtin_isnan((float)acc[e]);
    }
  }
  auto raw_of = [&](int j) __attribute__((always_inline)) -> R {
    if constexpr (kTiles > 0) return lrow[j * kVerThreads + t];
    else return load_raw<kHalf>(row, min(j * kVerTile + 4 * t, V - 4));
  };
  auto entries = [&](int j, R x) __attribute__((always_inline)) -> f4 {
    f4 l = to_f4(x);
    if constexpr (kTiles == 0) {
      if (mode != kPlain)
        for (int e = 0; e < 4; ++e) l[e] = read_as(l[e], mode);
      if ((j + 1) * kVerTile > V && j * kVerTile + 4 * t >= V) l = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    }
    return l;
  };
  // f(four entries) over this lane's entries, four tiles' loads at a time; entries of the padding are -inf
  auto each4 = [&](auto&& f) __attribute__((always_inline)) {
    int j = 0;
    for (; j + 4 <= tiles; j += 4) {
      const R x0 = raw_of(j), x1 = raw_of(j + 1), x2 = raw_of(j + 2), x3 = raw_of(j + 3);
      f(entries(j, x0));
      f(entries(j + 1, x1));
      f(entries(j + 2, x2));
      f(entries(j + 3, x3));
    }
    for (; j < tiles; ++j) f(entries(j, raw_of(j)));
  };
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    each4([&](f4 x) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(x[e]);
    });
  };
  float lane_max = mx, oddf = odd ? 1.0f : 0.0f;
  block_max2(sh, par, mx, oddf);
  if (oddf > 0.0f) {
    // NaN or an infinity somewhere (masked entries, often): read the row another way
    bool nan = false;
    each([&](float l) { nan = nan || __builtin_isnan(l); });
    nan = block_max(sh, par, nan ? 1.0f : 0.0f) > 0.0f;
    mode = mx == INFINITY ? kInfOnly : nan ? kNanZero : mx == -INFINITY ? kAllLow : kPlain;
    if (mode != kPlain) {
      if constexpr (kTiles > 0) {
        for (int j = 0; j < tiles; ++j) {
          const int at = j * kVerTile + 4 * t;
          if (at >= V) continue;
          R x = lrow[j * kVerThreads + t];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = (E)read_as((float)x[e], mode);
          lrow[j * kVerThreads + t] = x;
        }
      }
      mx = -INFINITY;
      each([&](float l) { mx = fmaxf(mx, l); });
      lane_max = mx;
      mx = block_max(sh, par, mx);
      mn = fminf(mn, 0.0f);
    }
  }
  const double mxd = (double)mx;
  auto weight = [&](float l) __attribute__((always_inline)) { return exp2_neg((double)l - mxd, p.scale, p.d_min); };

  RowStat st;
  st.max = mx;
  st.tau = -INFINITY;
  st.comp = 1.0;
  st.ok = 0;
  st.mode = mode;
  uint32_t none = 0, none2 = 0;
  if (!p.truncate) {
    // the sums of the segments are kept for the draw
    double m = 0.0;
    double* const sums = p.sums + ((int64_t)b * T + i) * p.segs + wv;
    for (int j = 0; j < tiles; j += 4) {
      double s[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        s[u] = 0.0;
        if (j + u < tiles) {
          const f4 x = entries(j + u, raw_of(j + u));
          s[u] = (weight(x[0]) + weight(x[1])) + (weight(x[2]) + weight(x[3]));
        }
      }
      m += (s[0] + s[1]) + (s[2] + s[3]);
      const double w = wave_add4(s, lane);
      const int seg = (j + lane) * kVerWaves;
      if (lane < 4 && seg + wv < p.segs) sums[seg] = w;
    }
    st.z = block_sum(sh, par, m);
  } else {
    // floor: a value that tau cannot lie below; entries under it are left out of the search.  In each
    // wave the q-th largest of its lanes' maxima, q = ceil(top_k / 16), is at or below q of its
    // entries, so the smallest of the 16 waves' has top_k entries at or above it.
    float floor = -INFINITY;
    if (p.top_k <= kVerThreads) {
      const int q = (p.top_k + kVerWaves - 1) / kVerWaves;
      float lm = lane_max, at = -INFINITY;
      for (int k = 0; k < q; ++k) {
        at = wave_fmax(lm);
        const uint64_t hit = __ballot(lm == at);
        if (lane == (int)__builtin_ctzll(hit)) lm = -INFINITY;
      }
      floor = -at;
    }
    mn = -mn;
    block_max2(sh, par, floor, mn);
    floor = p.top_k <= kVerThreads ? -floor : -INFINITY;
    mn = -mn;
    // Histogram of (mx - l) in kVerBins equal steps: 32 per octave of the weight, or finer where the
    // entries from floor up span less.  Larger l never falls in a later bin.  The same pass adds up
    // the mass of the whole row, top_p's measure.
    const float far = mx - fmaxf(mn, floor);
    const float s = far > 0.0f ? fminf(fmaxf(p.bin_scale, (float)(kVerBins - 1) / far), FLT_MAX) : p.bin_scale;
    auto bin_at = [&](float l) __attribute__((always_inline)) { return fminf((mx - l) * s, (float)(kVerBins - 1)); };
    for (int k = t; k < kVerBins; k += kVerThreads) {
      sh.cnt[k] = 0;
      sh.mass[k] = 0;
    }
    if (t == 0) {
      sh.n_cand = 0;
      sh.bin = kVerBins;
    }
    __syncthreads();
    const bool by_count = p.top_k < V;
    double all = 0.0;
    floor = fmaxf(floor, -FLT_MAX);  // masked entries have no weight
    each4([&](f4 x) __attribute__((always_inline)) {
      double w[4];
      if (p.use_mass) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = weight(x[e]);
        all += (w[0] + w[1]) + (w[2] + w[3]);
      }
      if (__ballot(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= floor) == 0) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (x[e] >= floor) {
          const int k = (int)bin_at(x[e]);
          if (by_count) atomicAdd(&sh.cnt[k], 1u);
          if (p.use_mass) atomicAdd((unsigned long long*)&sh.mass[k], (unsigned long long)mass_of(w[e]));
        }
      }
    });
    all = block_sum(sh, par, all);  // its barrier also ends the histogram
    const double goal = p.top_p * all;  // in units of the largest weight
    auto enough = [&](uint32_t c, uint64_t m) {
      return c >= (uint32_t)p.top_k || (p.use_mass && (double)m * kMassUnit >= goal);
    };
    // inclusive prefix over the bins (two per lane) and the first bin that reaches the budget
    const uint32_t c0 = sh.cnt[2 * t], c1 = sh.cnt[2 * t + 1];
    const uint64_t m0 = sh.mass[2 * t], m1 = sh.mass[2 * t + 1];
    uint32_t ci = wave_scan(c0 + c1, lane);
    uint64_t mi = wave_scan(m0 + m1, lane);
    if (lane == 63) {
      sh.redc[par][wv] = ci;
      sh.redm[par][wv] = mi;
    }
    __syncthreads();
    ci += row_add((lane & 15) < wv ? sh.redc[par][lane & 15] : 0u);
    mi += row_add((lane & 15) < wv ? sh.redm[par][lane & 15] : (uint64_t)0);
    par ^= 1;
    if (enough(ci - c1, mi - m1)) {
      if (!enough(ci - c1 - c0, mi - m1 - m0)) {
        sh.bin = 2 * t;
        sh.before_c = ci - c1 - c0;
        sh.before_m = mi - m1 - m0;
      }
    } else if (enough(ci, mi)) {
      sh.bin = 2 * t + 1;
      sh.before_c = ci - c1;
      sh.before_m = mi - m1;
    }
    __syncthreads();
    // None: fewer entries than top_k have a weight at all (the others are masked); all of those are kept.
    const bool found = sh.bin < kVerBins;
    const int bin = found ? sh.bin : kVerBins - 1;
    const uint32_t before_c = found ? sh.before_c : 0;
    const uint64_t before_m = found ? sh.before_m : 0;
    if (found) {
      const float bf = (float)bin;
      // the bin's span in logits with room for rounding, so that most groups are passed over quickly
      const float room = 1.0e-5f * (fabsf(mx) + (float)kVerBins / s);
      const float top = bin == 0 ? mx : mx - bf / s + room;
      const float low = bin == kVerBins - 1 ? floor : fmaxf(floor, mx - (bf + 1.0f) / s - room);
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
            if (at < kVerCand) {
              sh.cand[at] = x[e];
              sh.candm[at] = p.use_mass ? mass_of(weight(x[e])) : 0;
            }
          }
        }
      });
    }
    __syncthreads();
    const int in_bin = found ? sh.n_cand : kVerCand + 1;
    if (!found) floor = -FLT_MAX;
    uint32_t ngt = 0, neq = 0;
    uint64_t mgt = 0;
    if (in_bin <= kVerCand) {
      uint32_t c = before_c;
      uint64_t m = before_m;
      float v = -INFINITY;
      if (t < 4 && in_bin + t < kVerCand) sh.cand[in_bin + t] = -INFINITY;  // fills the last group of four
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
      st.tau = block_max(sh, par, t < in_bin && enough(c, m) ? v : -INFINITY);
      ngt = t < in_bin && v > st.tau ? 1 : 0;
      neq = t < in_bin && v == st.tau ? 1 : 0;
      mgt = ngt ? sh.candm[t] : 0;
      block_add(sh, par, ngt, neq, mgt);
      ngt += before_c;
      mgt += before_m;
    } else {
      // many entries in one bin (ties, or a spread that outliers stretch): bisection over the keys of
      // every entry, at most 32 rounds, for the largest value with enough entries at or above it
      uint32_t lo = key_of(floor), hi = found ? key_of(mx) : lo;
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
        block_add(sh, par, c, none, m);
        if (enough(c, m)) lo = mid;
        else hi = mid - 1u;
      }
      // lo may lie below every entry: then tau is the smallest of them
      float least = -INFINITY;
      const float lov = of_key(lo);
      each([&](float l) { least = l >= lov ? fmaxf(least, -l) : least; });
      st.tau = -block_max(sh, par, least);
      each([&](float l) {
        ngt += l > st.tau ? 1 : 0;
        neq += l == st.tau ? 1 : 0;
        mgt += l > st.tau && p.use_mass ? mass_of(weight(l)) : 0;
      });
      block_add(sh, par, ngt, neq, mgt);
    }
    if (!p.use_mass) {  // the mass above tau was not needed so far
      mgt = 0;
      each4([&](f4 x) __attribute__((always_inline)) {
        if (__ballot(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > st.tau) == 0) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) mgt += x[e] > st.tau ? mass_of(weight(x[e])) : 0;
      });
      block_add(sh, par, none, none2, mgt);
    }
    const double x = weight(st.tau);
    double comp = by_count ? (double)((int64_t)p.top_k - (int64_t)ngt) / (double)neq : 1.0;
    if (p.use_mass) comp = fmin(comp, (goal - (double)mgt * kMassUnit) / (x * (double)neq));
    comp = fmax(fmin(comp, 1.0), 0.0);
    // no entry above tau: the kept ones are ties, whose common share does not matter
    st.comp = mgt == 0 ? 1.0 : comp;
    st.z = (double)mgt * kMassUnit + st.comp * x * (double)neq;
  }
  if (t == 0) {
    if (i < n) {
      const int d = p.drafts[(int64_t)b * p.K + i];
      const bool in = d >= 0 && d < V;
      const float l = in ? read_as(kHalf ? (float)reinterpret_cast<const _Float16*>(row)[d]
                                         : reinterpret_cast<const float*>(row)[d], mode) : 0.0f;
      const double pd = in ? kept_of(p, st, l) / st.z : 0.0;
      const double qd = p.q ? (in ? (double)p.q[((int64_t)b * p.K + i) * V + d] : 0.0) : 1.0;
      st.ok = (double)p.u[(int64_t)b * T + i] * qd < pd ? 1 : 0;
    }
    p.stat[(int64_t)b * T + i] = st;
  }
}

// What the two kernels behind the rows' share: the row a sequence stops at and the weights it draws from.
template <bool kHalf>
struct Stop {
  const VerifyArgs& p;
  int64_t id;      // row b (K + 1) + j
  int j, n, draft;
  const float* q;  // the drafter's row, where j is a rejected draft's and there is one
  bool beyond;     // draw from what p has beyond q
  RowStat st;
  double unit, unit_tau;  // of a weight above tau, and at it
  const void* row;

  __device__ __forceinline__ Stop(const VerifyArgs& a, int b, int n_, int lane) : p(a), n(n_) {
    const int T = p.K + 1;
    j = n;
    for (int k0 = 0; k0 < n; k0 += 64) {
      const uint64_t hit = __ballot(k0 + lane < n && !p.stat[(int64_t)b * T + k0 + lane].ok);
      if (hit) {
        j = k0 + __builtin_ctzll(hit);
        break;
      }
    }
    id = (int64_t)b * T + j;
    st = p.stat[id];
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
      if (st.mode != kPlain)
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

// The segments' sums of the row each sequence stops at (not where the rows' kernel left them: without
// a filter, all drafts accepted).  A workgroup takes 8 segments for each of its 4 waves.
constexpr int kPartSegs = 8;
template <bool kHalf>
__global__ __launch_bounds__(256) void verify_parts_kernel(VerifyArgs p) {
  const int parts = (p.segs + 4 * kPartSegs - 1) / (4 * kPartSegs);
  const int b = blockIdx.x / parts, part = blockIdx.x - b * parts, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  if (n < 0 || n > p.K) return;
  const Stop<kHalf> stop(p, b, n, lane);
  if (!p.truncate && !stop.beyond) return;
  const int seg0 = (part * 4 + wv) * kPartSegs;
  f4 l[kPartSegs], qv[kPartSegs];
#pragma unroll
  for (int k = 0; k < kPartSegs; ++k) {
    const int at = (seg0 + k) * kSeg + 4 * lane;
    l[k] = stop.load_l(at);
    qv[k] = stop.load_q(at);
  }
  double* const sums = p.sums + stop.id * p.segs + seg0;
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

constexpr int kDrawThreads = 256;
struct DrawShared {
  double sum[kMaxSegs];
  double red[4];
  int first, last;
};

// One workgroup per sequence: the segment that holds the target, then the entry.
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
  Stop<kHalf> stop(p, b, n, lane);
  const int j = stop.j;
  for (int k = t; k < T; k += kDrawThreads)
    if (k != j) out[k] = k < j ? p.drafts[(int64_t)b * p.K + k] : -1;
  if (t == 0) p.accepted[b] = j;
  // the sum of segment k by one wave (the rows' and parts' kernels' order of additions aside)
  auto segment = [&](int k) {
    double w[4];
    const int at = k * kSeg + 4 * lane;
    stop.weights(stop.load_l(at), stop.load_q(at), at, w);
    return wave_add((w[0] + w[1]) + (w[2] + w[3]));
  };
  const int per = (segs + kDrawThreads - 1) / kDrawThreads;  // segments per lane of the scan: at most 16
  const int k0 = min(t * per, segs), k1 = min(k0 + per, segs);
  double total, run0;
  for (bool again = false;; again = true) {
    if (again) {  // nothing beyond the drafter's probabilities: p itself, whose sums nobody has
      for (int k = wv; k < segs; k += 4) {
        const double s = segment(k);
        if (lane == 0) sh.sum[k] = s;
      }
    } else {
      // sums of the rows' kernel are in units of the largest weight and hold the rejected draft of a lookup
      const double unit = !p.truncate && !stop.q ? stop.unit : 1.0;
      const int own = !p.truncate && stop.draft >= 0 && stop.draft < p.V ? stop.draft / kSeg : -1;
      const double* src = p.sums + stop.id * segs;
      for (int k = t; k < segs; k += kDrawThreads)
        if (k != own) sh.sum[k] = src[k] * unit;
      if (own >= 0 && wv == 0) {
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
    const double r0 = sh.red[0], r1 = sh.red[1], r2 = sh.red[2], r3 = sh.red[3];
    total = (r0 + r1) + (r2 + r3);
    run0 = (wv == 0 ? 0.0 : wv == 1 ? r0 : wv == 2 ? r0 + r1 : r0 + r1 + r2) + incl - s;
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
    if (first < segs) atomicMin(&sh.first, first);
    if (last >= 0) atomicMax(&sh.last, last);
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

// Rows of up to 128 KiB stay in LDS (one workgroup per CU then; up to 32 KiB two), longer ones are
// re-read from memory.
template <bool kHalf>
void launch_verify(const VerifyArgs& a, int B, hipStream_t s) {
  constexpr int kTileBytes = kVerTile * (kHalf ? 2 : 4);
  constexpr int kSmall = (32 << 10) / kTileBytes, kLarge = (128 << 10) / kTileBytes;
  const dim3 grid(B * (a.K + 1)), block(kVerThreads);
  const int tiles = (a.V + kVerTile - 1) / kVerTile;
  if (tiles <= kSmall) hipLaunchKernelGGL((verify_rows_kernel<kHalf, kSmall>), grid, block, 0, s, a);
  else if (tiles <= kLarge) hipLaunchKernelGGL((verify_rows_kernel<kHalf, kLarge>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((verify_rows_kernel<kHalf, 0>), grid, block, 0, s, a);
  if (a.truncate || a.q)
    hipLaunchKernelGGL(verify_parts_kernel<kHalf>, dim3(B * ((a.segs + 4 * kPartSegs - 1) / (4 * kPartSegs))), dim3(256), 0,
                       s, a);
  hipLaunchKernelGGL(verify_draw_kernel<kHalf>, dim3(B), dim3(kDrawThreads), 0, s, a);
}

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int64_t vkwr_sampling_verify_workspace_bytes(int B, int K, int V) {
  if (B <= 0 || K < 0 || V <= 0) return 0;
  const int64_t rows = (int64_t)B * ((int64_t)K + 1);
  return rows * ((int64_t)sizeof(RowStat) + (V + kSeg - 1) / kSeg * (int64_t)sizeof(double));
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
  VK_REQUIRE((int64_t)B * ((int64_t)K + 1) <= 0x7fffffff && B <= (1 << 24), "%s: B or B*(K+1) too large", fn);
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
  a.stat = reinterpret_cast<RowStat*>(workspace);
  a.segs = (V + kSeg - 1) / kSeg;
  a.sums = reinterpret_cast<double*>(a.stat + (int64_t)B * ((int64_t)K + 1));
  a.scale = 1.4426950408889634 / temperature;
  a.d_min = -1023.0 / a.scale;
  a.bin_scale = (float)(32.0 * a.scale);
  a.top_k = top_k;
  a.top_p = top_p;
  a.use_mass = top_p < 1.0;
  a.truncate = top_k < V || a.use_mass;
  if (logits_f16) launch_verify<true>(a, B, (hipStream_t)stream);
  else launch_verify<false>(a, B, (hipStream_t)stream);
  return check_launch(fn);
}
