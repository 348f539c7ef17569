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
// 64 bits: weights by a polynomial of relative error 3e-13, masses as integers in units of 2^-43
// (sums of up to 2^20 weights <= 1 do not overflow, and integer sums do not depend on their order),
// the draw's prefix sums in fp64.  A token differs from that of exact arithmetic only where a
// uniform lies within ~1e-11 of a border.
//
// Two launches: one workgroup per row finds max, tau, comp and Z and tests the row's draft; one
// workgroup per sequence finds its first rejected row and draws.

#include <cfloat>

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

constexpr int kVerThreads = 1024;
constexpr int kVerWaves = kVerThreads / 64;
constexpr int kVerBins = 2048;   // histogram of (max - l) for the threshold
constexpr int kVerCand = 1024;   // entries of one bin that are ranked directly
constexpr int kVerTile = 4 * kVerThreads;  // consecutive entries a workgroup reads at once
constexpr int kVerMaxV = 1 << 20;
constexpr int kVerMaxTiles = kVerMaxV / kVerTile;
constexpr double kMassUnit = 1.0 / 8796093022208.0;  // 2^-43

struct RowStat {
  double z, comp;
  float max, tau;
  int ok, pad;
};
static_assert(sizeof(RowStat) == 32, "row stat size");

struct VerifyArgs {
  int K, V;
  const void* logits;
  const int32_t *drafts, *n_draft;
  const float *q, *u;
  int32_t *tokens, *accepted;
  RowStat* stat;
  double scale;  // log2(e) / temperature
  float bin_scale;
  int top_k;
  double top_p;
  int use_mass, truncate;
};

__device__ __forceinline__ float sf(float x) {
  const float y = __builtin_isnan(x) ? 0.0f : x;
  return fminf(fmaxf(y, -FLT_MAX), FLT_MAX);
}

// 2^x for x <= 0: x = n + f with |f| <= 1/2, the degree-10 Taylor polynomial of e^{f ln 2} (remainder
// (0.3466)^11 / 11! = 2.2e-13), an exact power of two.
__device__ __forceinline__ double exp2_neg(double x) {
  x = fmax(x, -2000.0);  // -inf (padding) too; the result is 0
  const double n = __builtin_rint(x);
  const double f = x - n;
  double p = 7.054911620801123e-09;
  p = __builtin_fma(p, f, 1.0178086009239701e-07);
  p = __builtin_fma(p, f, 1.3215486790144309e-06);
  p = __builtin_fma(p, f, 1.5252733804059841e-05);
  p = __builtin_fma(p, f, 1.5403530393381609e-04);
  p = __builtin_fma(p, f, 1.3333558146428443e-03);
  p = __builtin_fma(p, f, 9.6181291076284771e-03);
  p = __builtin_fma(p, f, 5.5504108664821580e-02);
  p = __builtin_fma(p, f, 2.4022650695910071e-01);
  p = __builtin_fma(p, f, 6.9314718055994531e-01);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// A weight in [0, 1] as a whole number of 2^-43: 512 + x has that spacing.
__device__ __forceinline__ uint64_t mass_of(double x) {
  return __builtin_bit_cast(uint64_t, 512.0 + x) - __builtin_bit_cast(uint64_t, 512.0);
}

template <class X>
__device__ __forceinline__ X wave_add(X v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
__device__ __forceinline__ float wave_fmax(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

struct StatShared {
  uint64_t mass[kVerBins];
  uint32_t cnt[kVerBins];
  uint64_t red64[kVerWaves];
  uint64_t redm[kVerWaves];
  uint32_t redc[kVerWaves], redd[kVerWaves];
  float redf[kVerWaves];
  float cand[kVerCand];
  uint64_t candm[kVerCand];
  int n_cand, bin;
  uint32_t before_c;
  uint64_t before_m;
};

// Block reductions: every lane gets the result; two barriers.
__device__ __forceinline__ float block_fmax(StatShared& sh, float v) {
  v = wave_fmax(v);
  if ((threadIdx.x & 63) == 0) sh.redf[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = sh.redf[0];
#pragma unroll
  for (int w = 1; w < kVerWaves; ++w) r = fmaxf(r, sh.redf[w]);
  __syncthreads();
  return r;
}
__device__ __forceinline__ void block_add(StatShared& sh, uint32_t& a, uint32_t& b, uint64_t& m) {
  a = wave_add(a);
  b = wave_add(b);
  m = wave_add(m);
  if ((threadIdx.x & 63) == 0) {
    const int w = threadIdx.x >> 6;
    sh.redc[w] = a;
    sh.redd[w] = b;
    sh.redm[w] = m;
  }
  __syncthreads();
  a = b = 0;
  m = 0;
#pragma unroll
  for (int w = 0; w < kVerWaves; ++w) {
    a += sh.redc[w];
    b += sh.redd[w];
    m += sh.redm[w];
  }
  __syncthreads();
}

// Order-preserving key of a finite float.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 -> +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// Four consecutive entries of a row.
template <bool kHalf>
__device__ __forceinline__ f4 load4(const void* row, int i) {
  if constexpr (kHalf) {
    typedef _Float16 hv4 __attribute__((ext_vector_type(4)));
    const hv4 x = *reinterpret_cast<const hv4*>(reinterpret_cast<const _Float16*>(row) + i);
    return f4{sf((float)x[0]), sf((float)x[1]), sf((float)x[2]), sf((float)x[3])};
  } else {
    const f4 x = *reinterpret_cast<const f4*>(reinterpret_cast<const float*>(row) + i);
    return f4{sf(x[0]), sf(x[1]), sf(x[2]), sf(x[3])};
  }
}
template <bool kHalf>
__device__ __forceinline__ const void* row_at(const VerifyArgs& p, int64_t row) {
  return reinterpret_cast<const char*>(p.logits) + row * p.V * (kHalf ? 2 : 4);
}
template <bool kHalf>
__device__ __forceinline__ float load1(const void* row, int i) {
  if constexpr (kHalf) return sf((float)reinterpret_cast<const _Float16*>(row)[i]);
  else return sf(reinterpret_cast<const float*>(row)[i]);
}

// The kept weight of logit l in units of its row's largest weight.
__device__ __forceinline__ double kept_of(double scale, const RowStat& st, float l) {
  if (!(l >= st.tau)) return 0.0;
  const double x = exp2_neg(((double)l - (double)st.max) * scale);
  return l > st.tau ? x : x * st.comp;
}

// J > 0: the row's J tiles stay in registers (V <= J * kVerTile); J == 0: re-read in every pass.
template <bool kHalf, int J>
__global__ __launch_bounds__(kVerThreads) void verify_rows_kernel(VerifyArgs p) {
  __shared__ StatShared sh;
  const int T = p.K + 1;
  const int b = blockIdx.x / T, i = blockIdx.x - b * T;
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  if (n < 0 || n > p.K || i > n) return;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = p.V;
  const void* row = row_at<kHalf>(p, (int64_t)b * T + i);
  const int tiles = (V + kVerTile - 1) / kVerTile;
  f4 reg[J > 0 ? J : 1];
  const f4 kNone = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if constexpr (J > 0) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int at = j * kVerTile + 4 * t;
      reg[j] = at < V ? load4<kHalf>(row, at) : kNone;
    }
  }
  // f(entry) over this lane's entries; padding entries are -inf
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    if constexpr (J > 0) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) f(reg[j][e]);
    } else {
      for (int j = 0; j < tiles; ++j) {
        const int at = j * kVerTile + 4 * t;
        const f4 x = at < V ? load4<kHalf>(row, at) : kNone;
#pragma unroll
        for (int e = 0; e < 4; ++e) f(x[e]);
      }
    }
  };

  float mx = -INFINITY;
  each([&](float l) { mx = fmaxf(mx, l); });
  mx = block_fmax(sh, mx);
  const double mxd = (double)mx;
  auto weight = [&](float l) { return exp2_neg(((double)l - mxd) * p.scale); };

  RowStat st;
  st.max = mx;
  st.tau = -INFINITY;
  st.comp = 1.0;
  st.ok = st.pad = 0;
  if (!p.truncate) {
    uint64_t m = 0;
    uint32_t u0 = 0, u1 = 0;
    each([&](float l) { m += mass_of(weight(l)); });
    block_add(sh, u0, u1, m);
    st.z = (double)m * kMassUnit;
  } else {
    // Histogram of (max - l) in kVerBins equal steps: 32 per octave of the weight, or finer where
    // the entries of weight 2^-64 and more span less than that.  Larger l never falls in a later bin.
    float far = 0.0f;
    each([&](float l) {
      const float d = mx - l;
      far = fmaxf(far, d * p.bin_scale <= (float)kVerBins ? d : 0.0f);
    });
    far = block_fmax(sh, far);
    const float s = far > 0.0f ? fminf(fmaxf(p.bin_scale, (float)(kVerBins - 1) / far), FLT_MAX) : p.bin_scale;
    auto bin_of = [&](float l) { return (int)fminf((mx - l) * s, (float)(kVerBins - 1)); };
    for (int k = t; k < kVerBins; k += kVerThreads) {
      sh.cnt[k] = 0;
      sh.mass[k] = 0;
    }
    if (t == 0) sh.n_cand = 0;
    __syncthreads();
    each([&](float l) {
      if (l > -INFINITY) {
        const int k = bin_of(l);
        atomicAdd(&sh.cnt[k], 1u);
        atomicAdd((unsigned long long*)&sh.mass[k], (unsigned long long)mass_of(weight(l)));
      }
    });
    __syncthreads();
    // inclusive prefix over the bins (two per lane) and the first bin that reaches the budget
    const uint32_t c0 = sh.cnt[2 * t], c1 = sh.cnt[2 * t + 1];
    const uint64_t m0 = sh.mass[2 * t], m1 = sh.mass[2 * t + 1];
    uint32_t ci = c0 + c1;
    uint64_t mi = m0 + m1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t co = __shfl_up(ci, d, 64);
      const uint64_t mo = __shfl_up(mi, d, 64);
      if (lane >= d) {
        ci += co;
        mi += mo;
      }
    }
    if (lane == 63) {
      sh.redc[wv] = ci;
      sh.redm[wv] = mi;
    }
    if (t == 0) sh.bin = kVerBins;
    __syncthreads();
    uint64_t all = 0;
    for (int w = 0; w < kVerWaves; ++w) {
      if (w < wv) {
        ci += sh.redc[w];
        mi += sh.redm[w];
      }
      all += sh.redm[w];
    }
    const double goal = p.top_p * (double)all;
    auto enough = [&](uint32_t c, uint64_t m) { return c >= (uint32_t)p.top_k || (p.use_mass && (double)m >= goal); };
    if (enough(ci - c1, mi - m1)) atomicMin(&sh.bin, 2 * t);
    else if (enough(ci, mi)) atomicMin(&sh.bin, 2 * t + 1);
    __syncthreads();
    const int bin = sh.bin;  // exists: the count over all bins is V >= top_k
    if (bin == 2 * t) {
      sh.before_c = ci - c1 - c0;
      sh.before_m = mi - m1 - m0;
    } else if (bin == 2 * t + 1) {
      sh.before_c = ci - c1;
      sh.before_m = mi - m1;
    }
    __syncthreads();
    const uint32_t before_c = sh.before_c;
    const uint64_t before_m = sh.before_m;
    const int in_bin = (int)sh.cnt[bin];
    if (in_bin <= kVerCand) {
      each([&](float l) {
        if (l > -INFINITY && bin_of(l) == bin) {
          const int at = atomicAdd(&sh.n_cand, 1);  // any order: only sums and a maximum follow
          sh.cand[at] = l;
          sh.candm[at] = mass_of(weight(l));
        }
      });
      __syncthreads();
      float best = -INFINITY;
      if (t < in_bin) {
        const float v = sh.cand[t];
        uint32_t c = before_c;
        uint64_t m = before_m;
        for (int k = 0; k < in_bin; ++k) {
          const bool ge = sh.cand[k] >= v;
          c += ge ? 1u : 0u;
          m += ge ? sh.candm[k] : 0;
        }
        if (enough(c, m)) best = v;
      }
      st.tau = block_fmax(sh, best);
    } else {
      // many entries in one bin (ties, or a spread that outliers stretch): bisection over keys
      uint32_t lo = 0xffffffffu, hi = 0;
      each([&](float l) {
        if (l > -INFINITY && bin_of(l) == bin) {
          lo = min(lo, key_of(l));
          hi = max(hi, key_of(l));
        }
      });
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, m, 64));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, m, 64));
      }
      if (lane == 0) {
        sh.redc[wv] = lo;
        sh.redd[wv] = hi;
      }
      __syncthreads();
      for (int w = 0; w < kVerWaves; ++w) {
        lo = min(lo, sh.redc[w]);
        hi = max(hi, sh.redd[w]);
      }
      __syncthreads();
      while (lo < hi) {  // the largest key with enough entries at or above it: at most 32 rounds
        const uint32_t mid = lo + (hi - lo) / 2u + 1u;
        const float v = of_key(mid);
        uint32_t c = 0, unused = 0;
        uint64_t m = 0;
        each([&](float l) {
          if (l >= v) {
            c += 1;
            m += p.use_mass ? mass_of(weight(l)) : 0;
          }
        });
        block_add(sh, c, unused, m);
        if (enough(c, m)) lo = mid;
        else hi = mid - 1u;
      }
      st.tau = of_key(lo);
    }
    // entries above and at tau
    uint32_t ngt = 0, neq = 0;
    uint64_t mgt = 0;
    each([&](float l) {
      if (l > st.tau) {
        ngt += 1;
        mgt += mass_of(weight(l));
      }
      neq += l == st.tau ? 1 : 0;
    });
    block_add(sh, ngt, neq, mgt);
    const double x = weight(st.tau);
    double comp = (double)((int64_t)p.top_k - (int64_t)ngt) / (double)neq;
    if (p.use_mass) comp = fmin(comp, (goal - (double)mgt) * kMassUnit / (x * (double)neq));
    comp = fmax(fmin(comp, 1.0), 0.0);
    // no entry above tau: the kept ones are ties, whose common share does not matter
    st.comp = ngt == 0 ? 1.0 : comp;
    st.z = (double)mgt * kMassUnit + st.comp * x * (double)neq;
  }
  if (t == 0) {
    if (i < n) {
      const int d = p.drafts[(int64_t)b * p.K + i];
      const bool in = d >= 0 && d < V;
      const double pd = in ? kept_of(p.scale, st, load1<kHalf>(row, d)) / st.z : 0.0;
      const double qd = p.q ? (in ? (double)p.q[((int64_t)b * p.K + i) * V + d] : 0.0) : 1.0;
      st.ok = (double)p.u[(int64_t)b * T + i] * qd < pd ? 1 : 0;
    }
    p.stat[(int64_t)b * T + i] = st;
  }
}

struct DrawShared {
  double sum[kVerMaxTiles * kVerWaves];  // mass of each tile's 256 entries per wave
  double red[kVerWaves];
  int first, last;
};

template <bool kHalf>
__global__ __launch_bounds__(kVerThreads) void verify_draw_kernel(VerifyArgs p) {
  __shared__ DrawShared sh;
  const int T = p.K + 1, b = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = t >> 6, V = p.V;
  const int n = p.n_draft ? p.n_draft[b] : p.K;
  int32_t* out = p.tokens + (int64_t)b * T;
  if (n < 0 || n > p.K) {
    for (int k = t; k < T; k += kVerThreads) out[k] = -1;
    if (t == 0) p.accepted[b] = -1;
    return;
  }
  int j = 0;
  while (j < n && p.stat[(int64_t)b * T + j].ok) ++j;
  const RowStat st = p.stat[(int64_t)b * T + j];
  const void* row = row_at<kHalf>(p, (int64_t)b * T + j);
  const float* q = p.q && j < n ? p.q + ((int64_t)b * p.K + j) * V : nullptr;
  const int draft = j < n && !p.q ? p.drafts[(int64_t)b * p.K + j] : -1;
  const int tiles = (V + kVerTile - 1) / kVerTile, n_sum = tiles * kVerWaves;
  const double inv_z = 1.0 / st.z;
  bool beyond = j < n;  // draw from what p has beyond q
  // weights of the four entries at `at`
  auto weights = [&](int at, double* w) {
    const f4 l = load4<kHalf>(row, at);
    f4 qv = f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (q && beyond) qv = *reinterpret_cast<const f4*>(q + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      double x = kept_of(p.scale, st, l[e]) * inv_z;
      if (beyond) x = p.q ? fmax(x - (double)qv[e], 0.0) : (at + e == draft ? 0.0 : x);
      w[e] = x;
    }
  };
  double total, lane_total;
  for (;;) {
    for (int k = 0; k < tiles; ++k) {
      const int at = k * kVerTile + 4 * t;
      double w[4] = {0.0, 0.0, 0.0, 0.0};
      if (at < V) weights(at, w);
      const double s = wave_add((w[0] + w[1]) + (w[2] + w[3]));
      if (lane == 0) sh.sum[k * kVerWaves + wv] = s;
    }
    __syncthreads();
    // prefix over the wave sums, ceil(n_sum / 1024) <= 4 consecutive ones per lane
    const int per = (n_sum + kVerThreads - 1) / kVerThreads;
    double s = 0.0;
    for (int k = t * per; k < min((t + 1) * per, n_sum); ++k) s += sh.sum[k];
    double incl = s;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(incl, d, 64);
      if (lane >= d) incl += o;
    }
    if (lane == 63) sh.red[wv] = incl;
    if (t == 0) {
      sh.first = n_sum;
      sh.last = -1;
    }
    __syncthreads();
    total = 0.0;
    double pre = 0.0;
    for (int w = 0; w < kVerWaves; ++w) {
      if (w == wv) pre = total;
      total += sh.red[w];
    }
    lane_total = pre + incl - s;
    if (total > 0.0 || !beyond) break;
    beyond = false;
    __syncthreads();
  }
  const double target = (double)p.u[(int64_t)b * T + p.K] * total;
  {
    const int per = (n_sum + kVerThreads - 1) / kVerThreads;
    double run = lane_total;
    int first = n_sum, last = -1;
    for (int k = t * per; k < min((t + 1) * per, n_sum); ++k) {
      const double s = sh.sum[k];
      if (s > 0.0) {
        last = k;
        if (run + s > target && first == n_sum) first = k;
      }
      run += s;
    }
    if (first < n_sum) atomicMin(&sh.first, first);
    if (last >= 0) atomicMax(&sh.last, last);
  }
  __syncthreads();
  for (int k = t; k < T; k += kVerThreads)
    if (k != j) out[k] = k < j ? p.drafts[(int64_t)b * p.K + k] : -1;
  if (t == 0) p.accepted[b] = j;
  // the 256 entries that hold the target (rounding short of the end: the last with weight), by one wave
  const int seg = sh.first < n_sum ? sh.first : sh.last;
  if (wv != 0 || seg < 0) {
    if (seg < 0 && t == 0) out[j] = -1;
    return;
  }
  double before = 0.0;
  // the prefix before the segment again, in the order that found it
  {
    const int per = (n_sum + kVerThreads - 1) / kVerThreads;
    (void)per;
    for (int k = lane; k < seg; k += 64) before += sh.sum[k];
    before = wave_add(before);
  }
  const int at = (seg / kVerWaves) * kVerTile + (seg % kVerWaves) * 256 + 4 * lane;
  double w[4] = {0.0, 0.0, 0.0, 0.0};
  if (at < V) weights(at, w);
  double incl = (w[0] + w[1]) + (w[2] + w[3]);
  const double mine = incl;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  double run = before + incl - mine;
  int pick = -1, last = -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    run += w[e];
    if (w[e] > 0.0) {
      last = at + e;
      if (pick < 0 && run > target) pick = at + e;
    }
  }
  const uint64_t hit = __ballot(pick >= 0), any = __ballot(last >= 0);
  if (hit) {
    if (lane == __builtin_ctzll(hit)) out[j] = pick;
  } else if (any) {
    if (lane == 63 - __builtin_clzll(any)) out[j] = last;
  }
}

template <bool kHalf>
void launch_verify(const VerifyArgs& a, int B, hipStream_t s) {
  const dim3 grid(B * (a.K + 1)), block(kVerThreads);
  const int tiles = (a.V + kVerTile - 1) / kVerTile;
  if (tiles <= 4) hipLaunchKernelGGL((verify_rows_kernel<kHalf, 4>), grid, block, 0, s, a);
  else if (tiles <= 16) hipLaunchKernelGGL((verify_rows_kernel<kHalf, 16>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((verify_rows_kernel<kHalf, 0>), grid, block, 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel<kHalf>, dim3(B), block, 0, s, a);
}

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int64_t vkwr_sampling_verify_workspace_bytes(int B, int K, int V) {
  (void)V;
  return B > 0 && K >= 0 ? (int64_t)B * ((int64_t)K + 1) * (int64_t)sizeof(RowStat) : 0;
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
  VK_REQUIRE((int64_t)B * ((int64_t)K + 1) <= 0x7fffffff, "%s: B*(K+1) too large", fn);
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
  a.scale = 1.4426950408889634 / temperature;
  a.bin_scale = (float)(32.0 * a.scale);
  a.top_k = top_k;
  a.top_p = top_p;
  a.use_mass = top_p < 1.0;
  a.truncate = top_k < V || a.use_mass;
  if (logits_f16) launch_verify<true>(a, B, (hipStream_t)stream);
  else launch_verify<false>(a, B, (hipStream_t)stream);
  return check_launch(fn);
}
