// One step of beam search: the best continuations of every request's beams, and the recurrent
// states that follow them.
//
// Selection.  A live beam b offers every token v with raw = score_b + l_v - log sum_u exp(l_u), a
// finished one itself (token `end`, raw = score_b); the W best of a request by raw * length^-alpha
// go on.  Within a beam that order is the order of the logits, so a beam's W largest logits are
// enough, and they and the sum are found in one pass: beam_rows_kernel cuts each row into groups
// that a workgroup holds in registers, and writes the group's W largest entries, its maximum and
// its sum; beam_merge_kernel joins the groups and beams of a request.  The scores of different beams
// are compared across sums over the vocabulary: sums are joined, and scores formed and compared, in
// fp64 (a lane's sum of 16 terms is fp32).
//
// States.  beam_reorder_kernel renames slots where it can: the first child of a beam keeps its
// parent's slot, every further one gets a copy in a slot whose beam has no child.  A source is
// never a destination, so the copies need no order and no second buffer.
#include <hip/hip_runtime.h>

#include <float.h>

#include <algorithm>
#include <type_traits>

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

typedef _Float16 hv8 __attribute__((ext_vector_type(8)));
typedef float fv4 __attribute__((ext_vector_type(4)));
typedef uint32_t uv4 __attribute__((ext_vector_type(4)));

constexpr int kMaxBeams = 32;
constexpr int kMaxVocab = 1 << 20;
constexpr int kRowThreads = 512, kPer = 16, kGroup = kRowThreads * kPer;  // entries of a group
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kListCap = 512;     // entries above the bound that are ranked at once
constexpr int kMergeKeys = 4096;  // keys that a merge pass holds (32 beams x 128 groups: one row)
constexpr int kRankThreads = 512, kMergeThreads = kRankThreads + 64;

// Entries in the order (value descending, index ascending); 0 is below every entry.
__device__ __forceinline__ uint64_t entry_key(float v, uint32_t i) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // (-0 equals 0)
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)o << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return ~(uint32_t)k; }

constexpr float kNone = -__builtin_huge_valf();

struct RowStat {
  float max;  // of the group's entries; -inf: none
  float pad;
  double sum;  // of exp(l - max)
};

struct BeamArgs {
  const void* logits;
  const float* scores;
  const int32_t* lengths;
  const int32_t* ended;
  int32_t *tokens, *parents;
  float* scores_out;
  int32_t *lengths_out, *ended_out;
  uint64_t* keys;   // [rows][groups][W]
  RowStat* stats;   // [rows][groups]
  int W, V, groups, end;
  float alpha;
};

// max over the wave, in every lane: six steps from lane to lane and a broadcast
__device__ __forceinline__ float wave_max(float v) {
  auto step = [&](auto ctrl) __attribute__((always_inline)) {
    const int o = __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), decltype(ctrl)::value,
                                              0xf, 0xf, false);
    v = fmaxf(v, __builtin_bit_cast(float, o));
  };
  step(std::integral_constant<int, 0xB1>{});   // quad_perm 1 0 3 2
  step(std::integral_constant<int, 0x4E>{});   // quad_perm 2 3 0 1
  step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  step(std::integral_constant<int, 0x140>{});  // row_mirror: every lane of a row of 16 has the row's
  step(std::integral_constant<int, 0x142>{});  // row_bcast15
  step(std::integral_constant<int, 0x143>{});  // row_bcast31: lane 63 has the wave's
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// sum over the wave, in lane 63, by the same steps
__device__ __forceinline__ double wave_sum64(double v) {
  auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    // lanes that the step does not reach add 0
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  using All = std::integral_constant<int, 0xf>;
  step(std::integral_constant<int, 0xB1>{}, All{});
  step(std::integral_constant<int, 0x4E>{}, All{});
  step(std::integral_constant<int, 0x141>{}, All{});
  step(std::integral_constant<int, 0x140>{}, All{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // rows 1 and 3
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // rows 2 and 3
  return v;
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor(v, m, 64);
    v = o > v ? o : v;
  }
  return v;
}

// blockIdx.x: group of the row, blockIdx.y: row.  Lane t holds the pieces (8 fp16 or 4 fp32)
// t, t + 512, ... of the group.  Bound by memory where the logits are many (64 x 8 beams of 65536 fp32: 29.5 us,
// 4.6 TB/s; reads alone have reached 6.1); at 16 x 8 of fp16 (10.5 us; the bytes are 3.5) by its own instructions,
// an exponential of each entry above all, behind one load per lane; at 1 x 4 (4.9 us) by that trip and four
// barriers.  Groups of 8192 (us of a whole step at 1 x 4, 16 x 8, 64 x 8: 9.3, 14.8, 33.1): of 4096 9.2, 18.5, 44.3,
// of 16384 10.3, 14.2, 35.1.
template <bool kHalf>
__global__ __launch_bounds__(kRowThreads) void beam_rows_kernel(BeamArgs a) {
  constexpr int kPiece = kHalf ? 8 : 4;
  __shared__ float wmax[kRowWaves], wbound[kRowWaves];
  __shared__ double wsum[kRowWaves];
  __shared__ uint64_t list[kListCap], wkey[kRowWaves];
  __shared__ int count;
  const int64_t row = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int i0 = blockIdx.x * kGroup, W = a.W, V = a.V;
  const int over = a.ended[row];
  const float score = a.scores[row];
  auto index_of = [&](int e) { return i0 + ((e / kPiece) * kRowThreads + tid) * kPiece + e % kPiece; };

  typedef typename std::conditional<kHalf, hv8, fv4>::type Piece;
  typedef typename std::conditional<kHalf, _Float16, float>::type Elem;
  const Elem* const l = (const Elem*)a.logits + row * V;
  constexpr Elem kLow = (Elem)kNone;
  Piece p[kPer / kPiece];
#pragma unroll
  for (int j = 0; j < kPer / kPiece; ++j) {
    const int i = index_of(j * kPiece);
    if (i + kPiece <= V) {
      __builtin_memcpy(&p[j], l + i, 16);  // (a row need not start on 16 bytes)
    } else {
#pragma unroll
      for (int e = 0; e < kPiece; ++e) {
        p[j][e] = kLow;
        if (i + e < V) p[j][e] = l[i + e];
      }
    }
    if (j == 0 && (over || !(score > kNone))) return;  // (the merge leaves such rows out)
  }
  Piece tops = kLow;
#pragma unroll
  for (int j = 0; j < kPer / kPiece; ++j) {
    p[j] = __builtin_elementwise_max(p[j], (Piece)kLow);  // a NaN is never chosen
    tops = __builtin_elementwise_max(tops, p[j]);
  }
  float top = (float)tops[0];
#pragma unroll
  for (int e = 1; e < kPiece; ++e) top = fmaxf(top, (float)tops[e]);
  auto value = [&](int e) __attribute__((always_inline)) { return (float)p[e / kPiece][e % kPiece]; };
  // A bound that at least W entries reach: in each of n waves whose lanes all hold entries (or the
  // one there is) the q-th largest of the lanes' maxima, n q >= W, and the smallest of those.
  const int whole = min(kRowWaves, max(1, (min(V - i0, kGroup) + kPiece - 1) / kPiece / 64));
  const int q = (W + whole - 1) / whole;
  float left = top, bound = kNone, most = kNone;
  for (int s = 0; s < q; ++s) {
    bound = wave_max(left);
    if (s == 0) most = bound;
    const uint64_t at = __ballot(left == bound);
    if (lane == __builtin_ctzll(at)) left = kNone;
  }
  if (lane == 0) wmax[wave] = most, wbound[wave] = wave < whole ? bound : __builtin_huge_valf();
  if (tid == 0) count = 0;
  __syncthreads();
  float mx = wmax[0];
  bound = wbound[0];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) mx = fmaxf(mx, wmax[w]), bound = fminf(bound, wbound[w]);
  bound = fmaxf(bound, -FLT_MAX);  // (-inf is not an entry)
  if (__ballot(top >= bound)) {
    int mine = 0;  // entries of the wave
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += __popcll(__ballot(value(e) >= bound));
    int at = 0;
    if (lane == 0) at = atomicAdd(&count, mine);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const uint64_t b = __ballot(value(e) >= bound);
      if (b == 0) continue;
      const int n = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
      if (value(e) >= bound && n < kListCap) list[n] = entry_key(value(e), (uint32_t)index_of(e));
      at += __popcll(b);
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e)  // (at an infinite maximum the entries that are infinite themselves count 1 each)
    sum += __expf(fminf(value(e) - mx, 0.0f));
  if (!(mx > kNone)) sum = 0.0f;
  const double ws = wave_sum64((double)sum);
  if (lane == 63) wsum[wave] = ws;
  __syncthreads();
  const int64_t g = row * a.groups + blockIdx.x;
  if (tid == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) all += wsum[w];
    a.stats[g] = RowStat{mx, 0.0f, all};
  }
  uint64_t* const out = a.keys + g * W;
  const int n = count;
  if (n <= kListCap) {
    for (int i = tid; i < n; i += kRowThreads) {
      const uint64_t k = list[i];
      int better = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) better += list[j] > k;
      if (better < W) out[better] = k;
    }
    for (int i = n + tid; i < W; i += kRowThreads) out[i] = 0;
    return;
  }
  // many equal entries: one entry after the other
  uint64_t last = ~0ull;
  for (int s = 0; s < W; ++s) {
    uint64_t best = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const uint64_t k = value(e) > kNone ? entry_key(value(e), (uint32_t)index_of(e)) : 0;
      if (k < last && k > best) best = k;
    }
    best = wave_max_key(best);
    if (lane == 0) wkey[wave] = best;
    __syncthreads();
    last = wkey[0];
#pragma unroll
    for (int w = 1; w < kRowWaves; ++w) last = wkey[w] > last ? wkey[w] : last;
    if (tid == 0) out[s] = last;
    __syncthreads();
  }
}

// e^x for x <= 0 in fp64: 2^n e^t with |t| <= ln(2) / 2, e^t by its series to t^11 / 11! (the rest is below
// 7e-15).  Written out, as is the logarithm below: the merge runs once a step and waits for its own
// instructions, of which the library's functions have three times as many.
__device__ __forceinline__ double exp64(double x) {
  x = x > -1100.0 ? x : -1100.0;
  const double n = __builtin_rint(x * 1.4426950408889634);
  const double t = __builtin_fma(n, 0x1.8432a1b0e2634p-43, __builtin_fma(n, -0x1.62e42fefa4000p-1, x));  // ln 2 in 40 bits and the rest
  double p = 1.0;
#pragma unroll
  for (int k = 11; k >= 1; --k) p = __builtin_fma(t * (1.0 / k), p, 1.0);
  return __builtin_ldexp(p, (int)n);
}
// log x for x >= 1: fp32's, and one step of Newton's with the next term
__device__ __forceinline__ double log64(double x) {
  const double y = (double)__logf((float)x);
  const double r = __builtin_fma(x, exp64(-y), -1.0);
  return y + (r - 0.5 * r * r);
}

// One workgroup per request.  All it reads is requested at once; then the last wave joins the groups'
// sums while the others rank each row's keys (a key's place is the number of keys above it),
// and all rank the W x W
// scores.  Of a row's groups only the W with the largest first keys can hold
// one of its W largest.  Bound by its own chain of steps: 4.4 us at 1 x 4 beams of 65536, 5.8 at 64 x 8.
__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(BeamArgs a) {
  constexpr int kKeep = (kMergeKeys + kMergeThreads - 1) / kMergeThreads;  // keys per lane
  __shared__ uint64_t keys[kMergeKeys];
  __shared__ uint64_t cand[kMaxBeams * kMaxBeams];  // [beam][W], sorted
  __shared__ double rank[kMaxBeams * kMaxBeams], raw[kMaxBeams * kMaxBeams];
  __shared__ double base[kMaxBeams], factor[kMaxBeams], gsum[kMergeKeys];
  __shared__ float rmax[kMaxBeams], gmax[kMergeKeys];
  __shared__ int before[kMaxBeams * kMaxBeams], live[kMaxBeams], len0[kMaxBeams], valid;  // live: 0 offers nothing, 1 live, 2 finished
  const int tid = threadIdx.x, W = a.W, G = a.groups;
  const int64_t r0 = (int64_t)blockIdx.x * W;
  const int per_row = G * W, rows = kMergeKeys / per_row > W ? W : kMergeKeys / per_row;  // rows of a pass (at least 1)
  // all loads of the first pass before anything waits for one
  uint64_t kr[kKeep];
  RowStat sr{};
  float score = kNone;
  int over0 = 0, length = 0;
  auto load_keys = [&](int w0, int n) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kKeep; ++u) {
      const int i = u * kMergeThreads + tid;
      if (i < n) kr[u] = a.keys[(r0 + w0) * per_row + i];
    }
  };
  load_keys(0, rows * per_row);
  if (tid < W * G) sr = a.stats[r0 * G + tid];
  if (tid < W) {
    score = a.scores[r0 + tid];
    over0 = a.ended[r0 + tid];
    length = a.lengths[r0 + tid];
  }
  for (int i = tid; i < W * W; i += kMergeThreads) cand[i] = 0;
  for (int i = tid + kMergeThreads; i < W * G; i += kMergeThreads) {
    const RowStat st = a.stats[r0 * G + i];
    gmax[i] = st.max;
    gsum[i] = st.sum;
  }
  if (tid < W * G) {
    gmax[tid] = sr.max;
    gsum[tid] = sr.sum;
  }
  if (tid < W) {
    live[tid] = score > kNone ? (over0 ? 2 : 1) : 0;
    len0[tid] = length;
    base[tid] = (double)score;
    if (tid == 0) valid = 0;
  }
  for (int w0 = 0; w0 < W; w0 += rows) {
    const int n = (W - w0 < rows ? W - w0 : rows) * per_row;
    if (w0 > 0) load_keys(w0, n);
#pragma unroll
    for (int u = 0; u < kKeep; ++u)
      if (u * kMergeThreads + tid < n) keys[u * kMergeThreads + tid] = kr[u];
    __syncthreads();
    if (tid >= kRankThreads) {
      if (w0 == 0) {
        const int lane = tid - kRankThreads;
        // a group's sum relative to the row's maximum, a lane each, then a row's, a lane each
        for (int i = lane; i < W * G; i += 64) {
          const int w = i / G;
          float mx = kNone;
#pragma unroll 8
          for (int g = 0; g < G; ++g) mx = fmaxf(mx, gmax[w * G + g]);
          const float m = gmax[i];
          // (a row that offers nothing has what the workspace held: it is not used)
          gsum[i] = m == mx ? gsum[i] : m > kNone ? gsum[i] * exp64((double)m - (double)mx) : 0.0;
          if (i == w * G) rmax[w] = mx;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (lane < W) {
          const int w = lane;
          const bool over = live[w] == 2;
          if (live[w] == 1 && rmax[w] > kNone) {  // (where not one token is allowed there are no keys either)
            double sum = 0.0;
#pragma unroll 8
            for (int g = 0; g < G; ++g) sum += gsum[w * G + g];
            base[w] -= log64(sum);
          }
          const int len = len0[w] + (over ? 0 : 1);
          factor[w] = a.alpha == 0.0f || len <= 1 ? 1.0 : exp64(-(double)a.alpha * log64((double)len));
        }
      }
    } else {
      for (int i = tid; i < n; i += kRankThreads) {
        const int wl = i / per_row, at = i - wl * per_row, mine = at / W;
        const uint64_t* const row = keys + wl * per_row;
        const uint64_t k = row[at];
        if (live[w0 + wl] != 1 || k == 0) continue;
        if (G > W) {
          const uint64_t head = row[mine * W];
          int before = 0;
#pragma unroll 8
          for (int g = 0; g < G; ++g) before += row[g * W] > head;
          if (before >= W) continue;
        }
        int better = 0;
        if (per_row <= 256) {
#pragma unroll 8
          for (int j = 0; j < per_row; ++j) better += row[j] > k;
        } else {
          better = at - mine * W;
          for (int g = 0; g < G && better < W; ++g) {
            if (g == mine) continue;
            for (int j = 0; j < W && row[g * W + j] > k; ++j) ++better;
          }
        }
        if (better < W) cand[(w0 + wl) * W + better] = k;
      }
    }
    __syncthreads();
  }
  if (tid < W && live[tid] == 2) cand[tid * W] = entry_key(0.0f, (uint32_t)a.end);
  __syncthreads();
  constexpr double kBottom = -__builtin_huge_val();
  for (int i = tid; i < W * W; i += kMergeThreads) {
    const int w = i / W;
    const uint64_t k = cand[i];
    double r = kBottom;
    if (k != 0) {
      const float l = key_value(k);
      r = base[w] + (live[w] == 2 || l == rmax[w] ? 0.0 : (double)l - (double)rmax[w]);
    }
    raw[i] = r;
    rank[i] = r * factor[w];
    before[i] = rank[i] > kBottom ? i - w * W : W;  // in its own beam's list; W: does not count
    if (rank[i] > kBottom) atomicAdd(&valid, 1);
  }
  __syncthreads();
  // of the other beams' lists, by halving: those above, and among equals those of lower beams
  for (int u = tid; u < W * W * W; u += kMergeThreads) {
    const int i = u / W, o = u - i * W;
    if (before[i] >= W || o == i / W) continue;
    const double mine = rank[i];
    int lo = 0, hi = W;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const double r = rank[o * W + mid];
      if (r > mine || (r == mine && o * W < i)) lo = mid + 1;
      else hi = mid;
    }
    if (lo > 0) atomicAdd(&before[i], lo);
  }
  __syncthreads();
  for (int i = tid; i < W * W; i += kMergeThreads) {
    const int better = before[i];
    if (better >= W) continue;
    const int w = i / W, token = (int)key_index(cand[i]);
    const bool over = live[w] == 2;
    const int64_t o = r0 + better;
    a.tokens[o] = token;
    a.parents[o] = w;
    a.scores_out[o] = (float)raw[i];
    a.lengths_out[o] = len0[w] + (over ? 0 : 1);
    a.ended_out[o] = over || token == a.end;
  }
  if (tid < W && tid >= valid) {
    const int64_t o = r0 + tid;
    a.tokens[o] = -1;
    a.parents[o] = -1;
    a.scores_out[o] = kNone;
    a.lengths_out[o] = 0;
    a.ended_out[o] = 1;
  }
}

// ---------------------------------------------------------------- states behind the beams

constexpr int kMaxPools = 8, kFewPools = 3;
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = 16384;  // of a work item: one 64 x 64 fp32 block
constexpr int kMaxChildren = 4096;

struct RPool {
  char* base;
  int64_t layer_stride, slot_bytes;  // slot_bytes: of one layer; slots are that far apart
  int layers, pieces;                // work items of a layer's slot
};
// Room for N pools: the host takes longer for more bytes of arguments (3 pools 2.9 us, 8 pools 3.2).
template <int N>
struct RArgs {
  int W, children, n_slots;
  const int32_t *slots, *parents, *skip;
  int32_t* slots_out;
  int items;  // work items of a slot: all pools, all layers
  RPool p[N];
};

// Every workgroup works the copies out by itself (up to 4096 children, in LDS: a launch of its own for that
// would cost more), then they share the work items out evenly.  Bound by memory: 16 x 8 beams of a 24-layer state, 1.13 GB
// moved, 237 us at 4.77 TB/s, which is what a large copy reaches; a small one by its launch (4.7 - 6 us).
template <int N>
__global__ __launch_bounds__(kCopyThreads) void beam_reorder_kernel(RArgs<N> a) {
  extern __shared__ __attribute__((aligned(16))) int lds[];
  int* const par = lds;                   // [children]: parent, or -1 where no state goes along
  int2* const moves = reinterpret_cast<int2*>(lds + ((a.children + 1) & ~1));  // [children]: from slot, to slot
  __shared__ int wcount[kCopyThreads / 64], total;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = a.W;
  if (tid == 0) total = 0;
  for (int i = tid; i < a.children; i += kCopyThreads) {
    const int p = a.parents[i];
    par[i] = p >= 0 && p < W && !(a.skip && a.skip[i]) ? p : -1;
  }
  __syncthreads();
  for (int i0 = 0; i0 < a.children; i0 += kCopyThreads) {
    const int i = i0 + tid;
    bool copy = false;
    int from = 0, to = 0;
    if (i < a.children) {
      const int r0 = i / W * W, c = i - r0, mine = par[i];
      uint32_t used = 0;   // beams with a child that carries its state on
      int others = 0;      // children before this one that take a slot that is left over
      bool keeps = false;
      for (int j = 0; j < W; ++j) {
        const int p = par[r0 + j];
        const bool first = p >= 0 && !(used >> p & 1);
        if (first) used |= 1u << p;
        if (j < c) others += !first;
        if (j == c) keeps = first;
      }
      if (keeps) {
        to = a.slots[r0 + mine];
      } else {
        uint32_t rest = ~used;
        for (int j = 0; j < others; ++j) rest &= rest - 1;
        to = a.slots[r0 + __builtin_ctz(rest)];
        if (mine >= 0) {
          from = a.slots[r0 + mine];
          copy = from >= 0 && from < a.n_slots && to >= 0 && to < a.n_slots && from != to;
        }
      }
      if (blockIdx.x == 0) a.slots_out[i] = to;
    }
    const uint64_t bal = __ballot(copy);
    if (lane == 0) wcount[wave] = __popcll(bal);
    __syncthreads();
    int at = total + __popcll(bal & ((1ull << lane) - 1));
    for (int w = 0; w < wave; ++w) at += wcount[w];
    if (copy) moves[at] = int2{from, to};
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < kCopyThreads / 64; ++w) total += wcount[w];
    __syncthreads();
  }
  const int64_t work = (int64_t)total * a.items;
  for (int64_t u = blockIdx.x; u < work; u += gridDim.x) {
    const int2 mv = moves[u / a.items];
    int item = (int)(u % a.items), pi = 0;
    while (item >= a.p[pi].layers * a.p[pi].pieces) item -= a.p[pi].layers * a.p[pi].pieces, ++pi;
    const RPool& P = a.p[pi];
    const int layer = item / P.pieces, piece = item - layer * P.pieces;
    char* const b = P.base + layer * P.layer_stride + (int64_t)piece * kCopyBytes;
    const int64_t bytes = P.slot_bytes - (int64_t)piece * kCopyBytes;
    const char* const src = b + mv.x * P.slot_bytes;
    char* const dst = b + mv.y * P.slot_bytes;
    uv4 t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = (j * kCopyThreads + tid) * 16;
      if (o < bytes) t[j] = *reinterpret_cast<const uv4*>(src + o);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = (j * kCopyThreads + tid) * 16;
      if (o < bytes) *reinterpret_cast<uv4*>(dst + o) = t[j];
    }
  }
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  return na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

int groups_of(int V) { return (V + kGroup - 1) / kGroup; }

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int64_t vkwr_beam_workspace_bytes(int B, int W, int V) {
  if (B < 0 || W < 1 || W > kMaxBeams || V < 1 || V > kMaxVocab) return -1;
  return (int64_t)B * W * groups_of(V) * (int64_t)(W * sizeof(uint64_t) + sizeof(RowStat));
}

extern "C" int vkwr_beam_select(int B, int W, int V, const void* logits, int logits_f16, const float* scores,
                                const int32_t* lengths, const int32_t* ended, int32_t* tokens, int32_t* parents,
                                float* scores_out, int32_t* lengths_out, int32_t* ended_out, int end,
                                float length_penalty, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "vkwr_beam_select";
  VK_REQUIRE(B >= 0 && W >= 1 && W <= kMaxBeams && V >= 1 && V <= kMaxVocab,
             "%s: bad size B=%d W=%d V=%d (1 to %d beams, vocabularies up to %d)", fn, B, W, V, kMaxBeams, kMaxVocab);
  VK_REQUIRE(length_penalty >= 0.0f && length_penalty <= 16.0f, "%s: length penalty %g is not between 0 and 16", fn,
             (double)length_penalty);
  VK_REQUIRE(end >= -1 && end < V, "%s: end token %d of %d", fn, end, V);
  if (B == 0) return VKWR_OK;
  const int64_t rows = (int64_t)B * W;
  VK_REQUIRE(rows <= 65535, "%s: %lld rows, at most 65535", fn, (long long)rows);
  VK_REQUIRE(logits && scores && lengths && ended && tokens && parents && scores_out && lengths_out && ended_out,
             "%s: null pointer", fn);
  const int64_t need = vkwr_beam_workspace_bytes(B, W, V);
  VK_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need,
             "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", fn, (long long)need,
             (long long)workspace_bytes);
  const void* const ins[] = {scores, lengths, ended};
  void* const outs[] = {tokens, parents, scores_out, lengths_out, ended_out};
  const int64_t logits_bytes = rows * V * (logits_f16 ? 2 : 4);
  for (const void* in : ins) VK_REQUIRE(!overlap(in, 4 * rows, workspace, need), "%s: an input overlaps the workspace", fn);
  VK_REQUIRE(!overlap(logits, logits_bytes, workspace, need), "%s: the logits overlap the workspace", fn);
  for (int i = 0; i < 5; ++i) {
    for (const void* in : ins) VK_REQUIRE(!overlap(outs[i], 4 * rows, in, 4 * rows), "%s: an output overlaps an input", fn);
    for (int j = 0; j < i; ++j) VK_REQUIRE(!overlap(outs[i], 4 * rows, outs[j], 4 * rows), "%s: outputs overlap", fn);
    VK_REQUIRE(!overlap(outs[i], 4 * rows, workspace, need) && !overlap(outs[i], 4 * rows, logits, logits_bytes),
               "%s: an output overlaps the workspace or the logits", fn);
  }
  BeamArgs a{};
  a.logits = logits;
  a.scores = scores;
  a.lengths = lengths;
  a.ended = ended;
  a.tokens = tokens;
  a.parents = parents;
  a.scores_out = scores_out;
  a.lengths_out = lengths_out;
  a.ended_out = ended_out;
  a.W = W;
  a.V = V;
  a.groups = groups_of(V);
  a.end = end;
  a.alpha = length_penalty;
  a.stats = reinterpret_cast<RowStat*>(workspace);
  a.keys = reinterpret_cast<uint64_t*>(a.stats + rows * a.groups);
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)a.groups, (unsigned)rows), block(kRowThreads);
  if (logits_f16) hipLaunchKernelGGL(beam_rows_kernel<true>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(beam_rows_kernel<false>, grid, block, 0, s, a);
  if (int e = check_launch(fn)) return e;
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)B), dim3(kMergeThreads), 0, s, a);
  return check_launch(fn);
}

extern "C" int vkwr_beam_reorder(int B, int W, int n_slots, const int32_t* slots, const int32_t* parents,
                                 const int32_t* skip, int32_t* slots_out, int n_pools, const vkwr_beam_pool* pools,
                                 void* stream) {
  clear_error();
  const char* fn = "vkwr_beam_reorder";
  VK_REQUIRE(B >= 0 && W >= 1 && W <= kMaxBeams && (int64_t)B * W <= kMaxChildren,
             "%s: bad size B=%d W=%d (1 to %d beams, at most %d together)", fn, B, W, kMaxBeams, kMaxChildren);
  VK_REQUIRE(n_slots >= 0 && n_pools >= 0 && n_pools <= kMaxPools && (n_pools == 0 || pools), "%s: %d pools (at most %d) of %d slots",
             fn, n_pools, kMaxPools, n_slots);
  if (B == 0) return VKWR_OK;
  const int64_t nb = 4ll * B * W;
  VK_REQUIRE(slots && parents && slots_out, "%s: null pointer", fn);
  VK_REQUIRE(!overlap(slots_out, nb, slots, nb) && !overlap(slots_out, nb, parents, nb) &&
                 !(skip && overlap(slots_out, nb, skip, nb)),
             "%s: slots_out overlaps an input", fn);
  RArgs<kMaxPools> a{};
  a.W = W;
  a.children = B * W;
  a.n_slots = n_slots;
  a.slots = slots;
  a.parents = parents;
  a.skip = skip;
  a.slots_out = slots_out;
  int64_t items = 0;
  for (int i = 0; i < n_pools; ++i) {
    const vkwr_beam_pool& p = pools[i];
    VK_REQUIRE(p.layers >= 0 && p.slot_bytes >= 0 && p.slot_bytes % 16 == 0 && p.slot_bytes <= (1ll << 36) &&
                   p.layers <= (1 << 20),
               "%s: pool %d: %lld layers of %lld bytes a slot (a multiple of 16)", fn, i, (long long)p.layers,
               (long long)p.slot_bytes);
    if (p.layers == 0 || p.slot_bytes == 0 || n_slots == 0) continue;
    VK_REQUIRE(p.base && (uintptr_t)p.base % 16 == 0, "%s: pool %d: null pointer, or not 16-byte aligned", fn, i);
    VK_REQUIRE(p.layers * p.slot_bytes <= (1ll << 48) / n_slots, "%s: slots too large", fn);  // (no such memory, and no overflow below)
    const int64_t whole = p.layers * p.slot_bytes * n_slots;
    VK_REQUIRE(!overlap(slots_out, nb, p.base, whole) && !overlap(slots, nb, p.base, whole) &&
                   !overlap(parents, nb, p.base, whole) && !(skip && overlap(skip, nb, p.base, whole)),
               "%s: pool %d overlaps the tables", fn, i);
    for (int j = 0; j < i; ++j)
      VK_REQUIRE(!overlap(p.base, whole, pools[j].base, pools[j].layers * pools[j].slot_bytes * n_slots),
                 "%s: pools %d and %d overlap", fn, j, i);
    RPool& r = a.p[i];
    r.base = static_cast<char*>(p.base);
    r.slot_bytes = p.slot_bytes;
    r.layer_stride = p.slot_bytes * n_slots;
    r.layers = (int)p.layers;
    r.pieces = (int)((p.slot_bytes + kCopyBytes - 1) / kCopyBytes);
    items += (int64_t)r.layers * r.pieces;
    VK_REQUIRE(items < (1ll << 31), "%s: slots too large", fn);
  }
  a.items = (int)items;
  const int64_t most = items * (int64_t)B * std::max(0, W - 1);
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, 8 * device_cus()));
  const size_t lds = (size_t)((a.children + 1) & ~1) * 4 + (size_t)a.children * 8;
  if (n_pools <= kFewPools) {
    RArgs<kFewPools> few{a.W, a.children, a.n_slots, slots, parents, skip, slots_out, a.items, {}};
    std::copy(a.p, a.p + kFewPools, few.p);
    hipLaunchKernelGGL(beam_reorder_kernel<kFewPools>, dim3(grid), dim3(kCopyThreads), lds, (hipStream_t)stream, few);
  } else {
    hipLaunchKernelGGL(beam_reorder_kernel<kMaxPools>, dim3(grid), dim3(kCopyThreads), lds, (hipStream_t)stream, a);
  }
  return check_launch(fn);
}
