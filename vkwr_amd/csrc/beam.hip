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
// fp64 (lane sums of 32 terms are fp32).
//
// States.  beam_reorder_kernel renames slots where it can: the first child of a beam keeps its
// parent's slot, every further one gets a copy in a slot whose beam has no child.  A source is
// never a destination, so the copies need no order and no second buffer.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

typedef _Float16 hv8 __attribute__((ext_vector_type(8)));
typedef float fv4 __attribute__((ext_vector_type(4)));
typedef uint32_t uv4 __attribute__((ext_vector_type(4)));

constexpr int kMaxBeams = 32;
constexpr int kMaxVocab = 1 << 20;
constexpr int kRowThreads = 256, kPer = 32, kGroup = kRowThreads * kPer;  // entries of a group
constexpr int kListCap = 512;    // entries above the bound that are ranked at once
constexpr int kMergeKeys = 4096;  // keys that a merge pass holds: 32 beams x 128 groups

// Entries in the order (value descending, index ascending); 0 is below every entry.
__device__ __forceinline__ uint64_t entry_key(float v, uint32_t i) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
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

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
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

// blockIdx.x: group of the row, blockIdx.y: row.  kVec: rows are 16-byte aligned; lane t then holds
// the 16-byte pieces t, t + 256, ... of the group, else its entries t, t + 256, ...
template <bool kHalf, bool kVec>
__global__ __launch_bounds__(kRowThreads) void beam_rows_kernel(BeamArgs a) {
  __shared__ float wmax[4], wbound[4];
  __shared__ double wsum[4];
  __shared__ uint64_t list[kListCap], wkey[4];
  __shared__ int count;
  const int64_t row = blockIdx.y;
  if (a.ended[row] || !(a.scores[row] > kNone)) return;  // (the merge leaves such rows out)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int i0 = blockIdx.x * kGroup, W = a.W;
  constexpr int kPiece = kVec ? (kHalf ? 8 : 4) : 1;
  auto index_of = [&](int e) { return i0 + ((e / kPiece) * kRowThreads + tid) * kPiece + e % kPiece; };

  float v[kPer];
#pragma unroll
  for (int j = 0; j < kPer / kPiece; ++j) {
    const int i = index_of(j * kPiece);
    if constexpr (kVec) {
      if (i < a.V) {  // V is a multiple of a piece
        if constexpr (kHalf) {
          const hv8 h = *reinterpret_cast<const hv8*>((const _Float16*)a.logits + row * a.V + i);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j * 8 + e] = (float)h[e];
        } else {
          const fv4 f = *reinterpret_cast<const fv4*>((const float*)a.logits + row * a.V + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j * 4 + e] = f[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) v[j * kPiece + e] = kNone;
      }
    } else {
      v[j] = kNone;
      if (i < a.V) v[j] = kHalf ? (float)((const _Float16*)a.logits)[row * a.V + i] : ((const float*)a.logits)[row * a.V + i];
    }
  }
  float top = kNone;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    v[e] = v[e] != v[e] ? kNone : v[e] + 0.0f;  // a NaN is never chosen; -0 equals 0
    top = fmaxf(top, v[e]);
  }
  // A bound that at least W entries reach: in each wave the q-th largest of the lanes' maxima,
  // 4 q >= W, and the smallest of the four.
  const int q = (W + 3) / 4;
  float left = top, bound = kNone, most = kNone;
  for (int s = 0; s < q; ++s) {
    bound = wave_max(left);
    if (s == 0) most = bound;
    const uint64_t at = __ballot(left == bound);
    if (lane == __builtin_ctzll(at)) left = kNone;
  }
  if (lane == 0) wmax[wave] = most, wbound[wave] = bound;
  if (tid == 0) count = 0;
  __syncthreads();
  const float mx = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
  bound = fminf(fminf(wbound[0], wbound[1]), fminf(wbound[2], wbound[3]));
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    // (at an infinite maximum only the entries that are infinite themselves count)
    const float d = v[e] - mx;
    sum += v[e] == mx ? 1.0f : v[e] > kNone ? __expf(d) : 0.0f;
    if (v[e] >= bound && v[e] > kNone) {
      const int n = atomicAdd(&count, 1);
      if (n < kListCap) list[n] = entry_key(v[e], (uint32_t)index_of(e));
    }
  }
  if (!(mx > kNone)) sum = 0.0f;
  const double ws = wave_sum64((double)sum);
  if (lane == 0) wsum[wave] = ws;
  __syncthreads();
  const int64_t g = row * a.groups + blockIdx.x;
  if (tid == 0) a.stats[g] = RowStat{mx, 0.0f, (wsum[0] + wsum[1]) + (wsum[2] + wsum[3])};
  uint64_t* const out = a.keys + g * W;
  const int n = count;
  if (n <= kListCap) {
    for (int i = tid; i < n; i += kRowThreads) {
      const uint64_t k = list[i];
      int better = 0;
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
      const uint64_t k = v[e] > kNone ? entry_key(v[e], (uint32_t)index_of(e)) : 0;
      if (k < last && k > best) best = k;
    }
    best = wave_max_key(best);
    if (lane == 0) wkey[wave] = best;
    __syncthreads();
    const uint64_t b01 = wkey[0] > wkey[1] ? wkey[0] : wkey[1], b23 = wkey[2] > wkey[3] ? wkey[2] : wkey[3];
    last = b01 > b23 ? b01 : b23;
    if (tid == 0) out[s] = last;
    __syncthreads();
  }
}

// One workgroup per request.  Every list of keys is sorted, so an entry's rank among several lists is
// its place in its own plus the heads of the others above it, counted until W are.
__global__ __launch_bounds__(256) void beam_merge_kernel(BeamArgs a) {
  __shared__ uint64_t keys[kMergeKeys];
  __shared__ uint64_t cand[kMaxBeams * kMaxBeams];  // [beam][W], sorted
  __shared__ double rank[kMaxBeams * kMaxBeams], raw[kMaxBeams * kMaxBeams];
  __shared__ double base[kMaxBeams], factor[kMaxBeams];
  __shared__ float rmax[kMaxBeams];
  __shared__ int live[kMaxBeams], valid;  // 0: offers nothing, 1: live, 2: finished
  const int tid = threadIdx.x, W = a.W, G = a.groups;
  const int64_t r0 = (int64_t)blockIdx.x * W;
  if (tid == 0) valid = 0;
  if (tid < W) {
    const float score = a.scores[r0 + tid];
    const bool over = a.ended[r0 + tid] != 0;
    int kind = score > kNone ? (over ? 2 : 1) : 0;
    const int len = a.lengths[r0 + tid] + (over ? 0 : 1);
    float mx = kNone;
    double sum = 0.0;
    if (kind == 1) {
      const RowStat* const st = a.stats + (r0 + tid) * G;
      for (int g = 0; g < G; ++g) mx = fmaxf(mx, st[g].max);
      for (int g = 0; g < G; ++g)
        if (st[g].max > kNone) sum += st[g].max == mx ? st[g].sum : st[g].sum * exp((double)st[g].max - (double)mx);
      if (!(mx > kNone)) kind = 0;  // not one token is allowed
    }
    live[tid] = kind;
    rmax[tid] = mx;
    base[tid] = (double)score - (kind == 1 ? log(sum) : 0.0);
    factor[tid] = a.alpha == 0.0f ? 1.0 : pow((double)(len > 1 ? len : 1), -(double)a.alpha);
  }
  for (int i = tid; i < W * W; i += 256) cand[i] = 0;
  __syncthreads();
  const int per_row = G * W, rows = kMergeKeys / per_row > W ? W : kMergeKeys / per_row;  // rows of a pass (at least 1)
  for (int w0 = 0; w0 < W; w0 += rows) {
    const int n = (W - w0 < rows ? W - w0 : rows) * per_row;
    for (int i = tid; i < n; i += 256) keys[i] = live[w0 + i / per_row] == 1 ? a.keys[(r0 + w0) * per_row + i] : 0;
    __syncthreads();
    for (int i = tid; i < n; i += 256) {
      const uint64_t k = keys[i];
      if (k == 0) continue;
      const int w = i / per_row, at = i - w * per_row, mine = at / W;
      int better = at - mine * W;
      for (int g = 0; g < G && better < W; ++g) {
        if (g == mine) continue;
        const uint64_t* const l = keys + w * per_row + g * W;
        for (int j = 0; j < W && l[j] > k; ++j) ++better;
      }
      if (better < W) cand[(w0 + w) * W + better] = k;
    }
    __syncthreads();
  }
  if (tid < W && live[tid] == 2) cand[tid * W] = entry_key(0.0f, (uint32_t)a.end);
  __syncthreads();
  for (int i = tid; i < W * W; i += 256) {
    const int w = i / W;
    const uint64_t k = cand[i];
    double r = -__builtin_huge_val();
    if (k != 0) {
      const float l = key_value(k);
      r = base[w] + (live[w] == 2 || l == rmax[w] ? 0.0 : (double)l - (double)rmax[w]);
    }
    raw[i] = r;
    rank[i] = r * factor[w];
    if (rank[i] > -__builtin_huge_val()) atomicAdd(&valid, 1);
  }
  __syncthreads();
  for (int i = tid; i < W * W; i += 256) {
    const double mine = rank[i];
    if (!(mine > -__builtin_huge_val())) continue;
    const int w = i / W;
    int better = i - w * W;
    for (int o = 0; o < W && better < W; ++o) {
      if (o == w) continue;
      // beams before this one win ties
      for (int j = 0; j < W && (rank[o * W + j] > mine || (o < w && rank[o * W + j] == mine)); ++j) ++better;
    }
    if (better >= W) continue;
    const bool over = live[w] == 2;
    const int token = (int)key_index(cand[i]);
    const int64_t o = r0 + better;
    a.tokens[o] = token;
    a.parents[o] = w;
    a.scores_out[o] = (float)raw[i];
    a.lengths_out[o] = a.lengths[r0 + w] + (over ? 0 : 1);
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

constexpr int kMaxPools = 8;
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = 16384;  // of a work item: one 64 x 64 fp32 block
constexpr int kMaxChildren = 4096;

struct RPool {
  char* base;
  int64_t layer_stride, slot_bytes;  // slot_bytes: of one layer; slots are that far apart
  int layers, pieces;                // work items of a layer's slot
};
struct RArgs {
  int W, children, n_pools, n_slots;
  const int32_t *slots, *parents, *skip;
  int32_t* slots_out;
  int items;  // work items of a slot: all pools, all layers
  RPool p[kMaxPools];
};

// Every workgroup works the copies out by itself (a few hundred children at most are looked at), then
// they share the work items out evenly.
__global__ __launch_bounds__(kCopyThreads) void beam_reorder_kernel(RArgs a) {
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
  for (int i = 0; i < 5; ++i) {
    for (const void* in : ins) VK_REQUIRE(!overlap(outs[i], 4 * rows, in, 4 * rows), "%s: an output overlaps an input", fn);
    for (int j = 0; j < i; ++j) VK_REQUIRE(!overlap(outs[i], 4 * rows, outs[j], 4 * rows), "%s: outputs overlap", fn);
    VK_REQUIRE(!overlap(outs[i], 4 * rows, workspace, need) && !overlap(outs[i], 4 * rows, logits, rows * V * (logits_f16 ? 2 : 4)),
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
  const bool vec = (uintptr_t)logits % 16 == 0 && V % (logits_f16 ? 8 : 4) == 0;
  if (logits_f16 && vec) hipLaunchKernelGGL((beam_rows_kernel<true, true>), grid, block, 0, s, a);
  else if (logits_f16) hipLaunchKernelGGL((beam_rows_kernel<true, false>), grid, block, 0, s, a);
  else if (vec) hipLaunchKernelGGL((beam_rows_kernel<false, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((beam_rows_kernel<false, false>), grid, block, 0, s, a);
  if (int e = check_launch(fn)) return e;
  hipLaunchKernelGGL(beam_merge_kernel, dim3((unsigned)B), dim3(256), 0, s, a);
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
  RArgs a{};
  a.W = W;
  a.children = B * W;
  a.n_pools = n_pools;
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
  hipLaunchKernelGGL(beam_reorder_kernel, dim3(grid), dim3(kCopyThreads), lds, (hipStream_t)stream, a);
  return check_launch(fn);
}
