// Low-rank adapters of many requests beside a shared projection.
//
//   y_i = epi(base_i + scale[g] (x_i A_g^T) B_g^T),  g = adapters[i]; no adapter (g < 0): y_i = epi(base_i)
//
// x [m, K], A [G, R, K], B [G, N, R], base and y [m, N] fp16; sums in fp32.
//
// Plan: the rows ordered by adapter and cut into tiles of at most kTileM rows of one adapter, made
// on the device from the step's adapter indices, once for every projection of the step.
// Two launches per set of projections:
//   shrink  h = x A^T for each tile, K cut into parts that fill the chip when there are few tiles
//           (a decode batch); fp32 parts go to scratch
//   expand  the parts added in order, y = epi(base + scale h B^T)
// Both run on the matrix cores with 16 rows of x (or h) as the columns of v_mfma_f32_16x16x32_f16,
// the adapter's rows as its rows.  h is not rounded to fp16: it enters the second product as a sum
// of two halves (fp16(h) and fp16(h - fp16(h)), a product each), after a power of two per row has brought its
// largest value to [2^14, 2^15), the top of fp16's range, as what is far below the largest leaves it at the
// lower end: 22 bits of each value, and never more than 2^-39 of the row's largest off.  (128 products with
// fp16 entries of B stay below 2^38 in the fp32 sums.)

#include <algorithm>

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

typedef _Float16 hv8 __attribute__((ext_vector_type(8)));
typedef float fv4 __attribute__((ext_vector_type(4)));

constexpr int kTileM = 64;         // rows of a tile: up to 4 columns blocks of 16
constexpr int kSub = kTileM / 16;
constexpr int kMaxTargets = 8;
constexpr int kMaxRank = 128;
constexpr int kMaxAdapters = 8192;
constexpr int kMaxTiles = 65535;   // rows of the grid
constexpr int kRankBlock = 64;     // ranks per shrink workgroup
constexpr int kExpandWaves = 4;
constexpr int kNone = -1, kBad = -2;

struct Tile {
  int adapter, row0, rows;
  int blocks;  // blocks of 16 rows that the adapter has, 4 of more: how the first product cuts K
};
struct PlanHead {
  int n_tiles;     // all tiles
  int n_adapter;   // those with an adapter (they come first)
  int m, G;        // what it was made for
};

__host__ __device__ inline int64_t max_tiles(int64_t m, int64_t G) { return (m < G + 2 ? m : G + 2) + m / kTileM; }

__device__ __forceinline__ const Tile* plan_tiles(const void* plan) {
  return reinterpret_cast<const Tile*>(reinterpret_cast<const char*>(plan) + sizeof(PlanHead));
}
// The rows' numbers, kTileM places per tile (those behind its rows hold anything): where a workgroup's rows
// are hangs on no other load.
__device__ __forceinline__ const int32_t* plan_order(const void* plan, int64_t tiles) {
  return reinterpret_cast<const int32_t*>(plan_tiles(plan) + tiles);
}

// One workgroup: counts per bin (adapters, then rows without one, then indices out of range), prefix
// sums of counts and tiles, tiles, and the rows' places.  Rows of one bin are placed in the order
// in which their waves get there, in any of the adapter's tiles; what is computed for a row does not depend
// on its place, as all tiles of an adapter cut K alike.  Bound by the
// latency of its dozen dependent steps: 4 us up to 4096 rows.
__global__ __launch_bounds__(1024) void lora_plan_kernel(int64_t m, int G, const int32_t* adapters, void* plan,
                                                         int64_t tiles_cap) {
  extern __shared__ int lds[];
  int* const cnt = lds;          // [G + 2] counts, then next free place (of the tiles' kTileM each)
  int* const red = lds + G + 2;  // [32]
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, nb = G + 2;
  Tile* const tiles = const_cast<Tile*>(plan_tiles(plan));
  int32_t* const order = const_cast<int32_t*>(plan_order(plan, tiles_cap));
  auto bin_of = [&](int64_t i) {
    const int g = adapters[i];
    return g < 0 ? G : g < G ? g : G + 1;
  };
  // this lane's place among `take` consecutive ones of its bin; one atomic where a wave agrees
  auto place = [&](bool live, int bin) {
    const int first = __builtin_amdgcn_readfirstlane(bin);
    if (__ballot(live && bin == first) == ~0ull) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&cnt[bin], 64);
      return __builtin_amdgcn_readfirstlane(at) + lane;
    }
    return live ? atomicAdd(&cnt[bin], 1) : 0;
  };
  // the first 4096 rows' bins stay in registers between the two passes
  constexpr int kHeld = 4;
  int held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) held[u] = u * 1024 + t < m ? bin_of(u * 1024 + t) : -1;
  for (int k = t; k < nb; k += 1024) cnt[k] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u * 1024 < m) place(held[u] >= 0, held[u] >= 0 ? held[u] : 0);
  for (int64_t i0 = kHeld * 1024; i0 < m; i0 += 1024) {
    const bool live = i0 + t < m;
    place(live, live ? bin_of(i0 + t) : 0);
  }
  __syncthreads();
  const int per = (nb + 1023) / 1024, k0 = min(t * per, nb), k1 = min(k0 + per, nb);
  int rows = 0, tl = 0;
  for (int k = k0; k < k1; ++k) {
    rows += cnt[k];
    tl += (cnt[k] + kTileM - 1) / kTileM;
  }
  int ri = rows, ti = tl;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(ri, d, 64), b = __shfl_up(ti, d, 64);
    if (lane >= d) {
      ri += a;
      ti += b;
    }
  }
  if (lane == 63) {
    red[wv] = ri;
    red[16 + wv] = ti;
  }
  __syncthreads();
  int row = ri - rows, tile = ti - tl;
  for (int w = 0; w < wv; ++w) {
    row += red[w];
    tile += red[16 + w];
  }
  PlanHead* const head = reinterpret_cast<PlanHead*>(plan);
  if (t == 0) {
    head->m = (int)m;
    head->G = G;
  }
  for (int k = k0; k < k1; ++k) {
    const int c = cnt[k];
    if (k == G) head->n_adapter = tile;
    for (int r = 0; r < c; r += kTileM)
      tiles[tile++] = Tile{k < G ? k : k == G ? kNone : kBad, row + r, min(kTileM, c - r), min((c + 15) / 16, kSub)};
    if (k == nb - 1) head->n_tiles = tile;
    cnt[k] = (tile - (c + kTileM - 1) / kTileM) * kTileM;  // its first tile's first place
    row += c;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    if (u * 1024 >= m) break;
    const int at = place(held[u] >= 0, held[u] >= 0 ? held[u] : 0);
    if (held[u] >= 0) order[at] = u * 1024 + t;
  }
  for (int64_t i0 = kHeld * 1024; i0 < m; i0 += 1024) {
    const bool live = i0 + t < m;
    const int at = place(live, live ? bin_of(i0 + t) : 0);
    if (live) order[at] = (int32_t)(i0 + t);
  }
}

struct Target {
  const _Float16 *x, *a, *b, *base;
  _Float16* y;
  int n, k;
  int relu2;
};
struct LoraArgs {
  const void* plan;
  int64_t tiles_cap, m;
  int G;
  const float* scale;
  float* h;        // [parts][target][m][rank_pad]
  int rank, rank_pad, n_targets, parts, cols;
  Target t[kMaxTargets];
};

// What a workgroup is to do: the arguments in one round of scalar loads, the plan's in a second.  (Left to
// the compiler they came one by one where they are used, a dozen round trips one after the other.)
struct Work {
  const _Float16 *x, *a, *b, *base;
  _Float16* y;
  int n, k, relu2;
  const float* scale;
  float* h;
  int64_t m;
  int rank, rank_pad, n_targets, parts, cols;
  int tiles, adapter_tiles;  // 0: a plan for something else
  Tile tile;
  const int32_t* order;
  int mine;  // lane l: row number l of the tile
};
__device__ __forceinline__ Work work_of(const LoraArgs& p) {
  const Target& t = p.t[blockIdx.z];
  Work w{t.x,    t.a,        t.b,         t.base,  t.y,    t.n, t.k, t.relu2, p.scale, p.h, p.m,
         p.rank, p.rank_pad, p.n_targets, p.parts, p.cols, 0,   0,   {},      nullptr, 0};
  const void* plan = p.plan;
  const int64_t cap = p.tiles_cap;
  const int G = p.G;
  asm volatile("" ::"s"(w.x), "s"(w.a), "s"(w.b), "s"(w.base), "s"(w.y), "s"(w.n), "s"(w.k), "s"(w.relu2), "s"(w.scale),
               "s"(w.h), "s"(w.m), "s"(w.rank), "s"(w.rank_pad), "s"(w.n_targets), "s"(w.parts), "s"(w.cols), "s"(plan),
               "s"(cap), "s"(G));
  w.order = plan_order(plan, cap) + (int64_t)blockIdx.y * kTileM;
  w.mine = __hip_atomic_load(w.order + (threadIdx.x & 63), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
  const PlanHead head = *reinterpret_cast<const PlanHead*>(plan);
  w.tile = plan_tiles(plan)[blockIdx.y];  // blockIdx.y < tiles_cap: inside the plan, stale or not
  asm volatile("" ::"s"(head.n_tiles), "s"(head.n_adapter), "s"(head.m), "s"(head.G), "s"(w.tile.adapter), "s"(w.tile.row0),
               "s"(w.tile.rows), "s"(w.tile.blocks));
  const bool ours = head.m == w.m && head.G == G;
  w.tiles = ours ? head.n_tiles : 0;
  w.adapter_tiles = ours ? head.n_adapter : 0;
  return w;
}

__device__ __forceinline__ fv4 mfma(hv8 a, hv8 b, fv4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// x A^T of 16 rows over the 32-deep steps s0 .. s1 - 1: two steps' loads together, up to 32 ranks
// requested while the two before are multiplied.
template <int RT>
__device__ __forceinline__ void shrink_steps(const _Float16* xr, const _Float16* const* ar, int kg, int K, int s0, int s1,
                                             fv4 (&acc)[RT]) {
  const hv8 zero = {};
  struct Pair {
    hv8 a[2][RT], b[2];
  };
  auto load = [&](Pair& f, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int k = 32 * (st + u) + kg;
      const bool in = st + u < s1 && k < K;
      f.b[u] = in ? *reinterpret_cast<const hv8*>(xr + k) : zero;
#pragma unroll
      for (int j = 0; j < RT; ++j) f.a[u][j] = in ? *reinterpret_cast<const hv8*>(ar[j] + k) : zero;
    }
  };
  auto multiply = [&](const Pair& f) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < RT; ++j) acc[j] = mfma(f.a[u][j], f.b[u], acc[j]);
  };
  Pair p;
  if constexpr (RT > 2) {  // no registers for two pairs
    for (int st = s0; st < s1; st += 2) {
      load(p, st);
      multiply(p);
    }
    return;
  }
  Pair q;
  load(p, s0);
  for (int st = s0; st < s1; st += 4) {
    if (st + 2 < s1) load(q, st + 2);
    multiply(p);
    if (st + 2 >= s1) break;
    if (st + 4 < s1) load(p, st + 4);
    multiply(q);
  }
}

// Grid: x = rank block * parts + part, y = tile, z = target.  A wave takes one block of 16 rows; the
// eight waves cut the part's K in 8 for one block, in 4 for two, in 2 for three or four.  The waves' sums
// are added in K order through LDS.
//
// Tiles of three or four blocks (prompt chunks) go through LDS: the 16 rows of an operand, 2 K bytes apart,
// fall on the same sets of the vector cache, so that operands loaded straight into registers, 64 bytes of
// a row at a time, came in twice (four projections of 2304 rows, K = 4096, rank 64: 107 us; through LDS
// 34, 4.2 TB/s of the 142 MB that x and A are).  Stages of 64 k -- 64 rows of x and 64 of A, 128 bytes each,
// written by DMA, row r's 16-byte chunk c at place c ^ (r & 7) -- in a ring of four, three of them in flight.
constexpr int kShrinkWaves = 8;
constexpr int kStageK = 64, kStages = 4;
constexpr int kStageHalfs = 2 * kTileM * kStageK;
template <int RT>
__global__ __launch_bounds__(64 * kShrinkWaves, 4) void lora_shrink_kernel(LoraArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[kStages * kStageHalfs * 2];  // the ring, then the waves' sums
  fv4(*const lds)[RT][64] = reinterpret_cast<fv4(*)[RT][64]>(smem);
  static_assert((kShrinkWaves - 1) * kRankBlock / 16 * 1024 <= kStages * kStageHalfs * 2, "the sums fit");
  const Work tg = work_of(p);
  const Tile tile = tg.tile;
  if ((int)blockIdx.y >= tg.adapter_tiles) return;
  auto row_of = [&](int r) { return (int64_t)__shfl(tg.mine, min(r, tile.rows - 1), 64); };
  const int rb = (int)blockIdx.x >= tg.parts ? 1 : 0, part = (int)blockIdx.x - rb * tg.parts, r0 = rb * kRankBlock;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int K = tg.k, ns = tile.blocks;
  const int li = lane & 15, kg = 8 * (lane >> 4);
  const int rbits = ns == 1 ? 0 : ns == 2 ? 1 : 2;  // 2^rbits waves along the rows
  const int ri = wv & ((1 << rbits) - 1), ki = wv >> rbits;
  const int r = 16 * ri + li;
  const _Float16* xr = tg.x + row_of(r) * K;
  const _Float16* ar[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j)
    ar[j] = tg.a + ((int64_t)tile.adapter * tg.rank + min(r0 + 16 * j + li, tg.rank - 1)) * K;
  // this wave's 32-deep steps of the part
  const int steps = (K + 31) >> 5, chunks = (kShrinkWaves >> rbits) * tg.parts;
  const int c = (kShrinkWaves >> rbits) * part + ki;
  const int s0 = (int)((int64_t)steps * c / chunks), s1 = (int)((int64_t)steps * (c + 1) / chunks);
  fv4 acc[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j] = fv4{0.0f, 0.0f, 0.0f, 0.0f};
  if (rbits < 2) {
    if (ri < ns) shrink_steps<RT>(xr, ar, kg, K, s0, s1, acc);
  } else {
    const int blocks = (K + kStageK - 1) / kStageK;
    const int b0 = (int)((int64_t)blocks * part / tg.parts);
    const int b1 = (int)((int64_t)blocks * (part + 1) / tg.parts);
    // DMA instruction: 8 rows; wave w fills rows 8 w .. of x and rows 8 (w mod 2 RT) .. of A
    _Float16* const ring = reinterpret_cast<_Float16*>(smem);
    const int w = __builtin_amdgcn_readfirstlane(wv), aw = w % (2 * RT);
    const int xrow = 8 * w + (lane >> 3), arow = 8 * aw + (lane >> 3);
    const _Float16* const xs = tg.x + row_of(xrow) * K;
    const _Float16* const as = tg.a + ((int64_t)tile.adapter * tg.rank + min(r0 + arow, tg.rank - 1)) * K;
    const int xc = 8 * ((lane & 7) ^ (xrow & 7)), ac = 8 * ((lane & 7) ^ (arow & 7));
    auto issue = [&](int blk) __attribute__((always_inline)) {
      _Float16* const to = ring + ((blk - b0) % kStages) * kStageHalfs;
      // chunks past the end of K: the row's last one, made zero when they are read
      dma16(xs + min(blk * kStageK + xc, K - 8), to + w * 512);
      dma16(as + min(blk * kStageK + ac, K - 8), to + kTileM * kStageK + aw * 512);
    };
    for (int b = b0; b < min(b0 + kStages - 1, b1); ++b) issue(b);
    const int cc = 4 * ki + (lane >> 4);  // this lane's chunk: wave half ki multiplies 32 of the 64 k
    for (int b = b0; b < b1; ++b) {
      // stage b has landed once at most the two stages behind it are outstanding (two DMA each); the
      // barrier also ends the reads of the buffer that is filled next
      if (b + 2 < b1) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else if (b + 1 < b1) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (b + kStages - 1 < b1) issue(b + kStages - 1);
      const _Float16* const st = ring + ((b - b0) % kStages) * kStageHalfs;
      const hv8 zero = {};
      const bool in = b * kStageK + 8 * cc < K;
      hv8 fb = *reinterpret_cast<const hv8*>(st + r * kStageK + 8 * (cc ^ (r & 7)));
      fb = in ? fb : zero;
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        const int row = 16 * j + li;
        const hv8 fa = *reinterpret_cast<const hv8*>(st + (kTileM + row) * kStageK + 8 * (cc ^ (row & 7)));
        acc[j] = mfma(in ? fa : zero, fb, acc[j]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the ring is read
  }
  if (ki > 0) {
#pragma unroll
    for (int j = 0; j < RT; ++j) lds[((ki - 1) << rbits) + ri][j][lane] = acc[j];
  }
  __syncthreads();
  if (ki > 0 || r >= tile.rows) return;
  // lane (row li, ranks 16 j + 4 (lane / 16) ..): four consecutive ranks
  float* h = tg.h + ((int64_t)(part * tg.n_targets + (int)blockIdx.z) * tg.m + tile.row0) * tg.rank_pad + r0;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    if (r0 + 16 * j >= tg.rank_pad) break;
    for (int k = 0; k < (kShrinkWaves >> rbits) - 1; ++k) acc[j] += lds[(k << rbits) + ri][j][lane];
    *reinterpret_cast<fv4*>(h + (int64_t)r * tg.rank_pad + 16 * j + 4 * (lane >> 4)) = acc[j];
  }
}

__device__ __forceinline__ float relu2(float f) {
  f = f > 0.0f ? f : (f != f ? f : 0.0f);
  return f * f;
}

// Grid: x = block of cols columns, y = tile, z = target.  Up to 16 rows: the waves take 64 columns
// each at a time; more: half of the waves for each half of the row blocks.  Bound by memory where there are
// many rows (2304 rows, four projections of N = 4096, rank 64, 32 adapters: 66 us for 218 MB of base, y and
// B), else by its chain of loads: tile, row numbers, h's parts, B and base.  A fragment of B for each of four
// waves along the rows instead of two (6 waves per SIMD) took 103 us, base and y past the caches 81.
__global__ __launch_bounds__(64 * kExpandWaves, 4) void lora_expand_kernel(LoraArgs p) {
  extern __shared__ char dyn[];
  const Work tg = work_of(p);
  const Tile tile = tg.tile;
  const int N = tg.n, c0 = (int)blockIdx.x * tg.cols, c1 = min(c0 + tg.cols, N);
  if ((int)blockIdx.y >= tg.tiles || c0 >= N) return;
  const int32_t* const order = tg.order;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  if (tile.adapter < 0) {
    // no adapter: the epilogue alone; an index out of range: NaN
    if (tile.adapter == kNone && !tg.relu2 && tg.base == tg.y) return;
    const int per_row = (c1 - c0) >> 3;
    for (int i = tid; i < tile.rows * per_row; i += 64 * kExpandWaves) {
      const int r = i / per_row;
      const int64_t at = (int64_t)order[r] * N + c0 + 8 * (i - r * per_row);
      h8 v = ld8(tg.base + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (tile.adapter == kBad) v.v[e] = (_Float16)__builtin_nanf("");
        else if (tg.relu2) v.v[e] = f16_of(relu2((float)v.v[e]));
      }
      st8(tg.y + at, v);
    }
    return;
  }
  const int ns = (tile.rows + 15) >> 4, chunks = (tg.rank + 31) >> 5;
  const int li = lane & 15, grp = lane >> 4;
  const _Float16* const bw = tg.b + (int64_t)tile.adapter * N * tg.rank;
  const hv8 zero = {};
  // Product row li of column tile t is output column cw + 32 (t / 2) + 8 (li / 4) + 4 (t % 2) + li % 4, so that
  // a lane of group grp ends up with the columns cw + 32 q + 8 grp .. + 7 (q = 0, 1): four lanes cover 64
  // consecutive bytes of a row.
  auto weights = [&](int cw, int ch, hv8 (&fa)[4]) __attribute__((always_inline)) {
    const int rk = 32 * ch + 8 * grp;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int col = cw + 32 * (t >> 1) + 8 * (li >> 2) + 4 * (t & 1) + (li & 3);
      fa[t] = rk < tg.rank && col < c1 ? *reinterpret_cast<const hv8*>(bw + (int64_t)col * tg.rank + rk) : zero;
    }
  };
  const int rw = ns > 1 ? 2 : 1, per = (ns + rw - 1) / rw;  // waves along the rows; row blocks per wave
  const int ri = wv % rw, ci = wv / rw, pass = 64 * (kExpandWaves / rw);
  int64_t rows[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) rows[s] = (int64_t)__shfl(tg.mine, min(16 * (ri * per + s) + li, tile.rows - 1), 64) * N;
  // requested before h is waited for: the first pass's weights and base
  hv8 fa[4];
  h8 base[2][2];
  auto load_base = [&](int cw) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= per) break;
      const int64_t at = rows[s] + cw + 8 * grp;
      if (cw + 8 * grp < c1) base[s][0] = ld8(tg.base + at);
      if (cw + 8 * grp + 32 < c1) base[s][1] = ld8(tg.base + at + 32);
    }
  };

  hv8* const hf = reinterpret_cast<hv8*>(dyn);                          // [chunk][sub][half][lane]
  int* const back = reinterpret_cast<int*>(hf + chunks * kSub * 128);    // [kTileM] powers of two taken out of the rows
  // h = scale * (sum of the parts, in order), 8 ranks of a row per item, at most 4 items a lane; a row's
  // items lie in neighbouring lanes (rank_pad / 8, a power of two)
  const float sc = tg.scale ? tg.scale[tile.adapter] : 1.0f;
  const int groups = tg.rank_pad >> 3, gbits = 31 - __builtin_clz(groups);
  const float* h0 = tg.h + ((int64_t)blockIdx.z * tg.m + tile.row0) * tg.rank_pad;
  const int64_t plane = (int64_t)tg.n_targets * tg.m * tg.rank_pad;
  struct Parts {
    fv4 x[4], y[4];
  };
  auto load_parts = [&](Parts& f, int i, int q0) __attribute__((always_inline)) {  // four parts together
    const float* src = h0 + (int64_t)min(i >> gbits, tile.rows - 1) * tg.rank_pad + 8 * (i & (groups - 1));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float* at = src + min(q0 + q, tg.parts - 1) * plane;
      f.x[q] = *reinterpret_cast<const fv4*>(at);
      f.y[q] = *reinterpret_cast<const fv4*>(at + 4);
    }
  };
  auto live_at = [&](int i) { return (i >> gbits) < tile.rows && 8 * (i & (groups - 1)) < tg.rank; };
  // requested first, as the others wait for it
  Parts ph;
  if (live_at(tid)) load_parts(ph, tid, 0);
  weights(c0 + 64 * ci, 0, fa);
  load_base(c0 + 64 * ci);
  for (int i = tid; i - tid < 16 * ns * groups; i += 64 * kExpandWaves) {
    const int r = i >> gbits, gr = i & (groups - 1);
    float hv[8];
    uint32_t mx = 0;
    const bool live = r < tile.rows && 8 * gr < tg.rank;  // rows behind the tile's and ranks of the padding: 0
    {
      fv4 lo = fv4{0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
      if (live) {
        for (int q0 = 0; q0 < tg.parts; q0 += 4) {
          if (i != tid || q0 > 0) load_parts(ph, i, q0);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (q0 + q >= tg.parts) break;
            lo += ph.x[q];
            hi += ph.y[q];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        hv[e] = live ? (e < 4 ? lo[e & 3] : hi[e & 3]) * sc : 0.0f;
        const uint32_t size = __builtin_bit_cast(uint32_t, hv[e]) & 0x7fffffffu;
        mx = max(mx, size < 0x7f800000u ? size : 0);  // the largest finite one: infinities, NaN pass as they are
      }
    }
    for (int d = 1; d < groups; d <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d, 64));
    const int sh = 141 - max((int)(mx >> 23), 1);  // its biased exponent becomes that of [2^14, 2^15)
    if (r < kTileM && gr == 0) back[r] = -sh;
    hv8 vh, vl;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = __builtin_ldexpf(hv[e], sh);
      vh[e] = (_Float16)f;
      // an infinity has no second half
      vl[e] = __builtin_isinf((float)vh[e]) ? (_Float16)0.0f : (_Float16)(f - (float)vh[e]);
    }
    if (r < kTileM && (gr >> 2) < chunks) {
      hv8* d = hf + ((gr >> 2) * kSub + (r >> 4)) * 128 + 16 * (gr & 3) + (r & 15);
      d[0] = vh;
      d[64] = vl;
    }
  }
  __syncthreads();
  for (int cw = c0 + 64 * ci; cw < c1; cw += pass) {
    const bool in0 = cw + 8 * grp < c1, in1 = cw + 8 * grp + 32 < c1;
    fv4 acc[2][4];
    if (cw != c0 + 64 * ci) load_base(cw);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[s][t] = fv4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int ch = 0; ch < chunks; ++ch) {
      if (ch > 0 || cw != c0 + 64 * ci) weights(cw, ch, fa);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (s >= per) break;
        const hv8* fb = hf + (ch * kSub + min(ri * per + s, kSub - 1)) * 128 + lane;
        const hv8 hi = fb[0], lo = fb[64];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[s][t] = mfma(fa[t], hi, acc[s][t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[s][t] = mfma(fa[t], lo, acc[s][t]);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= per) break;
      const int r = 16 * (ri * per + s) + li;
      if (r >= tile.rows) continue;
      const int bk = back[r];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (!(q ? in1 : in0)) continue;
        h8 v = base[s][q];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = (float)v.v[e] + __builtin_ldexpf(acc[s][2 * q + (e >> 2)][e & 3], bk);
          v.v[e] = f16_of(tg.relu2 ? relu2(f) : f);
        }
        st8(tg.y + rows[s] + cw + 8 * grp + 32 * q, v);
      }
    }
  }
}

struct LoraPlan {
  int parts, rank_pad, rank_blocks, cols;
  int64_t bytes;
};

// K parts of the first product: enough workgroups for the chip, at least 512 deep each, or 256 where that
// leaves fewer than 128 (128 rows, 40 adapters, rank 32, K = 2048, N = 8192: 16.0 us with 4 parts, 16.5 with 8,
// which the second product has to add; 434 rows of K = 8192: 16.7 with 8, 15.8 with 16; 27 rows of 7 adapters, K =
// 2560: 15.2 with 4, 14.3 with 8).  Columns of the
// second product per workgroup: 256, or 128 where that leaves few workgroups (423 rows, 2 adapters of 16, N =
// 2048: 18.6 us, 21.0 with 256; 128 rows, 40 adapters, N = 8192: 21.1 and 18.4, as each adds h's parts up
// anew; wider ones expose their later columns' loads: 2304 rows, 4 of 4096, 67 us, 72 with 1024 columns and
// eight waves).  The number of tiles is known on the device only; the rows of a step that has them scattered
// make one per adapter.
LoraPlan lora_split(int64_t m, int G, int rank, int n_targets, int64_t k_min, int64_t n_max) {
  LoraPlan s{};
  s.rank_pad = 32;  // a power of two, so that a row's groups of 8 lie in neighbouring lanes
  while (s.rank_pad < rank) s.rank_pad *= 2;
  s.rank_blocks = (rank + kRankBlock - 1) / kRankBlock;
  const int64_t tiles = std::min<int64_t>(m, G) + m / kTileM;
  const int64_t each = tiles * n_targets * s.rank_blocks;
  int64_t parts = 1;
  while (parts < 16 && parts * each < 512 && k_min / (2 * parts) >= (parts * each < 128 ? 256 : 512)) parts *= 2;
  s.parts = (int)parts;
  s.cols = 256;
  while (s.cols > 128 && tiles * n_targets * (n_max / s.cols) < 512) s.cols /= 2;
  s.bytes = parts * n_targets * m * s.rank_pad * 4;
  return s;
}

int check_lora(const char* fn, int64_t m, int G, int rank, int n_targets, const vkwr_lora_target* t) {
  VK_REQUIRE(m >= 0 && m <= 0x7fffffff - 64, "%s: bad row count %lld", fn, (long long)m);
  VK_REQUIRE(G >= 1 && G <= kMaxAdapters, "%s: 1 to %d adapters, got %d", fn, kMaxAdapters, G);
  VK_REQUIRE(rank >= 8 && rank <= kMaxRank && rank % 8 == 0, "%s: rank must be a multiple of 8 up to %d, got %d", fn,
             kMaxRank, rank);
  VK_REQUIRE(n_targets >= 1 && n_targets <= kMaxTargets && t, "%s: 1 to %d targets, got %d", fn, kMaxTargets,
             n_targets);
  for (int i = 0; i < n_targets; ++i) {
    VK_REQUIRE(t[i].n >= 8 && t[i].n % 8 == 0 && t[i].n <= (1 << 20) && t[i].k >= 8 && t[i].k % 8 == 0 &&
                   t[i].k <= (1 << 20),
               "%s: target %d: n and k must be multiples of 8 up to 2^20, got n=%lld k=%lld", fn, i,
               (long long)t[i].n, (long long)t[i].k);
    VK_REQUIRE(t[i].epilogue == VKWR_GEMM_EPI_NONE || t[i].epilogue == VKWR_GEMM_EPI_RELU_SQUARE,
               "%s: target %d: unsupported epilogue %d", fn, i, t[i].epilogue);
  }
  return VKWR_OK;
}

int64_t least_k(int n_targets, const vkwr_lora_target* t) {
  int64_t k = t[0].k;
  for (int i = 1; i < n_targets; ++i) k = t[i].k < k ? t[i].k : k;
  return k;
}

int64_t most_n(int n_targets, const vkwr_lora_target* t) {
  int64_t n = t[0].n;
  for (int i = 1; i < n_targets; ++i) n = std::max(n, t[i].n);
  return n;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int64_t vkwr_lora_plan_bytes(int64_t m, int n_adapters) {
  if (m < 0 || n_adapters < 1 || n_adapters > kMaxAdapters || max_tiles(m, n_adapters) > kMaxTiles) return -1;
  return (int64_t)sizeof(PlanHead) + max_tiles(m, n_adapters) * (int64_t)(sizeof(Tile) + 4 * kTileM);
}

extern "C" int vkwr_lora_plan(int64_t m, int n_adapters, const int32_t* adapters, void* plan, int64_t plan_bytes,
                              void* stream) {
  clear_error();
  const char* fn = "vkwr_lora_plan";
  const int64_t need = vkwr_lora_plan_bytes(m, n_adapters);
  VK_REQUIRE(need >= 0, "%s: bad size (m=%lld, %d adapters; at most %d adapters and %d row tiles)", fn, (long long)m,
             n_adapters, kMaxAdapters, kMaxTiles);
  VK_REQUIRE(m == 0 || adapters, "%s: null pointer", fn);
  VK_REQUIRE(plan && plan_bytes >= need && (uintptr_t)plan % 16 == 0,
             "%s: needs a 16-byte aligned plan of %lld bytes, got %lld", fn, (long long)need, (long long)plan_bytes);
  hipLaunchKernelGGL(lora_plan_kernel, dim3(1), dim3(1024), (n_adapters + 2 + 32) * sizeof(int), (hipStream_t)stream, m,
                     n_adapters, adapters, plan, max_tiles(m, n_adapters));
  return check_launch(fn);
}

extern "C" int64_t vkwr_lora_workspace_bytes(int64_t m, int n_adapters, int rank, int n_targets,
                                             const vkwr_lora_target* targets) {
  clear_error();
  if (check_lora("vkwr_lora_workspace_bytes", m, n_adapters, rank, n_targets, targets)) return -1;
  const int64_t k = least_k(n_targets, targets), n = most_n(n_targets, targets);
  // Fewer rows can be cut into more parts (a power of two up to 16, which never grows with the rows), so for each
  // number of parts the most rows that have it.
  int64_t most = 0;
  for (int64_t rows = m; rows > 0;) {
    const LoraPlan s = lora_split(rows, n_adapters, rank, n_targets, k, n);
    most = std::max(most, s.bytes);
    int64_t lo = 0, hi = rows;  // the most rows with more parts: [lo, hi)
    while (hi - lo > 1) {
      const int64_t mid = lo + (hi - lo) / 2;
      (lora_split(mid, n_adapters, rank, n_targets, k, n).parts > s.parts ? lo : hi) = mid;
    }
    rows = lo;
  }
  return most;
}

extern "C" int vkwr_lora_f16(int64_t m, int n_adapters, int rank, const float* scale, const void* plan,
                             int n_targets, const vkwr_lora_target* targets, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "vkwr_lora_f16";
  if (int e = check_lora(fn, m, n_adapters, rank, n_targets, targets)) return e;
  if (m == 0) return VKWR_OK;
  const LoraPlan sp =
      lora_split(m, n_adapters, rank, n_targets, least_k(n_targets, targets), most_n(n_targets, targets));
  VK_REQUIRE(plan && (uintptr_t)plan % 16 == 0, "%s: null or misaligned plan", fn);
  VK_REQUIRE(workspace && workspace_bytes >= sp.bytes && (uintptr_t)workspace % 16 == 0,
             "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", fn, (long long)sp.bytes,
             (long long)workspace_bytes);
  LoraArgs a{};
  a.plan = plan;
  a.tiles_cap = max_tiles(m, n_adapters);
  a.m = m;
  a.G = n_adapters;
  a.scale = scale;
  a.h = reinterpret_cast<float*>(workspace);
  a.rank = rank;
  a.rank_pad = sp.rank_pad;
  a.n_targets = n_targets;
  a.parts = sp.parts;
  a.cols = sp.cols;
  int64_t widest = 0;
  for (int i = 0; i < n_targets; ++i) {
    const vkwr_lora_target& t = targets[i];
    const uint16_t* base = t.base ? t.base : t.y;
    VK_REQUIRE(t.x && t.a && t.b && t.y, "%s: target %d: null pointer", fn, i);
    VK_REQUIRE(((uintptr_t)t.x | (uintptr_t)t.a | (uintptr_t)t.b | (uintptr_t)t.y | (uintptr_t)base) % 16 == 0,
               "%s: target %d: pointers must be 16-byte aligned", fn, i);
    VK_REQUIRE(base == t.y || !overlap(base, 2 * m * t.n, t.y, 2 * m * t.n), "%s: target %d: base overlaps y", fn, i);
    for (int j = 0; j < n_targets; ++j) {
      VK_REQUIRE(!overlap(targets[j].x, 2 * m * targets[j].k, t.y, 2 * m * t.n), "%s: y of target %d overlaps x of %d",
                 fn, i, j);
      VK_REQUIRE(j == i || (!overlap(targets[j].y, 2 * m * targets[j].n, t.y, 2 * m * t.n) &&
                            !(targets[j].base && overlap(targets[j].base, 2 * m * targets[j].n, t.y, 2 * m * t.n))),
                 "%s: y of target %d overlaps y or base of %d", fn, i, j);
    }
    a.t[i] = Target{reinterpret_cast<const _Float16*>(t.x), reinterpret_cast<const _Float16*>(t.a),
                    reinterpret_cast<const _Float16*>(t.b), reinterpret_cast<const _Float16*>(base),
                    reinterpret_cast<_Float16*>(t.y), (int)t.n, (int)t.k,
                    t.epilogue == VKWR_GEMM_EPI_RELU_SQUARE};
    widest = std::max(widest, t.n);
  }
  VK_REQUIRE(a.tiles_cap <= kMaxTiles, "%s: %lld row tiles, at most %d", fn, (long long)a.tiles_cap, kMaxTiles);
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid(sp.parts * sp.rank_blocks, (unsigned)a.tiles_cap, n_targets);
  const int rt = (std::min(rank, kRankBlock) + 15) / 16;
  if (rt == 1) hipLaunchKernelGGL(lora_shrink_kernel<1>, grid, dim3(64 * kShrinkWaves), 0, s, a);
  else if (rt == 2) hipLaunchKernelGGL(lora_shrink_kernel<2>, grid, dim3(64 * kShrinkWaves), 0, s, a);
  else hipLaunchKernelGGL(lora_shrink_kernel<4>, grid, dim3(64 * kShrinkWaves), 0, s, a);
  const dim3 egrid((unsigned)((widest + sp.cols - 1) / sp.cols), (unsigned)a.tiles_cap, n_targets);
  const int lds = (rank + 31) / 32 * kSub * 2048 + kTileM * 4;
  hipLaunchKernelGGL(lora_expand_kernel, egrid, dim3(64 * kExpandWaves), lds, s, a);
  return check_launch(fn);
}
