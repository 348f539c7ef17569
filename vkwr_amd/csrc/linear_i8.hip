// Linear layers with 8-bit weights: y = f(s_i t_j sum_k q_ik w_jk [+ bias_j]).
//
// q_ik = round_half_even(127 x_ik / max|x_i|), s_i = max|x_i| / 127: each row of fp16 activations
// with a scale of its own; w_jk 8-bit weights with a scale t_j per output channel.  The sum over k
// is exact in int32 (127^2 2^17 < 2^31), so neither the order of the products nor a cut of K
// changes a bit of y.
//
// Both operands are held in the fragment order of v_mfma_i32_32x32x32_i8: the 32 rows x 32 k of
// one operand are one contiguous kilobyte, lane l holding row l % 32, k 16 (l / 32) .. + 15.
// Weights are packed once; the activations are written that way as they are rounded.  Every wave
// load, and every copy into LDS, is then one contiguous kilobyte, and every LDS read conflict-free.
// The weights are the first operand of a product, so that a lane's results are consecutive
// outputs of one row of y.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

typedef int iv4 __attribute__((ext_vector_type(4)));
typedef int iv16 __attribute__((ext_vector_type(16)));
typedef _Float16 hv8 __attribute__((ext_vector_type(8)));
typedef uint32_t uv4 __attribute__((ext_vector_type(4)));

constexpr int kMaxI8 = 8;          // problems per call
constexpr int kI8Rows = 32;        // rows of a block of packed 8-bit values
constexpr int kI8Pad = 128;        // K is padded to multiples of this, with zeros
constexpr int64_t kI8MaxK = 131072;   // 127^2 k < 2^31
constexpr int64_t kI8MaxRows = 1 << 22;  // of a matrix, and of all the activations of a call (launch sizes)

__host__ __device__ inline int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Byte of element (r, k) of a packed matrix with `steps` = padded K / 32.
__device__ __forceinline__ int64_t i8_index(int64_t r, int64_t k, int64_t steps) {
  return ((r >> 5) * steps + (k >> 5)) * 1024 + (((k >> 4) & 1) * 32 + (r & 31)) * 16 + (k & 15);
}

// The problems of a launch, with room for N.  A launch of one carries that one only: the host takes 2.7 us for
// 80 bytes of arguments and 3.4 for 700.
template <typename Prob, int N>
struct BatchOf {
  int n;
  Prob p[N];
};

// The problem that a workgroup belongs to: problems of equally many workgroups have a row of the grid each
// (kGridRows; a launch of one too), others are searched for by their first workgroups.  Kernels that live for a
// few microseconds read all of its fields in one round of loads (an empty asm holds them above
// the first branch): left alone the compiler reads each where it is used, one trip after another.
template <bool kGridRows, typename Prob, int N>
__device__ __forceinline__ int problem_of(const BatchOf<Prob, N>& bt, int b) {
  if constexpr (N == 1) return 0;
  if constexpr (kGridRows) return blockIdx.y;
  int pi = 0;
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (i < bt.n && b >= bt.p[i].wg_begin) pi = i;
  return pi;
}

// ---------------------------------------------------------------- rounding rows to 8 bits

struct QProb {
  const _Float16* x;
  int8_t* q;
  float* s;
  int m, k, steps;
  int wg_begin;  // first workgroup
};
typedef BatchOf<QProb, kMaxI8> QBatch;

// The 8 bits of 127 x / top for 16 values, halves to even.  127 x is exact in fp32; one correction
// of the product with 1 / top makes the quotient exact wherever it is representable, so that a
// quotient ending in .5 is seen as one, and every other is at least 2^-19 of itself away from
// a half (x and top have 11 bits each).  Adding 1.5 2^23 rounds to an integer in the low bits.
__device__ __forceinline__ uint32_t quant4(const float (&v)[4], float top, float inv) {
  uint32_t o = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = 127.0f * v[e];
    const float q0 = t * inv;
    const float q = __builtin_fmaf(__builtin_fmaf(-q0, top, t), inv, q0);
    o |= (__builtin_bit_cast(uint32_t, q + 12582912.0f) & 0xffu) << (8 * e);
  }
  return o;
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  typedef uint16_t u2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u2, a), __builtin_bit_cast(u2, b)));
}

// 8 values of a row from k0, zeros past K.  Rows that do not start on 16 bytes are loaded the same way
// (an unaligned load: one value at a time took 13 us for 77 rows of 2501, this 4).
__device__ __forceinline__ uv4 load8(const _Float16* x, int64_t k0, int k) {
  uv4 v = {0, 0, 0, 0};
  if (k0 + 8 <= k) {
    __builtin_memcpy(&v, x + k0, 16);
  } else if (k0 < k) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < k) v[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, x[k0 + e]) << (16 * (e & 1));
  }
  return v;
}

// 16 values of row x from k0.
__device__ __forceinline__ void load16(const _Float16* x, int64_t k0, int k, uv4 (&v)[2]) {
  v[0] = load8(x, k0, k);
  v[1] = load8(x, k0 + 8, k);
}

__device__ __forceinline__ uint32_t top_bits(uint32_t top, const uv4 (&v)[2]) {
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max_u16x2(top, v[w >> 2][w & 3] & 0x7fff7fffu);
  return top;
}

__device__ __forceinline__ iv4 quant16(const uv4 (&v)[2], float top, float inv) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  iv4 o;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const h2 a = __builtin_bit_cast(h2, (uint32_t)v[w >> 1][2 * (w & 1)]), b = __builtin_bit_cast(h2, (uint32_t)v[w >> 1][2 * (w & 1) + 1]);
    const float f[4] = {(float)a.x, (float)a.y, (float)b.x, (float)b.y};
    o[w] = (int)quant4(f, top, inv);
  }
  return o;
}

// T lanes per row, 256 / T rows per workgroup (T = 512: one row): so many that a lane holds 16 values, or 32 of
// rows past 4096, and a few hundred rows reach every CU (us: 128 rows of 2048 3.1, with 32 a lane 3.3; 433 of
// 8192 4.8, one wave per row 9.0; 2304 of 4096 9.0, of 16384 28 at 4.1 TB/s).  The 32 rows of
// a block go to one XCD (workgroup b runs on XCD b % 8), whose L2 joins the 16-byte pieces that they
// write into common lines.  Rows longer than 16384 are read twice.  |x| is compared as an integer, where an
// infinity or a NaN exceeds every number: such a row gets the scale NaN and zeros.
template <int T, int kKeep, bool kGridRows, int N>
__global__ __launch_bounds__(T < 256 ? 256 : T) void i8_rows_kernel(BatchOf<QProb, N> bt) {
  constexpr int kThreads = T < 256 ? 256 : T, kRows = kThreads / T, kWaves = T / 64;
  __shared__ uint32_t wtop[kThreads / 64];
  const QProb P = bt.p[problem_of<kGridRows>(bt, blockIdx.x)];
  asm volatile("" ::"s"(P.x), "s"(P.q), "s"(P.s), "s"(P.m), "s"(P.k), "s"(P.steps), "s"(P.wg_begin));
  const int u = (int)blockIdx.x - (kGridRows ? 0 : P.wg_begin), per = 32 / kRows;  // workgroups of a block of rows
  const int idx = u >> 3;
  const int64_t row = ((int64_t)(idx / per) * 8 + (u & 7)) * 32 + idx % per * kRows + threadIdx.x / T;
  const int t = threadIdx.x % T, wave = threadIdx.x >> 6;
  const int k = row < P.m ? P.k : 0, chunks = row < P.m ? P.steps * 2 : 0;  // chunks of 16
  const _Float16* const x = P.x + row * P.k;
  uv4 v[kKeep][2];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < kKeep; ++c) load16(x, (int64_t)(c * T + t) * 16, k, v[c]);
#pragma unroll
  for (int c = 0; c < kKeep; ++c) top = top_bits(top, v[c]);
  for (int c = kKeep * T + t; c < chunks; c += T) {
    uv4 w[2];
    load16(x, (int64_t)c * 16, k, w);
    top = top_bits(top, w);
  }
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
  if constexpr (kWaves > 1) {
    if ((threadIdx.x & 63) == 0) wtop[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = max(top, wtop[wave / kWaves * kWaves + w]);
  }
  if (row >= P.m) return;
  const bool finite = top < 0x7c00u;
  const float a = finite ? h2f((uint16_t)top) : 0.0f;
  const float inv = a > 0.0f ? 1.0f / a : 0.0f;
  if (t == 0) P.s[row] = finite ? a / 127.0f : __builtin_nanf("");
  int8_t* const q = P.q + i8_index(row, 0, P.steps);
  auto put = [&](int c, const uv4(&w)[2]) __attribute__((always_inline)) {
    const iv4 o = a > 0.0f ? quant16(w, a, inv) : iv4{0, 0, 0, 0};
    *reinterpret_cast<iv4*>(q + (int64_t)c * 512) = o;  // chunk c: 512 bytes on
  };
#pragma unroll
  for (int c = 0; c < kKeep; ++c)
    if (c * T + t < chunks) put(c * T + t, v[c]);
  for (int c = kKeep * T + t; c < chunks; c += T) {
    uv4 w[2];
    load16(x, (int64_t)c * 16, k, w);
    put(c, w);
  }
}

// Row-major 8-bit values into the packed order, one 16-byte chunk per lane.
__global__ __launch_bounds__(256) void i8_pack_kernel(int64_t rows, int64_t k, const int8_t* src, int64_t steps,
                                                      int64_t chunks, int8_t* dst) {
  const int64_t stride = (int64_t)gridDim.x * 256;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < chunks; c += stride) {
    const int lane = (int)(c & 63);
    const int64_t b = c >> 6, r = b / steps * 32 + (lane & 31), k0 = b % steps * 32 + (lane >> 5) * 16;
    iv4 o = {0, 0, 0, 0};
    if (r < rows && k0 + 16 <= k) {
      __builtin_memcpy(&o, src + r * k + k0, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (r < rows && k0 + e < k) o[e >> 2] |= (int)((uint32_t)(uint8_t)src[r * k + k0 + e] << (8 * (e & 3)));
    }
    *reinterpret_cast<iv4*>(dst + c * 16) = o;
  }
}

// ---------------------------------------------------------------- products

struct IProb {
  const int8_t* q;       // packed activations
  const float* s;        // their scales
  const int8_t* w;       // packed weights
  const float* t;        // their scales
  const _Float16* bias;
  _Float16* y;
  int m, n, steps;
  int epi;
  int nmb, ncol;         // row and column tiles
  int wg_begin;
};
typedef BatchOf<IProb, kMaxI8> IBatch;

// A weight scale as the products use it: within 2^86, so that s t and the scaled sum stay finite (s < 2^10,
// |sum| < 2^31), and neither a sum of 0 nor a negative one under the square meets an infinity.  No output
// changes: from a scale of 2^86 on every other sum (s >= 2^-31) scales to 2^55 and more, which each epilogue takes
// to the end of its range.  (Two instructions; NaN stays.)
__device__ __forceinline__ float column_scale(float t) {
  return __builtin_elementwise_maximum(__builtin_elementwise_minimum(t, 0x1p86f), -0x1p86f);
}

// N outputs: the sums scaled in fp32 (+ bias), the epilogue, one rounding to fp16.  Every kernel finishes its
// sums here, so that a row's bits do not depend on which one ran.  One branch for all N: with one for
// each, the code of the functions lay N times between the outputs.
template <int N, typename H>
__device__ __forceinline__ void i8_finish(const int (&a)[N], float s, const float (&t)[N], int epi, const float (&bias)[N],
                                          H& h) {
  float f[N];
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = (float)a[e] * (s * t[e]);
  if (epi == VKWR_GEMM_EPI_RELU_SQUARE) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = __builtin_fmaf(f[e], __builtin_fmaxf(f[e], 0.0f), 0.0f);  // (NaN stays; no -0)
  } else if (epi == VKWR_GEMM_EPI_BIAS) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] += bias[e];
  } else if (epi == VKWR_GEMM_EPI_TANH) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = tanhf(f[e]);
  } else if (epi == VKWR_GEMM_EPI_SIGMOID) {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = sigmoidf(f[e]);
  }
#pragma unroll
  for (int e = 0; e < N; ++e) h[e] = f16_of(f[e]);
}

// Up to eight outputs of a row, in one store where there are eight (of any alignment).
typedef _Float16 __attribute__((address_space(1)))* gptr;
__device__ __forceinline__ void store8(gptr o, const hv8& h, int left) {
  typedef hv8 __attribute__((aligned(2))) hv8u;
  if (left >= 8) {
    *reinterpret_cast<__attribute__((address_space(1))) hv8u*>(o) = h;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) o[e] = h[e];
  }
}

// (S TM) rows x (S TN) outputs per workgroup, S = 16 or 32 (the matrix instruction's), over the whole of K: the NW
// waves take the blocks of KS k-steps w, w + NW, ... with NB blocks' loads in flight, straight into registers, and the NW partial
// tiles are added through LDS: no operand is read twice by a workgroup, and no wave waits for another before
// the end.  Bound by what a CU takes from its L2 (K 8192, N 2048, m = 433: 1 MiB a
// workgroup, 15.4 us, 36 - 45 bytes a clock and CU of the 62 that a loop of nothing but loads reaches; the rounding in
// front of it takes 5), and where K is short by the trips at its ends (K 2048, N 8192, m = 128: 7.9).
template <int S, int TM, int TN, int NW, int KS, int NB, bool kGridRows, int N>
__global__ __launch_bounds__(NW * 64) void i8_stream_kernel(BatchOf<IProb, N> bt) {
  constexpr int kTiles = TM * TN, kG = 64 + 4 / TN;  // 16-byte cells of a group of 4 results, padded: reads hit all banks
  constexpr int kRegs = S * S / 64, kGroups = kRegs / 4, kOuts = S / 8;  // of a tile: a lane's results, groups; a row's eights
  constexpr int kStep = 1024 / S;                                        // k of an instruction
  static_assert(kTiles * S * kOuts <= NW * 64, "one piece of the output per thread");
  typedef int Acc __attribute__((ext_vector_type(kRegs)));
  __shared__ __attribute__((aligned(16))) iv4 red[NW * kTiles * kGroups * kG];
  const IProb P = bt.p[problem_of<kGridRows>(bt, blockIdx.x)];
  asm volatile("" ::"s"(P.q), "s"(P.s), "s"(P.w), "s"(P.t), "s"(P.bias), "s"(P.y), "s"(P.m), "s"(P.n), "s"(P.steps), "s"(P.epi),
               "s"(P.nmb), "s"(P.ncol), "s"(P.wg_begin));
  const int lt = (int)blockIdx.x - (kGridRows ? 0 : P.wg_begin);
  // the row tiles of a column tile run on one XCD, eight ids apart, and share its weights' one trip to the L2
  const int mb = (lt >> 3) % P.nmb, cb = (lt >> 3) / P.nmb * 8 + (lt & 7);
  if (cb >= P.ncol) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = P.steps * 32 / kStep, mblk = (P.m + S - 1) / S, nblk = (P.n + S - 1) / S;
  // this thread's eight outputs, and their scales, requested before everything else
  const int og = threadIdx.x % kOuts, ot = threadIdx.x / kOuts % TN + threadIdx.x / (kOuts * TN * S) * TN;
  const int orow = threadIdx.x / (kOuts * TN) % S;
  const int row = (mb * TM + ot / TN) * S + orow, col = (cb * TN + ot % TN) * S + 8 * og;
  const bool out = threadIdx.x < kTiles * S * kOuts && row < P.m && col < P.n;
  float os = 0.0f, ts[8], bs[8] = {};
  if (out) {
    os = P.s[row];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = min(col + e, P.n - 1);
      ts[e] = P.t[c];
      if (P.epi == VKWR_GEMM_EPI_BIAS) bs[e] = (float)P.bias[c];
    }
  }
  // block u's first operand (S = 16: lane l holds row l % 16, k 16 (l / 16) .. + 15, of two packed blocks); blocks
  // past the last are read as the last
  auto operand = [&](const int8_t* q, int u) __attribute__((always_inline)) {
    if constexpr (S == 32) return q + (int64_t)u * P.steps * 1024 + lane * 16;
    else return q + (int64_t)(u >> 1) * P.steps * 1024 + (lane >> 4) * 512 + ((u & 1) * 16 + (lane & 15)) * 16;
  };
  const int8_t *xp[TM], *wp[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) xp[i] = operand(P.q, min(mb * TM + i, mblk - 1));
#pragma unroll
  for (int j = 0; j < TN; ++j) wp[j] = operand(P.w, min(cb * TN + j, nblk - 1));
  Acc acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = Acc{0};
  iv4 fx[NB][KS][TM], fw[NB][KS][TN];
  auto load = [&](int buf, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int64_t o = ((int64_t)(wave + b * NW) * KS + s) * (kStep * 32);
#pragma unroll
      for (int j = 0; j < TN; ++j) fw[buf][s][j] = *reinterpret_cast<const iv4*>(wp[j] + o);
#pragma unroll
      for (int i = 0; i < TM; ++i) fx[buf][s][i] = *reinterpret_cast<const iv4*>(xp[i] + o);
    }
  };
  auto compute = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if constexpr (S == 32) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[buf][s][j], fx[buf][s][i], acc[i][j], 0, 0, 0);
          else acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[buf][s][j], fx[buf][s][i], acc[i][j], 0, 0, 0);
        }
  };
  static_assert(kI8Pad % (kStep * KS) == 0, "whole blocks");
  const int blocks = steps / KS, nb = (blocks - wave + NW - 1) / NW;  // this wave's blocks
  if (nb >= NB) {
    // no load here or in the loop is behind a condition, so that the waits in it are exact: with the first
    // loads under conditions the compiler waited for all that were out before every round
#pragma unroll
    for (int u = 0; u < NB; ++u) load(u, u);
    __builtin_amdgcn_sched_barrier(0);
    int b = 0;
    for (; b + 2 * NB <= nb; b += NB) {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        compute(u);
        __builtin_amdgcn_sched_barrier(0);
        load(u, b + NB + u);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      compute(u);
      if (b + NB + u < nb) load(u, b + NB + u);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int u = 0; u + 1 < NB; ++u)
      if (b + NB + u < nb) compute(u);
  } else {
#pragma unroll
    for (int u = 0; u + 1 < NB; ++u)
      if (u < nb) load(u, u);
#pragma unroll
    for (int u = 0; u + 1 < NB; ++u)
      if (u < nb) compute(u);
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const Acc& a = acc[t / TN][t % TN];
      red[((wave * kTiles + t) * kGroups + g) * kG + lane] = iv4{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
    }
  __syncthreads();
  if (!out) return;
  // eight outputs are two cells: S lanes apart in group og, or in the one group there is
  iv4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int at = (w * kTiles + ot) * kGroups * kG + (S == 32 ? og * kG : 2 * og * S) + orow;
    lo += red[at];
    hi += red[at + S];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) ts[e] = column_scale(ts[e]);
  const int sum[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  hv8 h;
  i8_finish(sum, os, ts, P.epi, bs, h);
  store8((gptr)(P.y + (int64_t)row * P.n + col), h, P.n - col);
}

// ---- few rows: rounded by the kernel that multiplies them
//
// One workgroup per 32 outputs, whose eight waves share K.  The rows (up to 8, up to 32768 values
// together) are rounded by every workgroup itself, in LDS, while its first weights are on the way: that
// costs less than a launch in front of this one.  One row is multiplied four k an instruction, a lane holding 16 k of one
// output and reading the row's 16 values as a broadcast; more by the matrix cores, most of whose columns repeat the
// last row (with four k an instruction 4 rows of K 8192, N 2048 took 9.0 us, so 7.8).  Bound by the weights from
// memory where they are large (a row of K 4096, N 16384: 13.6 us, 4.9 TB/s with what the last-level cache holds), by one
// trip to memory and the rounding behind it where they are small (three of K = N = 2048: 4.8 us, of which
// the bytes are 2.7).
constexpr int kGemvRows = 8;
constexpr int kGemvKeep = 8;                    // 16-byte pieces of x per lane
constexpr int kGemvMost = kGemvKeep * 512 * 8;  // values of all rows together

struct GProb {
  const _Float16* x;
  const int8_t* w;
  const float* t;
  const _Float16* bias;
  _Float16* y;
  int m, n, k, steps, epi, wg_begin;
};
typedef BatchOf<GProb, kMaxI8> GBatch;

template <int M, bool kGridRows, int N>
__global__ __launch_bounds__(512) void i8_gemv_kernel(BatchOf<GProb, N> bt) {
  constexpr int kWaves = 8, kPer = kWaves / M, kAhead = 8;  // waves of a row; blocks of weights in flight
  constexpr int kSkew = 32;  // bytes between rows, so that a read of a block's 32 k of 8 rows hits all banks
  __shared__ __attribute__((aligned(16))) int8_t xq[kGemvMost + M * (kI8Pad + kSkew)];
  __shared__ uint32_t wtop[kWaves];
  __shared__ __attribute__((aligned(16))) int part[kWaves][M][32];
  const GProb P = bt.p[problem_of<kGridRows>(bt, blockIdx.x)];
  asm volatile("" ::"s"(P.x), "s"(P.w), "s"(P.t), "s"(P.bias), "s"(P.y), "s"(P.m), "s"(P.n), "s"(P.k), "s"(P.steps), "s"(P.epi),
               "s"(P.wg_begin));
  const int cb = (int)blockIdx.x - (kGridRows ? 0 : P.wg_begin);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int steps = P.steps, k = P.k, kpad = steps * 32;
  const int8_t* const w = P.w + (int64_t)cb * steps * 1024 + lane * 16;
  const int orow = tid >> 5, ocol = cb * 32 + (tid & 31);  // this thread's output, if it has one
  const bool out = tid < 32 * M && orow < P.m && ocol < P.n;
  float ts[1], bs[1] = {0.0f};
  if (out) {
    ts[0] = P.t[ocol];
    if (P.epi == VKWR_GEMM_EPI_BIAS) bs[0] = (float)P.bias[ocol];
  }
  // ---- this wave's pieces of 8 values of its row
  const int row = min(wave / kPer, P.m - 1), w0 = wave % kPer, pieces = kpad / 8;
  const _Float16* const x = P.x + (int64_t)row * k;
  uv4 v[kGemvKeep];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kGemvKeep; ++i) {
    const int c = (i * kPer + w0) * 64 + lane;
    v[i] = load8(x, (int64_t)c * 8, k);
  }
  // (behind the row, whose values are waited for first: loads come back in order)
  __builtin_amdgcn_sched_barrier(0);
  iv4 fw[kAhead];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const int st = min(wave + a * kWaves, steps - 1);
    fw[a] = *reinterpret_cast<const iv4*>(w + (int64_t)st * 1024);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < kGemvKeep; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max_u16x2(top, v[i][e] & 0x7fff7fffu);
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
  if (lane == 0) wtop[wave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) top = max(top, wtop[wave / kPer * kPer + i]);
  {
    const float a = top < 0x7c00u ? h2f((uint16_t)top) : 0.0f, inv = a > 0.0f ? 1.0f / a : 0.0f;
#pragma unroll
    for (int i = 0; i < kGemvKeep; ++i) {
      const int c = (i * kPer + w0) * 64 + lane;
      if (c < pieces) {
        typedef _Float16 h2v __attribute__((ext_vector_type(2)));
        uint32_t o[2] = {0, 0};
        if (a > 0.0f) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const h2v lo = __builtin_bit_cast(h2v, (uint32_t)v[i][2 * h]), hi = __builtin_bit_cast(h2v, (uint32_t)v[i][2 * h + 1]);
            const float f[4] = {(float)lo.x, (float)lo.y, (float)hi.x, (float)hi.y};
            o[h] = quant4(f, a, inv);
          }
        }
        *reinterpret_cast<uint64_t*>(xq + wave / kPer * (kpad + kSkew) + c * 8) = (uint64_t)o[1] << 32 | o[0];
      }
    }
  }
  __syncthreads();
  typename std::conditional<M == 1, int, iv16>::type acc = {0};
  const int8_t* const xl = xq + min(lane & 31, M - 1) * (kpad + kSkew) + (lane >> 5) * 16;
  auto dot = [&](const iv4& b, int st) __attribute__((always_inline)) {
    const iv4 a = *reinterpret_cast<const iv4*>(xl + st * 32);
    if constexpr (M == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_sdot4(a[e], b[e], acc, false);
    } else {
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(b, a, acc, 0, 0, 0);
    }
  };
  // a block's registers take the block kAhead rounds further as soon as it is done (a row of K 16384, N 4096: 16.1 us;
  // asking for kAhead at once when the last are done 19.6); loads past the end read the last block again
  int s0 = wave;
  for (; s0 + kAhead * kWaves < steps; s0 += kAhead * kWaves) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      dot(fw[a], s0 + a * kWaves);
      __builtin_amdgcn_sched_barrier(0);
      const int st = min(s0 + (kAhead + a) * kWaves, steps - 1);
      fw[a] = *reinterpret_cast<const iv4*>(w + (int64_t)st * 1024);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
    if (s0 + a * kWaves < steps) dot(fw[a], s0 + a * kWaves);
  if constexpr (M == 1) {
    acc += __shfl_xor(acc, 32, 64);
    if (lane < 32) part[wave][0][lane] = acc;
  } else if ((lane & 31) < M) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<iv4*>(&part[wave][lane & 31][8 * g + 4 * (lane >> 5)]) =
          iv4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
  }
  __syncthreads();
  if (!out) return;
  int sums[1] = {0};
#pragma unroll
  for (int q = 0; q < kWaves; ++q) sums[0] += part[q][orow][tid & 31];
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) all = max(all, wtop[orow * kPer + i]);
  const float s = all < 0x7c00u ? h2f((uint16_t)all) / 127.0f : __builtin_nanf("");
  ts[0] = column_scale(ts[0]);
  _Float16 h[1];
  i8_finish(sums, s, ts, P.epi, bs, h);
  P.y[(int64_t)orow * P.n + ocol] = h[0];
}

// ---- many rows: tiles through LDS, bound by the matrix cores
//
// (64 TM) x (64 TN) outputs per workgroup, four waves of (32 TM) x (32 TN) in registers.  K advances
// 64 per stage through a ring of NBUF LDS buffers; both operands being in fragment order, a stage is a row of
// 2 KiB pieces, copied straight to LDS, and read back lane by lane.  One barrier per stage, before the
// second of its two groups of products, whose operands are then in registers: behind it the buffer is free and
// the copies of the stage NBUF further go out between the products, so that they neither hold those up
// nor arrive late.  The copies are written in assembly, as the compiler would make every LDS read wait for all of
// them; the waits are placed here.  (Stages of 128 k with two groups of copies each took 5 % more: 147 us instead
// of 138 for three of K = N = 4096, m = 2304.  From three buffers on their number makes no difference.)
// What bounds it: 2.1 POPS where every CU is busy, at 2.0 GHz (the card's power), the LDS at 75 - 85 % of its
// rate; 2.5 where 192 CUs are (K = N = 4096, m = 2304).
template <int TM, int TN>
struct I8Tile {
  static constexpr int kX = 4 * TM, kW = 4 * TN, kBlocks = kX + kW;  // kilobytes of a stage
  static constexpr int kCopies = TM + TN;                            // per wave
  static constexpr int kOutRow = 144;                                // bytes of a staged row of 64 outputs
};

__device__ __forceinline__ const void* uniform_ptr(const void* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const void*)(uintptr_t)((uint64_t)hi << 32 | lo);
}

// 16 bytes per lane: global (base + off) -> LDS (lds + 16 lane); base and lds wave-uniform
__device__ __forceinline__ void copy16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}

template <int TM, int TN, int kEpi>
__device__ __forceinline__ void i8_store(char* st, const IProb& P, const iv16 (&acc)[TM][TN], int row0, int col0, int lane) {
  constexpr int kRow = I8Tile<TM, TN>::kOutRow, kBuf = 32 * kRow;
  const int lr = lane & 31, lh = lane >> 5, r8 = lane >> 3, c8 = 8 * (lane & 7);
  int m = P.m, n = P.n;
  gptr y = (gptr)P.y;
  // (global address-space pointers, so that the accesses stay global, not flat, ones)
  typedef const float __attribute__((address_space(1)))* gcf;
  gcf sp = (gcf)P.s, tp = (gcf)P.t;
  const _Float16 __attribute__((address_space(1)))* bp = (const _Float16 __attribute__((address_space(1)))*)P.bias;
  asm("" : "+s"(m), "+s"(n), "+s"(y), "+s"(sp), "+s"(tp), "+s"(bp));
  // the columns' scales (and biases) behind the two strips
  float* const tl = reinterpret_cast<float*>(st + 2 * kBuf);
#pragma unroll
  for (int c = 0; c < 32 * TN; c += 64) {
    if (c + lane < 32 * TN) {
      const int col = min(col0 + c + lane, n - 1);
      tl[c + lane] = column_scale(tp[col]);
      if constexpr (kEpi == VKWR_GEMM_EPI_BIAS) tl[32 * TN + c + lane] = (float)bp[col];
    }
  }
  __builtin_amdgcn_wave_barrier();
  float s[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) s[i] = sp[min(row0 + 32 * i + lr, m - 1)];
  constexpr int kStrips = TM * TN / 2;
  auto write = [&](int p) __attribute__((always_inline)) {
    const int i = p % TM, j0 = p / TM * 2;
    char* const o = st + (p & 1) * kBuf + lr * kRow;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = (j0 + jj) * 32 + 8 * g + 4 * lh;
        const f4 t = *reinterpret_cast<const f4*>(tl + c);
        f4 b = {0, 0, 0, 0};
        if constexpr (kEpi == VKWR_GEMM_EPI_BIAS) b = *reinterpret_cast<const f4*>(tl + 32 * TN + c);
        typedef _Float16 hv4 __attribute__((ext_vector_type(4)));
        hv4 h;
        const iv16& c16 = acc[i][j0 + jj];
        const int sums[4] = {c16[4 * g], c16[4 * g + 1], c16[4 * g + 2], c16[4 * g + 3]};
        const float ts[4] = {t[0], t[1], t[2], t[3]}, bs[4] = {b[0], b[1], b[2], b[3]};
        i8_finish(sums, s[i], ts, kEpi, bs, h);
        *reinterpret_cast<hv4*>(o + (jj * 32 + 8 * g + 4 * lh) * 2) = h;
      }
  };
  auto send = [&](int p) __attribute__((always_inline)) {
    const int i = p % TM, col = col0 + p / TM * 64 + c8;
    const char* const o = st + (p & 1) * kBuf + r8 * kRow + c8 * 2;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const hv8 v = *reinterpret_cast<const hv8*>(o + 8 * h * kRow);
      const int row = row0 + 32 * i + 8 * h + r8;
      if (row >= m || col >= n) continue;
      store8(y + (int64_t)row * n + col, v, n - col);
    }
  };
  write(0);
#pragma unroll
  for (int p = 1; p < kStrips; ++p) {
    write(p);
    send(p - 1);
  }
  send(kStrips - 1);
}

template <int TM, int TN, int NBUF>
__global__ __launch_bounds__(256, 1) void i8_tile_kernel(IBatch bt, int tiles) {
  using T = I8Tile<TM, TN>;
  constexpr int ND = T::kCopies;
  constexpr int kOut = 4 * (2 * 32 * T::kOutRow + 2 * 32 * TN * 4);
  constexpr int kBuf = T::kBlocks * 1024, kRing = NBUF * kBuf;
  static_assert(kOut <= kRing, "the outputs are staged where the operands were");
  __shared__ __attribute__((aligned(1024))) char sm[kRing];
  // workgroup b runs on XCD b % 8: each takes a contiguous range of tiles, in groups of 4 tile rows
  int L;
  {
    const int b = blockIdx.x, x = b & 7, q8 = tiles >> 3, r8 = tiles & 7;
    L = (x < r8 ? x * (q8 + 1) : r8 * (q8 + 1) + (x - r8) * q8) + (b >> 3);
  }
  const IProb& P = bt.p[problem_of<false>(bt, L)];
  const int lt = L - P.wg_begin, per = 4 * P.ncol, grp = lt / per, in = lt - grp * per;
  const int g0 = grp * 4, gs = min(4, P.nmb - g0);
  const int mb = g0 + in % gs, cb = in / gs;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wm = w >> 1, wn = w & 1;
  const int steps = P.steps, ns = steps >> 1;
  const int mlast = ((P.m + 31) >> 5) - 1 - mb * 2 * TM, nlast = ((P.n + 31) >> 5) - 1 - cb * 2 * TN;
  // copy d of wave w: k step w % 2 of the stage, of block 2 d + w / 2 of x, then of the weights
  uint32_t off[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int blk = d < TM ? min(2 * d + (w >> 1), mlast) : min(2 * (d - TM) + (w >> 1), nlast);
    off[d] = (uint32_t)((blk * steps + (w & 1)) * 1024 + lane * 16);
  }
  const char* const px = (const char*)uniform_ptr(P.q + (int64_t)mb * 2 * TM * steps * 1024);
  const char* const pw = (const char*)uniform_ptr(P.w + (int64_t)cb * 2 * TN * steps * 1024);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(VK_LDS void*)&sm[0] + w * 1024);
  auto copies = [&](int buf, int st) __attribute__((always_inline)) {
    const int64_t k0 = (int64_t)min(st, ns - 1) * 2048;  // past the end: the last stage once more, unused
    const void *xb = uniform_ptr(px + k0), *wb = uniform_ptr(pw + k0);
#pragma unroll
    for (int d = 0; d < ND; ++d) copy16(d < TM ? xb : wb, off[d], lds0 + buf * kBuf + d * 4096);
  };
  const char* const fxp = sm + wm * TM * 2048 + lane * 16;
  const char* const fwp = sm + (T::kX + wn * TN * 2) * 1024 + lane * 16;
  iv4 fx[2][TM], fw[2][TN];
  auto fread = [&](int buf, int kk, int set) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i) fx[set][i] = *reinterpret_cast<const iv4*>(fxp + buf * kBuf + (i * 2 + kk) * 1024);
#pragma unroll
    for (int j = 0; j < TN; ++j) fw[set][j] = *reinterpret_cast<const iv4*>(fwp + buf * kBuf + (j * 2 + kk) * 1024);
  };
  iv16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = iv16{0};
  // the products of a group with the next group's reads between them
  auto products = [&](int set) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[set][j], fx[set][i], acc[i][j], 0, 0, 0);
    constexpr int kReads = TM + TN < TM * TN ? TM + TN : TM * TN;
#pragma unroll
    for (int q = 0; q < kReads; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, TM + TN - kReads, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, TM * TN - kReads, 0);
  };
  // the products of a group with the copies of stage st between them
  auto products_copies = [&](int set, int buf, int st) __attribute__((always_inline)) {
    const int64_t k0 = (int64_t)min(st, ns - 1) * 2048;
    const void *xb = uniform_ptr(px + k0), *wb = uniform_ptr(pw + k0);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[set][j], fx[set][i], acc[i][j], 0, 0, 0);
        const int p = i * TN + j;
#pragma unroll
        for (int d = 0; d < ND; ++d)
          if (d * TM * TN / ND == p) copy16(d < TM ? xb : wb, off[d], lds0 + buf * kBuf + d * 4096);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  // all but the newest n stages' copies have landed, and this wave's reads have returned
#define VK_I8_LANDED(n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((n) * ND) : "memory")
#pragma unroll
  for (int u = 0; u < NBUF; ++u) copies(u, u);
  VK_I8_LANDED(NBUF - 1);
  fread(0, 0, 0);
  int cur = 0;
  for (int s = 0; s < ns; ++s) {
    const int nxt = cur + 1 == NBUF ? 0 : cur + 1;
    fread(cur, 1, 1);
    products(0);
    __builtin_amdgcn_sched_barrier(0);
    VK_I8_LANDED(NBUF - 2);  // stage s + 1 is there, and this one is read, for every wave
    fread(nxt, 0, 0);
    products_copies(1, cur, s + NBUF);
    __builtin_amdgcn_sched_barrier(0);
    cur = nxt;
  }
  // the last copies have landed and every wave's reads are done
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  char* const st = sm + w * (kOut / 4);
  const int row0 = mb * 64 * TM + wm * 32 * TM, col0 = cb * 64 * TN + wn * 32 * TN;
  switch (P.epi) {
    case VKWR_GEMM_EPI_RELU_SQUARE: i8_store<TM, TN, VKWR_GEMM_EPI_RELU_SQUARE>(st, P, acc, row0, col0, lane); break;
    case VKWR_GEMM_EPI_BIAS: i8_store<TM, TN, VKWR_GEMM_EPI_BIAS>(st, P, acc, row0, col0, lane); break;
    case VKWR_GEMM_EPI_TANH: i8_store<TM, TN, VKWR_GEMM_EPI_TANH>(st, P, acc, row0, col0, lane); break;
    case VKWR_GEMM_EPI_SIGMOID: i8_store<TM, TN, VKWR_GEMM_EPI_SIGMOID>(st, P, acc, row0, col0, lane); break;
    default: i8_store<TM, TN, VKWR_GEMM_EPI_NONE>(st, P, acc, row0, col0, lane); break;
  }
}

// ---------------------------------------------------------------- host

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  return na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

int64_t packed_bytes(int64_t rows, int64_t k) { return up(rows, kI8Rows) * up(k, kI8Pad); }

int check_problems(const char* fn, int n, const vkwr_i8_problem* p) {
  VK_REQUIRE(n >= 1 && n <= kMaxI8 && p, "%s: 1 to %d problems, got %d", fn, kMaxI8, n);
  int64_t rows = 0;
  for (int i = 0; i < n; ++i) {
    VK_REQUIRE(p[i].m >= 0 && p[i].m <= kI8MaxRows && p[i].n >= 1 && p[i].n <= kI8MaxRows && p[i].k >= 1 &&
                   p[i].k <= kI8MaxK,
               "%s: problem %d: sizes m=%lld n=%lld k=%lld (m and n up to 2^22, k up to %lld)", fn, i,
               (long long)p[i].m, (long long)p[i].n, (long long)p[i].k, (long long)kI8MaxK);
    VK_REQUIRE(p[i].epilogue == VKWR_GEMM_EPI_NONE || p[i].epilogue == VKWR_GEMM_EPI_RELU_SQUARE ||
                   p[i].epilogue == VKWR_GEMM_EPI_BIAS || p[i].epilogue == VKWR_GEMM_EPI_TANH ||
                   p[i].epilogue == VKWR_GEMM_EPI_SIGMOID,
               "%s: problem %d: unsupported epilogue %d", fn, i, p[i].epilogue);
    rows += p[i].m;
  }
  VK_REQUIRE(rows <= kI8MaxRows, "%s: sizes: %lld rows together, at most 2^22", fn, (long long)rows);
  return VKWR_OK;
}

// Where each problem's 8-bit rows and scales lie in the workspace; problems of one call that read the
// same rows share them.
struct I8Scratch {
  int from[kMaxI8];
  int64_t q[kMaxI8], s[kMaxI8], bytes;
};
I8Scratch scratch_of(int n, const vkwr_i8_problem* p) {
  I8Scratch c{};
  for (int i = 0; i < n; ++i) {
    c.from[i] = i;
    for (int j = 0; j < i && c.from[i] == i; ++j)
      if (p[j].x == p[i].x && p[j].m == p[i].m && p[j].k == p[i].k) c.from[i] = j;
    if (c.from[i] != i) {
      c.q[i] = c.q[c.from[i]], c.s[i] = c.s[c.from[i]];
      continue;
    }
    c.q[i] = c.bytes;
    c.bytes += packed_bytes(p[i].m, p[i].k);
    c.s[i] = c.bytes;
    c.bytes += up(4 * p[i].m, 16);
  }
  return c;
}

// Launches `kernel` (template arguments kGridRows and N last) on batch b of `total` workgroups of `threads`: a row
// of the grid per problem where they have equally many workgroups.
#define VK_I8_LAUNCH(b, total, threads, stream, ...)                                                            \
  do {                                                                                                          \
    bool by_row;                                                                                                \
    const dim3 g = grid_of(b, total, &by_row), th(threads);                                                     \
    if (b.n == 1) {                                                                                             \
      const BatchOf<std::decay_t<decltype(b.p[0])>, 1> one{1, {b.p[0]}};                                        \
      hipLaunchKernelGGL((__VA_ARGS__, true, 1 >), g, th, 0, stream, one);                                      \
    } else if (by_row) {                                                                                        \
      hipLaunchKernelGGL((__VA_ARGS__, true, kMaxI8 >), g, th, 0, stream, b);                                   \
    } else {                                                                                                    \
      hipLaunchKernelGGL((__VA_ARGS__, false, kMaxI8 >), g, th, 0, stream, b);                                  \
    }                                                                                                           \
  } while (0)

// That grid; problems begin at wg_begin.
template <typename Batch>
dim3 grid_of(const Batch& b, int64_t total, bool* rows) {
  *rows = total % b.n == 0;
  for (int i = 0; i < b.n; ++i) *rows = *rows && b.p[i].wg_begin == i * (total / b.n);
  return *rows ? dim3((unsigned)(total / b.n), (unsigned)b.n) : dim3((unsigned)total);
}

// Rounds the rows of every problem of `b` (wg_begin filled in here).
void launch_rows(QBatch& b, hipStream_t s) {
  int most = 0;
  for (int i = 0; i < b.n; ++i) most = std::max(most, b.p[i].steps);
  const int T = most <= 32 ? 64 : most <= 64 ? 128 : most <= 256 ? 256 : 512;  // lanes per row
  unsigned grid = 0;
  for (int i = 0; i < b.n; ++i) {
    b.p[i].wg_begin = (int)grid;
    grid += (unsigned)up((b.p[i].m + 31) / 32, 8) * 32 / std::max(1, 256 / T);
  }
  if (grid == 0) return;
  if (T == 64) VK_I8_LAUNCH(b, grid, 256, s, i8_rows_kernel<64, 1);
  else if (T == 128) VK_I8_LAUNCH(b, grid, 256, s, i8_rows_kernel<128, 1);
  else if (most <= 128) VK_I8_LAUNCH(b, grid, 256, s, i8_rows_kernel<256, 1);
  else if (T == 256) VK_I8_LAUNCH(b, grid, 256, s, i8_rows_kernel<256, 2);
  else VK_I8_LAUNCH(b, grid, 512, s, i8_rows_kernel<512, 2);
}

QProb row_problem(const uint16_t* x, int64_t m, int64_t k, int8_t* q, float* s) {
  QProb p{};
  p.x = reinterpret_cast<const _Float16*>(x);
  p.q = q;
  p.s = s;
  p.m = (int)m;
  p.k = (int)k;
  p.steps = (int)(up(k, kI8Pad) / 32);
  return p;
}

// The tile that a batch runs with: the smallest whose workgroups fit the (256) CUs at once.  A second
// round mostly costs more than larger tiles that leave CUs idle, and larger tiles than that
// leave bandwidth.  us of a whole call, this tile against its neighbours:
//   16 x 16    K 8192, N 2048, m = 9     8.7; 16 x 32 9.7, 32 x 32 10.7
//              K 16384, N 4096, m = 9    17.7; 16 x 32 19.9, 32 x 32 23.9
//   16 x 32    K 16384, N 4096, m = 32   20.8; 16 x 16 22.6, 32 x 32 25.6
//   32 x 32    K 8192, N 2048, m = 128   12.6; 32 x 64 14.9, 64 x 64 18.3
//   32 x 64    K = N = 4096, m = 128     10.6; 32 x 32 11.6, 64 x 64 12.6
//   64 x 64    K 2048, N 8192, m = 128   10.2; 32 x 64 11.2, 64 x 128 11.8
//              K 8192, N 2048, m = 433   20.7; 64 x 128 25.3, 128 x 128 34.0
//   64 x 128   K = N = 4096, m = 433     17.2; 64 x 64 21.0, 128 x 128 21.6
//   128 x 128  K 8192, N 2048, m = 1100  36.2; 64 x 128 44.0, 128 x 256 49.1
//   128 x 256  K = N = 4096, m = 1100    31.3; 128 x 128 41.3, 192 x 256 41.0
//   192 x 256  K = N = 4096, m = 2304    48.7; 128 x 256 63.2, 256 x 256 58.6
//   256 x 256  K = N = 4096, m = 4096    76.8; 192 x 256 88.6
// Where it loses, up to a seventh: few rows of many outputs, whose smaller tiles take two to five rounds
// (K 4096, the rule's / the best of 16 x 16 to 128 x 128):
//   16 rows    N 12288  32 x 64 13.2 / 16 x 16 12.5; N 16384 15.6 / 14.7; N 16448 64 x 128 16.5 / 16 x 16 15.6; N 20480 19.4 / 17.0
//   32 rows    N 16448  64 x 128 17.1 (64 x 64 20.9); N 20480 21.1 / 32 x 32 20.0
//   64 rows    N 12288  64 x 64 15.8 / 32 x 32 14.6; N 16384 19.2 / 32 x 64 17.2; N 16448 64 x 128 17.3 (64 x 64 24.1)
//              three of N 4096  64 x 64 16.6 / 32 x 32 15.6 (48 rows 15.9 / 15.2)
// Beyond one round of the largest: whichever of the last two takes less by its rounds, one of 192
// rows counted as 0.77 (K 4096, N 16384, m = 2304: three rounds each, 145, 179; three of N 4096: 576 tiles
// in three rounds 142, 432 in two 135).
// Up to 8 rows of 32768 values together are rounded by the kernel that multiplies them: three of K = N = 2048, 1 row
// 4.8 us, on tiles 7.1; 8 rows 6.0 and 7.4; 5 of K = N = 4096 7.1 and 7.8; 4 of K 8192, N 2048 7.8 and 8.5.  With
// twice as many values (8 rows of K 8192: 10.1 and 8.7) the rounding costs more than its launch.
// Up to 64 x 64, weights and rows go straight into registers (stream kernel).
enum { kRouteGemv, kRouteStream, kRouteTile };
struct I8Route {
  int kind, rows, cols;  // of a workgroup's tile
};
constexpr I8Route kI8Routes[] = {{kRouteStream, 16, 16}, {kRouteStream, 16, 32}, {kRouteStream, 32, 32}, {kRouteStream, 32, 64},
                                 {kRouteStream, 64, 64}, {kRouteTile, 64, 128},  {kRouteTile, 128, 128}, {kRouteTile, 128, 256},
                                 {kRouteTile, 192, 256}, {kRouteTile, 256, 256}};
constexpr int kI8RouteCount = sizeof(kI8Routes) / sizeof(kI8Routes[0]);

I8Route pick_route(int n, const vkwr_i8_problem* p) {
  int64_t most = 0;
  for (int i = 0; i < n; ++i) most = std::max(most, p[i].m);
  if (most <= kGemvRows) {
    int64_t values = 0;
    for (int i = 0; i < n; ++i)
      if (p[i].m > 0) values = std::max(values, (most <= 2 ? most : most <= 4 ? 4 : 8) * up(p[i].k, kI8Pad));
    if (values <= kGemvMost) return {kRouteGemv, kGemvRows, 32};
  }
  const int64_t cus = device_cus();
  int64_t tiles[kI8RouteCount];
  for (int r = 0; r < kI8RouteCount; ++r) {
    tiles[r] = 0;
    for (int i = 0; i < n; ++i) tiles[r] += up(p[i].m, kI8Routes[r].rows) / kI8Routes[r].rows * (up(p[i].n, kI8Routes[r].cols) / kI8Routes[r].cols);
    if (tiles[r] <= cus) return kI8Routes[r];
  }
  constexpr int a = kI8RouteCount - 2, b = kI8RouteCount - 1;
  return kI8Routes[0.77 * (double)((tiles[a] + cus - 1) / cus) < (double)((tiles[b] + cus - 1) / cus) ? a : b];
}

#define VK_I8_TILE(tm, tn, nbuf) \
  hipLaunchKernelGGL((i8_tile_kernel<tm, tn, nbuf>), dim3((unsigned)wgs), dim3(256), 0, s, b, wgs)

void launch_products(const I8Route& r, const IBatch& b, int wgs, hipStream_t s) {
  if (r.kind == kRouteStream) {
    if (r.rows == 64) VK_I8_LAUNCH(b, wgs, 512, s, i8_stream_kernel<32, 2, 2, 8, 1, 4);
    else if (r.cols == 64) VK_I8_LAUNCH(b, wgs, 512, s, i8_stream_kernel<32, 1, 2, 8, 2, 4);
    else if (r.rows == 32) VK_I8_LAUNCH(b, wgs, 512, s, i8_stream_kernel<32, 1, 1, 8, 2, 4);
    else if (r.cols == 32) VK_I8_LAUNCH(b, wgs, 512, s, i8_stream_kernel<16, 1, 2, 8, 2, 4);
    else VK_I8_LAUNCH(b, wgs, 512, s, i8_stream_kernel<16, 1, 1, 8, 2, 4);
  } else if (r.rows == 64) {
    VK_I8_TILE(1, 2, 6);
  } else if (r.rows == 128) {
    if (r.cols == 128) VK_I8_TILE(2, 2, 6);
    else VK_I8_TILE(2, 4, 4);
  } else if (r.rows == 192) {
    VK_I8_TILE(3, 4, 4);
  } else {
    VK_I8_TILE(4, 4, 4);
  }
}

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int64_t vkwr_i8_packed_bytes(int64_t rows, int64_t k) {
  if (rows < 0 || rows > kI8MaxRows || k < 1 || k > kI8MaxK) return -1;
  return packed_bytes(rows, k);
}

extern "C" int vkwr_i8_pack(int64_t rows, int64_t k, const int8_t* src, int8_t* dst, void* stream) {
  clear_error();
  const char* fn = "vkwr_i8_pack";
  const int64_t bytes = vkwr_i8_packed_bytes(rows, k);
  VK_REQUIRE(bytes >= 0, "%s: bad size (rows=%lld, k=%lld)", fn, (long long)rows, (long long)k);
  if (bytes == 0) return VKWR_OK;
  VK_REQUIRE(src && dst && (uintptr_t)dst % 16 == 0, "%s: null pointer, or dst not 16-byte aligned", fn);
  VK_REQUIRE(!overlap(src, rows * k, dst, bytes), "%s: dst overlaps src", fn);
  const int64_t chunks = bytes / 16;
  hipLaunchKernelGGL(i8_pack_kernel, dim3((unsigned)std::min<int64_t>((chunks + 255) / 256, 8192)), dim3(256), 0,
                     (hipStream_t)stream, rows, k, src, up(k, kI8Pad) / 32, chunks, dst);
  return check_launch(fn);
}

extern "C" int vkwr_i8_quantize_rows_f16(int64_t rows, int64_t k, const uint16_t* x, int8_t* q, float* scale,
                                         void* stream) {
  clear_error();
  const char* fn = "vkwr_i8_quantize_rows_f16";
  const int64_t bytes = vkwr_i8_packed_bytes(rows, k);
  VK_REQUIRE(bytes >= 0, "%s: bad size (rows=%lld, k=%lld)", fn, (long long)rows, (long long)k);
  if (bytes == 0) return VKWR_OK;
  VK_REQUIRE(x && q && scale && (uintptr_t)q % 16 == 0, "%s: null pointer, or q not 16-byte aligned", fn);
  VK_REQUIRE(!overlap(x, 2 * rows * k, q, bytes) && !overlap(x, 2 * rows * k, scale, 4 * rows) &&
                 !overlap(q, bytes, scale, 4 * rows),
             "%s: x, q and scale overlap", fn);
  QBatch b{};
  b.n = 1;
  b.p[0] = row_problem(x, rows, k, q, scale);
  launch_rows(b, (hipStream_t)stream);
  return check_launch(fn);
}

extern "C" int64_t vkwr_linear_i8_workspace_bytes(int n_problems, const vkwr_i8_problem* problems) {
  clear_error();
  if (check_problems("vkwr_linear_i8_workspace_bytes", n_problems, problems)) return -1;
  int64_t bytes = 0;  // as if no two problems read the same rows: a smaller m may tell them apart
  for (int i = 0; i < n_problems; ++i) bytes += packed_bytes(problems[i].m, problems[i].k) + up(4 * problems[i].m, 16);
  return bytes;
}

extern "C" int vkwr_linear_i8_f16(int n_problems, const vkwr_i8_problem* problems, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "vkwr_linear_i8_f16";
  const vkwr_i8_problem* const p = problems;
  const int n = n_problems;
  if (int e = check_problems(fn, n, p)) return e;
  const int64_t need = vkwr_linear_i8_workspace_bytes(n, p);
  if (need == 0) return VKWR_OK;  // no rows
  VK_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need,
             "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", fn, (long long)need,
             (long long)workspace_bytes);
  for (int i = 0; i < n; ++i) {
    if (p[i].m == 0) continue;
    VK_REQUIRE(p[i].x && p[i].w && p[i].w_scale && p[i].y && (p[i].epilogue != VKWR_GEMM_EPI_BIAS || p[i].bias),
               "%s: problem %d: null pointer", fn, i);
    VK_REQUIRE((uintptr_t)p[i].w % 16 == 0, "%s: problem %d: w must be 16-byte aligned", fn, i);
    const int64_t ny = 2 * p[i].m * p[i].n;
    VK_REQUIRE(!overlap(p[i].y, ny, workspace, need) && !overlap(p[i].x, 2 * p[i].m * p[i].k, workspace, need) &&
                   !overlap(p[i].w, packed_bytes(p[i].n, p[i].k), workspace, need) &&
                   !overlap(p[i].w_scale, 4 * p[i].n, workspace, need) &&
                   !(p[i].epilogue == VKWR_GEMM_EPI_BIAS && overlap(p[i].bias, 2 * p[i].n, workspace, need)),
               "%s: problem %d: a tensor overlaps the workspace", fn, i);
    for (int j = 0; j < n; ++j) {
      if (p[j].m == 0) continue;
      VK_REQUIRE(!overlap(p[i].y, ny, p[j].x, 2 * p[j].m * p[j].k) &&
                     !overlap(p[i].y, ny, p[j].w, packed_bytes(p[j].n, p[j].k)) &&
                     !overlap(p[i].y, ny, p[j].w_scale, 4 * p[j].n) &&
                     !(p[j].epilogue == VKWR_GEMM_EPI_BIAS && overlap(p[i].y, ny, p[j].bias, 2 * p[j].n)) &&
                     (i == j || !overlap(p[i].y, ny, p[j].y, 2 * p[j].m * p[j].n)),
                 "%s: y of problem %d overlaps what problem %d reads or writes", fn, i, j);
    }
  }
  const hipStream_t st = (hipStream_t)stream;
  const I8Route route = pick_route(n, p);
  if (route.kind == kRouteGemv) {
    GBatch gb{};
    int64_t wgs = 0;
    int most = 0;
    for (int i = 0; i < n; ++i) {
      if (p[i].m == 0) continue;
      GProb& P = gb.p[gb.n++];
      P.x = reinterpret_cast<const _Float16*>(p[i].x);
      P.w = p[i].w;
      P.t = p[i].w_scale;
      P.bias = reinterpret_cast<const _Float16*>(p[i].bias);
      P.y = reinterpret_cast<_Float16*>(p[i].y);
      P.m = (int)p[i].m;
      P.n = (int)p[i].n;
      P.k = (int)p[i].k;
      P.steps = (int)(up(p[i].k, kI8Pad) / 32);
      P.epi = p[i].epilogue;
      P.wg_begin = (int)wgs;
      wgs += (p[i].n + 31) / 32;
      most = std::max(most, P.m);
    }
    if (most == 1) VK_I8_LAUNCH(gb, wgs, 512, st, i8_gemv_kernel<1);
    else if (most == 2) VK_I8_LAUNCH(gb, wgs, 512, st, i8_gemv_kernel<2);
    else if (most <= 4) VK_I8_LAUNCH(gb, wgs, 512, st, i8_gemv_kernel<4);
    else VK_I8_LAUNCH(gb, wgs, 512, st, i8_gemv_kernel<8);
    return check_launch(fn);
  }
  const I8Scratch c = scratch_of(n, p);
  char* const ws = static_cast<char*>(workspace);
  QBatch qb{};
  IBatch ib{};
  int64_t wgs = 0;
  for (int i = 0; i < n; ++i) {
    if (p[i].m == 0) continue;
    int8_t* const q = reinterpret_cast<int8_t*>(ws + c.q[i]);
    float* const s = reinterpret_cast<float*>(ws + c.s[i]);
    if (c.from[i] == i) qb.p[qb.n++] = row_problem(p[i].x, p[i].m, p[i].k, q, s);
    IProb& P = ib.p[ib.n++];
    P.q = q;
    P.s = s;
    P.w = p[i].w;
    P.t = p[i].w_scale;
    P.bias = reinterpret_cast<const _Float16*>(p[i].bias);
    P.y = reinterpret_cast<_Float16*>(p[i].y);
    P.m = (int)p[i].m;
    P.n = (int)p[i].n;
    P.steps = (int)(up(p[i].k, kI8Pad) / 32);
    P.epi = p[i].epilogue;
    P.nmb = (P.m + route.rows - 1) / route.rows;
    P.ncol = (P.n + route.cols - 1) / route.cols;
    P.wg_begin = (int)wgs;
    wgs += (int64_t)P.nmb * (route.kind == kRouteStream ? up(P.ncol, 8) : P.ncol);
    VK_REQUIRE(wgs < (1 << 22), "%s: too many tiles", fn);
  }
  launch_rows(qb, st);
  if (int e = check_launch(fn)) return e;
  launch_products(route, ib, (int)wgs, st);
  return check_launch(fn);
}
