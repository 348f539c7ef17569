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
constexpr int64_t kI8MaxK = 131072;  // 127^2 k < 2^31

__host__ __device__ inline int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Byte of element (r, k) of a packed matrix with `steps` = padded K / 32.
__device__ __forceinline__ int64_t i8_index(int64_t r, int64_t k, int64_t steps) {
  return ((r >> 5) * steps + (k >> 5)) * 1024 + (((k >> 4) & 1) * 32 + (r & 31)) * 16 + (k & 15);
}

// ---------------------------------------------------------------- rounding rows to 8 bits

struct QProb {
  const _Float16* x;
  int8_t* q;
  float* s;
  int m, k, steps;
  int vec;       // rows of x are 16-byte aligned
  int wg_begin;  // first workgroup
};
struct QBatch {
  int n;
  QProb p[kMaxI8];
};

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

// 16 values of row x from k0, zeros past K.
template <bool kVec>
__device__ __forceinline__ void load16(const _Float16* x, int64_t k0, int k, uv4 (&v)[2]) {
  if constexpr (kVec) {
    const uv4* p = reinterpret_cast<const uv4*>(x + k0);
    v[0] = k0 + 8 <= k ? p[0] : uv4{0, 0, 0, 0};
    v[1] = k0 + 16 <= k ? p[1] : uv4{0, 0, 0, 0};
  } else {
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int64_t k1 = k0 + 2 * w;
      const uint32_t lo = k1 < k ? __builtin_bit_cast(uint16_t, x[k1]) : 0;
      const uint32_t hi = k1 + 1 < k ? __builtin_bit_cast(uint16_t, x[k1 + 1]) : 0;
      v[w >> 2][w & 3] = lo | hi << 16;
    }
  }
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

// One row per wave, eight rows per workgroup: the rows of a 128-byte line of the packed matrix.
// The row is kept in registers between its maximum and its rounding where it has at most
// 1024 kKeep values, else read again.  |x| is compared as an integer, where an infinity or a NaN
// exceeds every number: such a row gets the scale NaN and zeros.
template <int kKeep, bool kVec>
__global__ __launch_bounds__(512) void i8_rows_kernel(QBatch bt) {
  int pi = 0;
#pragma unroll
  for (int i = 1; i < kMaxI8; ++i)
    if (i < bt.n && (int)blockIdx.x >= bt.p[i].wg_begin) pi = i;
  const QProb& P = bt.p[pi];
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)((int)blockIdx.x - P.wg_begin) * 8 + (threadIdx.x >> 6);
  if (row >= P.m) return;
  const _Float16* const x = P.x + row * P.k;
  const int k = P.k, chunks = P.steps * 2;  // chunks of 16
  uv4 v[kKeep][2];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < kKeep; ++c) load16<kVec>(x, (int64_t)(c * 64 + lane) * 16, k, v[c]);
#pragma unroll
  for (int c = 0; c < kKeep; ++c) top = top_bits(top, v[c]);
  for (int c = kKeep * 64 + lane; c < chunks; c += 64) {
    uv4 u[2];
    load16<kVec>(x, (int64_t)c * 16, k, u);
    top = top_bits(top, u);
  }
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
  const bool finite = top < 0x7c00u;
  const float a = finite ? h2f((uint16_t)top) : 0.0f;
  const float inv = a > 0.0f ? 1.0f / a : 0.0f;
  if (lane == 0) P.s[row] = finite ? a / 127.0f : __builtin_nanf("");
  int8_t* const q = P.q + i8_index(row, 0, P.steps);
  auto put = [&](int c, const uv4(&u)[2]) __attribute__((always_inline)) {
    const iv4 o = a > 0.0f ? quant16(u, a, inv) : iv4{0, 0, 0, 0};
    *reinterpret_cast<iv4*>(q + (int64_t)c * 512) = o;  // chunk c: 512 bytes on
  };
#pragma unroll
  for (int c = 0; c < kKeep; ++c)
    if (c * 64 + lane < chunks) put(c * 64 + lane, v[c]);
  for (int c = kKeep * 64 + lane; c < chunks; c += 64) {
    uv4 u[2];
    load16<kVec>(x, (int64_t)c * 16, k, u);
    put(c, u);
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
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (r < rows && k0 + e < k) o[e >> 2] |= (int)((uint32_t)(uint8_t)src[r * k + k0 + e] << (8 * (e & 3)));
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
  int epi, vec;          // vec: rows of y are 16-byte aligned
  int nmb, ncol;         // row and column tiles
  int wg_begin;
};
struct IBatch {
  int n;
  IProb p[kMaxI8];
};

__device__ __forceinline__ float i8_act(int epi, float v) {
  if (epi == VKWR_GEMM_EPI_RELU_SQUARE) return v > 0.0f ? v * v : (v != v ? v : 0.0f);  // NaN stays
  if (epi == VKWR_GEMM_EPI_TANH) return tanhf(v);
  if (epi == VKWR_GEMM_EPI_SIGMOID) return sigmoidf(v);
  return v;
}

// Eight consecutive outputs of a row: the sums scaled in fp32, the epilogue, one rounding to fp16.
__device__ __forceinline__ void i8_finish8(const int (&a)[8], int row, int col, int m, int n, int epi, int vec, float s,
                                           const float* t, const _Float16* bias, _Float16* y) {
  if (row >= m || col >= n) return;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = col + e < n ? col + e : n - 1;
    f[e] = (float)a[e] * (s * t[c]);
    if (epi == VKWR_GEMM_EPI_BIAS) f[e] += (float)bias[c];
    f[e] = i8_act(epi, f[e]);
  }
  _Float16* const o = y + (int64_t)row * n + col;
  if (vec) {
    hv8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = f16_of(f[e]);
    *reinterpret_cast<hv8*>(o) = h;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < n) o[e] = f16_of(f[e]);
  }
}

// (32 TM) rows x (32 TN) outputs per workgroup over the whole of K: the NW waves take the blocks of
// KS k-steps w, w + NW, ... with the next block's loads in flight, and the NW partial
// tiles are added through LDS.
template <int TM, int TN, int NW, int KS>
__global__ __launch_bounds__(NW * 64) void i8_stream_kernel(IBatch bt) {
  constexpr int kTiles = TM * TN, kG = 65;  // 16-byte cells of a group of 4 results: 64 lanes and one of padding
  __shared__ __attribute__((aligned(16))) iv4 red[NW * kTiles * 4 * kG];
  int pi = 0;
#pragma unroll
  for (int i = 1; i < kMaxI8; ++i)
    if (i < bt.n && (int)blockIdx.x >= bt.p[i].wg_begin) pi = i;
  const IProb& P = bt.p[pi];
  const int lt = (int)blockIdx.x - P.wg_begin;
  const int mb = lt % P.nmb, cb = lt / P.nmb;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int steps = P.steps, mblk = (P.m + 31) >> 5, nblk = (P.n + 31) >> 5;
  const int8_t *xp[TM], *wp[TN];  // blocks past the last are read as the last
#pragma unroll
  for (int i = 0; i < TM; ++i) xp[i] = P.q + (int64_t)min(mb * TM + i, mblk - 1) * steps * 1024 + lane * 16;
#pragma unroll
  for (int j = 0; j < TN; ++j) wp[j] = P.w + (int64_t)min(cb * TN + j, nblk - 1) * steps * 1024 + lane * 16;
  iv16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = iv16{0};
  iv4 fx[2][KS][TM], fw[2][KS][TN];
  auto load = [&](int buf, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int64_t o = ((int64_t)b * KS + s) * 1024;
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
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[buf][s][j], fx[buf][s][i], acc[i][j], 0, 0, 0);
  };
  const int blocks = steps / KS;  // K is padded to 4 steps
  static_assert(kI8Pad % (32 * KS) == 0, "whole blocks");
  int b = wave;
  if (b < blocks) load(0, b);
  for (; b + 2 * NW < blocks; b += 2 * NW) {
    load(1, b + NW);
    __builtin_amdgcn_sched_barrier(0);
    compute(0);
    __builtin_amdgcn_sched_barrier(0);
    load(0, b + 2 * NW);
    __builtin_amdgcn_sched_barrier(0);
    compute(1);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (b + NW < blocks) {
    load(1, b + NW);
    __builtin_amdgcn_sched_barrier(0);
    compute(0);
    compute(1);
  } else if (b < blocks) {
    compute(0);
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const iv16& a = acc[t / TN][t % TN];
      red[((wave * kTiles + t) * 4 + g) * kG + lane] = iv4{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
    }
  __syncthreads();
  for (int u = threadIdx.x; u < kTiles * 128; u += NW * 64) {
    const int g = u & 3, t = (u >> 2) % TN + (u / (4 * TN * 32)) * TN, r = (u / (4 * TN)) & 31;
    iv4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      lo += red[((w * kTiles + t) * 4 + g) * kG + r];
      hi += red[((w * kTiles + t) * 4 + g) * kG + r + 32];
    }
    const int row = (mb * TM + t / TN) * 32 + r, col = (cb * TN + t % TN) * 32 + 8 * g;
    const int a[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (row < P.m) i8_finish8(a, row, col, P.m, P.n, P.epi, P.vec, P.s[row], P.t, P.bias, P.y);
  }
}

// ---------------------------------------------------------------- host

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  return na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

int64_t packed_bytes(int64_t rows, int64_t k) { return up(rows, kI8Rows) * up(k, kI8Pad); }

int check_problems(const char* fn, int n, const vkwr_i8_problem* p) {
  VK_REQUIRE(n >= 1 && n <= kMaxI8 && p, "%s: 1 to %d problems, got %d", fn, kMaxI8, n);
  for (int i = 0; i < n; ++i) {
    VK_REQUIRE(p[i].m >= 0 && p[i].m <= (1 << 22) && p[i].n >= 1 && p[i].n <= (1 << 24) && p[i].k >= 1 &&
                   p[i].k <= kI8MaxK,
               "%s: problem %d: sizes m=%lld n=%lld k=%lld (m up to 2^22, n up to 2^24, k up to %lld)", fn, i,
               (long long)p[i].m, (long long)p[i].n, (long long)p[i].k, (long long)kI8MaxK);
    VK_REQUIRE(p[i].epilogue == VKWR_GEMM_EPI_NONE || p[i].epilogue == VKWR_GEMM_EPI_RELU_SQUARE ||
                   p[i].epilogue == VKWR_GEMM_EPI_BIAS || p[i].epilogue == VKWR_GEMM_EPI_TANH ||
                   p[i].epilogue == VKWR_GEMM_EPI_SIGMOID,
               "%s: problem %d: unsupported epilogue %d", fn, i, p[i].epilogue);
  }
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

template <int kKeep>
void launch_rows_vec(bool vec, unsigned grid, hipStream_t s, const QBatch& b) {
  if (vec) hipLaunchKernelGGL((i8_rows_kernel<kKeep, true>), dim3(grid), dim3(512), 0, s, b);
  else hipLaunchKernelGGL((i8_rows_kernel<kKeep, false>), dim3(grid), dim3(512), 0, s, b);
}

// Rounds the rows of every problem of `b` (wg_begin filled in here).
void launch_rows(QBatch& b, hipStream_t s) {
  unsigned grid = 0;
  int most = 0;
  bool vec = true;
  for (int i = 0; i < b.n; ++i) {
    b.p[i].wg_begin = (int)grid;
    grid += (unsigned)((b.p[i].m + 7) / 8);
    most = std::max(most, b.p[i].steps);
    vec = vec && b.p[i].vec;
  }
  if (grid == 0) return;
  if (most <= 32) launch_rows_vec<1>(vec, grid, s, b);
  else if (most <= 64) launch_rows_vec<2>(vec, grid, s, b);
  else if (most <= 128) launch_rows_vec<4>(vec, grid, s, b);
  else launch_rows_vec<8>(vec, grid, s, b);
}

QProb row_problem(const uint16_t* x, int64_t m, int64_t k, int8_t* q, float* s) {
  QProb p{};
  p.x = reinterpret_cast<const _Float16*>(x);
  p.q = q;
  p.s = s;
  p.m = (int)m;
  p.k = (int)k;
  p.steps = (int)(up(k, kI8Pad) / 32);
  p.vec = (uintptr_t)x % 16 == 0 && k % 8 == 0;
  return p;
}

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int64_t vkwr_i8_packed_bytes(int64_t rows, int64_t k) {
  if (rows < 0 || rows > (1 << 24) || k < 1 || k > kI8MaxK) return -1;
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
    VK_REQUIRE(!overlap(p[i].y, ny, workspace, need) && !overlap(p[i].x, 2 * p[i].m * p[i].k, workspace, need),
               "%s: problem %d: x or y overlaps the workspace", fn, i);
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
  const I8Scratch c = scratch_of(n, p);
  char* const ws = static_cast<char*>(workspace);
  QBatch qb{};
  IBatch ib{};
  constexpr int TM = 2, TN = 2;
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
    P.vec = (uintptr_t)p[i].y % 16 == 0 && p[i].n % 8 == 0;
    P.nmb = (P.m + 32 * TM - 1) / (32 * TM);
    P.ncol = (P.n + 32 * TN - 1) / (32 * TN);
    P.wg_begin = (int)wgs;
    wgs += (int64_t)P.nmb * P.ncol;
    VK_REQUIRE(wgs < (1 << 23), "%s: too many tiles", fn);
  }
  launch_rows(qb, (hipStream_t)stream);
  if (int e = check_launch(fn)) return e;
  hipLaunchKernelGGL((i8_stream_kernel<TM, TN, 8, 2>), dim3((unsigned)wgs), dim3(512), 0, (hipStream_t)stream, ib);
  return check_launch(fn);
}
