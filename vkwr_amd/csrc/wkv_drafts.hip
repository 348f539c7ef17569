// WKV-7 over drafted tokens (speculative decoding of a recurrent model).
//
// A step runs every sequence over T tokens of which only some will be kept.  A cache drops
// rejected positions; a recurrent state cannot, so the state is written one step late:
//
//   S = pool[slot]
//   for t < kept:   S = S diag(d_t) + (S a_t) b_t^T + v_t k_t^T     with the vectors of the step before
//   pool[slot] = S                                                  (kept > 0)
//   for t < T:      the same with this step's vectors, y_t = S r_t  (S is not written)
//
// One launch reads and writes each state once, as a plain decode step does, whatever T is; the
// alternatives move more: T states written per step and one of them kept, or the kept tokens
// run by a launch of their own (one read more).
//
// The state rows are independent recurrences (row i: S_i. <- S_i. d + (S_i. . a) b + v_i k), so a
// (sequence, head) is split over lanes by rows and columns only: lane (g = lane & 7, q = lane >> 3)
// of wave wv owns kRPL rows at columns 4g..4g+3 and 32+4g..32+4g+3.  A dot product is eight 8-term
// FMA chains and a butterfly over the eight lanes of the row -- the order of the row-split prefill
// and decode kernels, so a draft's y and state are their bits whatever the split.
//
// Token vectors are staged in LDS as fp32 in chunks of kDraftTC tokens, the kept and the new tokens as one
// sequence; the decay is computed once per token and channel, with a channel on every lane (as one of six
// vectors in 16-byte pieces, a sixth of each wave's lanes computed eight of them while the others waited).

#include "vk_capi.h"
#include "vk_common.cuh"

namespace vk {
namespace {

typedef _Float16 hv8 __attribute__((ext_vector_type(8)));

constexpr int kDraftTC = 16;   // tokens per staged chunk
constexpr int kDraftVecs = 6;  // r, decay, k, v, a, b

struct DraftArgs {
  int P, T, C, H, n_slots, n_pending;
  float* pool;
  const int32_t *slots, *kept, *pending_rows;
  const _Float16 *pend[5];                 // w, k, v, a, b of the pending tokens, [n_pending, P, C]
  const _Float16 *r, *w, *k, *v, *a, *b;   // [B, T, C]
  _Float16* y;
};

// Sum over the 8 lanes 8m..8m+7, ((p0+p1)+(p2+p3)) + ((p4+p5)+(p6+p7)) in every lane.
__device__ __forceinline__ float row_sum8(float x) {
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xB1, 0xF, 0xF, false));
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4E, 0xF, 0xF, false));
  x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x141, 0xF, 0xF, false));
  return x;
}

// kRPL state rows per lane: 8 / kRPL waves per (sequence, head).  Few chains (up to two per CU) are bound by
// the latency of one and take kRPL = 1 (one sequence of 32 heads, 5 + 5 tokens: 5.3 us against 6.7 with 2),
// the others 2, bound by the states' traffic (128 sequences of 64 heads, 5 + 5 tokens, in a replayed graph:
// 76 us, 4.2 TB/s; in the run that compared them 69 with 2, 83 with 1, 82 with 4, 120 with 8, whose single wave
// has nothing beside it to cover its loads).  116 VGPRs leave four waves per SIMD; held to 96 for a fifth, the
// spills cost more (90 us in that run).
template <int kRPL>
__global__ __launch_bounds__(64 * (8 / kRPL)) void wkv7_fp32_drafts_kernel(DraftArgs p) {
  constexpr int kThreads = 64 * (8 / kRPL);
  __shared__ f4 vl[kDraftTC * kDraftVecs * 16];  // [token][vector][16 x f4]
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int g = lane & 7, q = lane >> 3;
  const int bi = blockIdx.x / p.H, h = blockIdx.x - bi * p.H;
  const int i0 = 8 * kRPL * wv + kRPL * q;
  const size_t ytok = (size_t)bi * p.T * p.C + (size_t)h * kHead;

  const int slot = p.slots[bi];
  const int nk = p.kept ? p.kept[bi] : 0;
  const int prow = p.pending_rows ? p.pending_rows[bi] : bi;
  if (slot < 0 || slot >= p.n_slots || nk < 0 || nk > p.P || (nk > 0 && (prow < 0 || prow >= p.n_pending))) {
    for (int i = tid; i < p.T * kHead; i += kThreads)
      p.y[ytok + (size_t)(i / kHead) * p.C + (i % kHead)] = (_Float16)__builtin_nanf("");
    return;
  }
  const int total = nk + p.T;
  if (total == 0) return;
  float* S = p.pool + ((size_t)slot * p.H + h) * (kHead * kHead);
  float s[kRPL][8];
#pragma unroll
  for (int rr = 0; rr < kRPL; ++rr) {
    const float* row = S + (i0 + rr) * kHead;
    const f4 lo = *reinterpret_cast<const f4*>(row + 4 * g);
    const f4 hi = *reinterpret_cast<const f4*>(row + 32 + 4 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[rr][e] = lo[e];
      s[rr][4 + e] = hi[e];
    }
  }
  auto write_state = [&]() {
#pragma unroll
    for (int rr = 0; rr < kRPL; ++rr) {
      float* row = S + (i0 + rr) * kHead;
      *reinterpret_cast<f4*>(row + 4 * g) = f4{s[rr][0], s[rr][1], s[rr][2], s[rr][3]};
      *reinterpret_cast<f4*>(row + 32 + 4 * g) = f4{s[rr][4], s[rr][5], s[rr][6], s[rr][7]};
    }
  };
  const size_t pend0 = (size_t)(nk > 0 ? prow : 0) * p.P * p.C + (size_t)h * kHead;

  for (int c0 = 0; c0 < total; c0 += kDraftTC) {
    const int n = min(kDraftTC, total - c0);
    if (c0 > 0) __syncthreads();  // the chunk before is read
    // r, k, v, a, b in pieces of 8 channels, w channel by channel: all loads, then all stores
    constexpr int kPieces = (kDraftTC * 40 + kThreads - 1) / kThreads, kChannels = kDraftTC * kHead / kThreads;
    hv8 x[kPieces];
    _Float16 xw[kChannels];
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int piece = tid + u * kThreads, tv = piece >> 3, tt = tv / 5, vec = tv - tt * 5, t = c0 + tt;
      if (tt >= n || (t < nk && vec == 0)) continue;  // kept tokens need no r
      const _Float16* src = t < nk ? (vec == 1 ? p.pend[1] : vec == 2 ? p.pend[2] : vec == 3 ? p.pend[3] : p.pend[4]) +
                                         pend0 + (size_t)t * p.C
                                   : (vec == 0 ? p.r : vec == 1 ? p.k : vec == 2 ? p.v : vec == 3 ? p.a : p.b) + ytok +
                                         (size_t)(t - nk) * p.C;
      x[u] = *reinterpret_cast<const hv8*>(src + (piece & 7) * 8);
    }
#pragma unroll
    for (int u = 0; u < kChannels; ++u) {
      const int e = tid + u * kThreads, tt = e >> 6, t = c0 + tt;
      if (tt >= n) continue;
      xw[u] = t < nk ? p.pend[0][pend0 + (size_t)t * p.C + (e & 63)] : p.w[ytok + (size_t)(t - nk) * p.C + (e & 63)];
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int piece = tid + u * kThreads, tv = piece >> 3, tt = tv / 5, vec = tv - tt * 5;
      if (tt >= n || (c0 + tt < nk && vec == 0)) continue;
      f4* d = &vl[(tt * kDraftVecs + vec + (vec > 0 ? 1 : 0)) * 16 + (piece & 7) * 2];
      d[0] = f4{(float)x[u][0], (float)x[u][1], (float)x[u][2], (float)x[u][3]};
      d[1] = f4{(float)x[u][4], (float)x[u][5], (float)x[u][6], (float)x[u][7]};
    }
#pragma unroll
    for (int u = 0; u < kChannels; ++u) {
      const int e = tid + u * kThreads, tt = e >> 6;
      if (tt < n) reinterpret_cast<float*>(&vl[(tt * kDraftVecs + 1) * 16])[e & 63] = decay((float)xw[u]);
    }
    __syncthreads();
    for (int tt = 0; tt < n; ++tt) {
      const int t = c0 + tt;
      if (t == nk && nk > 0) write_state();
      const f4* base = &vl[tt * kDraftVecs * 16];
      const f4 d0 = base[1 * 16 + g], d1 = base[1 * 16 + 8 + g], k0 = base[2 * 16 + g], k1 = base[2 * 16 + 8 + g];
      const f4 a0 = base[4 * 16 + g], a1 = base[4 * 16 + 8 + g], b0 = base[5 * 16 + g], b1 = base[5 * 16 + 8 + g];
      const float* vv = reinterpret_cast<const float*>(base + 3 * 16) + i0;
#pragma unroll
      for (int rr = 0; rr < kRPL; ++rr) {
        float sa = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sa = __builtin_fmaf(s[rr][e], e < 4 ? a0[e & 3] : a1[e & 3], sa);
        sa = row_sum8(sa);
        const float vi = vv[rr];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = s[rr][e] * (e < 4 ? d0[e & 3] : d1[e & 3]);
          x = __builtin_fmaf(sa, e < 4 ? b0[e & 3] : b1[e & 3], x);
          s[rr][e] = __builtin_fmaf(e < 4 ? k0[e & 3] : k1[e & 3], vi, x);
        }
      }
      if (t >= nk) {
        const f4 r0 = base[g], r1 = base[8 + g];
        float yv = 0.0f;
#pragma unroll
        for (int rr = 0; rr < kRPL; ++rr) {
          float acc = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc = __builtin_fmaf(s[rr][e], e < 4 ? r0[e & 3] : r1[e & 3], acc);
          acc = row_sum8(acc);
          yv = g == rr ? acc : yv;  // lane g < kRPL keeps row i0 + g
        }
        if (g < kRPL) p.y[ytok + (size_t)(t - nk) * p.C + i0 + g] = f16_of(yv);
      }
    }
  }
  if (total == nk) write_state();
}

}  // namespace
}  // namespace vk

using namespace vk;

extern "C" int vkwr_wkv7_fp32_drafts_slots(int B, int P, int T, int C, int H, float* pool, int n_slots,
                                           const int32_t* slots, const int32_t* kept, int n_pending,
                                           const int32_t* pending_rows, const uint16_t* pw, const uint16_t* pk,
                                           const uint16_t* pv, const uint16_t* pa, const uint16_t* pb,
                                           const uint16_t* r, const uint16_t* w, const uint16_t* k,
                                           const uint16_t* v, const uint16_t* a, const uint16_t* b, uint16_t* y,
                                           void* stream) {
  clear_error();
  const char* fn = "vkwr_wkv7_fp32_drafts_slots";
  VK_REQUIRE(B >= 0 && P >= 0 && T >= 0 && H >= 0 && n_slots >= 0 && n_pending >= 0,
             "%s: negative size (B=%d P=%d T=%d H=%d n_slots=%d n_pending=%d)", fn, B, P, T, H, n_slots, n_pending);
  VK_REQUIRE(C == (int64_t)H * kHead, "%s: only head size 64 is supported (C=%d H=%d)", fn, C, H);
  VK_REQUIRE((int64_t)B * H < (1 << 23) && (int64_t)P + T <= (1 << 24), "%s: B*H or P+T too large", fn);
  VK_REQUIRE((kept != nullptr) == (P > 0), "%s: kept must be given exactly when P > 0", fn);
  if (B == 0 || H == 0 || P + T == 0) return VKWR_OK;
  VK_REQUIRE(pool && slots, "%s: null pointer", fn);
  VK_REQUIRE(P == 0 || (pw && pk && pv && pa && pb), "%s: null pending pointer", fn);
  VK_REQUIRE(P == 0 || pending_rows || n_pending >= B, "%s: %d pending rows for %d sequences", fn, n_pending, B);
  VK_REQUIRE(T == 0 || (r && w && k && v && a && b && y), "%s: null pointer", fn);
  const uintptr_t bits = (uintptr_t)pool | (uintptr_t)pw | (uintptr_t)pk | (uintptr_t)pv | (uintptr_t)pa |
                         (uintptr_t)pb | (uintptr_t)r | (uintptr_t)w | (uintptr_t)k | (uintptr_t)v |
                         (uintptr_t)a | (uintptr_t)b;
  VK_REQUIRE(bits % 16 == 0, "%s: pool and token vectors must be 16-byte aligned", fn);
  auto h16 = [](const uint16_t* x) { return reinterpret_cast<const _Float16*>(x); };
  DraftArgs p{P, T, C, H, n_slots, n_pending, pool, slots, kept, pending_rows,
              {h16(pw), h16(pk), h16(pv), h16(pa), h16(pb)}, h16(r), h16(w), h16(k), h16(v), h16(a), h16(b),
              reinterpret_cast<_Float16*>(y)};
  if ((int64_t)B * H <= 2 * (int64_t)device_cus())
    hipLaunchKernelGGL(wkv7_fp32_drafts_kernel<1>, dim3(B * H), dim3(512), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(wkv7_fp32_drafts_kernel<2>, dim3(B * H), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch(fn);
}
