// The grouping of the MoE router's pairs by expert: shared by the launch that does
// nothing else (moe_experts.hip) and the one that rounds the tokens' rows beside it
// (mx4_quantize.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave_ops.h"

namespace hi_rocm {

constexpr int kMoeMaxExperts = 2048;
constexpr int kMoeMaxPairs = 1 << 22;
constexpr int kMoeFewPairs = 8192;  // up to so many by four waves with four loads each, else by 16 with eight

// Workgroup e takes expert e's pairs (e = experts: those with an id outside
// [0, experts), which come last and belong to no group).  Every workgroup
// counts the ids below its own, so none waits for another; its waves own
// consecutive stretches of the pairs, lane l of a stretch 4 consecutive pairs
// at a time, so places follow the pairs' order.  A stretch of up to 256 L pairs
// is read once, all loads at once, and kept in registers.  What bounds it is
// the latency of the loads, two scans and a barrier: 64 pairs 2.8 us.  Four
// waves with 4 loads each, or 16 with 8, us for 4,096, 8,192 and 32,768 pairs of
// 64 experts: 3.6, 5.1, 14.1 and 6.2, 6.4, 8.1.
template <int W, int L>
__device__ __forceinline__ void moe_group_pairs(const uint32_t* ids, int pairs, int experts, int32_t* order,
                                                int32_t* slots, int32_t* offsets, int e) {
  constexpr int kTile = 256 * L;
  __shared__ int less[W], equal[W];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int per = ((pairs + W - 1) / W + 3) & ~3;
  const int p0 = min(wid * per, pairs), p1 = min(p0 + per, pairs), tiles = (p1 - p0 + kTile - 1) / kTile;
  // range-checked: this wave's stretch
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc((void*)(ids + p0), 0, (p1 - p0) * 4, kBufferConfig);
  i32x4_t v[L];
  auto load = [&](int tile) {
    #pragma unroll
    for (int j = 0; j < L; ++j)
      v[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, tile * (kTile * 4) + (j * 64 + lane) * 16, 0, 0);
  };
  // the expert of element q of load j (past the stretch: none, above all)
  auto expert = [&](int tile, int j, int q) {
    const int p = p0 + tile * kTile + (j * 64 + lane) * 4 + q;
    const int id = (uint32_t)v[j][q] < (uint32_t)experts ? v[j][q] : experts;
    return p < p1 ? id : experts + 1;
  };
  int lt = 0, eq = 0;
  for (int t = 0; t < tiles; ++t) {
    load(t);
    #pragma unroll
    for (int j = 0; j < L; ++j)
      #pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int x = expert(t, j, q);
        lt += x < e;
        eq += x == e;
      }
  }
  lt = __builtin_amdgcn_readlane((int)wave_incl_scan_u32((uint32_t)lt), 63);
  eq = __builtin_amdgcn_readlane((int)wave_incl_scan_u32((uint32_t)eq), 63);
  if (lane == 0) { less[wid] = lt; equal[wid] = eq; }
  __syncthreads();
  int at = 0;
  #pragma unroll
  for (int w = 0; w < W; ++w) at += less[w];
  if (threadIdx.x == 0) offsets[e] = at;  // (offsets[experts]: where the groups end)
  if (eq == 0) return;
  for (int w = 0; w < wid; ++w) at += equal[w];
  for (int t = 0; t < tiles; ++t) {
    if (tiles > 1) load(t);
    #pragma unroll
    for (int j = 0; j < L; ++j) {
      int n = 0;
      bool mine[4];
      #pragma unroll
      for (int q = 0; q < 4; ++q) {
        mine[q] = expert(t, j, q) == e;
        n += mine[q];
      }
      if (__ballot(n != 0) == 0ull) continue;
      const int incl = (int)wave_incl_scan_u32((uint32_t)n);
      int i = at + incl - n;
      const int p = p0 + t * kTile + (j * 64 + lane) * 4;
      #pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (mine[q]) {
          order[i] = p + q;
          slots[p + q] = i;
          ++i;
        }
      }
      at += __builtin_amdgcn_readlane(incl, 63);
    }
  }
}

}  // namespace hi_rocm
