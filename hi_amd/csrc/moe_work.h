// How products grouped by expert split their work over workgroups, and the
// gate's function: shared by the bf16 and the 4-bit expert products.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "wave_ops.h"

namespace hi_rocm {

// The groups are cut into tiles of BM places, and the work is (tile, block of
// columns).  A workgroup finds its own from the offsets (64 experts a wave
// scan), so one launch of the largest possible grid serves any raggedness.
// Workgroups go round the 8 XCDs by their number; each XCD takes a contiguous
// stretch of the work, in which an expert's tiles of one block of columns
// follow each other, so that its L2 sees a block of weights once and an
// expert's rows while they are in use.
constexpr int kXcds = 8;

struct MoeWork {
  int expert, i0, i1, block;  // places [i0, i1), column block
};

template <int BM, typename Args>
__device__ __forceinline__ bool moe_work(const Args& a, int blocks, MoeWork& wk) {
  const int lane = threadIdx.x & 63;
  // (past the last expert: none, without a branch that a load would wait behind)
  auto count = [&](int e, int& s) {
    const int from = a.offsets[min(e, a.experts)], to = a.offsets[min(e + 1, a.experts)];
    s = min(max(from, 0), a.places);
    return max(min(to, a.places) - s, 0);
  };
  // the first 256 experts' counts, asked for together and kept
  constexpr int kKept = 4;
  int start_of[kKept], count_of[kKept];
  #pragma unroll
  for (int c = 0; c < kKept; ++c) count_of[c] = count(c * 64 + lane, start_of[c]);
  int tiles = 0;
  #pragma unroll
  for (int c = 0; c < kKept; ++c) tiles += (count_of[c] + BM - 1) / BM;
  for (int e0 = 64 * kKept; e0 < a.experts; e0 += 64) {
    int s;
    tiles += (count(e0 + lane, s) + BM - 1) / BM;
  }
  tiles = (int)wave_incl_scan_u32((uint32_t)tiles);
  tiles = __builtin_amdgcn_readlane(tiles, 63);
  const int64_t total = (int64_t)tiles * blocks, per = (total + kXcds - 1) / kXcds;
  const int64_t slot = blockIdx.x / kXcds, w = blockIdx.x % kXcds * per + slot;
  if (slot >= per || w >= total) return false;
  int before = 0;  // tiles of the experts before e0
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    int s, n = 0;
    if (e0 < 64 * kKept) {
      #pragma unroll
      for (int c = 0; c < kKept; ++c) {
        s = e0 == c * 64 ? start_of[c] : s;
        n = e0 == c * 64 ? count_of[c] : n;
      }
    } else {
      n = count(e0 + lane, s);
    }
    const int mine = (n + BM - 1) / BM;
    const int incl = before + (int)wave_incl_scan_u32((uint32_t)mine);
    const uint64_t hit = __ballot((int64_t)incl * blocks > w && (int64_t)(incl - mine) * blocks <= w);
    if (hit != 0ull) {
      const int l = __builtin_ctzll(hit);
      const int first = __builtin_amdgcn_readlane(incl - mine, l), nt = __builtin_amdgcn_readlane(mine, l);
      const int start = __builtin_amdgcn_readlane(s, l), places = __builtin_amdgcn_readlane(n, l);
      const int local = (int)(w - (int64_t)first * blocks);
      // tiles of one size, a multiple of 16 places
      const int size = ((places + nt - 1) / nt + 15) & ~15;
      wk.expert = e0 + l;
      wk.block = local / nt;
      wk.i0 = start + min(local % nt * size, places);
      wk.i1 = min(wk.i0 + size, start + places);
      return wk.i0 < wk.i1;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// silu(g) * u.  exp(-g) as 2^t (1 + ln 2 * what t = -g log2 e lost to its
// rounding): within a few units of the last place, in a third of expf's and the
// division's instructions (the product kernels repeat this for every register).
// Where 2^t overflows (g from -88.73 down) there is nothing to correct, as inf
// times what was lost would be NaN: the result is -0 there (|silu(g)| < 2^-121),
// and may be from g = -87.34, where 1 / (1 + exp(-g)) is no normal number.
__device__ __forceinline__ float moe_silu_mul(float g, float u) {
  constexpr float kLog2e = 1.44269502e+00f, kLog2eLo = 1.92596299e-08f, kLn2 = 6.93147182e-01f;
  const float t = -g * kLog2e;
  const float lost = fmaf(-g, kLog2eLo, fmaf(-g, kLog2e, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  const float e = fabsf(t) < 128.f ? fmaf(p, lost * kLn2, p) : p;  // (beyond: p is 0 or inf, or NaN)
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// ---- what the product kernels' loops through LDS are made of ----

// (a chunk past the end of k)
static __device__ const uint4 moe_zero = {0u, 0u, 0u, 0u};

typedef __attribute__((address_space(3))) void moe_lds;
typedef const __attribute__((address_space(1))) void moe_global;

// The barrier alone, with nothing moved across it (__syncthreads would also
// wait for the loads in flight).
__device__ __forceinline__ void moe_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}
// vmcnt <= N, lgkmcnt 0
template <int N>
__device__ __forceinline__ void moe_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | 7 << 4);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// lgkmcnt 0
__device__ __forceinline__ void moe_wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// vmcnt <= N alone: what was read from LDS may still be on its way.
template <int N>
__device__ __forceinline__ void moe_wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | 7 << 4 | 15 << 8);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// The largest grid that any split of the places over the experts needs (every
// expert ends in at most one short tile).
template <typename Args>
int64_t moe_grid(const Args& a, int bm, int bn) {
  const int64_t tiles = a.places / bm + std::min(a.experts, a.places);
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols, per = a.swiglu ? bn / 2 : bn;
  return (tiles * ((cols_out + per - 1) / per) + kXcds - 1) / kXcds * kXcds;
}

// (a launch holds less than 2^32 threads)
inline bool moe_grid_fits(int64_t grid, int threads) { return grid <= UINT32_MAX / threads; }

}  // namespace hi_rocm
