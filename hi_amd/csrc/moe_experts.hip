// The experts behind the MoE router (moe_router.hip): the router's (token,
// slot) pairs grouped by expert, matrix products over the groups, and the
// weighted sum of a token's experts.  (The reference runs its experts' row
// products one token at a time; no grouped counterpart there.)
//
// Pair p = token * top_k + slot.  hi_rocm_moe_group sorts the pairs by expert,
// stably: order[i] = the pair in place i, slots[p] = its place, offsets[e] ..
// offsets[e + 1] = expert e's places.  A product takes place i's row of x
// times its expert's weights:
//     y[i][c] = sum_k x[row(i)][k] * w[e][c][k]
// with row(i) = order[i] / top_k, or i itself where x is already in the
// groups' order; the combination sums a token's places in slot order.
// Nothing depends on the order in which workgroups run.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "hi_rocm.h"
#include "sampler_internal.h"
#include "wave_ops.h"

namespace hi_rocm {
hipError_t ensure_lds(const void* fn, size_t bytes);  // sampler_chunked.hip

namespace {

typedef __bf16 moe_bf16x8 __attribute__((ext_vector_type(8)));
typedef float moe_f32x4 __attribute__((ext_vector_type(4)));

constexpr int kMoeMaxExperts = 2048;
constexpr int kMoeMaxPairs = 1 << 22;

// ---- grouping -------------------------------------------------------------

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
__global__ void __launch_bounds__(64 * W) moe_group_kernel(const uint32_t* ids, int pairs, int experts, int32_t* order,
                                                           int32_t* slots, int32_t* offsets) {
  constexpr int kTile = 256 * L;
  __shared__ int less[W], equal[W];
  const int e = blockIdx.x, lane = threadIdx.x & 63;
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

// ---- products -------------------------------------------------------------

struct GroupedArgs {
  const __bf16* x;         // [x_rows][x_stride]
  int64_t x_stride;
  const int32_t* order;    // or null: place i's row is i
  const int32_t* offsets;  // [experts + 1]
  const __bf16* w;         // [experts][cols][k]
  void* out;               // [places][out_stride]
  int64_t out_stride;
  int x_rows, top_k, places, experts, cols, k, swiglu, out_bf16;
  int out_vec;  // rows of out start on 16 bytes (32,768 rows of 2048 bf16, k 512: 93 us, else 173)
};

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

template <int BM>
__device__ __forceinline__ bool moe_work(const GroupedArgs& a, int blocks, MoeWork& wk) {
  const int lane = threadIdx.x & 63;
  auto count = [&](int e, int& s) {
    s = 0;
    if (e >= a.experts) return 0;
    s = min(max(a.offsets[e], 0), a.places);
    return max(min(a.offsets[e + 1], a.places) - s, 0);
  };
  int tiles = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
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
    int s;
    const int n = count(e0 + lane, s), mine = (n + BM - 1) / BM;
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

// The row of x behind place i.
__device__ __forceinline__ const __bf16* moe_row(const GroupedArgs& a, int i) {
  const int row = a.order ? a.order[i] / a.top_k : i;
  return a.x + (int64_t)min(max(row, 0), a.x_rows - 1) * a.x_stride;
}

// Four columns c .. c + 3 of place p.
__device__ __forceinline__ void moe_store(const GroupedArgs& a, int p, int c, int cols_out, const moe_f32x4& y) {
  const int64_t at = (int64_t)p * a.out_stride + c;
  if (c + 4 <= cols_out && a.out_vec) {
    if (a.out_bf16) {
      typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<bf16x4*>((__bf16*)a.out + at) = __builtin_convertvector(y, bf16x4);
    } else {
      *reinterpret_cast<moe_f32x4*>((float*)a.out + at) = y;
    }
    return;
  }
  #pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (c + q >= cols_out) break;
    if (a.out_bf16) ((__bf16*)a.out)[at + q] = (__bf16)y[q];
    else ((float*)a.out)[at + q] = y[q];
  }
}

__device__ __forceinline__ moe_bf16x8 moe_ld(const __bf16* p) { return *reinterpret_cast<const moe_bf16x8*>(p); }

// Both product kernels multiply with MFMA 16x16x32 bf16 (lane l = 16 g + r: A
// row r, elements 8 g .. + 7; B column r, the same; D rows 4 g .. + 3 of column
// r), the weights as A and the places as B: a lane ends with four neighbouring
// columns of one place.

// Few places an expert (decode): the weights are what is read.  The
// workgroup's waves split k; each streams 64 columns' rows straight into
// registers, two blocks of 64 ahead, and multiplies them with up to 16 MT
// places.  A lane loads 32 bytes of its row at element 16 g of a block, so a
// row's 128-byte line is read whole, and gives 16 to each of two MFMAs (both
// operands are taken in that order of k).  The waves' sums are added in wave
// order.  Bound by the weights' bytes: 8 tokens with 8 of 256 experts each, 2048
// x 1536, some 370 MB of weights: 61 us with the grouping, 5.9 TB/s; three
// workgroups a CU hide each other's beginnings (offsets, rows, first weights).
constexpr int kFewWaves = 4;
constexpr int kFewCols = 64;

template <int MT>
__global__ void __launch_bounds__(64 * kFewWaves) moe_few_kernel(GroupedArgs a) {
  __shared__ moe_f32x4 part[kFewWaves - 1][MT * 4][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols;
  const int per = a.swiglu ? kFewCols / 2 : kFewCols;
  MoeWork wk;
  if (!moe_work<16 * MT>(a, (cols_out + per - 1) / per, wk)) return;
  const int c0 = wk.block * per;
  const __bf16* wr[4];
  #pragma unroll
  for (int t = 0; t < 4; ++t) {  // with swiglu two tiles of gate columns, then the same of up columns
    const int c = a.swiglu ? min(c0 + (t & 1) * 16 + r, cols_out - 1) + (t >> 1) * cols_out
                           : min(c0 + t * 16 + r, cols_out - 1);
    wr[t] = a.w + ((int64_t)wk.expert * a.cols + c) * a.k + 16 * g;
  }
  const __bf16* xr[MT];
  #pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = moe_row(a, min(wk.i0 + 16 * m + r, wk.i1 - 1)) + 16 * g;
  moe_f32x4 acc[MT][4];
  #pragma unroll
  for (int m = 0; m < MT; ++m)
    #pragma unroll
    for (int t = 0; t < 4; ++t) acc[m][t] = moe_f32x4{0.f, 0.f, 0.f, 0.f};
  moe_bf16x8 wb[2][4][2], xb[2][MT][2];
  auto load = [&](int slot, int k) {
    #pragma unroll
    for (int t = 0; t < 4; ++t) { wb[slot][t][0] = moe_ld(wr[t] + k); wb[slot][t][1] = moe_ld(wr[t] + k + 8); }
    #pragma unroll
    for (int m = 0; m < MT; ++m) { xb[slot][m][0] = moe_ld(xr[m] + k); xb[slot][m][1] = moe_ld(xr[m] + k + 8); }
  };
  auto multiply = [&](int slot) {
    #pragma unroll
    for (int h = 0; h < 2; ++h)
      #pragma unroll
      for (int m = 0; m < MT; ++m)
        #pragma unroll
        for (int t = 0; t < 4; ++t)
          acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[slot][t][h], xb[slot][m][h], acc[m][t], 0, 0, 0);
  };
  // whole blocks of 64, a wave's share of them; the last wave also takes the rest
  const int nb = a.k >> 6, share = (nb + kFewWaves - 1) / kFewWaves;
  const int b0 = min(wid * share, nb), b1 = min(b0 + share, nb);
  if (b0 < b1) load(0, b0 * 64);
  if (b0 + 1 < b1) load(1, (b0 + 1) * 64);
  for (int b = b0; b < b1; b += 2) {
    multiply(0);
    if (b + 2 < b1) load(0, (b + 2) * 64);
    if (b + 1 < b1) {
      multiply(1);
      if (b + 3 < b1) load(1, (b + 3) * 64);
    }
  }
  if (wid == kFewWaves - 1 && (a.k & 63) != 0) {
    const int k = nb * 64, left = a.k - k - 16 * g;  // (a multiple of 8)
    const moe_bf16x8 zero = {};
    #pragma unroll
    for (int t = 0; t < 4; ++t) {
      wb[0][t][0] = left > 0 ? moe_ld(wr[t] + k) : zero;
      wb[0][t][1] = left > 8 ? moe_ld(wr[t] + k + 8) : zero;
    }
    #pragma unroll
    for (int m = 0; m < MT; ++m) {
      xb[0][m][0] = left > 0 ? moe_ld(xr[m] + k) : zero;
      xb[0][m][1] = left > 8 ? moe_ld(xr[m] + k + 8) : zero;
    }
    multiply(0);
  }
  if (wid > 0) {
    #pragma unroll
    for (int m = 0; m < MT; ++m)
      #pragma unroll
      for (int t = 0; t < 4; ++t) part[wid - 1][m * 4 + t][lane] = acc[m][t];
  }
  __syncthreads();
  if (wid > 0) return;
  #pragma unroll
  for (int m = 0; m < MT; ++m) {
    #pragma unroll
    for (int t = 0; t < 4; ++t)
      #pragma unroll
      for (int w = 0; w < kFewWaves - 1; ++w) acc[m][t] += part[w][m * 4 + t][lane];
    const int p = wk.i0 + 16 * m + r;
    if (p >= wk.i1) continue;
    if (a.swiglu) {
      #pragma unroll
      for (int t = 0; t < 2; ++t) {
        moe_f32x4 y;
        #pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = moe_silu_mul(acc[m][t][q], acc[m][t + 2][q]);
        if (c0 + t * 16 + 4 * g < cols_out) moe_store(a, p, c0 + t * 16 + 4 * g, cols_out, y);
      }
    } else {
      #pragma unroll
      for (int t = 0; t < 4; ++t)
        if (c0 + t * 16 + 4 * g < cols_out) moe_store(a, p, c0 + t * 16 + 4 * g, cols_out, acc[m][t]);
    }
  }
}

// Many places an expert (prefill): BM places times BN weight rows a workgroup
// of eight waves, two a SIMD, a wave (BM / WM) x (BN / WN) of them.
//
// k goes in steps of BK through NB LDS buffers that loads fill directly (the
// step NB - 1 ahead).  A step has two phases: read the step's operands from
// LDS and start the loads of a later step; multiply.  Waves 4 to 7 run one
// phase behind waves 0 to 3 (a barrier more before the first step), so on
// every SIMD one wave reads while the other multiplies.  Why no buffer is
// written while it is read: a wave's reads are done (lgkmcnt 0) before the
// barrier that ends its phase, the other waves read the same step at most one
// phase later, and the buffer of step s - 1 is filled again from step s's read
// phase on.  Why a step is there when it is read: each wave waits for its own
// loads of step s + 1 (all but the NB - 2 newest steps') before the barrier
// that ends its reading of step s.
//
// A row of a step is BK * 2 bytes; its 16-byte chunk c lies at c ^ (row & 7)
// (BK = 64) or c ^ (row / 2 & 3) (BK = 32), so that 16 rows' reads of a chunk
// meet all banks.  A load writes 64 lanes x 16 contiguous bytes; the lanes
// choose their global addresses so that the chunks land there.  Chunks past k
// come from a zero.
//
// What bounds it: 32,768 places of 8 experts, 2048 x 2048: 229 to 241 us from
// card to card, 1,140 to 1,200 TFLOP/s, of which the products of tiles in flight
// take 200 us (a large dense product of the same size 192) and the rest is
// beginnings and ends of workgroups, whose results all CUs write at about the
// same time.  With 64 experts of a router's sizes 311 to 340: tiles are not full,
// and the short ones end up in any round (experts of equal size: 254), and the
// weights come from memory once (537 MB) instead of from the L2s.  (Tried: five buffers instead of four;
// 64 of k in two buffers; 128 x 128 a wave with four waves; two workgroups a CU;
// workgroups that stay and load the next tile under this one's last steps;
// bodies for every 32 places: within 2% or slower.  In the loop reading the
// operands and filling the buffers take LDS as long as the products take the
// matrix cores, 1,024 cycles a step.  Weights straight to registers take a third
// of that off, but two waves then load the same weights: 323 us.)
__device__ const uint4 moe_zero = {0u, 0u, 0u, 0u};

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

template <int L>
struct MoeSources {
  const __bf16* p[L];
};

// The loads of a step's L rounds into `to` (this wave's part of the first).
// A pointer of its own for what the step reads from LDS and one for what the
// loads write: the compiler then knows that the reads need not wait for them.
template <int L, int T>
__device__ __forceinline__ void moe_fill(const MoeSources<L>& src, bool in, int k, char* to) {
  #pragma unroll
  for (int i = 0; i < L; ++i) {
    const void* from = in ? (const void*)(src.p[i] + k) : (const void*)&moe_zero;
    __builtin_amdgcn_global_load_lds((moe_global*)from, (moe_lds*)(to + i * T * 16), 16, 0, 0);
  }
}

template <int MT, int NT, int KH, int BK, int WM>
__device__ __forceinline__ void moe_read(const char* __restrict__ xb, const char* __restrict__ wb, int r, int g,
                                         moe_bf16x8 (&xf)[KH][MT], moe_bf16x8 (&wf)[KH][NT]) {
  #pragma unroll
  for (int h = 0; h < KH; ++h) {
    const int at = BK == 64 ? ((g + 4 * h) ^ (r & 7)) * 16 : (g ^ ((r >> 1) & 3)) * 16;
    #pragma unroll
    for (int t = 0; t < NT; ++t) wf[h][t] = *reinterpret_cast<const moe_bf16x8*>(wb + t * (32 * BK) + at);
    #pragma unroll
    for (int m = 0; m < MT; ++m)
      xf[h][m] = *reinterpret_cast<const moe_bf16x8*>(xb + m * (WM * 32 * BK) + at);
  }
}

// A wave's results, MT x 16 places (every WM-th 16 from p0) of NT x 16 columns
// (from c0, with swiglu half as many), by way of its own LDS: 64 places at a
// time in rows of 64 columns, written out 16 bytes a lane, a row's bytes next to each other.
// Stored from the lanes that hold them, each store would touch 16 rows, and
// the unrolled code would be ten times as long.
constexpr int kMoeOutBytes = 16384;

template <int MT, int NT, int WM>
__device__ __forceinline__ void moe_tile_out(const GroupedArgs& a, moe_f32x4 (&acc)[MT][NT], char* mem, int p0, int i1,
                                             int c0, int cols_out, int lane) {
  static_assert(NT == 4, "64 columns a wave");
  const int r = lane & 15, g = lane >> 4;
  if (a.swiglu) {
    #pragma unroll
    for (int m = 0; m < MT; ++m)
      #pragma unroll
      for (int t = 0; t < NT / 2; ++t)
        #pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][t][q] = moe_silu_mul(acc[m][t][q], acc[m][t + NT / 2][q]);
  }
  const int wide = a.swiglu ? 32 : 64;  // columns of a row
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  #pragma unroll
  for (int half = 0; half < (MT + 3) / 4; ++half) {
    if (p0 + half * (WM * 64) >= i1) return;
    // row j of 64 values: the 16-byte chunk c at c ^ (j & 7)
    #pragma unroll
    for (int m = half * 4; m < half * 4 + 4 && m < MT; ++m) {
      const int j = (m - half * 4) * 16 + r;
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (a.out_bf16)
          *reinterpret_cast<bf16x4*>(mem + j * 128 + ((t * 2 + (g >> 1)) ^ (j & 7)) * 16 + (g & 1) * 8) =
              __builtin_convertvector(acc[m][t], bf16x4);
        else
          *reinterpret_cast<moe_f32x4*>(mem + j * 256 + ((t * 4 + g) ^ (j & 7)) * 16) = acc[m][t];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int es = a.out_bf16 ? 2 : 4, n = 16 / es;    // bytes of a value, values of a chunk
    const int lanes = wide / n, rows = 64 / lanes;      // lanes of a row, rows at a time
    const int c = lane % lanes, col = c0 + c * n;
    #pragma unroll 1
    for (int j = lane / lanes; j < (MT < 4 ? MT * 16 : 64); j += rows) {
      const int p = p0 + half * (WM * 64) + (j >> 4) * (WM * 16) + (j & 15);
      if (p >= i1) break;
      const uint4 v = *reinterpret_cast<const uint4*>(mem + j * (64 * es) + (c ^ (j & 7)) * 16);
      char* to = (char*)a.out + ((int64_t)p * a.out_stride + col) * es;
      if (col + n <= cols_out && a.out_vec) {
        *reinterpret_cast<uint4*>(to) = v;
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        #pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (q >= n || col + q >= cols_out) break;
          if (a.out_bf16) ((uint16_t*)to)[q] = (uint16_t)(w[q >> 1] >> (q & 1) * 16);
          else ((uint32_t*)to)[q] = w[q & 3];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int BM, int BN, int MT, int BK, int NB>  // MT: of BM / 16 / WM, what the tile has places for
__device__ __forceinline__ void moe_many_tile(const GroupedArgs& a, const MoeWork& wk, char* moe_smem) {
  constexpr int T = 512, CH = BK / 8;                    // 16-byte chunks of a row
  constexpr int XL = BM * CH / T, WL = BN * CH / T;      // loads a thread
  constexpr int WN = BN / 64, WM = 8 / WN, NT = 4, KH = BK / 32;
  constexpr int ROW = BK * 2, STEP = (BM + BN) * ROW;
  static_assert(MT * WM * 16 <= BM && XL >= 1 && WL >= 1 && BM * CH % T == 0 && BN * CH % T == 0, "tile split");
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid % WM, wn = wid / WM;
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols;
  const int per = a.swiglu ? BN / 2 : BN;
  const int c0 = wk.block * per;
  // the column behind row j of the tile's weights: with swiglu each wave's
  // rows are half gate, half up
  constexpr int WR = BN / WN;
  auto column = [&](int j) {
    if (!a.swiglu) return min(c0 + j, cols_out - 1);
    const int in = j % WR;
    return min(c0 + j / WR * (WR / 2) + in % (WR / 2), cols_out - 1) + (in >= WR / 2 ? cols_out : 0);
  };
  // this thread's chunk of the rows it loads (the same in every round: a round
  // is a multiple of 8 rows)
  const int jr = tid / CH;
  const int chunk = (tid % CH) ^ (BK == 64 ? jr & 7 : jr >> 1 & 3);
  MoeSources<XL> xs;
  MoeSources<WL> ws;
  #pragma unroll
  for (int i = 0; i < XL; ++i) xs.p[i] = moe_row(a, min(wk.i0 + i * (T / CH) + jr, wk.i1 - 1)) + 8 * chunk;
  #pragma unroll
  for (int i = 0; i < WL; ++i)
    ws.p[i] = a.w + ((int64_t)wk.expert * a.cols + column(i * (T / CH) + jr)) * a.k + 8 * chunk;
  const int steps = (a.k + BK - 1) / BK;
  // Workgroups begin at different steps and come round: rows of weights lie a.k
  // apart, and with all workgroups at the same step of a power of two they
  // would ask the same few memory channels (16,384 places of 128 experts, 2048
  // x 1536: 171 us, so 161; never more than 2% slower).  The same step for all
  // places of an expert and a block: a row's sums do not depend on its place.
  int k = (wk.expert * 7 + wk.block * 2) % steps * BK;
  auto fill = [&](int step) {
    const bool in = step < steps && k + 8 * chunk < a.k;
    char* to = moe_smem + step % NB * STEP + wid * 1024;
    moe_fill<XL, T>(xs, in, k, to);
    moe_fill<WL, T>(ws, in, k, to + BM * ROW);
    k = k + BK < steps * BK ? k + BK : 0;
  };
  moe_f32x4 acc[MT][NT];
  #pragma unroll
  for (int m = 0; m < MT; ++m)
    #pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = moe_f32x4{0.f, 0.f, 0.f, 0.f};
  #pragma unroll
  for (int s = 0; s < NB - 1; ++s) fill(s);
  moe_wait<(XL + WL) * (NB - 2)>();
  moe_barrier();
  if (wid >= 4) moe_barrier();
  for (int s = 0; s < steps; ++s) {
    moe_bf16x8 xf[KH][MT], wf[KH][NT];
    const char* b = moe_smem + s % NB * STEP;
    moe_read<MT, NT, KH, BK, WM>(b + (wm * 16 + r) * ROW, b + BM * ROW + (wn * WR + r) * ROW, r, g, xf, wf);
    fill(s + NB - 1);
    moe_wait<(XL + WL) * (NB - 2)>();
    moe_barrier();
    __builtin_amdgcn_s_setprio(1);
    #pragma unroll
    for (int h = 0; h < KH; ++h)
      #pragma unroll
      for (int m = 0; m < MT; ++m)
        #pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[h][t], xf[h][m], acc[m][t], 0, 0, 0);
    __builtin_amdgcn_s_setprio(0);
    moe_barrier();
  }
  if (wid < 4) moe_barrier();
  moe_wait<0>();  // no load may still write LDS when it is used again, or the workgroup ends
  moe_barrier();
  moe_tile_out<MT, NT, WM>(a, acc, moe_smem + wid * kMoeOutBytes, wk.i0 + wm * 16, wk.i1,
                       c0 + wn * (a.swiglu ? WR / 2 : WR), cols_out, lane);
}

// WM waves share the places, every WM-th 16 of them, so a tile of fewer places
// than BM is multiplied as one of a quarter, a half or three quarters (with four
// waves, a half).  (32,768 places of 64 experts, 2048 x 2048: 311 us against 322
// with every tile multiplied whole.)
template <int BM, int BN, int BK, int NB>
__global__ void __launch_bounds__(512) moe_many_kernel(GroupedArgs a) {
  extern __shared__ __align__(16) char moe_smem[];
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols, per = a.swiglu ? BN / 2 : BN;
  MoeWork wk;
  if (!moe_work<BM>(a, (cols_out + per - 1) / per, wk)) return;
  constexpr int WM = 8 / (BN / 64), MT = BM / 16 / WM;
  switch ((wk.i1 - wk.i0 + BM / 4 - 1) / (BM / 4)) {
    case 1: return moe_many_tile<BM, BN, (MT + 3) / 4, BK, NB>(a, wk, moe_smem);
    case 2: return moe_many_tile<BM, BN, MT / 2, BK, NB>(a, wk, moe_smem);
    case 3: return moe_many_tile<BM, BN, (MT * 3 + 3) / 4, BK, NB>(a, wk, moe_smem);
    default: return moe_many_tile<BM, BN, MT, BK, NB>(a, wk, moe_smem);
  }
}

// The largest grid that any split of the places over the experts needs (every
// expert ends in at most one short tile).
int64_t moe_grid(const GroupedArgs& a, int bm, int bn) {
  const int64_t tiles = a.places / bm + std::min(a.experts, a.places);
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols, per = a.swiglu ? bn / 2 : bn;
  return (tiles * ((cols_out + per - 1) / per) + kXcds - 1) / kXcds * kXcds;
}

// (a launch holds less than 2^32 threads)
bool moe_grid_fits(int64_t grid, int threads) { return grid <= UINT32_MAX / threads; }

template <int MT>
hipError_t launch_few(const GroupedArgs& a, hipStream_t st) {
  const int64_t grid = moe_grid(a, 16 * MT, kFewCols);
  if (!moe_grid_fits(grid, 64 * kFewWaves)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(moe_few_kernel<MT>, dim3((unsigned)grid), dim3(64 * kFewWaves), 0, st, a);
  return hipGetLastError();
}

template <int BM, int BN, int BK, int NB>
hipError_t launch_many(const GroupedArgs& a, hipStream_t st) {
  constexpr size_t bytes = (size_t)NB * (BM + BN) * BK * 2;
  auto* kernel = moe_many_kernel<BM, BN, BK, NB>;
  const int64_t grid = moe_grid(a, BM, BN);
  if (!moe_grid_fits(grid, 512)) return hipErrorInvalidConfiguration;
  const hipError_t e = ensure_lds((const void*)kernel, bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(512), bytes, st, a);
  return hipGetLastError();
}

// By the places an expert has on average: up to 8 a wave's 16 places suffice,
// up to 20 its 32; above, the 64 would only gain where the next kernel leaves
// CUs idle.  us at 8, 16, 24 and 40 places each of
//   64 experts, 2048 x 2048:  16 places 96, 120, 149, 214; 32: 96, 107, 113, 168;
//     64: 101, 109, 116, 128; tiles of 128: 124, 124, 124, 126
//   128 experts, 1024 x 1536: 77, 92, 117, 166; 76, 82, 90, 135; 90, 94, 99, 108;
//     78, 77, 78, 82
// Where tiles of 128 x 256 would leave half the CUs idle, tiles of 128 x 128: us
// with 256 and 128 columns: 1,358 places of 8 experts, 1880 x 992: 30.5 and
// 23.6; 600 of 16, 2048 x 1024: 27.7 and 22.6; 800 of 16, 1024 x 512: 15.8 and
// 12.9.
// Tiles of 128 or of 256 places by the rounds that their workgroups, one a CU,
// make: up to two count whole, and a round of 256 as 7/4 of one of 128.  An
// expert's last tile counts as half a tile.  us at 128, 192, 256 and 512 places:
//   64 experts, 2048 x 2048:  tiles of 128 149, 177, 209, 341; of 256 150, 159, 223, 329
//   128 experts, 1024 x 1536: 124, 149, 180, 307; 116, 133, 175, 275
//   16 experts, 1024 x 2048:  21, 22, 36, 58; 25, 27, 30, 55
// The rule takes the slower side of some rows above: 128 experts of 128 and of 256
// places (124 for 116, 180 for 175), 16 of 512 (58 for 55), and 64 of 24 places
// (124 for 113, the bound of 20).
hipError_t launch_grouped(const GroupedArgs& a, hipStream_t st) {
  const int avg = a.places / a.experts;
  if (avg <= 8) return launch_few<1>(a, st);
  if (avg <= 20) return launch_few<2>(a, st);
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols, per = a.swiglu ? 128 : 256;
  auto wgs = [&](int bm) {
    const int64_t halves = avg < bm ? 2 * (int64_t)a.experts : 2 * (int64_t)a.places / bm + a.experts;
    return halves * ((cols_out + per - 1) / per) / 2;
  };
  auto rounds = [&](int bm) { return wgs(bm) <= 512 ? (wgs(bm) + 255) / 256 * 256 : wgs(bm); };
  if (wgs(128) <= 128) return launch_many<128, 128, 64, 4>(a, st);
  if (7 * rounds(256) < 4 * rounds(128)) return launch_many<256, 256, 32, 4>(a, st);
  return launch_many<128, 256, 64, 3>(a, st);
}

// ---- combination ----------------------------------------------------------

// One token: four columns a thread, the places and weights of eight slots at a
// time (uniform, so they come as scalars) and the eight rows' loads together.
// Bound by the rows' bytes: 2,048 tokens, 8 rows of 2048 f32 each, 143 MB: 24 us,
// 5.9 TB/s (partly from the last product's stores in cache); 200 tokens 2.7 us.
template <typename YT, typename OT, bool VEC>
__global__ void __launch_bounds__(256) moe_combine_kernel(const YT* y, int64_t y_stride, const int32_t* slots,
                                                          const int32_t* end, const float* weights, int top_k,
                                                          int places, int cols, OT* out, int64_t out_stride) {
  typedef YT yvec __attribute__((ext_vector_type(4)));
  typedef OT ovec __attribute__((ext_vector_type(4)));
  constexpr int S = 8;
  const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= cols) return;
  places = min(max(*end, 0), places);  // places behind the groups hold no product
  const int32_t* sl = slots + (int64_t)t * top_k;
  const float* wt = weights + (int64_t)t * top_k;
  moe_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const bool whole = VEC && c + 4 <= cols;
  for (int s0 = 0; s0 < top_k; s0 += S) {
    moe_f32x4 v[S];
    float w[S];
    #pragma unroll
    for (int s = 0; s < S; ++s) {
      v[s] = moe_f32x4{0.f, 0.f, 0.f, 0.f};
      w[s] = 0.f;
      if (s0 + s < top_k) {
        const int i = sl[s0 + s];
        if ((uint32_t)i < (uint32_t)places) {
          w[s] = wt[s0 + s];
          const YT* row = y + (int64_t)i * y_stride + c;
          if (whole) {
            v[s] = __builtin_convertvector(*reinterpret_cast<const yvec*>(row), moe_f32x4);
          } else {
            #pragma unroll
            for (int q = 0; q < 4; ++q)
              if (c + q < cols) v[s][q] = (float)row[q];
          }
        }
      }
    }
    #pragma unroll
    for (int s = 0; s < S; ++s) sum += w[s] * v[s];
  }
  OT* to = out + (int64_t)t * out_stride + c;
  if (whole) {
    *reinterpret_cast<ovec*>(to) = __builtin_convertvector(sum, ovec);
  } else {
    #pragma unroll
    for (int q = 0; q < 4; ++q)
      if (c + q < cols) to[q] = (OT)sum[q];
  }
}

template <typename YT, typename OT>
void launch_combine_types(const void* y, int64_t y_stride, const int32_t* slots, const int32_t* end,
                          const float* weights, int tokens, int top_k, int places, int cols, void* out,
                          int64_t out_stride, hipStream_t st) {
  const dim3 grid((unsigned)tokens, (unsigned)((cols + 1023) / 1024));
  // rows whose four columns can be loaded and stored at once (2,048 tokens: 24.4
  // us, one by one 32.4)
  const bool vec = (uintptr_t)y % (4 * sizeof(YT)) == 0 && (uintptr_t)out % (4 * sizeof(OT)) == 0 && y_stride % 4 == 0 &&
                   out_stride % 4 == 0;
  if (vec)
    hipLaunchKernelGGL((moe_combine_kernel<YT, OT, true>), grid, dim3(256), 0, st, (const YT*)y, y_stride, slots, end,
                       weights, top_k, places, cols, (OT*)out, out_stride);
  else
    hipLaunchKernelGGL((moe_combine_kernel<YT, OT, false>), grid, dim3(256), 0, st, (const YT*)y, y_stride, slots, end,
                       weights, top_k, places, cols, (OT*)out, out_stride);
}

template <typename YT>
void launch_combine(const void* y, int64_t y_stride, const int32_t* slots, const int32_t* end, const float* weights,
                    int tokens, int top_k, int places, int cols, void* out, int out_dtype, int64_t out_stride,
                    hipStream_t st) {
  if (out_dtype == HI_ROCM_DTYPE_BF16)
    launch_combine_types<YT, __bf16>(y, y_stride, slots, end, weights, tokens, top_k, places, cols, out, out_stride, st);
  else
    launch_combine_types<YT, float>(y, y_stride, slots, end, weights, tokens, top_k, places, cols, out, out_stride, st);
}

bool moe_dtype_ok(int d) { return d == HI_ROCM_DTYPE_F32 || d == HI_ROCM_DTYPE_BF16; }
int moe_size(int d) { return d == HI_ROCM_DTYPE_F32 ? 4 : 2; }

}  // namespace
}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_moe_group(const uint32_t* ids, int tokens, int top_k, int experts, int32_t* order, int32_t* slots,
                      int32_t* offsets, void* stream) {
  if (ids == nullptr || order == nullptr || slots == nullptr || offsets == nullptr || tokens <= 0 || top_k <= 0 ||
      experts <= 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_moe_group: invalid arguments");
  if (experts > kMoeMaxExperts || (int64_t)tokens * top_k > kMoeMaxPairs)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_moe_group: more than 2048 experts or 2^22 pairs");
  const int pairs = tokens * top_k;
  const dim3 grid((unsigned)(experts + 1));
  if (pairs <= 8192)
    hipLaunchKernelGGL((moe_group_kernel<4, 4>), grid, dim3(256), 0, (hipStream_t)stream, ids, pairs, experts, order, slots,
                       offsets);
  else
    hipLaunchKernelGGL((moe_group_kernel<16, 8>), grid, dim3(1024), 0, (hipStream_t)stream, ids, pairs, experts, order,
                       slots, offsets);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "moe group launch");
}

int hi_rocm_moe_grouped_product(const void* x, int x_rows, int64_t x_stride, const int32_t* order, int top_k,
                                const int32_t* offsets, int places, int experts, const void* weight, int cols, int k,
                                int swiglu, void* out, int out_dtype, int64_t out_stride, void* stream) {
  if (x == nullptr || offsets == nullptr || weight == nullptr || out == nullptr || x_rows <= 0 || places <= 0 ||
      experts <= 0 || cols <= 0 || k <= 0 || x_stride < k || !moe_dtype_ok(out_dtype) || (order && top_k <= 0) ||
      (!order && x_rows < places) || (swiglu && cols % 2 != 0) || out_stride < (swiglu ? cols / 2 : cols))
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_moe_grouped_product: invalid arguments");
  if ((uintptr_t)out % moe_size(out_dtype) != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_moe_grouped_product: out not aligned to its type");
  if (experts > kMoeMaxExperts || places > kMoeMaxPairs || cols > (1 << 20) || k > (1 << 20))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_moe_grouped_product: more than 2048 experts, 2^22 places, or 2^20 columns or inputs");
  if (k % 8 != 0 || x_stride % 8 != 0 || (uintptr_t)x % 16 != 0 || (uintptr_t)weight % 16 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_moe_grouped_product: needs k a multiple of 8 and rows that start on 16 bytes");
  GroupedArgs a;
  memset(&a, 0, sizeof(a));
  a.x = (const __bf16*)x;
  a.x_stride = x_stride;
  a.order = order;
  a.offsets = offsets;
  a.w = (const __bf16*)weight;
  a.out = out;
  a.out_stride = out_stride;
  a.x_rows = x_rows;
  a.top_k = order ? top_k : 1;
  a.places = places;
  a.experts = experts;
  a.cols = cols;
  a.k = k;
  a.swiglu = swiglu != 0;
  a.out_bf16 = out_dtype == HI_ROCM_DTYPE_BF16;
  a.out_vec = (uintptr_t)out % 16 == 0 && out_stride * moe_size(out_dtype) % 16 == 0;
  const hipError_t e = launch_grouped(a, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_moe_grouped_product: too many places and columns for one launch");
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "moe grouped product launch");
}

int hi_rocm_moe_combine(const void* y, int y_dtype, int64_t y_stride, const int32_t* slots, const int32_t* offsets,
                        int experts, const float* weights, int tokens, int top_k, int cols, void* out, int out_dtype,
                        int64_t out_stride, void* stream) {
  if (y == nullptr || slots == nullptr || offsets == nullptr || weights == nullptr || out == nullptr || tokens <= 0 ||
      top_k <= 0 || experts <= 0 || cols <= 0 || y_stride < cols || out_stride < cols || !moe_dtype_ok(y_dtype) || !moe_dtype_ok(out_dtype))
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_moe_combine: invalid arguments");
  if ((uintptr_t)y % moe_size(y_dtype) != 0 || (uintptr_t)out % moe_size(out_dtype) != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_moe_combine: y or out not aligned to its type");
  if ((int64_t)tokens * top_k > kMoeMaxPairs || experts > kMoeMaxExperts || cols > (1 << 20))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_moe_combine: more than 2048 experts, 2^22 pairs or 2^20 columns");
  const int places = tokens * top_k;
  if (y_dtype == HI_ROCM_DTYPE_BF16)
    launch_combine<__bf16>(y, y_stride, slots, offsets + experts, weights, tokens, top_k, places, cols, out, out_dtype, out_stride,
                           (hipStream_t)stream);
  else
    launch_combine<float>(y, y_stride, slots, offsets + experts, weights, tokens, top_k, places, cols, out, out_dtype, out_stride,
                          (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "moe combine launch");
}

}  // extern "C"
