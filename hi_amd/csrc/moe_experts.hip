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
// consecutive stretches of the pairs, so places follow the pairs' order.
template <int W>
__global__ void __launch_bounds__(64 * W) moe_group_kernel(const uint32_t* ids, int pairs, int experts, int32_t* order,
                                                           int32_t* slots, int32_t* offsets) {
  __shared__ int less[W], equal[W];
  const int e = blockIdx.x, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int per = ((pairs + W - 1) / W + 63) & ~63;
  const int p0 = min(wid * per, pairs), p1 = min(p0 + per, pairs);
  int lt = 0, eq = 0;
  #pragma unroll 4
  for (int p = p0 + lane; p < p1; p += 64) {
    const uint32_t id = ids[p];
    const int v = id < (uint32_t)experts ? (int)id : experts;
    lt += v < e;
    eq += v == e;
  }
  #pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    lt += __shfl_xor(lt, o, 64);
    eq += __shfl_xor(eq, o, 64);
  }
  if (lane == 0) { less[wid] = lt; equal[wid] = eq; }
  __syncthreads();
  int at = 0;
  #pragma unroll
  for (int w = 0; w < W; ++w) at += less[w];
  if (threadIdx.x == 0) offsets[e] = at;  // (offsets[experts]: where the groups end)
  for (int w = 0; w < wid; ++w) at += equal[w];
  if (equal[wid] == 0) return;
  for (int p = p0 + lane; p - lane < p1; p += 64) {
    const uint32_t id = p < p1 ? ids[p] : 0u;
    const int v = id < (uint32_t)experts ? (int)id : experts;
    const bool mine = p < p1 && v == e;
    const uint64_t b = __ballot(mine);
    if (mine) {
      const int i = at + __popcll(b & ((1ull << lane) - 1ull));
      order[i] = p;
      slots[p] = i;
    }
    at += __popcll(b);
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
  int out_vec;  // four columns of out can be stored at once
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
      wk.expert = e0 + l;
      wk.block = local / nt;
      wk.i0 = start + local % nt * BM;
      wk.i1 = min(wk.i0 + BM, start + places);
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

__device__ __forceinline__ float moe_silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

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
// order.
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

// Many places an expert (prefill): BM places times BN weight rows a workgroup,
// k in steps of 64 through two LDS buffers.  A wave multiplies (BM / WM) x (BN
// / WN).  A step's operands are loaded into registers while the step before it
// multiplies, then written to the other buffer; rows of 128 bytes with the
// 16-byte chunk c of row j at c ^ (j & 7), so that 16 rows' reads of one chunk
// meet all banks.
template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) moe_many_kernel(GroupedArgs a) {
  constexpr int T = 64 * WM * WN, XL = BM * 8 / T, WL = BN * 8 / T, MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int STEP = (BM + BN) * 128;
  static_assert(BM * 8 % T == 0 && BN * 8 % T == 0 && NT % 2 == 0, "tile split");
  extern __shared__ __align__(16) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, r = lane & 15, g = lane >> 4;
  const int wm = wid % WM, wn = wid / WM;
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols;
  const int per = a.swiglu ? BN / 2 : BN;
  MoeWork wk;
  if (!moe_work<BM>(a, (cols_out + per - 1) / per, wk)) return;
  const int c0 = wk.block * per;
  // the column behind row j of the tile's weights: with swiglu each wave's
  // rows are half gate, half up
  constexpr int WR = BN / WN;
  auto column = [&](int j) {
    if (!a.swiglu) return min(c0 + j, cols_out - 1);
    const int in = j % WR;
    return min(c0 + j / WR * (WR / 2) + in % (WR / 2), cols_out - 1) + (in >= WR / 2 ? cols_out : 0);
  };
  const int chunk = (tid & 7) ^ ((tid >> 3) & 7);  // (T / 8 rows a round: a multiple of 8)
  const __bf16 *xp[XL], *wp[WL];
  #pragma unroll
  for (int i = 0; i < XL; ++i) xp[i] = moe_row(a, min(wk.i0 + (i * T + tid) / 8, wk.i1 - 1)) + 8 * chunk;
  #pragma unroll
  for (int i = 0; i < WL; ++i)
    wp[i] = a.w + ((int64_t)wk.expert * a.cols + column((i * T + tid) / 8)) * a.k + 8 * chunk;
  moe_bf16x8 xs[XL], ws[WL];
  auto load = [&](int k) {
    const bool in = k + 8 * chunk < a.k;
    const moe_bf16x8 zero = {};
    #pragma unroll
    for (int i = 0; i < XL; ++i) xs[i] = in ? moe_ld(xp[i] + k) : zero;
    #pragma unroll
    for (int i = 0; i < WL; ++i) ws[i] = in ? moe_ld(wp[i] + k) : zero;
  };
  auto stage = [&](int buf) {
    unsigned char* b = lds + buf * STEP;
    #pragma unroll
    for (int i = 0; i < XL; ++i) *reinterpret_cast<moe_bf16x8*>(b + (i * T + tid) * 16) = xs[i];
    #pragma unroll
    for (int i = 0; i < WL; ++i) *reinterpret_cast<moe_bf16x8*>(b + BM * 128 + (i * T + tid) * 16) = ws[i];
  };
  moe_f32x4 acc[MT][NT];
  #pragma unroll
  for (int m = 0; m < MT; ++m)
    #pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = moe_f32x4{0.f, 0.f, 0.f, 0.f};
  const bool busy = wk.i0 + wm * (BM / WM) < wk.i1;  // this wave has places
  const int steps = (a.k + 63) / 64;
  load(0);
  stage(0);
  __syncthreads();
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps) load((s + 1) * 64);
    if (busy) {
      const unsigned char* b = lds + (s & 1) * STEP;
      const unsigned char* xb = b + (wm * (BM / WM) + r) * 128;
      const unsigned char* wb = b + BM * 128 + (wn * WR + r) * 128;
      #pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = ((g + 4 * h) ^ (r & 7)) * 16;
        moe_bf16x8 wf[NT], xf[MT];
        #pragma unroll
        for (int t = 0; t < NT; ++t) wf[t] = *reinterpret_cast<const moe_bf16x8*>(wb + t * 2048 + at);
        #pragma unroll
        for (int m = 0; m < MT; ++m) xf[m] = *reinterpret_cast<const moe_bf16x8*>(xb + m * 2048 + at);
        #pragma unroll
        for (int m = 0; m < MT; ++m)
          #pragma unroll
          for (int t = 0; t < NT; ++t)
            acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[t], xf[m], acc[m][t], 0, 0, 0);
      }
    }
    if (s + 1 < steps) stage((s + 1) & 1);
    __syncthreads();
  }
  if (!busy) return;
  #pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int p = wk.i0 + wm * (BM / WM) + 16 * m + r;
    if (p >= wk.i1) continue;
    if (a.swiglu) {
      #pragma unroll
      for (int t = 0; t < NT / 2; ++t) {
        moe_f32x4 y;
        #pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = moe_silu_mul(acc[m][t][q], acc[m][t + NT / 2][q]);
        const int c = c0 + wn * (WR / 2) + t * 16 + 4 * g;
        if (c < cols_out) moe_store(a, p, c, cols_out, y);
      }
    } else {
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int c = c0 + wn * WR + t * 16 + 4 * g;
        if (c < cols_out) moe_store(a, p, c, cols_out, acc[m][t]);
      }
    }
  }
}

// The largest grid that any split of the places over the experts needs (every
// expert ends in at most one short tile).
int64_t moe_grid(const GroupedArgs& a, int bm, int bn) {
  const int64_t tiles = a.places / bm + std::min(a.experts, a.places);
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols, per = a.swiglu ? bn / 2 : bn;
  return (tiles * ((cols_out + per - 1) / per) + kXcds - 1) / kXcds * kXcds;
}

template <int MT>
hipError_t launch_few(const GroupedArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(moe_few_kernel<MT>, dim3((unsigned)moe_grid(a, 16 * MT, kFewCols)), dim3(64 * kFewWaves), 0, st, a);
  return hipGetLastError();
}

template <int BM, int BN, int WM, int WN>
hipError_t launch_many(const GroupedArgs& a, hipStream_t st) {
  constexpr size_t bytes = 2 * (BM + BN) * 128;
  auto* kernel = moe_many_kernel<BM, BN, WM, WN>;
  const hipError_t e = ensure_lds((const void*)kernel, bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)moe_grid(a, BM, BN)), dim3(64 * WM * WN), bytes, st, a);
  return hipGetLastError();
}

hipError_t launch_grouped(const GroupedArgs& a, hipStream_t st) {
  const int avg = a.places / a.experts;
  if (avg <= 8) return launch_few<1>(a, st);
  if (avg <= 20) return launch_few<2>(a, st);
  if (avg <= 40) return launch_few<4>(a, st);
  if (avg <= 256) return launch_many<128, 256, 2, 4>(a, st);
  return launch_many<256, 256, 2, 4>(a, st);
}

// ---- combination ----------------------------------------------------------

template <typename YT, typename OT>
__global__ void __launch_bounds__(256) moe_combine_kernel(const YT* y, int64_t y_stride, const int32_t* slots,
                                                          const int32_t* end, const float* weights, int top_k,
                                                          int places, int cols, OT* out, int64_t out_stride) {
  const int t = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;
  if (c >= cols) return;
  places = min(max(*end, 0), places);  // places behind the groups hold no product
  float sum = 0.f;
  for (int s = 0; s < top_k; ++s) {
    const int i = slots[(int64_t)t * top_k + s];
    if ((uint32_t)i < (uint32_t)places) sum += weights[(int64_t)t * top_k + s] * (float)y[(int64_t)i * y_stride + c];
  }
  out[(int64_t)t * out_stride + c] = (OT)sum;
}

template <typename YT>
void launch_combine(const void* y, int64_t y_stride, const int32_t* slots, const int32_t* end, const float* weights,
                    int tokens, int top_k, int places, int cols, void* out, int out_dtype, int64_t out_stride,
                    hipStream_t st) {
  const dim3 grid((unsigned)tokens, (unsigned)((cols + 255) / 256));
  if (out_dtype == HI_ROCM_DTYPE_BF16)
    hipLaunchKernelGGL((moe_combine_kernel<YT, __bf16>), grid, dim3(256), 0, st, (const YT*)y, y_stride, slots, end,
                       weights, top_k, places, cols, (__bf16*)out, out_stride);
  else
    hipLaunchKernelGGL((moe_combine_kernel<YT, float>), grid, dim3(256), 0, st, (const YT*)y, y_stride, slots, end,
                       weights, top_k, places, cols, (float*)out, out_stride);
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
  if (pairs <= 4096)
    hipLaunchKernelGGL(moe_group_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, ids, pairs, experts, order, slots,
                       offsets);
  else
    hipLaunchKernelGGL(moe_group_kernel<16>, grid, dim3(1024), 0, (hipStream_t)stream, ids, pairs, experts, order,
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
  a.out_vec = (uintptr_t)out % (4 * moe_size(out_dtype)) == 0 && out_stride % 4 == 0;
  if (moe_grid(a, 16, 32) > INT32_MAX)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_moe_grouped_product: too many places and columns");
  const hipError_t e = launch_grouped(a, (hipStream_t)stream);
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
