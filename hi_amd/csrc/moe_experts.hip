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
};

// Tile t of the groups cut into tiles of BM places: its expert and its first
// place and end (false: there are fewer tiles).  Every wave finds it from the
// offsets, 64 experts at a time.
template <int BM>
__device__ __forceinline__ bool moe_tile(const GroupedArgs& a, int t, int& expert, int& i0, int& i1) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    const int e = e0 + lane;
    int s = 0, n = 0;
    if (e < a.experts) {
      s = min(max(a.offsets[e], 0), a.places);
      n = max(min(a.offsets[e + 1], a.places) - s, 0);
    }
    const int tiles = (n + BM - 1) / BM;
    const int incl = (int)wave_incl_scan_u32((uint32_t)tiles) + before;
    const uint64_t hit = __ballot(incl > t && incl - tiles <= t);
    if (hit != 0ull) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int first = __shfl(incl - tiles, l, 64);
      const int start = __shfl(s, l, 64), count = __shfl(n, l, 64);
      expert = e0 + l;
      i0 = start + (t - first) * BM;
      i1 = min(i0 + BM, start + count);
      return true;
    }
    before = __shfl(incl, 63, 64);
  }
  return false;
}

__device__ __forceinline__ float moe_silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// One wave: 16 places times 64 columns (with swiglu 32 gate columns and the
// 32 up columns beside them), straight from memory.
__global__ void __launch_bounds__(256) moe_grouped_kernel(GroupedArgs a) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  int e, i0, i1;
  if (!moe_tile<16>(a, blockIdx.x, e, i0, i1)) return;
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols;
  const int per = a.swiglu ? 32 : 64;
  const int c0 = (blockIdx.y * 4 + wid) * per;
  if (c0 >= cols_out) return;
  const int i = min(i0 + r, i1 - 1);
  int row = a.order ? a.order[i] / a.top_k : i;
  row = min(max(row, 0), a.x_rows - 1);
  const __bf16* xr = a.x + (int64_t)row * a.x_stride;
  const __bf16* wr[4];
  #pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int c = a.swiglu ? min(c0 + (t & 1) * 16 + r, cols_out - 1) + (t >> 1) * cols_out
                           : min(c0 + t * 16 + r, cols_out - 1);
    wr[t] = a.w + ((int64_t)e * a.cols + c) * a.k;
  }
  moe_f32x4 acc[4];
  #pragma unroll
  for (int t = 0; t < 4; ++t) acc[t] = moe_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < a.k; k0 += 32) {
    const int k = k0 + 8 * g;
    moe_bf16x8 xa = {};
    if (k < a.k) xa = *reinterpret_cast<const moe_bf16x8*>(xr + k);
    #pragma unroll
    for (int t = 0; t < 4; ++t) {
      moe_bf16x8 b = {};
      if (k < a.k) b = *reinterpret_cast<const moe_bf16x8*>(wr[t] + k);
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa, b, acc[t], 0, 0, 0);
    }
  }
  #pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (a.swiglu && t >= 2) break;
    const int c = c0 + t * 16 + r;
    if (c >= cols_out) continue;
    #pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int p = i0 + 4 * g + q;
      if (p >= i1) continue;
      const float y = a.swiglu ? moe_silu_mul(acc[t][q], acc[t + 2 < 4 ? t + 2 : 3][q]) : acc[t][q];
      if (a.out_bf16) ((__bf16*)a.out)[(int64_t)p * a.out_stride + c] = (__bf16)y;
      else ((float*)a.out)[(int64_t)p * a.out_stride + c] = y;
    }
  }
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
  // every group ends in at most one short tile
  const int64_t tiles = places / 16 + std::min(experts, places);
  const int cols_out = swiglu ? cols / 2 : cols, per = swiglu ? 128 : 256;
  hipLaunchKernelGGL(moe_grouped_kernel, dim3((unsigned)tiles, (unsigned)((cols_out + per - 1) / per)), dim3(256), 0,
                     (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
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
