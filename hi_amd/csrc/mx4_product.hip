// Products with microscaled 4-bit weights (mx4.h): linear layers and the
// experts behind the MoE router (moe_experts.hip has the same in bf16, and the
// grouping and combination around both).
//
//     y[i][c] = sum_k Q(x[row(i)])[k] * w[e][c][k] (+ bias[c])
//
// Both operands go to the matrix cores as they lie in memory, 4 bits a value
// with a scale for 32: four times the bf16 rate, and no unpacking.  Q rounds x to
// the same format: beforehand ("rows"), or, for few rows, in registers as it is
// loaded, since a block is one lane's.  Products of two codes are multiples of
// 1/4 up to 36, so a block's sum is exact; the sums over blocks are f32.
//
// MFMA 16x16x128: A row r and B column r in lane 16 g + r, block g; D rows 4 g ..
// + 3 of column r.  Weights are A and places B: a lane ends with four
// neighbouring columns of one place.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "hi_rocm.h"
#include "moe_work.h"
#include "mx4.h"
#include "sampler_internal.h"

namespace hi_rocm {
hipError_t ensure_lds(const void* fn, size_t bytes);  // sampler_chunked.hip
hipError_t mx4_make_rows(const void* x, int dtype, int64_t rows, int k, int64_t x_stride, void* out,
                         hipStream_t st);  // mx4_quantize.hip

namespace {

struct Mx4Args {
  const uint8_t* x;          // bf16 rows, or codes
  int64_t x_stride;          // bytes
  const uint8_t* x_scales;   // with codes
  int64_t x_scale_stride;
  const int32_t* order;      // or null: place i's row is i
  const int32_t* offsets;    // [experts + 1], or null: one expert, all places
  const uint8_t* w;          // packed
  const uint8_t* w_scales;
  const float* bias;         // or null
  void* out;                 // [places][out_stride], or codes
  int64_t out_stride;        // values, or bytes of codes
  uint8_t* out_scales;       // with codes
  int64_t out_scale_stride;
  int x_rows, top_k, places, experts, cols, k, swiglu, out_dtype;
  int tiles, steps, quads;   // of an expert's packed weight
  int out_vec;               // rows of out start on 16 bytes
};

// This workgroup's tile of BM places and block of columns.
template <int BM>
__device__ __forceinline__ bool mx4_work(const Mx4Args& a, int blocks, MoeWork& wk) {
  if (a.offsets != nullptr) return moe_work<BM>(a, blocks, wk);
  const int nt = (a.places + BM - 1) / BM;
  const int64_t total = (int64_t)nt * blocks, per = (total + kXcds - 1) / kXcds;
  const int64_t slot = blockIdx.x / kXcds, w = blockIdx.x % kXcds * per + slot;
  if (slot >= per || w >= total) return false;
  wk.expert = 0;
  wk.block = (int)(w / nt);
  wk.i0 = (int)(w % nt) * BM;
  wk.i1 = min(wk.i0 + BM, a.places);
  return true;
}

// The row of x behind place i.
__device__ __forceinline__ int mx4_row(const Mx4Args& a, int i) {
  const int row = a.order ? a.order[i] / a.top_k : i;
  return min(max(row, 0), a.x_rows - 1);
}

// Four columns c .. c + 3 of place p.
__device__ __forceinline__ void mx4_store(const Mx4Args& a, int p, int c, int cols_out, const mx4_f32x4& y) {
  const int64_t at = (int64_t)p * a.out_stride + c;
  if (c + 4 <= cols_out && a.out_vec) {
    if (a.out_dtype == HI_ROCM_DTYPE_BF16) {
      typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<bf16x4*>((__bf16*)a.out + at) = __builtin_convertvector(y, bf16x4);
    } else {
      *reinterpret_cast<mx4_f32x4*>((float*)a.out + at) = y;
    }
    return;
  }
  #pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (c + q >= cols_out) break;
    if (a.out_dtype == HI_ROCM_DTYPE_BF16) ((__bf16*)a.out)[at + q] = (__bf16)y[q];
    else ((float*)a.out)[at + q] = y[q];
  }
}

// A block of 32 columns (from c, a multiple of 32) of place p as codes: lane 16
// g + r has columns 4 g .. + 3 of both halves.  All lanes of a place together.
__device__ __forceinline__ void mx4_store_codes(const Mx4Args& a, int p, bool in, int c, int g, const mx4_f32x4& lo,
                                                const mx4_f32x4& hi) {
  const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  uint32_t m = 0u;
  #pragma unroll
  for (int q = 0; q < 8; ++q) m = max(m, __float_as_uint(v[q]) & 0x7fffffffu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  const uint32_t s = mx4_scale_of(m >> 23), codes = mx4_codes(v, s);
  if (!in) return;
  uint8_t* to = (uint8_t*)a.out + (int64_t)p * a.out_stride + c / 2 + 2 * g;
  *reinterpret_cast<uint16_t*>(to) = (uint16_t)codes;
  *reinterpret_cast<uint16_t*>(to + 8) = (uint16_t)(codes >> 16);
  if (g == 0) a.out_scales[(int64_t)p * a.out_scale_stride + mx4_scale_at(c / kMx4Block)] = (uint8_t)s;
}

// Few places (decode): the weights are what is read.  The workgroup's waves
// split k; each streams 16 NT columns' blocks straight into registers, two steps
// ahead, and multiplies them with up to 16 MT places.  The waves' sums are added
// in wave order.
template <int MT, int NT, int W, bool CODES>
__global__ void __launch_bounds__(64 * W) mx4_few_kernel(Mx4Args a) {
  __shared__ mx4_f32x4 part[W - 1][MT * NT][64];
  constexpr int COLS = 16 * NT;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols;
  const int per = a.swiglu ? COLS / 2 : COLS;
  MoeWork wk;
  if (!mx4_work<16 * MT>(a, (cols_out + per - 1) / per, wk)) return;
  const int c0 = wk.block * per;
  const uint8_t* wp[NT];
  const uint8_t* sp[NT];
  #pragma unroll
  for (int t = 0; t < NT; ++t) {  // with swiglu tiles of gate columns, then the same of up columns
    int tile = c0 / 16 + t;
    if (a.swiglu) tile = c0 / 16 + t % (NT / 2) + (t >= NT / 2 ? cols_out / 16 : 0);
    const int64_t at = (int64_t)wk.expert * a.tiles + min(tile, a.tiles - 1);
    wp[t] = a.w + at * a.steps * 1024 + lane * 16;
    sp[t] = a.w_scales + at * a.quads * 256 + lane * 4;
  }
  const uint8_t* xp[MT];
  const uint8_t* xs[MT];
  #pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t row = mx4_row(a, min(wk.i0 + 16 * m + r, wk.i1 - 1));
    xp[m] = a.x + row * a.x_stride + g * (CODES ? 16 : 64);
    xs[m] = CODES ? a.x_scales + row * a.x_scale_stride + 4 * g : nullptr;
  }
  mx4_f32x4 acc[MT][NT];
  #pragma unroll
  for (int m = 0; m < MT; ++m)
    #pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = mx4_f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int XL = CODES ? 1 : 4;
  mx4_i32x4 wv[2][NT];
  int ws[2][NT];
  uint4 xv[2][MT][XL];
  uint32_t xsc[2][MT];
  auto load = [&](int slot, int step) {
    const bool in = step * kMx4Step + g * kMx4Block < a.k;
    #pragma unroll
    for (int t = 0; t < NT; ++t) {
      wv[slot][t] = *reinterpret_cast<const mx4_i32x4*>(wp[t] + (int64_t)step * 1024);
      ws[slot][t] = sp[t][(step >> 2) * 256 + (step & 3)];
    }
    #pragma unroll
    for (int m = 0; m < MT; ++m) {
      #pragma unroll
      for (int i = 0; i < XL; ++i)
        xv[slot][m][i] = in ? reinterpret_cast<const uint4*>(xp[m] + (int64_t)step * (CODES ? 64 : 256))[i]
                            : uint4{0u, 0u, 0u, 0u};
      xsc[slot][m] = CODES ? (in ? xs[m][(step >> 2) * 16 + (step & 3)] : 127u) : 0u;
    }
  };
  auto multiply = [&](int slot) {
    #pragma unroll
    for (int m = 0; m < MT; ++m) {
      mx4_i32x4 xc;
      uint32_t s;
      if constexpr (CODES) {
        xc = __builtin_bit_cast(mx4_i32x4, xv[slot][m][0]);
        s = xsc[slot][m];
      } else {
        s = mx4_scale_of(mx4_field(mx4_max_pair(mx4_max_pair(mx4_max_of(xv[slot][m][0]), mx4_max_of(xv[slot][m][1])),
                                                mx4_max_pair(mx4_max_of(xv[slot][m][2]), mx4_max_of(xv[slot][m][3])))));
        #pragma unroll
        for (int i = 0; i < 4; ++i) xc[i] = (int)mx4_codes(xv[slot][m][i], s);
      }
      #pragma unroll
      for (int t = 0; t < NT; ++t) acc[m][t] = mx4_mfma<0, 0>(wv[slot][t], xc, acc[m][t], ws[slot][t], (int)s);
    }
  };
  const int share = (a.steps + W - 1) / W;
  const int b0 = min(wid * share, a.steps), b1 = min(b0 + share, a.steps);
  if (b0 < b1) load(0, b0);
  if (b0 + 1 < b1) load(1, b0 + 1);
  for (int b = b0; b < b1; b += 2) {
    multiply(0);
    if (b + 2 < b1) load(0, b + 2);
    if (b + 1 < b1) {
      multiply(1);
      if (b + 3 < b1) load(1, b + 3);
    }
  }
  if (wid > 0) {
    #pragma unroll
    for (int m = 0; m < MT; ++m)
      #pragma unroll
      for (int t = 0; t < NT; ++t) part[wid - 1][m * NT + t][lane] = acc[m][t];
  }
  __syncthreads();
  if (wid > 0) return;
  #pragma unroll
  for (int m = 0; m < MT; ++m) {
    #pragma unroll
    for (int t = 0; t < NT; ++t)
      #pragma unroll
      for (int w = 0; w < W - 1; ++w) acc[m][t] += part[w][m * NT + t][lane];
    const int p = wk.i0 + 16 * m + r;
    const bool in = p < wk.i1;
    if (a.swiglu) {
      if constexpr (NT >= 2) {
        #pragma unroll
        for (int t = 0; t < NT / 2; ++t)
          #pragma unroll
          for (int q = 0; q < 4; ++q) acc[m][t][q] = moe_silu_mul(acc[m][t][q], acc[m][t + NT / 2][q]);
        if constexpr (NT == 4) {
          if (a.out_dtype == HI_ROCM_DTYPE_MX4) {
            mx4_store_codes(a, p, in, c0, g, acc[m][0], acc[m][1]);
            continue;
          }
        }
        #pragma unroll
        for (int t = 0; t < NT / 2; ++t)
          if (in && c0 + t * 16 + 4 * g < cols_out) mx4_store(a, p, c0 + t * 16 + 4 * g, cols_out, acc[m][t]);
      }
    } else {
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int c = c0 + t * 16 + 4 * g;
        if (!in || c >= cols_out) continue;
        if (a.bias != nullptr) {
          #pragma unroll
          for (int q = 0; q < 4; ++q) acc[m][t][q] += c + q < cols_out ? a.bias[c + q] : 0.f;
        }
        mx4_store(a, p, c, cols_out, acc[m][t]);
      }
    }
  }
}

int64_t mx4_grid(const Mx4Args& a, int bm, int bn) {
  if (a.offsets != nullptr) return moe_grid(a, bm, bn);
  const int64_t nt = ((int64_t)a.places + bm - 1) / bm;
  return (nt * (((int64_t)a.cols + bn - 1) / bn) + kXcds - 1) / kXcds * kXcds;
}

template <int MT, int NT, int W, bool CODES>
hipError_t launch_few(const Mx4Args& a, hipStream_t st) {
  const int64_t grid = mx4_grid(a, 16 * MT, 16 * NT);
  if (!moe_grid_fits(grid, 64 * W)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((mx4_few_kernel<MT, NT, W, CODES>), dim3((unsigned)grid), dim3(64 * W), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_product(const Mx4Args& a, bool codes, hipStream_t st) {
  if (!codes) return launch_few<1, 4, 4, false>(a, st);
  return launch_few<4, 4, 4, true>(a, st);
}

bool mx4_float(int d) { return d == HI_ROCM_DTYPE_F32 || d == HI_ROCM_DTYPE_BF16; }
int mx4_size(int d) { return d == HI_ROCM_DTYPE_F32 ? 4 : 2; }

// x as a product reads it: "rows" given, bf16 rows as they are when they are
// few, or "rows" made of them in the workspace.
int mx4_take_x(const char* name, Mx4Args& a, const void* x, int x_dtype, int64_t x_rows, int64_t x_stride, void* ws,
               size_t ws_bytes, hipStream_t st, bool& codes) {
  const Mx4Rows L = mx4_rows_layout(x_rows, a.k);
  a.x_rows = (int)x_rows;
  codes = x_dtype == HI_ROCM_DTYPE_MX4 || x_rows > HI_ROCM_MX4_FEW_ROWS;
  if (!codes) {
    a.x = (const uint8_t*)x;
    a.x_stride = x_stride * 2;
    return HI_ROCM_OK;
  }
  if (x_dtype != HI_ROCM_DTYPE_MX4) {
    const hipError_t e = mx4_make_rows(x, x_dtype, x_rows, a.k, x_stride, ws, st);
    if (e != hipSuccess) return api_hip_fail(e, name);
    x = ws;
  }
  a.x = (const uint8_t*)x;
  a.x_stride = L.code_stride;
  a.x_scales = (const uint8_t*)x + L.scales;
  a.x_scale_stride = L.scale_stride;
  return HI_ROCM_OK;
}

int mx4_fail(int status, const char* name, const char* what) {
  char text[256];
  snprintf(text, sizeof(text), "%s: %s", name, what);
  return api_fail(status, text);
}

// What both products check of x and the weight.
int mx4_check(const char* name, const void* x, int x_dtype, int64_t x_rows, int64_t x_stride, const void* packed,
              size_t packed_bytes, int experts, int n, int k, const void* ws, size_t ws_bytes) {
  if (x == nullptr || packed == nullptr || x_rows <= 0 || n <= 0 || k <= 0 || experts <= 0 ||
      (x_dtype != HI_ROCM_DTYPE_BF16 && x_dtype != HI_ROCM_DTYPE_MX4) || (x_dtype == HI_ROCM_DTYPE_BF16 && x_stride < k))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "invalid arguments");
  if (!mx4_weight_fits(experts, n, k) || x_rows > HI_ROCM_MX4_MAX_ROWS)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name,
                    "needs k a multiple of 32 up to 2^24, at most 2048 experts, 2^24 outputs, 2^35 weights, 2^22 rows");
  if ((uintptr_t)packed % 16 != 0 || packed_bytes < mx4_packed_layout(experts, n, k).total)
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "packed not on 16 bytes, or too small (hi_rocm_mx4_packed_bytes)");
  if ((uintptr_t)x % 16 != 0 || (x_dtype == HI_ROCM_DTYPE_BF16 && x_stride % 8 != 0))
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "needs rows that start on 16 bytes");
  if (x_dtype == HI_ROCM_DTYPE_BF16 && x_rows > HI_ROCM_MX4_FEW_ROWS &&
      (ws == nullptr || (uintptr_t)ws % 16 != 0 || ws_bytes < mx4_rows_layout(x_rows, k).total))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "workspace not on 16 bytes, or too small (hi_rocm_mx4_rows_bytes)");
  return HI_ROCM_OK;
}

void mx4_take_weight(Mx4Args& a, const void* packed, int experts, int n, int k) {
  const Mx4Packed L = mx4_packed_layout(experts, n, k);
  a.w = (const uint8_t*)packed;
  a.w_scales = (const uint8_t*)packed + L.scales;
  a.experts = experts;
  a.cols = n;
  a.k = k;
  a.tiles = (int)L.tiles;
  a.steps = (int)L.steps;
  a.quads = (int)L.quads;
}

}  // namespace
}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_mx4_linear(const void* x, int x_dtype, int rows, int64_t x_stride, const void* packed, size_t packed_bytes,
                       int n, int k, const float* bias, void* out, int out_dtype, int64_t out_stride, void* workspace,
                       size_t workspace_bytes, void* stream) {
  const char* name = "hi_rocm_mx4_linear";
  const int bad = mx4_check(name, x, x_dtype, rows, x_stride, packed, packed_bytes, 1, n, k, workspace, workspace_bytes);
  if (bad != HI_ROCM_OK) return bad;
  if (out == nullptr || !mx4_float(out_dtype) || out_stride < n || (uintptr_t)out % mx4_size(out_dtype) != 0 ||
      (uintptr_t)bias % 4 != 0)
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "invalid arguments");
  Mx4Args a;
  memset(&a, 0, sizeof(a));
  mx4_take_weight(a, packed, 1, n, k);
  a.bias = bias;
  a.out = out;
  a.out_stride = out_stride;
  a.out_dtype = out_dtype;
  a.out_vec = (uintptr_t)out % 16 == 0 && out_stride * mx4_size(out_dtype) % 16 == 0;
  a.places = rows;
  a.top_k = 1;
  bool codes;
  const int rc = mx4_take_x(name, a, x, x_dtype, rows, x_stride, workspace, workspace_bytes, (hipStream_t)stream, codes);
  if (rc != HI_ROCM_OK) return rc;
  const hipError_t e = launch_product(a, codes, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "too many rows and outputs for one launch");
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 linear launch");
}

int hi_rocm_mx4_grouped_product(const void* x, int x_dtype, int x_rows, int64_t x_stride, const int32_t* order,
                                int top_k, const int32_t* offsets, int places, int experts, const void* packed,
                                size_t packed_bytes, int cols, int k, int swiglu, void* out, int out_dtype,
                                int64_t out_stride, size_t out_bytes, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const char* name = "hi_rocm_mx4_grouped_product";
  const int bad =
      mx4_check(name, x, x_dtype, x_rows, x_stride, packed, packed_bytes, experts, cols, k, workspace, workspace_bytes);
  if (bad != HI_ROCM_OK) return bad;
  const int wide = swiglu ? cols / 2 : cols;
  const bool to_rows = out_dtype == HI_ROCM_DTYPE_MX4;
  if (offsets == nullptr || out == nullptr || places <= 0 || (order && top_k <= 0) || (!order && x_rows < places) ||
      (!to_rows && (!mx4_float(out_dtype) || out_stride < wide || (uintptr_t)out % mx4_size(out_dtype) != 0)) ||
      (to_rows && !swiglu))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "invalid arguments");
  if (swiglu && cols % 64 != 0)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "needs gate and up halves of a multiple of 32 columns");
  if (places > HI_ROCM_MX4_MAX_ROWS)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "more than 2^22 places");
  if (to_rows && ((uintptr_t)out % 16 != 0 || out_bytes < mx4_rows_layout(places, wide).total))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "out not on 16 bytes, or too small (hi_rocm_mx4_rows_bytes)");
  Mx4Args a;
  memset(&a, 0, sizeof(a));
  mx4_take_weight(a, packed, experts, cols, k);
  a.order = order;
  a.offsets = offsets;
  a.out = out;
  a.out_stride = out_stride;
  a.out_dtype = out_dtype;
  if (to_rows) {
    const Mx4Rows L = mx4_rows_layout(places, wide);
    a.out_stride = L.code_stride;
    a.out_scales = (uint8_t*)out + L.scales;
    a.out_scale_stride = L.scale_stride;
  } else {
    a.out_vec = (uintptr_t)out % 16 == 0 && out_stride * mx4_size(out_dtype) % 16 == 0;
  }
  a.places = places;
  a.top_k = order ? top_k : 1;
  a.swiglu = swiglu != 0;
  bool codes;
  const int rc =
      mx4_take_x(name, a, x, x_dtype, x_rows, x_stride, workspace, workspace_bytes, (hipStream_t)stream, codes);
  if (rc != HI_ROCM_OK) return rc;
  const hipError_t e = launch_product(a, codes, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "too many places and columns for one launch");
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 grouped product launch");
}

}  // extern "C"
