// Microscaled 4-bit floating point (mx4.h): rounding of rows to it, back to
// values, and the layouts that the products (mx4_product.hip) read.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hi_rocm.h"
#include "moe_group.h"
#include "mx4.h"
#include "sampler_internal.h"
#include "wave_ops.h"

namespace hi_rocm {
namespace {

constexpr int kMx4Units = 4;  // units a wave has in flight

// A unit is 512 values of a row, eight a lane: four lanes hold a block.
struct Mx4Unit {
  int64_t row;
  int quad, at;  // at: this lane's first value
  bool in;
};
__device__ __forceinline__ Mx4Unit mx4_unit(uint32_t u, uint32_t units, uint32_t quads, int k, int lane) {
  Mx4Unit x;
  const uint32_t row = u / quads;  // (units fit 28 bits: mx4_rows_fit)
  x.row = row;
  x.quad = (int)(u - row * quads);
  x.at = x.quad * kMx4Quad + lane * 8;
  x.in = u < units && x.at < k;
  return x;
}

// Rounds rows of x.  ROWS: scales in the order of "rows", else [rows][k / 32].
// Bound by the bytes: 2 or 4 read and 0.53 written a value; 16,384 x 4,096 f32 57 to 63
// us, 5.4 to 4.8 TB/s, bf16 32 (5.3).  A unit is one row's, so a row that ends inside one
// leaves lanes idle: 65,536 x 544 f32 31 us (5.2 TB/s), 262,144 x 128 32 (4.8; bf16 24,
// 3.5), 2,097,152 x 32 191 (1.6).
template <typename T>
struct Mx4Quantize {
  const T* x;
  int64_t x_stride;
  uint32_t units;
  int quads, k;
  uint8_t* codes;
  int64_t code_stride;
  uint8_t* scales;
  int64_t scale_stride;
};
template <typename T, bool ROWS>
__device__ __forceinline__ void mx4_quantize_units(const Mx4Quantize<T>& q, uint32_t u0) {
  const T* x = q.x;
  const int64_t x_stride = q.x_stride, code_stride = q.code_stride, scale_stride = q.scale_stride;
  const uint32_t units = q.units;
  const int quads = q.quads, k = q.k;
  uint8_t *codes = q.codes, *scales = q.scales;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int L = F32 ? 2 : 1;
  const int lane = threadIdx.x & 63;
  uint4 v[kMx4Units][L];
  #pragma unroll
  for (int i = 0; i < kMx4Units; ++i) {
    const Mx4Unit un = mx4_unit(u0 + i, units, quads, k, lane);
    #pragma unroll
    for (int j = 0; j < L; ++j)
      v[i][j] = un.in ? reinterpret_cast<const uint4*>(x + un.row * x_stride + un.at)[j] : uint4{0u, 0u, 0u, 0u};
  }
  #pragma unroll
  for (int i = 0; i < kMx4Units; ++i) {
    const Mx4Unit un = mx4_unit(u0 + i, units, quads, k, lane);
    uint32_t a;
    float f[8];
    if constexpr (F32) {
      const uint32_t w[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
      a = 0u;
      #pragma unroll
      for (int q = 0; q < 8; ++q) {
        f[q] = __uint_as_float(w[q]);
        a = max(a, w[q] & 0x7fffffffu);
      }
    } else {
      a = mx4_max_of(v[i][0]);
      a = max(a >> 16, a & 0xffffu);
    }
    a = max(a, dpp32<kDppXor1>(a, a));
    a = max(a, dpp32<kDppXor2>(a, a));
    const uint32_t s = mx4_scale_of(a >> (F32 ? 23 : 7));
    uint32_t c;
    if constexpr (F32) c = mx4_codes(f, s);
    else c = mx4_codes(v[i][0], s);
    if (un.in) {
      *reinterpret_cast<uint32_t*>(codes + un.row * code_stride + un.at / 2) = c;
    }
    // (scales behind k: the unit's row is one of x's, its values are not)
    if ((lane & 3) == 0 && (un.in || (ROWS && u0 + i < units))) {
      const int b = un.at / kMx4Block;
      scales[un.row * scale_stride + (ROWS ? mx4_scale_at(b) : b)] = (uint8_t)(un.in ? s : 127u);
    }
  }
}

template <typename T, bool ROWS>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(Mx4Quantize<T> q) {
  mx4_quantize_units<T, ROWS>(q, (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kMx4Units);
}

// The expert layer's first launch: workgroups 0 .. experts group the pairs, the
// others round the tokens' rows, which need no group (200 tokens of 1440: 3.8 us,
// in two launches 3.2 and 3.5).
template <int W, int L>
__global__ void __launch_bounds__(64 * W) mx4_prepare_kernel(const uint32_t* ids, int pairs, int experts, int32_t* order,
                                                             int32_t* slots, int32_t* offsets, Mx4Quantize<__bf16> q) {
  const int b = (int)blockIdx.x - (experts + 1);
  if (b < 0) moe_group_pairs<W, L>(ids, pairs, experts, order, slots, offsets, blockIdx.x);
  else mx4_quantize_units<__bf16, true>(q, ((uint32_t)b * W + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kMx4Units);
}

// Back to values, in f32 or bf16 (exact but for bf16's range: code times power
// of two has two bits).  16,384 x 4,096 to bf16: 32 us (5.3 TB/s) into one place again
// and again, 39 (4.4) into three in turn.  Rows that end inside a unit: 65,536 x 544 32 us
// (2.8), 262,144 x 128 56 (1.5).
template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, uint32_t units,
                                                             int quads, int k, T* out, int64_t out_stride) {
  const int lane = threadIdx.x & 63;
  const uint32_t u0 = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kMx4Units;
  uint32_t c[kMx4Units], s[kMx4Units];
  #pragma unroll
  for (int i = 0; i < kMx4Units; ++i) {
    const Mx4Unit un = mx4_unit(u0 + i, units, quads, k, lane);
    c[i] = un.in ? *reinterpret_cast<const uint32_t*>(codes + un.row * (k / 2) + un.at / 2) : 0u;
    s[i] = un.in ? scales[un.row * (k / kMx4Block) + un.at / kMx4Block] : 127u;
  }
  #pragma unroll
  for (int i = 0; i < kMx4Units; ++i) {
    const Mx4Unit un = mx4_unit(u0 + i, units, quads, k, lane);
    if (!un.in) continue;
    // 2^(s - 127): the subnormal 2^-127 for 0
    const float scale = s[i] == 255u ? __builtin_nanf("") : __uint_as_float(s[i] == 0u ? 1u << 22 : s[i] << 23);
    typedef T vec __attribute__((ext_vector_type(8)));
    vec y;
    #pragma unroll
    for (int q = 0; q < 8; ++q) {
      // half units: 0 1 2 3 4 6 8 12
      const uint32_t n = c[i] >> (4 * q), m = n & 7u;
      const uint32_t h = m < 4u ? m : (2u + (m & 1u)) << ((m >> 1) - 1u);
      const float f = (float)h * 0.5f * scale;
      y[q] = (T)((n & 8u) ? -f : f);
    }
    T* to = out + un.row * out_stride + un.at;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<vec*>(to) = y;
    } else {
      reinterpret_cast<mx4_f32x4*>(to)[0] = __builtin_shufflevector(y, y, 0, 1, 2, 3);
      reinterpret_cast<mx4_f32x4*>(to)[1] = __builtin_shufflevector(y, y, 4, 5, 6, 7);
    }
  }
}

// Weights into "packed" order, once: 16 bytes of codes a thread.
__global__ void __launch_bounds__(256) mx4_pack_kernel(const uint8_t* codes, int n, int k, int64_t tiles, int64_t steps,
                                                       int64_t count, uint4* out) {
  const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (w >= count) return;
  const int lane = (int)(w & 63);
  const int64_t block = w >> 6, step = block % steps, tile = block / steps % tiles, e = block / steps / tiles;
  const int64_t row = tile * 16 + (lane & 15), at = step * kMx4Step + (lane >> 4) * kMx4Block;
  uint4 v = {0u, 0u, 0u, 0u};
  if (row < n && at < k) v = *reinterpret_cast<const uint4*>(codes + (e * n + row) * (k / 2) + at / 2);
  out[w] = v;
}
__global__ void __launch_bounds__(256) mx4_pack_scales_kernel(const uint8_t* scales, int n, int blocks, int64_t tiles,
                                                              int64_t quads, int64_t count, uint32_t* out) {
  const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (w >= count) return;
  const int r = (int)(w >> 2) & 15, g = (int)(w & 3);
  const int64_t block = w >> 6, quad = block % quads, tile = block / quads % tiles, e = block / quads / tiles;
  const int64_t row = tile * 16 + r;
  uint32_t v = 0u;
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t b = quad * 16 + j * 4 + g;
    const uint32_t s = row < n && b < blocks ? scales[(e * n + row) * blocks + b] : 127u;
    v |= s << (8 * j);
  }
  out[w] = v;
}

bool mx4_float(int dtype) { return dtype == HI_ROCM_DTYPE_F32 || dtype == HI_ROCM_DTYPE_BF16; }
int mx4_size(int dtype) { return dtype == HI_ROCM_DTYPE_F32 ? 4 : 2; }

template <bool ROWS>
hipError_t launch_quantize(const void* x, int dtype, int64_t rows, int k, int64_t x_stride, uint8_t* codes,
                           int64_t code_stride, uint8_t* scales, int64_t scale_stride, hipStream_t st) {
  const int quads = (k + kMx4Quad - 1) / kMx4Quad;
  const uint32_t units = (uint32_t)(rows * quads);
  const dim3 grid((unsigned)((units + 4 * kMx4Units - 1) / (4 * kMx4Units)));
  if (dtype == HI_ROCM_DTYPE_F32)
    hipLaunchKernelGGL((mx4_quantize_kernel<float, ROWS>), grid, dim3(256), 0, st,
                       Mx4Quantize<float>{(const float*)x, x_stride, units, quads, k, codes, code_stride, scales, scale_stride});
  else
    hipLaunchKernelGGL((mx4_quantize_kernel<__bf16, ROWS>), grid, dim3(256), 0, st,
                       Mx4Quantize<__bf16>{(const __bf16*)x, x_stride, units, quads, k, codes, code_stride, scales, scale_stride});
  return hipGetLastError();
}

// (rows in one launch of 256 threads for 16 units)
bool mx4_rows_fit(int64_t rows, int k) {
  const int64_t quads = ((int64_t)k + kMx4Quad - 1) / kMx4Quad;
  return rows <= INT64_MAX / 65536 / quads && (rows * quads + 15) / 16 <= UINT32_MAX / 256;
}

}  // namespace

// Rows for the products (mx4_product.hip), arguments checked there.
hipError_t mx4_make_rows(const void* x, int dtype, int64_t rows, int k, int64_t x_stride, void* out, hipStream_t st) {
  const Mx4Rows L = mx4_rows_layout(rows, k);
  return launch_quantize<true>(x, dtype, rows, k, x_stride, (uint8_t*)out, L.code_stride, (uint8_t*)out + L.scales,
                               L.scale_stride, st);
}

}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_mx4_quantize(const void* x, int dtype, int64_t rows, int k, int64_t x_stride, uint8_t* codes,
                         uint8_t* scales, void* stream) {
  if (x == nullptr || codes == nullptr || scales == nullptr || rows <= 0 || k <= 0 || !mx4_float(dtype) || x_stride < k)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_quantize: invalid arguments");
  if (k % kMx4Block != 0 || (uintptr_t)x % 16 != 0 || x_stride * mx4_size(dtype) % 16 != 0 || (uintptr_t)codes % 16 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_mx4_quantize: needs k a multiple of 32, rows and codes that start on 16 bytes");
  if (k > HI_ROCM_MX4_MAX_K || !mx4_rows_fit(rows, k))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_quantize: more than 2^24 inputs, or too many rows");
  const hipError_t e = launch_quantize<false>(x, dtype, rows, k, x_stride, codes, k / 2, scales, k / kMx4Block,
                                              (hipStream_t)stream);
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 quantize launch");
}

int hi_rocm_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int k, void* out, int out_dtype,
                           int64_t out_stride, void* stream) {
  if (codes == nullptr || scales == nullptr || out == nullptr || rows <= 0 || k <= 0 || !mx4_float(out_dtype) ||
      out_stride < k)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_dequantize: invalid arguments");
  if (k % kMx4Block != 0 || (uintptr_t)out % 16 != 0 || out_stride * mx4_size(out_dtype) % 16 != 0 ||
      (uintptr_t)codes % 16 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_mx4_dequantize: needs k a multiple of 32, rows and codes that start on 16 bytes");
  if (k > HI_ROCM_MX4_MAX_K || !mx4_rows_fit(rows, k))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_dequantize: more than 2^24 inputs, or too many rows");
  const int quads = (k + kMx4Quad - 1) / kMx4Quad;
  const uint32_t units = (uint32_t)(rows * quads);
  const dim3 grid((unsigned)((units + 4 * kMx4Units - 1) / (4 * kMx4Units)));
  if (out_dtype == HI_ROCM_DTYPE_F32)
    hipLaunchKernelGGL((mx4_dequantize_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, codes, scales, units,
                       quads, k, (float*)out, out_stride);
  else
    hipLaunchKernelGGL((mx4_dequantize_kernel<__bf16>), grid, dim3(256), 0, (hipStream_t)stream, codes, scales, units,
                       quads, k, (__bf16*)out, out_stride);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 dequantize launch");
}

int hi_rocm_mx4_rows_bytes(int64_t rows, int k, size_t* out_bytes) {
  if (rows <= 0 || k <= 0 || out_bytes == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_rows_bytes: invalid arguments");
  if (k % kMx4Block != 0 || k > HI_ROCM_MX4_MAX_K || !mx4_rows_fit(rows, k))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_rows_bytes: needs k a multiple of 32 up to 2^24, fewer rows");
  *out_bytes = mx4_rows_layout(rows, k).total;
  return HI_ROCM_OK;
}

int hi_rocm_mx4_rows(const void* x, int dtype, int64_t rows, int k, int64_t x_stride, void* out, size_t out_bytes,
                     void* stream) {
  if (x == nullptr || out == nullptr || rows <= 0 || k <= 0 || !mx4_float(dtype) || x_stride < k)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_rows: invalid arguments");
  if (k % kMx4Block != 0 || (uintptr_t)x % 16 != 0 || x_stride * mx4_size(dtype) % 16 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_rows: needs k a multiple of 32 and rows that start on 16 bytes");
  if (k > HI_ROCM_MX4_MAX_K || !mx4_rows_fit(rows, k))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_rows: more than 2^24 inputs, or too many rows");
  if ((uintptr_t)out % 16 != 0 || out_bytes < mx4_rows_layout(rows, k).total)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_rows: out not on 16 bytes, or too small (hi_rocm_mx4_rows_bytes)");
  const hipError_t e = mx4_make_rows(x, dtype, rows, k, x_stride, out, (hipStream_t)stream);
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 rows launch");
}

int hi_rocm_mx4_moe_prepare(const uint32_t* ids, int tokens, int top_k, int experts, int32_t* order, int32_t* slots,
                            int32_t* offsets, const void* x, int k, int64_t x_stride, void* out, size_t out_bytes,
                            void* stream) {
  if (ids == nullptr || order == nullptr || slots == nullptr || offsets == nullptr || x == nullptr || out == nullptr ||
      tokens <= 0 || top_k <= 0 || experts <= 0 || k <= 0 || x_stride < k)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_moe_prepare: invalid arguments");
  if (experts > kMoeMaxExperts || (int64_t)tokens * top_k > kMoeMaxPairs)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_moe_prepare: more than 2048 experts or 2^22 pairs");
  if (k % kMx4Block != 0 || (uintptr_t)x % 16 != 0 || x_stride % 8 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_mx4_moe_prepare: needs k a multiple of 32 and rows that start on 16 bytes");
  if (k > HI_ROCM_MX4_MAX_K || !mx4_rows_fit(tokens, k))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_moe_prepare: more than 2^24 inputs, or too many rows");
  const Mx4Rows R = mx4_rows_layout(tokens, k);
  if ((uintptr_t)out % 16 != 0 || out_bytes < R.total)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_moe_prepare: out not on 16 bytes, or too small (hi_rocm_mx4_rows_bytes)");
  const int pairs = tokens * top_k, quads = (k + kMx4Quad - 1) / kMx4Quad;
  const Mx4Quantize<__bf16> q{(const __bf16*)x, x_stride, (uint32_t)(tokens * quads), quads, k, (uint8_t*)out, R.code_stride,
                              (uint8_t*)out + R.scales, R.scale_stride};
  const int waves = pairs <= kMoeFewPairs ? 4 : 16;
  const int64_t groups = experts + 1 + ((int64_t)q.units + waves * kMx4Units - 1) / (waves * kMx4Units);
  if (groups > UINT32_MAX / (64 * waves))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_mx4_moe_prepare: too many rows for one launch");
  if (waves == 4)
    hipLaunchKernelGGL((mx4_prepare_kernel<4, 4>), dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, ids, pairs,
                       experts, order, slots, offsets, q);
  else
    hipLaunchKernelGGL((mx4_prepare_kernel<16, 8>), dim3((unsigned)groups), dim3(1024), 0, (hipStream_t)stream, ids, pairs,
                       experts, order, slots, offsets, q);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 moe prepare launch");
}

int hi_rocm_mx4_packed_bytes(int experts, int n, int k, size_t* out_bytes) {
  if (experts <= 0 || n <= 0 || k <= 0 || out_bytes == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_packed_bytes: invalid arguments");
  if (!mx4_weight_fits(experts, n, k))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_mx4_packed_bytes: needs k a multiple of 32 up to 2^24, at most 2048 experts, 2^24 outputs "
                    "and 2^35 weights");
  *out_bytes = mx4_packed_layout(experts, n, k).total;
  return HI_ROCM_OK;
}

int hi_rocm_mx4_pack(const uint8_t* codes, const uint8_t* scales, int experts, int n, int k, void* packed,
                     size_t packed_bytes, void* stream) {
  if (codes == nullptr || scales == nullptr || packed == nullptr || experts <= 0 || n <= 0 || k <= 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_pack: invalid arguments");
  if (!mx4_weight_fits(experts, n, k) || (uintptr_t)codes % 16 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_mx4_pack: needs k a multiple of 32 up to 2^24, at most 2048 experts, 2^24 outputs and 2^35 "
                    "weights, codes that start on 16 bytes");
  const Mx4Packed L = mx4_packed_layout(experts, n, k);
  if ((uintptr_t)packed % 16 != 0 || packed_bytes < L.total)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_pack: packed not on 16 bytes, or too small (hi_rocm_mx4_packed_bytes)");
  const int64_t words = (int64_t)experts * L.tiles * L.steps * 64, sw = (int64_t)experts * L.tiles * L.quads * 64;
  hipLaunchKernelGGL(mx4_pack_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, (hipStream_t)stream, codes, n,
                     k, L.tiles, L.steps, words, (uint4*)packed);
  hipLaunchKernelGGL(mx4_pack_scales_kernel, dim3((unsigned)((sw + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                     scales, n, k / kMx4Block, L.tiles, L.quads, sw, (uint32_t*)((char*)packed + L.scales));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 pack launch");
}

}  // extern "C"
