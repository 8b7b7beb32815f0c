// Products with 4-bit weights and group scales, for the few rows of a decode
// step (the reference's models are quantised in groups; its 4-bit row
// products start at crates/hi-cuda/src/kernels.cu:8658).
//
//     w[n][k] = (q[n][k] - z[n][k / G]) * s[n][k / G],   q in 0 .. 15
//     y[m][n] = sum_k x[m][k] * w[n][k] + bias[n]
//
// The weights meet the matrix cores as 16 + q in bf16, which is exact (16 has
// exponent 4, so the upper four mantissa bits count in ones) and costs a shift
// and an and-or for two weights.  A group's product with the rows, d = sum x
// (16 + q), and the rows' sums over the group, e = sum x (a product with ones,
// in the same layout), give
//     y += s * (d - (16 + z) * e)
// in f32: the weights are never rounded.  (An offset of 128, which needs no
// shift for the first pair, would lose three more bits to the difference.)
//
// hi_rocm_w4_pack lays the weights out once: blocks of 16 outputs x 128 inputs
// in the order in which the lanes of a wave hold them, so a wave reads 1 KB
// of contiguous memory a block; the blocks of 16 outputs follow each other
// along k.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "hi_rocm.h"
#include "sampler_internal.h"

namespace hi_rocm {
namespace {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4Block = 128;   // inputs of a block
constexpr int kW4Waves = 4;     // waves of a workgroup, splitting k

struct W4Layout {
  int64_t n_tiles, k_blocks;
  size_t scales, zeros, total;
};
W4Layout w4_layout(int n, int k, int group, int scale_dtype, bool zeros) {
  auto align = [](size_t x) { return (x + 255) & ~(size_t)255; };
  W4Layout L;
  L.n_tiles = ((int64_t)n + 15) / 16;
  L.k_blocks = ((int64_t)k + kW4Block - 1) / kW4Block;
  const size_t blocks = (size_t)L.n_tiles * L.k_blocks;
  const size_t per = 16 * (kW4Block / group) * (scale_dtype == HI_ROCM_DTYPE_BF16 ? 2 : 4);
  L.scales = align(blocks * 1024);
  L.zeros = L.scales + align(blocks * per);
  L.total = zeros ? L.zeros + align(blocks * per) : L.zeros;
  return L;
}

// Lane (g, r) = 16 g + r of a block holds output r's inputs 32 i + 8 g .. + 7
// in word i; input 2 p of the eight in nibble p, input 2 p + 1 in nibble p + 4,
// so one shift and one mask give a pair.
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* q, int n, int k, int64_t k_blocks,
                                                      int64_t words, uint32_t* out) {
  const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (w >= words) return;
  const int64_t block = w >> 8;
  const int i = (int)(w & 3), lane = (int)(w >> 2) & 63, r = lane & 15, g = lane >> 4;
  const int64_t row = block / k_blocks * 16 + r, k0 = block % k_blocks * kW4Block + 32 * i + 8 * g;
  uint32_t v = 0u;
  if (row < n && k0 < k) {
    const uint8_t* p = q + row * (k / 2) + k0 / 2;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = p[j];
      v |= (b & 15u) << (4 * j) | (b >> 4) << (4 * j + 16);
    }
  }
  out[w] = v;
}

// Scales (or zeros): [n][k / G] to [block][16][128 / G].  Places past n or k
// hold 0: a scale of 0 drops their products.
template <typename T>
__global__ void __launch_bounds__(256) w4_pack_scales_kernel(const T* in, int n, int groups, int gpb, int64_t k_blocks,
                                                             int64_t count, T* out) {
  const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (w >= count) return;
  const int64_t block = w / (16 * gpb);
  const int j = (int)(w % gpb), r = (int)(w / gpb) & 15;
  const int64_t row = block / k_blocks * 16 + r, grp = block % k_blocks * gpb + j;
  out[w] = row < n && grp < groups ? in[row * groups + grp] : (T)0.f;
}

struct W4Args {
  const __bf16* x;        // [rows][x_stride]
  int64_t x_stride;
  const uint32_t* q;      // packed blocks
  const void* scales;
  const void* zeros;      // or null: 8
  const float* bias;      // or null
  void* out;
  int64_t out_stride;
  int rows, n, k, out_bf16;
  int n_tiles, k_blocks;
};

// The eight weights of a word as 16 + q in bf16.
__device__ __forceinline__ w4_bf16x8 w4_unpack(uint32_t w) {
  w4_u32x4 v;
  v[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
  v[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
  v[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
  v[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
  return __builtin_bit_cast(w4_bf16x8, v);
}

template <typename T>
__device__ __forceinline__ float w4_float(T v) { return (float)v; }

// MT tiles of 16 rows times one tile of 16 outputs; the workgroup's waves
// split the blocks of k, and their sums are added in wave order.
// MFMA 16x16x32 bf16 (lane l = 16 g + r): A row r, elements 8 g .. 8 g + 7;
// B column r, the same elements; D rows 4 g .. 4 g + 3 of column r.
template <int MT, int G, typename ST>
__global__ void __launch_bounds__(64 * kW4Waves) w4_linear_kernel(W4Args a) {
  constexpr int GPB = kW4Block / G, CH = G / 32;  // groups a block, MFMAs a group
  __shared__ float part[kW4Waves - 1][MT * 4][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int nt = blockIdx.x, m0 = blockIdx.y * (16 * MT);
  const int per = (a.k_blocks + kW4Waves - 1) / kW4Waves;
  const int kb0 = wid * per, kb1 = min(kb0 + per, a.k_blocks);
  const __bf16* xr[MT];
  #pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = m0 + 16 * t + r;
    xr[t] = a.x + (int64_t)(m < a.rows ? m : 0) * a.x_stride;
  }
  w4_bf16x8 ones;
  #pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.0f;
  w4_f32x4 acc[MT];
  #pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
  const ST* sp = (const ST*)a.scales;
  const ST* zp = (const ST*)a.zeros;
  for (int kb = kb0; kb < kb1; ++kb) {
    const int64_t block = (int64_t)nt * a.k_blocks + kb;
    const w4_u32x4 w = *reinterpret_cast<const w4_u32x4*>(a.q + block * 256 + lane * 4);
    float s[GPB], z[GPB];
    #pragma unroll
    for (int j = 0; j < GPB; ++j) {
      s[j] = w4_float(sp[(block * 16 + r) * GPB + j]);
      z[j] = 16.f + (zp ? w4_float(zp[(block * 16 + r) * GPB + j]) : 8.f);
    }
    w4_bf16x8 b[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = w4_unpack(w[i]);
    #pragma unroll
    for (int t = 0; t < MT; ++t) {
      #pragma unroll
      for (int j = 0; j < GPB; ++j) {
        w4_f32x4 d = {0.f, 0.f, 0.f, 0.f}, e = {0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int i = j * CH; i < (j + 1) * CH; ++i) {
          const int kk = kb * kW4Block + 32 * i + 8 * g;
          w4_bf16x8 xa = {};
          if (kk < a.k) xa = *reinterpret_cast<const w4_bf16x8*>(xr[t] + kk);
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa, b[i], d, 0, 0, 0);
          e = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa, ones, e, 0, 0, 0);
        }
        #pragma unroll
        for (int q = 0; q < 4; ++q) acc[t][q] = fmaf(s[j], fmaf(-z[j], e[q], d[q]), acc[t][q]);
      }
    }
  }
  if (wid > 0) {
    #pragma unroll
    for (int t = 0; t < MT; ++t)
      #pragma unroll
      for (int q = 0; q < 4; ++q) part[wid - 1][t * 4 + q][lane] = acc[t][q];
  }
  __syncthreads();
  if (wid > 0) return;
  const int n = nt * 16 + r;
  if (n >= a.n) return;
  const float bias = a.bias ? a.bias[n] : 0.f;
  #pragma unroll
  for (int t = 0; t < MT; ++t) {
    #pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = m0 + 16 * t + 4 * g + q;
      if (m >= a.rows) continue;
      float y = acc[t][q];
      #pragma unroll
      for (int w = 0; w < kW4Waves - 1; ++w) y += part[w][t * 4 + q][lane];
      if (a.bias) y += bias;
      if (a.out_bf16) ((__bf16*)a.out)[(int64_t)m * a.out_stride + n] = (__bf16)y;
      else ((float*)a.out)[(int64_t)m * a.out_stride + n] = y;
    }
  }
}

template <int MT, int G, typename ST>
void launch_w4(const W4Args& a, hipStream_t st) {
  const dim3 grid((unsigned)a.n_tiles, (unsigned)((a.rows + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((w4_linear_kernel<MT, G, ST>), grid, dim3(64 * kW4Waves), 0, st, a);
}
template <int G, typename ST>
void launch_w4_rows(const W4Args& a, hipStream_t st) {
  if (a.rows <= 16) launch_w4<1, G, ST>(a, st);
  else if (a.rows <= 32) launch_w4<2, G, ST>(a, st);
  else launch_w4<4, G, ST>(a, st);
}
template <typename ST>
void launch_w4_group(const W4Args& a, int group, hipStream_t st) {
  if (group == 32) launch_w4_rows<32, ST>(a, st);
  else if (group == 64) launch_w4_rows<64, ST>(a, st);
  else launch_w4_rows<128, ST>(a, st);
}

// Sizes and types of a packed weight: HI_ROCM_OK, or a status with a message.
int w4_check(int n, int k, int group, int scale_dtype, const char* what_args, const char* what_sizes) {
  if (n <= 0 || k <= 0 || group <= 0 || (scale_dtype != HI_ROCM_DTYPE_F32 && scale_dtype != HI_ROCM_DTYPE_BF16))
    return api_fail(HI_ROCM_ERR_ARGS, what_args);
  if ((group != 32 && group != 64 && group != 128) || k % group != 0 || n > (1 << 24) || k > (1 << 24))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, what_sizes);
  return HI_ROCM_OK;
}

}  // namespace
}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_w4_packed_bytes(int n, int k, int group, int scale_dtype, int has_zeros, size_t* out_bytes) {
  if (out_bytes == nullptr) return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_packed_bytes: invalid arguments");
  const int rc = w4_check(n, k, group, scale_dtype, "hi_rocm_w4_packed_bytes: invalid arguments",
                          "hi_rocm_w4_packed_bytes: needs groups of 32, 64 or 128, k a multiple of them, n and k up to 2^24");
  if (rc != HI_ROCM_OK) return rc;
  *out_bytes = w4_layout(n, k, group, scale_dtype, has_zeros != 0).total;
  return HI_ROCM_OK;
}

int hi_rocm_w4_pack(const void* q, const void* scales, const void* zeros, int scale_dtype, int n, int k, int group,
                    void* packed, size_t packed_bytes, void* stream) {
  if (q == nullptr || scales == nullptr || packed == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_pack: invalid arguments");
  const int rc = w4_check(n, k, group, scale_dtype, "hi_rocm_w4_pack: invalid arguments",
                          "hi_rocm_w4_pack: needs groups of 32, 64 or 128, k a multiple of them, n and k up to 2^24");
  if (rc != HI_ROCM_OK) return rc;
  const W4Layout L = w4_layout(n, k, group, scale_dtype, zeros != nullptr);
  if (packed_bytes < L.total || (uintptr_t)packed % 16 != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_pack: packed buffer too small or not 16-byte aligned");
  if ((uintptr_t)scales % (scale_dtype == HI_ROCM_DTYPE_BF16 ? 2 : 4) != 0 ||
      (uintptr_t)zeros % (scale_dtype == HI_ROCM_DTYPE_BF16 ? 2 : 4) != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_pack: scales not aligned to their type");
  const int64_t blocks = L.n_tiles * L.k_blocks, words = blocks * 256;
  const int gpb = kW4Block / group;
  const int64_t count = blocks * 16 * gpb;
  if ((words + 255) / 256 > INT32_MAX)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_w4_pack: more than 2^31 blocks");
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(w4_pack_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, st, (const uint8_t*)q, n, k,
                     L.k_blocks, words, (uint32_t*)packed);
  for (int i = 0; i < (zeros ? 2 : 1); ++i) {
    const void* in = i ? zeros : scales;
    char* out = (char*)packed + (i ? L.zeros : L.scales);
    const dim3 grid((unsigned)((count + 255) / 256));
    if (scale_dtype == HI_ROCM_DTYPE_BF16)
      hipLaunchKernelGGL(w4_pack_scales_kernel<__bf16>, grid, dim3(256), 0, st, (const __bf16*)in, n, k / group, gpb,
                         L.k_blocks, count, (__bf16*)out);
    else
      hipLaunchKernelGGL(w4_pack_scales_kernel<float>, grid, dim3(256), 0, st, (const float*)in, n, k / group, gpb,
                         L.k_blocks, count, (float*)out);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "w4 pack launch");
}

int hi_rocm_w4_linear(const void* x, int rows, int64_t x_stride, const void* packed, size_t packed_bytes,
                      int scale_dtype, int has_zeros, int n, int k, int group, const float* bias, void* out,
                      int out_dtype, int64_t out_stride, void* stream) {
  if (x == nullptr || packed == nullptr || out == nullptr || rows <= 0 || x_stride < k || out_stride < n ||
      (out_dtype != HI_ROCM_DTYPE_F32 && out_dtype != HI_ROCM_DTYPE_BF16))
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_linear: invalid arguments");
  const int rc = w4_check(n, k, group, scale_dtype, "hi_rocm_w4_linear: invalid arguments",
                          "hi_rocm_w4_linear: needs groups of 32, 64 or 128, k a multiple of them, n and k up to 2^24");
  if (rc != HI_ROCM_OK) return rc;
  if (rows > 1 << 20) return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_w4_linear: more than 2^20 rows");
  if ((uintptr_t)x % 16 != 0 || x_stride % 8 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_w4_linear: needs rows of x that start on 16 bytes");
  if ((uintptr_t)out % (out_dtype == HI_ROCM_DTYPE_F32 ? 4 : 2) != 0 || (uintptr_t)bias % 4 != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_linear: out or bias not aligned to its type");
  const W4Layout L = w4_layout(n, k, group, scale_dtype, has_zeros != 0);
  if (packed_bytes < L.total || (uintptr_t)packed % 16 != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_linear: packed buffer too small or not 16-byte aligned");
  W4Args a;
  memset(&a, 0, sizeof(a));
  a.x = (const __bf16*)x;
  a.x_stride = x_stride;
  a.q = (const uint32_t*)packed;
  a.scales = (const char*)packed + L.scales;
  a.zeros = has_zeros ? (const char*)packed + L.zeros : nullptr;
  a.bias = bias;
  a.out = out;
  a.out_stride = out_stride;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.out_bf16 = out_dtype == HI_ROCM_DTYPE_BF16;
  a.n_tiles = (int)L.n_tiles;
  a.k_blocks = (int)L.k_blocks;
  if (scale_dtype == HI_ROCM_DTYPE_BF16) launch_w4_group<__bf16>(a, group, (hipStream_t)stream);
  else launch_w4_group<float>(a, group, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "w4 linear launch");
}

}  // extern "C"
