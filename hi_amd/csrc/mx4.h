// Microscaled 4-bit floating point (the Open Compute Project's MX formats
// 1.0, MXFP4): blocks of 32 values along k, each an E2M1 code (sign, then 0, 0.5,
// 1, 1.5, 2, 3, 4, 6) times a power of two that the block shares, E8M0 byte s:
// 2^(s - 127), 255 NaN.
//
// The matrix cores take 128 values of k a step: lane 16 g + r holds row r's
// block g of the step as 16 bytes (value j in nibble j) and that block's scale
// in a byte of a register, so a block and its scale are one lane's.  Four
// steps' scales share a register; which byte counts is part of the instruction.
//
// Two layouts follow that.  "Rows" (what a product reads as x): codes
// [rows][k / 2], then scales [rows][quads][16] with block 4 (4 q + j) + g of k
// in byte 4 g + j of quad q, a lane's four steps in one word; scales behind k are
// one.  "Packed" (weights): codes [tile of 16 rows][step][lane][16 bytes], then
// scales [tile][quad][row][16], padded with zero codes and scales of one.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hi_rocm.h"

namespace hi_rocm {

constexpr int kMx4Block = 32;    // values that share a scale
constexpr int kMx4Step = 128;    // values of k a matrix instruction takes
constexpr int kMx4Quad = 512;    // values of k whose scales share a word

typedef int mx4_i32x4 __attribute__((ext_vector_type(4)));
typedef int mx4_i32x8 __attribute__((ext_vector_type(8)));
typedef float mx4_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 mx4_bf16x2 __attribute__((ext_vector_type(2)));

struct Mx4Rows {
  int64_t code_stride, scale_stride;  // bytes of a row
  size_t scales, total;               // where the scales begin, bytes in all
};
inline Mx4Rows mx4_rows_layout(int64_t rows, int k) {
  Mx4Rows L;
  L.code_stride = k / 2;
  L.scale_stride = ((int64_t)k + kMx4Quad - 1) / kMx4Quad * 16;
  L.scales = (size_t)rows * L.code_stride;
  L.total = L.scales + (size_t)rows * L.scale_stride + kMx4Quad / 2;  // (a last quad's codes may be read whole)
  return L;
}

struct Mx4Packed {
  int64_t tiles, steps, quads;  // of one expert
  size_t scales, total;
};
inline Mx4Packed mx4_packed_layout(int experts, int n, int k) {
  Mx4Packed L;
  L.tiles = ((int64_t)n + 15) / 16;
  L.steps = ((int64_t)k + kMx4Step - 1) / kMx4Step;
  L.quads = ((int64_t)k + kMx4Quad - 1) / kMx4Quad;
  L.scales = (size_t)experts * L.tiles * L.steps * 1024;
  L.total = L.scales + (size_t)experts * L.tiles * L.quads * 256;
  return L;
}

// What the calls take: words of a packed weight in one launch (less than 2^32
// threads, also with n and k padded to tiles), byte offsets within 64 bits.
inline bool mx4_weight_fits(int experts, int n, int k) {
  if (k % kMx4Block != 0 || k > HI_ROCM_MX4_MAX_K || experts > 2048 || n > (1 << 24)) return false;
  const Mx4Packed L = mx4_packed_layout(experts, n, k);
  return experts * L.tiles <= ((int64_t)1 << 35) / 2048 / L.steps;
}

// The scale of a block from the exponent field of its largest magnitude (f32
// or bf16): 2^(floor(log2 a) - 2), so that a lies in [4, 8) of it; what is above
// 6 becomes 6.  Subnormal magnitudes have field 0 and the smallest scale, as
// have those up to 2^-125; infinity and NaN give NaN.
__device__ __forceinline__ uint32_t mx4_scale_of(uint32_t field) {
  return field == 255u ? 255u : (uint32_t)max((int)field - 2, 0);
}

// Eight values of a block with scale byte s as codes.  The conversion takes its
// scale from a float's exponent field, rounds to nearest even, saturates at 6
// and keeps the sign (checked on the card for every scale at the borders,
// subnormal values among them).
__device__ __forceinline__ uint32_t mx4_codes(const float (&v)[8], uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  uint32_t c = 0u;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  return s == 255u ? 0u : c;
}
// The same from bf16 pairs.
__device__ __forceinline__ uint32_t mx4_codes(const uint4& v, uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  uint32_t c = 0u;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, v.x), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, v.y), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, v.z), scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx4_bf16x2, v.w), scale, 3);
  return s == 255u ? 0u : c;
}

// The larger magnitudes of two bf16 pairs, half by half.
__device__ __forceinline__ uint32_t mx4_max_pair(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
constexpr uint32_t kMx4Abs = 0x7fff7fffu;
__device__ __forceinline__ uint32_t mx4_max_of(const uint4& v) {
  return mx4_max_pair(mx4_max_pair(v.x & kMx4Abs, v.y & kMx4Abs), mx4_max_pair(v.z & kMx4Abs, v.w & kMx4Abs));
}
// The exponent field of the larger half.
__device__ __forceinline__ uint32_t mx4_field(uint32_t pair) { return max(pair >> 16, pair & 0xffffu) >> 7; }

// Where block b's scale lies in a row of "rows".
__host__ __device__ __forceinline__ int mx4_scale_at(int b) { return (b >> 4) * 16 + (b & 3) * 4 + (b >> 2 & 3); }

// D = A B + C over 128 values of k, both operands 4-bit, the scales in the low bytes
// of sa and sb.
__device__ __forceinline__ mx4_f32x4 mx4_mfma(const mx4_i32x4& a, const mx4_i32x4& b, const mx4_f32x4& c, int sa, int sb) {
  const mx4_i32x8 wa = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const mx4_i32x8 wb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

}  // namespace hi_rocm
