// fp4.cuh -- the 4-bit block formats: constants, the scale layout and the conversions that the
// quantisation, the products and the expert layer share.
//
//   mxfp4  32 values share a power of two (e8m0: byte b stands for 2^(b - 127), 255 for NaN)
//   nvfp4  16 values share an e4m3 number; one fp32 global scale multiplies the whole matrix
// A value is an e2m1 number, one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign; two of them share a
// byte, the one with the lower index in the low half.
//
// Scales lie as the tensor cores read them: tiles of 128 rows x 4 blocks, 512 bytes each, tile
// (row / 128, block / 4) in row-major order; the byte of (row, block) inside its tile is
// (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4. Bytes past the matrix's edge are zero.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fmoe.h"

namespace fmoe {
namespace fp4 {

constexpr int kTileRows = 128;
constexpr int kTileBytes = 512;

__host__ __device__ constexpr int block_of(int format) { return format == FMOE_MXFP4 ? 32 : 16; }
// columns that one 512-byte scale tile covers
__host__ __device__ constexpr int tile_cols(int format) { return 4 * block_of(format); }
__host__ __device__ constexpr int64_t tiles_down(int64_t rows) {
  return (rows + kTileRows - 1) / kTileRows;
}
__host__ __device__ constexpr int tiles_across(int cols, int format) {
  return (cols + tile_cols(format) - 1) / tile_cols(format);
}
__host__ __device__ constexpr int scale_offset(int row, int block) {
  return (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4;
}

// Eight values to eight codes: round to nearest, ties to the even code, 6 at most.
__device__ __forceinline__ uint32_t encode8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight codes to eight values.
__device__ __forceinline__ void decode8(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// e4m3 byte of a non-negative value, round to nearest even, 448 at most; and back.
__device__ __forceinline__ uint32_t e4m3_byte(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0xffu;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  uint32_t h;
  const uint16_t b = (uint16_t)byte;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(b));
  return __half22float2(*reinterpret_cast<const __half2*>(&h)).x;
}
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  // 2^-127 is below the normal range
  return byte == 255 ? __int_as_float(0x7fffffff)
                     : __int_as_float(byte == 0 ? 0x00400000 : (int)(byte << 23));
}
template <int kFormat>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return kFormat == FMOE_MXFP4 ? e8m0_value(byte) : e4m3_value(byte);
}

// The scale byte of a block whose largest magnitude has the bits `top` (sign cleared; the
// bits order like the magnitudes, with the infinity and NaN above them), and the number that
// the values are divided by (`divide`, nvfp4) or multiplied by (mxfp4) to be encoded.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top, float& multiply) {
  // 2^(floor(log2 top) - 2): the exponent field less 2, at least 2^-127
  const uint32_t field = top >> 23;
  const uint32_t byte = field > 2 ? field - 2 : 0;
  multiply = __int_as_float((int)((254 - byte) << 23));
  return top >= 0x7f800000u ? 255u : byte;
}
// The correctly rounded quotient x / d from the rounded reciprocal r of d by one residual step,
// q = x r, q + (x - q d) r (Markstein 1990), where these stay finite.
__device__ __forceinline__ float quotient(float x, float d, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-q, d, x), r, q);
}
__device__ __forceinline__ bool tame(float d) { return d > 0x1p-100f && d < 0x1p100f; }

// The divisor 6 g of a block's largest magnitude, and its reciprocal: once per matrix.
struct NvDivisor {
  float global, six, r;
};
__device__ __forceinline__ NvDivisor nv_divisor(float global) {
  const float six = __fmul_rn(6.0f, global);
  return {global, six, __frcp_rn(six)};
}
__device__ __forceinline__ uint32_t nv_scale(uint32_t top, const NvDivisor& n, float& divide) {
  const float t = __int_as_float((int)top);
  const float s = tame(n.six) && t < 0x1p20f ? quotient(t, n.six, n.r) : __fdiv_rn(t, n.six);
  const uint32_t byte = e4m3_byte(fminf(s, 448.0f));
  divide = __fmul_rn(e4m3_value(byte), n.global);
  return top >= 0x7f800000u ? 127u : byte;
}

// Encodes 16 values (an nvfp4 block, or half an mxfp4 block whose largest magnitude both halves
// know): the codes of v[0..7] and v[8..15] and the block's scale byte. The quotients are the
// correctly rounded ones of the definition.
template <int kFormat>
__device__ __forceinline__ uint32_t encode16(float (&v)[16], uint32_t top, const NvDivisor& n,
                                             uint32_t& lo, uint32_t& hi) {
  uint32_t byte, flip = 0;
  float by;
  if constexpr (kFormat == FMOE_MXFP4) {
    byte = mx_scale(top, by);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __fmul_rn(v[i], by);
  } else {
    byte = nv_scale(top, n, by);
    const float r = __frcp_rn(by);
    if (tame(by) && __int_as_float((int)top) * r < 0x1p20f) {
      // Two at a time: each half of a packed operation rounds like the single one. With -r for r
      // all signs are turned, and a zero keeps its own (the residual step adds +0 to it, which
      // would take it from -0).
      const float2 r2 = make_float2(-r, -r), d2 = make_float2(by, by);
      flip = 0x88888888u;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float2 x = make_float2(v[i], v[i + 1]);
        const float2 q = __fmul2_rn(x, r2);
        const float2 y = __ffma2_rn(__ffma2_rn(q, d2, x), r2, q);
        v[i] = y.x;
        v[i + 1] = y.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] = by > 0.0f ? __fdiv_rn(v[i], by) : __fmul_rn(v[i], 0.0f);
    }
  }
  const float a[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
  const float b[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
  lo = encode8(a) ^ flip;
  hi = encode8(b) ^ flip;
  return byte;
}

// gate * silu(up) with the fast exponential and division: a few units in the last place, far
// below the 4 bits that it is rounded to
__device__ __forceinline__ float swiglu(float gate, float up) {
  return gate * __fdividef(up, 1.0f + __expf(-up));
}

}  // namespace fp4
}  // namespace fmoe
