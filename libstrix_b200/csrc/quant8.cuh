// What the kernels that end in 8 bits share: the gate functions, the scale of a
// group, and the rounding of eight values to packed bytes.
//
//   scale = amax / top (448 for e4m3, 127 for int8), 1 where that is below the
//           smallest normal number (an all-zero group, or one too small to scale);
//   q     = y * (1 / scale) rounded to the nearest value, ties to even.
// A NaN in a group makes its scale NaN, an infinity makes it infinite, so that
// neither disappears in the bytes (max.NaN below; a plain fmaxf drops NaN).
#pragma once

#include "common.cuh"

namespace strix {
namespace quant8 {

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float abs_max8(const float (&y)[8]) {
  const float a = max_nan(fabsf(y[0]), fabsf(y[1]), fabsf(y[2])), b = max_nan(fabsf(y[3]), fabsf(y[4]), fabsf(y[5]));
  return max_nan(max_nan(a, b), fabsf(y[6]), fabsf(y[7]));
}

__device__ __forceinline__ float rcp(float x) {   // within a step of fp32
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float kTopF8 = 448.f, kTopI8 = 127.f;
constexpr float kSmallestNormal = 1.17549435e-38f;

// amax / TOP, as a product with the constant's reciprocal: a step or two of fp32 off the
// quotient, which the values are then divided by (an IEEE division in each of a group's 16
// lanes costs a tenth of act_mul_quant's instructions).
__device__ __forceinline__ float scale_of(float amax, float top) {
  const float s = amax * (1.f / top);
  return s < kSmallestNormal ? 1.f : s;   // NaN compares false and stays
}

__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}

// Four values times inv, |product| at most 127 (and a last bit), as bytes. Added to 1.5 x
// 2^23 the product rounds to a whole number, to nearest even, in the sum's low bits.
__device__ __forceinline__ uint32_t pack_i8x4(float a, float b, float c, float d, float inv) {
  constexpr float kMagic = 12582912.f;
  const uint32_t qa = __float_as_uint(fmaf(a, inv, kMagic)), qb = __float_as_uint(fmaf(b, inv, kMagic));
  const uint32_t qc = __float_as_uint(fmaf(c, inv, kMagic)), qd = __float_as_uint(fmaf(d, inv, kMagic));
  return prmt(prmt(qa, qb, 0x0040), prmt(qc, qd, 0x0040), 0x5410);
}

template <bool F8>
__device__ __forceinline__ uint2 pack8(const float (&y)[8], float inv) {
  if constexpr (F8)
    return make_uint2(pack_e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv),
                      pack_e4m3x4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv));
  else
    return make_uint2(pack_i8x4(y[0], y[1], y[2], y[3], inv), pack_i8x4(y[4], y[5], y[6], y[7], inv));
}

// Eight 16-bit values (bf16, or fp16) as fp32.
template <bool F16>
__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ws[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = bf16_lo(ws[i]), v[2 * i + 1] = bf16_hi(ws[i]);
    }
  }
}

// silu(g) = g / (1 + e^-g); gelu with tanh(u) written as 2 sigmoid(2u) - 1:
// 0.5 g (1 + tanh(u)) = g / (1 + e^-2u), u = sqrt(2 / pi) (g + 0.044715 g^3). Both
// through one exponential: a tanh under fast-math holds 11 bits only.
template <bool GELU>
__device__ __forceinline__ float gate(float g) {
  const float u = GELU ? 1.5957691216057308f * (g + 0.044715f * g * g * g) : g;
  return g * rcp(1.f + __expf(-u));
}
// The same, chosen at run time by a selection of the exponent: a branch around each of an
// epilogue's 64 gates costs the FP8 product 3 %.
__device__ __forceinline__ float gate(float g, int act) {
  const float u = act == 1 ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return g * rcp(1.f + __expf(-u));
}

}  // namespace quant8
}  // namespace strix
