// The 8-bit paged cache: e4m3 codes with one fp32 scale per page and KV head, value = code * scale.
//
// Scales are powers of two.  A floating-point code loses nothing by that (its relative step is the
// same at every magnitude; a finer scale would only move the largest value closer to the end of the
// range), dividing by it is exact, and when a page's scale has to grow its old codes move down by whole
// exponents: exact unless they fall below 2^-6, where e4m3 has no more exponents to give.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace b200moe {

constexpr int kCodeHeadDim = 128;
// Scales lie in [2^-32, 2^32]: the floor is what the smallest fp16 value needs, and with the range
// closed on both sides no quotient of two scales leaves fp32.
constexpr float kScaleMin = 2.3283064365386963e-10f;  // 2^-32
constexpr float kScaleMax = 4294967296.f;             // 2^32

// A scale as the kernels use it: a page that was never stored to (0, or anything) counts as the floor.
__device__ __forceinline__ float usable_scale(float s) { return fminf(fmaxf(s, kScaleMin), kScaleMax); }

// Smallest power of two s with amax <= 448 s, within the range; amax is given by its bits.
__device__ __forceinline__ float scale_for(uint32_t amax_bits) {
  // 448 = 1.75 * 2^8, and 1.75 has the mantissa 0x600000.
  int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, -32), 32);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Four codes -> fp16 pairs of the two in the low and the two in the high half (exact).  Written as one
// block so that the halves of the word are register halves and not masks and shifts.
__device__ __forceinline__ void codes_to_half2(uint32_t codes, uint32_t& low, uint32_t& high) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(low), "=r"(high)
      : "r"(codes));
}

// Four fp32 values -> four codes, round to nearest even, too large values to the largest code.
__device__ __forceinline__ uint32_t to_codes4(float x0, float x1, float x2, float x3) {
  uint32_t codes;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h};\n\t}"
      : "=r"(codes)
      : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
  return codes;
}

// Four codes multiplied by `ratio` and rounded again.
__device__ __forceinline__ uint32_t rescale_codes4(uint32_t codes, float ratio) {
  uint32_t a, b;
  codes_to_half2(codes, a, b);
  const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
  return to_codes4(fa.x * ratio, fa.y * ratio, fb.x * ratio, fb.y * ratio);
}

}  // namespace b200moe
