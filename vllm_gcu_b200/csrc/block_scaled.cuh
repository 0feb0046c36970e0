// Codes of a key / value cache held in 8 bits with a scale for each block of tokens and head (block_scaled.cu writes and
// expands it, attention_block_scaled.cu reads it): fp8 e4m3 or int8, what a code stands for is code * scale.
//
// Scales are powers of two.  An e4m3 code has the same relative step at every size, so that a power of two costs nothing
// (its 17 binades below the largest code are enough for a block's numbers), and int8 loses half a bit on the mean.  In
// return division by a scale is exact, so that a code is the input's one rounding; a block that outgrows its scale has its
// codes halved as often as it takes, which e4m3 does without rounding but for the smallest ones; and every code times its
// scale is a bf16 number.
#pragma once

#include "common.cuh"

namespace b200 {
namespace block_scaled {

constexpr int kLowExponent = -100, kHighExponent = 121;   // of scales

// Exponent of the least scale whose largest code reaches `top` (finite, >= 0): 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.
template <bool kInt8>
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 127;
  const uint32_t frac = bits & 0x7fffffu;
  const int need = kInt8 ? e - 6 + (frac > 0x7e0000u) : e - 8 + (frac > 0x600000u);
  return max(kLowExponent, min(kHighExponent, need));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Magnitude that counts for a block's scale: infinities take the largest code and NaN the code 0, whatever the scale.
__device__ __forceinline__ float finite_size(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

// Four numbers in units of their scale -> four codes.  NaN becomes 0: a masked place of a block must not reach the rows
// that do not see it, and a request whose keys are NaN has queries that are NaN as well.
template <bool kInt8>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  constexpr float kTop = kInt8 ? 127.0f : 448.0f;
  float v[4] = {a, b, c, d};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = v[i] == v[i] ? v[i] : 0.0f;
    v[i] = fminf(fmaxf(v[i], -kTop), kTop);
  }
  if constexpr (kInt8) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (static_cast<uint32_t>(__float2int_rn(v[i])) & 0xffu) << (8 * i);
    return r;
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
}

// The same for numbers that are finite and reach no further than the largest code, without a look at each of them.  int8: in
// 1.5 * 2^23 + x the last bits are x rounded to a whole number (one instruction with the product in front, where a
// conversion has a quarter of the rate).
template <bool kInt8>
__device__ __forceinline__ uint32_t codes4_of(const float (&x)[4], float unit) {
  if constexpr (kInt8) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(fmaf(x[i], unit, 12582912.0f));
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  } else {
    uint32_t r;
    asm("{\n\t"
        ".reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t"
        "}"
        : "=r"(r)
        : "f"(x[0] * unit), "f"(x[1] * unit), "f"(x[2] * unit), "f"(x[3] * unit));
    return r;
  }
}

// Four codes of a word -> two pairs of fp16, exact: `lo` holds bytes 0 and 1, `hi` bytes 2 and 3.  int8: with the sign
// bit turned a byte u is the last part of the fp16 number 1024 + u, less 1152 the code.
template <bool kInt8>
__device__ __forceinline__ void unpack4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kInt8) {
    w ^= 0x80808080u;
    const uint32_t bias = 0x64806480u;         // 1152
    uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&l), *reinterpret_cast<const __half2*>(&bias));
    const __half2 b = __hsub2(*reinterpret_cast<__half2*>(&h), *reinterpret_cast<const __half2*>(&bias));
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    asm("{\n\t"
        ".reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t"
        "}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}
__device__ __forceinline__ float2 half_pair(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

}  // namespace block_scaled
}  // namespace b200
