// Device helpers shared by the 8-bit paged K/V cache kernels: the two code formats (e4m3 and
// int8) and power-of-two scales.
//
// Layout of a cache: codes [num_pages, kv_heads, page_size, head_dim] (one byte each), one
// fp32 scale per (page, kv head), a power of two within [2^-60, 2^60]; value = code * scale.
// A page of one head is contiguous, so a tile of keys is one rectangle for TMA.
//
// Why powers of two: scaling a value is then exact, so a page whose scale grows is rescaled
// without a second rounding of e4m3 codes (only codes that underflow lose bits), the stored
// codes do not depend on how the division was carried out, and attention can fold log2 of
// the value scale into the logit. Cost: int8 codes use 64..127 of their range instead of 127.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <string>

#include "common.cuh"

namespace nmb {

// Numbers in error messages: plain text, so that no iostream formatting is involved in code
// built by nvcc (it crashed with this project's toolchain).
inline std::string num(int64_t v) { return std::to_string(v); }

namespace kv {

constexpr int kScaleExpMin = -60;
constexpr int kScaleExpMax = 60;

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float s) {
  return ((__float_as_int(s) >> 23) & 255) - 127;
}

// Smallest e with amax <= qmax * 2^e, clamped (0 gives the lower end). qmax is 448 =
// 0.875 * 2^9 or 127 = 0.9921875 * 2^7: compare the mantissas, then it is exponent arithmetic.
template <bool INT8>
__device__ __forceinline__ int scale_exponent(float amax) {
  constexpr int kBits = INT8 ? 7 : 9;
  constexpr int kMant = INT8 ? 0x7E0000 : 0x600000;  // 0.9921875 * 2 and 0.875 * 2, below 1.
  const int bits = __float_as_int(amax);
  // amax = m * 2^x with m in [0.5, 1): x = biased exponent - 126. Subnormals clamp anyway.
  const int x = (bits >> 23) - 126;
  const int e = x - kBits + ((bits & 0x7FFFFF) > kMant ? 1 : 0);
  return min(max(e, kScaleExpMin), kScaleExpMax);
}

// Codes of four values already divided by the scale: rounded to nearest even, saturated
// (infinities too); NaN stays NaN in e4m3 and becomes 0 in int8, which has none.
template <bool INT8>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if (INT8) {
    const int ia = min(max(__float2int_rn(a), -127), 127), ib = min(max(__float2int_rn(b), -127), 127);
    const int ic = min(max(__float2int_rn(c), -127), 127), id = min(max(__float2int_rn(d), -127), 127);
    return (ia & 255) | ((ib & 255) << 8) | ((ic & 255) << 16) | (static_cast<uint32_t>(id) << 24);
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Four codes as two f16x2 (bytes 0,1 and 2,3), exact in both formats. int8: a byte c ^ 0x80 in the low mantissa bits
// of 1024 gives 1024 + 128 + c exactly; subtract 1152.
template <bool INT8>
__device__ __forceinline__ void decode4(uint32_t v, uint32_t& lo, uint32_t& hi) {
  if (INT8) {
    const uint32_t x = v ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    __half2 hb = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<uint32_t*>(&ha);
    hi = *reinterpret_cast<uint32_t*>(&hb);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(v));
  }
}

// 0x80 in each byte of `v` that is the NaN of e4m3 (0x7F or 0xFF).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) {
  return ((v & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}

__device__ __forceinline__ float2 f16x2_to_float2(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

}  // namespace kv
}  // namespace nmb
