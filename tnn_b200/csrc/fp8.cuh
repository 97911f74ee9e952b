// Block-scaled e4m3: 128 consecutive values of a row share one fp32 scale.  A value v of a block whose largest magnitude
// is amax is stored as the code e4m3(v * (448 / amax)) and stands for code * (amax / 448); the quotient, the product and the
// scale are each rounded once in 32 bits, the code once to e4m3 (nearest even).
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {
namespace fp8 {

constexpr int kBlock = 128;                  // values per scale
constexpr float kMax = 448.f;                // largest e4m3 magnitude
constexpr float kMinAmax = 9.094947e-13f;    // 2^-40: a block of smaller values (zeros among them) is scaled as if this were its amax

// Magnitudes are compared as integers, in which a NaN is larger than an infinity and that than any number: a block that
// holds one gets a scale of NaN or infinity and stands for no finite value.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ float amax_of_bits(uint32_t bits) {
    const uint32_t least = __float_as_uint(kMinAmax);
    return __uint_as_float(bits > least ? bits : least);
}
// max(m, |a|, |b|) for m >= 0, a NaN if there is one (0x7FFFFFFF: the largest magnitude as an integer too)
__device__ __forceinline__ float amax3(float m, float a, float b) {
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float encode_scale(float amax) { return __fdiv_rn(kMax, amax); }
__device__ __forceinline__ float decode_scale(float amax) { return __fdiv_rn(amax, kMax); }

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

}  // namespace fp8
}  // namespace b200
