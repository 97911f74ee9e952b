// Shared by the two 8-bit GEMM kernels (tiles in linear_fp8.cu, a few rows in linear_fp8_rows.cu).
#pragma once
#include "linear_common.cuh"

namespace b200 {
namespace lin {

constexpr int kFewRows = 64;   // the kernel for a few rows takes no more
bool few_rows_pay(const B200LinearFp8Desc& d, int sms);
int launch_linear_fp8_rows(const B200LinearFp8Desc& d, cudaStream_t stream, int sms);

// GELU, x Phi(x) = max(x, 0) - u Q(u) with u = |x| and the normal tail Q(u) = exp(-u^2 / 2) P(u).  P, half the Mills ratio scaled
// by sqrt(2 / pi), is smooth; a polynomial of degree 7 fitted to it on [0, 6] with the weight u exp(-u^2 / 2) leaves the result
// 3.0e-6 off at most over all x (evaluated in fp32; the tail beyond 6 is under 6e-9).  The tanh form that half-precision results
// get away with (3e-5, tanh.approx) moved enough e4m3 codes to show: error of a feed-forward pair 6.9e-4 with it, 2.8e-4 exact.
// One MUFU instruction per value, everything else on packed pairs.  x + |x| keeps a NaN.
__device__ __forceinline__ void gelu_tail_x2(float& a, float& b) {
    const float ua = fabsf(a), ub = fabsf(b);
    const uint64_t u = pack_f32x2(fminf(ua, 6.0f), fminf(ub, 6.0f));
    uint64_t q = pack_f32x2(-9.496552e-5f, -9.496552e-5f);
    const float c[7] = {1.505126e-3f, -1.03997699e-2f, 4.23175171e-2f, -1.17116407e-1f, 2.42861018e-1f, -3.9737156e-1f, 4.99881923e-1f};
#pragma unroll
    for (int i = 0; i < 7; ++i) q = fma_f32x2(q, u, pack_f32x2(c[i], c[i]));
    float ta, tb;
    unpack_f32x2(mul_f32x2(mul_f32x2(u, u), pack_f32x2(-0.72134752f, -0.72134752f)), ta, tb);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ta) : "f"(ta));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(tb) : "f"(tb));
    const uint64_t tail = mul_f32x2(mul_f32x2(q, pack_f32x2(ta, tb)), u);
    const uint64_t sum = add_f32x2(pack_f32x2(a, b), pack_f32x2(ua, ub));
    unpack_f32x2(fma_f32x2(tail, pack_f32x2(-1.f, -1.f), mul_f32x2(sum, pack_f32x2(0.5f, 0.5f))), a, b);
}

}  // namespace lin
}  // namespace b200
