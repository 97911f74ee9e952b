// Shared by the two 8-bit GEMM kernels (tiles in linear_fp8.cu, a few rows in linear_fp8_rows.cu).
#pragma once
#include "linear_common.cuh"

namespace b200 {
namespace lin {

constexpr int kFewRows = 128;   // the kernel for a few rows takes no more
bool few_rows_pay(const B200LinearFp8Desc& d, int sms);
int launch_linear_fp8_rows(const B200LinearFp8Desc& d, cudaStream_t stream, int sms);

// GELU, x Phi(x) = max(x, 0) - u Q(u) with u = |x| and the normal tail Q(u) = exp(-u^2 / 2) P(u).  P, half the Mills ratio scaled
// by sqrt(2 / pi), is smooth; a polynomial of degree 7 fitted to it on [0, 6] with the weight u exp(-u^2 / 2) leaves the result
// 3.0e-6 off at most over all x (evaluated in fp32; the tail beyond 6 is under 6e-9).  The tanh form that half-precision results
// get away with (3e-5, tanh.approx) moved enough e4m3 codes to show: error of a feed-forward pair 6.9e-4 with it, 2.8e-4 exact.
// In v = u sqrt(log2(e) / 2), exp(-u^2 / 2) is 2^(-v^2).  One MUFU instruction per value and eleven packed ones per pair, which
// bound it (fourteen before the change of variable).  max.NaN keeps a NaN.
__device__ __forceinline__ void gelu_tail_x2(float& a, float& b) {
    const uint64_t v = mul_f32x2(pack_f32x2(fminf(fabsf(a), 6.0f), fminf(fabsf(b), 6.0f)), pack_f32x2(0.84932180f, 0.84932180f));
    uint64_t q = pack_f32x2(3.50742003e-4f, 3.50742003e-4f);   // -P u / v
    const float c[7] = {-4.72135826e-3f, 2.7707038e-2f, -9.57544178e-2f, 0.225075723f, -0.396406709f, 0.550873953f, -0.588565986f};
#pragma unroll
    for (int i = 0; i < 7; ++i) q = fma_f32x2(q, v, pack_f32x2(c[i], c[i]));
    float ta, tb;
    unpack_f32x2(mul_f32x2(v, v), ta, tb);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ta) : "f"(-ta));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(tb) : "f"(-tb));
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(a));
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(b));
    unpack_f32x2(fma_f32x2(mul_f32x2(q, pack_f32x2(ta, tb)), v, pack_f32x2(a, b)), a, b);
}

}  // namespace lin
}  // namespace b200
