// The 8-bit GEMM of linear_fp8.cu for a few rows (tokens being generated, short requests): bound by the weights' bytes and by
// latency, not by the tensor pipe, so there is no tile pipeline here.  A CTA owns NT x 8 columns of 8 or 16 rows; its W warps
// share the k-blocks (warp w takes w, w + W, ...), read their part of w and x with 16-byte loads straight into registers and
// multiply with mma.sync m16n8k32 (e4m3, fp32 accumulation: 7e-8 from 64 bits).  Each warp has two k-blocks in flight.
// 16 x 4096 x 4096: 5.8 us in a graph, weights in L2 (from HBM their bytes take 2.6); 11.4 with one k-block in flight and the codes
// widened to fp16 for m16n8k16, 8.3 with two.
//
// No shuffling of operands: a product sums over k in any order as long as both sides agree, so lane (r = lane / 4, c = lane % 4)
// holds the 16 consecutive codes 16 c .. 16 c + 15 of a 64-wide chunk for weight row r and for x rows r and r + 8, and each of
// two MMAs takes eight codes of a lane.  A k-block's sum is scaled and added to the warp's fp32 sums; the warps' sums meet in
// shared memory, in the order of the warps.
//
// e4m3 output: a scale block is 128 columns, 8 CTAs' worth of 16.  They form a cluster and exchange their rows' largest
// magnitudes through distributed shared memory.
#include "fp8.cuh"
#include "linear_fp8.cuh"
#include "ptx.cuh"

namespace b200 {
namespace lin {
namespace {

struct RowsParams {
    const uint8_t* x;
    const uint8_t* w;
    const float* x_scale;
    const float* w_scale;
    const float* bias;
    const void* residual;
    void* y;
    float* y_scale;
    int M, N, K, k_blocks;
    long long ldx, ldw, ldr, ldy, ld_xs, ld_ys;
    int out_dtype, res_dtype, epilogue;
};

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr, uint32_t rank) {
    uint32_t v;
    asm volatile("{\n\t.reg .b32 remote;\n\tmapa.shared::cluster.u32 remote, %1, %2;\n\tld.shared::cluster.u32 %0, [remote];\n\t}"
                 : "=r"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// XR = 8-row halves of x's one 16-row tile in use, NT = 8-column tiles per CTA, W = warps.  F8: e4m3 output, clusters of 8 CTAs
// (NT = 2).
template <int XR, int NT, int W, bool F8>
__global__ void __launch_bounds__(32 * W, 16 / W) linear_fp8_rows_kernel(const RowsParams p) {
    constexpr int ROWS = XR * 8, COLS = NT * 8, kWarps = W;
    __shared__ float sums[kWarps][ROWS * COLS];
    __shared__ uint32_t amax_s[ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.x * COLS, m0 = blockIdx.y * ROWS;
    pdl_launch_dependents();
    pdl_wait();

    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    const float* ws = p.w_scale + static_cast<long long>(min(n0, p.N - 1) / fp8::kBlock) * p.k_blocks;
    // codes of one k-block: two chunks of 64, for NT weight rows and XR rows of x
    struct Codes {
        uint4 w[2][NT], x[2][XR];
        float xs[XR], ws;
    };
    auto fetch = [&](int kb, Codes& q) {
        if (kb >= p.k_blocks) return;                          // (not multiplied either)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = kb * 128 + h * 64 + c * 16;          // K is a multiple of 16: a lane's codes are all there or none
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int row = n0 + n * 8 + r;
                q.w[h][n] = k < p.K && row < p.N ? __ldg(reinterpret_cast<const uint4*>(p.w + row * p.ldw + k)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int t = 0; t < XR; ++t) {
                const int row = m0 + t * 8 + r;
                q.x[h][t] = k < p.K && row < p.M ? __ldg(reinterpret_cast<const uint4*>(p.x + row * p.ldx + k)) : make_uint4(0, 0, 0, 0);
            }
        }
        q.ws = __ldg(ws + kb);
#pragma unroll
        for (int t = 0; t < XR; ++t) q.xs[t] = m0 + t * 8 + r < p.M ? __ldg(p.x_scale + kb * p.ld_xs + m0 + t * 8 + r) : 0.f;
    };
    auto multiply = [&](const Codes& q) {
        float part[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[n][e] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {                      // eight codes of each lane
                const uint4 &lo = q.x[h][0], &hi = q.x[h][XR - 1];
                const uint32_t a0 = i == 0 ? lo.x : lo.z, a2 = i == 0 ? lo.y : lo.w;
                const uint32_t a1 = XR == 2 ? (i == 0 ? hi.x : hi.z) : 0u, a3 = XR == 2 ? (i == 0 ? hi.y : hi.w) : 0u;
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    mma_e4m3(part[n], a0, a1, a2, a3, i == 0 ? q.w[h][n].x : q.w[h][n].z, i == 0 ? q.w[h][n].y : q.w[h][n].w);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2 * XR; ++e) acc[n][e] = fmaf(part[n][e], q.xs[e >> 1] * q.ws, acc[n][e]);
    };
    {
        Codes q[2];                                            // this k-block's and the next one's
        fetch(warp, q[0]);
        fetch(warp + kWarps, q[1]);
        for (int kb = warp; kb < p.k_blocks; kb += 2 * kWarps) {
            multiply(q[0]);
            fetch(kb + 2 * kWarps, q[0]);
            if (kb + kWarps < p.k_blocks) multiply(q[1]);
            fetch(kb + 3 * kWarps, q[1]);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2 * XR; ++e) sums[warp][(r + (e >> 1) * 8) * COLS + n * 8 + c * 2 + (e & 1)] = acc[n][e];
    if (F8 && threadIdx.x < ROWS) amax_s[threadIdx.x] = 0;
    __syncthreads();

    // a thread per pair of columns of a row
    constexpr int PAIRS = ROWS * COLS / 2;
    constexpr int PER = (PAIRS + 32 * kWarps - 1) / (32 * kWarps);
    float v[PER][2];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = threadIdx.x + i * 32 * kWarps;
        const int at_row = at / (COLS / 2), row = m0 + at_row, col = at % (COLS / 2) * 2, n = n0 + col;
        v[i][0] = v[i][1] = 0.f;
        if (at >= PAIRS || row >= p.M || n >= p.N) continue;   // (N is even)
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 s = *reinterpret_cast<const float2*>(&sums[w][at_row * COLS + col]);
            a += s.x;
            b += s.y;
        }
        if (p.bias != nullptr) {
            a += __ldg(p.bias + n);
            b += __ldg(p.bias + n + 1);
        }
        const bool f32 = !F8 && p.out_dtype == B200_F32;
        if (p.epilogue == B200_EPI_BIAS_GELU) {
            if (f32) {
                a = 0.5f * a * (1.0f + erff(a * 0.70710678118654752f));
                b = 0.5f * b * (1.0f + erff(b * 0.70710678118654752f));
            } else {
                gelu_tail_x2(a, b);
            }
        } else if (p.epilogue == B200_EPI_BIAS_TANH) {
            a = tanhf(a);
            b = tanhf(b);
        } else if (p.epilogue == B200_EPI_BIAS_RESIDUAL) {
            const float2 q = unpack2(*reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.residual) + row * p.ldr + n), p.res_dtype);
            a += q.x;
            b += q.y;
        }
        v[i][0] = a;
        v[i][1] = b;
        if (F8) {
            atomicMax(&amax_s[at_row], max(fp8::abs_bits(a), fp8::abs_bits(b)));   // (a maximum: its order changes nothing)
        } else if (f32) {
            *reinterpret_cast<float2*>(static_cast<float*>(p.y) + row * p.ldy + n) = make_float2(a, b);
        } else {
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.y) + row * p.ldy + n) = pack2(a, b, p.out_dtype);
        }
    }
    if (F8) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        const uint32_t amax_u = smem_u32(amax_s);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = threadIdx.x + i * 32 * kWarps;
            const int at_row = at / (COLS / 2), row = m0 + at_row, n = n0 + at % (COLS / 2) * 2;
            if (at >= PAIRS || row >= p.M || n >= p.N) continue;
            uint32_t bits = 0;
            for (uint32_t k = 0; k < 8; ++k) bits = max(bits, ld_cluster_u32(amax_u + at_row * 4, k));
            const float amax = fp8::amax_of_bits(bits);
            const float enc = fp8::encode_scale(amax);
            *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(p.y) + row * p.ldy + n) =
                static_cast<uint16_t>(fp8::pack4(v[i][0] * enc, v[i][1] * enc, 0.f, 0.f));
            if (n % fp8::kBlock == 0) p.y_scale[n / fp8::kBlock * p.ld_ys + row] = fp8::decode_scale(amax);
        }
        // nobody leaves while its maxima may be read
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <int XR, int NT, int W, bool F8>
int launch_rows(const RowsParams& p, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(F8 ? static_cast<unsigned>((p.N + 127) / 128) * 8 : static_cast<unsigned>((p.N + NT * 8 - 1) / (NT * 8)),
                       static_cast<unsigned>((p.M + XR * 8 - 1) / (XR * 8)));
    cfg.blockDim = dim3(32 * W);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (F8) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 8;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = static_cast<unsigned>(n);
    cudaLaunchKernelEx(&cfg, linear_fp8_rows_kernel<XR, NT, W, F8>, p);
    count_launch();
    return check_launch();
}

template <int XR>
int launch_tiles(const RowsParams& p, int sms, cudaStream_t stream) {
    if (p.out_dtype == B200_E4M3) return launch_rows<XR, 2, 8, true>(p, stream);
    // 8 columns per CTA while that does not make more CTAs than SMs: the more SMs fetch weights at once, the shorter each one's
    // share; sixteen warps where there are k-blocks for more than eight and an SM has but one CTA.
    const long long down = (p.M + XR * 8 - 1) / (XR * 8);
    const bool narrow = (p.N + 7) / 8 * down <= sms;
    if (p.k_blocks > 8 && (narrow || (p.N + 15) / 16 * down <= sms))
        return narrow ? launch_rows<XR, 1, 16, false>(p, stream) : launch_rows<XR, 2, 16, false>(p, stream);
    return narrow ? launch_rows<XR, 1, 8, false>(p, stream) : launch_rows<XR, 2, 8, false>(p, stream);
}

}  // namespace

// The kernel above pays while its CTAs, 16 rows by 16 columns, are at most 3.5 per SM; with clusters of 8, 1.75.  Beyond, tiles
// read x and w less often.  us per call in a graph, this kernel | tiles, N x K:
//   half output  2304 x 768:  M 1 2.3 | 4.5   M 32 2.9 | 4.6   M 64 4.6 | 4.7        1024 x 4096: M 16 3.6 | 12.1   M 64 6.0 | 12.2
//                4096 x 1024: M 32 4.9 | 5.3  M 48 6.7 | 5.3                         4096 x 4096: M 32 10.7 | 12.4  M 48 14.9 | 12.4
//                1024 x 1024: M 128 4.6 | 5.4  M 160 5.8 | 5.4                      1024 x 4096: M 128 10.7 | 12.4
//   e4m3 output  2304 x 768:  M 16 3.8 | 6.1  M 32 6.6 | 5.9                         4096 x 1024: M 16 4.8 | 6.8    M 24 7.4 | 6.8
//                2048 x 2048: M 32 5.6 | 9.0  M 48 9.4 | 9.1                         4096 x 4096: M 16 7.4 | 14.2   M 32 13.8 | 14.0
bool few_rows_pay(const B200LinearFp8Desc& d, int sms) {
    if (d.M > kFewRows) return false;
    const bool f8 = d.out_dtype == B200_E4M3;
    const long long across = f8 ? (d.N + 127) / 128 * 8 : (d.N + 15) / 16;
    return (d.M + 15) / 16 * across * 4 <= (f8 ? 7ll : 14ll) * sms;
}

int launch_linear_fp8_rows(const B200LinearFp8Desc& d, cudaStream_t stream, int sms) {
    RowsParams p;
    p.x = static_cast<const uint8_t*>(d.x);
    p.w = static_cast<const uint8_t*>(d.w_nk);
    p.x_scale = d.x_scale;
    p.w_scale = d.w_scale;
    p.bias = d.bias;
    p.residual = d.residual;
    p.y = d.y;
    p.y_scale = d.y_scale;
    p.M = static_cast<int>(d.M);
    p.N = static_cast<int>(d.N);
    p.K = static_cast<int>(d.K);
    p.k_blocks = (p.K + 127) / 128;
    p.ldx = d.ldx;
    p.ldw = d.ldw;
    p.ldr = d.ldr;
    p.ldy = d.ldy;
    p.ld_xs = d.ld_x_scale;
    p.ld_ys = d.ld_y_scale;
    p.out_dtype = d.out_dtype;
    p.res_dtype = d.res_dtype;
    p.epilogue = d.epilogue;
    return p.M <= 8 ? launch_tiles<1>(p, sms, stream) : launch_tiles<2>(p, sms, stream);
}

}  // namespace lin
}  // namespace b200
