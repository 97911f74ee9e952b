// What makes the 8-bit operands of linear_fp8.cu: the row quantizer, (residual +) LayerNorm with an 8-bit result, and the
// one-time weight pre-pack.  All HBM-bound: every input is read once, every output written once.
#include "fp8.cuh"
#include "linear_common.cuh"

namespace b200 {
namespace {

// ---------------------------------------------------------------- rows -> e4m3 + scales
// A group of 8 lanes owns one block of 128 values, 16 per lane: 16-byte loads and one 16-byte store per lane, the block's
// largest magnitude by three shuffles.  A warp holds four blocks, UNROLL of them per lane in flight.  65536 x 1024 bf16: 34.5 us,
// 0.90 of the measured copy rate; f32 56.9 us, 0.91.
template <int DT>
struct Raw16 {   // 16 consecutive elements as loaded
    static constexpr int Q = DT == B200_F32 ? 4 : 2;
    uint4 q[Q];
};
template <int DT>
__device__ __forceinline__ void decode16(const Raw16<DT>& r, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < Raw16<DT>::Q; ++i) {
        const uint32_t w[4] = {r.q[i].x, r.q[i].y, r.q[i].z, r.q[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == B200_F32) {
                v[i * 4 + e] = __uint_as_float(w[e]);
            } else {
                const float2 f = unpack2(w[e], DT);
                v[i * 8 + e * 2] = f.x;
                v[i * 8 + e * 2 + 1] = f.y;
            }
        }
    }
}

// Largest magnitude of 16 elements, as the bits of an fp32 value (ordered as integers, NaN above infinity).  Half-precision
// magnitudes are ordered the same way, so two at a time are compared before one is widened.
template <int DT>
__device__ __forceinline__ uint32_t amax_bits16(const Raw16<DT>& r) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < Raw16<DT>::Q; ++i) {
        const uint32_t w[4] = {r.q[i].x, r.q[i].y, r.q[i].z, r.q[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == B200_F32) m = max(m, w[e] & 0x7FFFFFFFu);
            else m = __vmaxu2(m, w[e] & 0x7FFF7FFFu);
        }
    }
    if constexpr (DT == B200_F32) return m;
    m = max(m & 0xFFFFu, m >> 16);
    return __float_as_uint(unpack2(m, DT).x);
}

// An item is a block of one row.  Items are dealt to the groups of all CTAs in turn; a group finds the row and block of its
// next item from those of the last one (a 64-bit division per item took as long as the item's bytes: 65536 x 1024 bf16
// 64.6 us).
template <int DT>
__global__ void __launch_bounds__(256) quantize_fp8_kernel(B200QuantizeFp8Desc d, int blocks) {
    constexpr int UNROLL = DT == B200_F32 ? 2 : 4;
    constexpr int kGroups = 32;   // blocks of 128 values per CTA and step
    pdl_launch_dependents();
    pdl_wait();
    const int sub = threadIdx.x & 7;
    const unsigned step = gridDim.x * kGroups, first = blockIdx.x * kGroups + (threadIdx.x >> 3);
    const int step_rows = static_cast<int>(step / blocks), step_blocks = static_cast<int>(step % blocks);
    long long row = first / blocks;
    int kb = static_cast<int>(first % blocks);
    while (__any_sync(0xffffffffu, row < d.rows)) {
        Raw16<DT> raw[UNROLL];
        long long rows[UNROLL];
        int kbs[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            rows[u] = row;
            kbs[u] = kb;
            const long long col = kb * fp8::kBlock + sub * 16;
#pragma unroll
            for (int k = 0; k < Raw16<DT>::Q; ++k) raw[u].q[k] = make_uint4(0, 0, 0, 0);
            if (row < d.rows && col < d.K) {
                const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(d.x) +
                                                                (row * d.ldx + col) * (DT == B200_F32 ? 4 : 2));
#pragma unroll
                for (int k = 0; k < Raw16<DT>::Q; ++k) raw[u].q[k] = __ldg(p + k);
            }
            row += step_rows;
            kb += step_blocks;
            if (kb >= blocks) {
                kb -= blocks;
                ++row;
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[16];
            decode16<DT>(raw[u], v);
            uint32_t bits = amax_bits16<DT>(raw[u]);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
            const float amax = fp8::amax_of_bits(bits);
            const float enc = fp8::encode_scale(amax);
            const int col = kbs[u] * fp8::kBlock + sub * 16;
            if (rows[u] < d.rows && col < d.K) {
                uint4 q;
                q.x = fp8::pack4(v[0] * enc, v[1] * enc, v[2] * enc, v[3] * enc);
                q.y = fp8::pack4(v[4] * enc, v[5] * enc, v[6] * enc, v[7] * enc);
                q.z = fp8::pack4(v[8] * enc, v[9] * enc, v[10] * enc, v[11] * enc);
                q.w = fp8::pack4(v[12] * enc, v[13] * enc, v[14] * enc, v[15] * enc);
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(d.q) + rows[u] * d.ldq + col) = q;
                if (sub == 0) d.scale[kbs[u] * d.ld_scale + rows[u]] = fp8::decode_scale(amax);
            }
        }
    }
}

// ---------------------------------------------------------------- (residual +) LayerNorm -> half and e4m3 + scales
// G warps per row; a lane holds NV groups of 8 consecutive elements (group g of lane l of warp w = elements
// ((g * G + w) * 32 + l) * 8 ..), so that 16 lanes hold a block of 128 and its largest magnitude is four shuffles away.  The 8-bit
// result is rounded from the 32-bit one, not from its half-precision copy.  gamma and beta in shared memory, the next row's loads
// in flight while this one is reduced.  With a residual 32768 x 768 f16 31.5 us, 0.85 of the measured copy rate; without one, or where a
// row does not fill its warps' lanes, bound by instructions and the latency of shuffles and shared memory (0.75; 2096 columns 0.53;
// two rows on their way were slower from 1024 columns on: 31 against 28 us).
__device__ __forceinline__ void decode8(const uint4& q, int dtype, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2(w[e], dtype);
        v[2 * e] = f.x;
        v[2 * e + 1] = f.y;
    }
}

template <int NV, int G, int DT, bool RESID>
__global__ void __launch_bounds__(256) add_layernorm_fp8_kernel(B200LayerNormFp8Desc d) {
    extern __shared__ float gb[];   // gamma, then beta: group-major, the 8 elements of a lane's group in two float4 planes
    __shared__ float part[2][8];    // the warps' sums and sums of squares, where a row has several warps
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp % G;
    const int H = static_cast<int>(d.H);
    const int groups = H >> 3;
    float* beta_s = gb + NV * G * 256;
    pdl_launch_dependents();
    pdl_wait();   // gamma and beta too may have been written by the kernel in front
    const long long step = static_cast<long long>(gridDim.x) * (8 / G);
    uint4 raw[NV], res[RESID ? NV : 1];
    auto fetch = [&](long long row) {
        if (row >= d.rows) return;
#pragma unroll
        for (int g = 0; g < NV; ++g) {
            const int gi = (g * G + w) * 32 + lane;
            raw[g] = make_uint4(0, 0, 0, 0);
            if (RESID) res[g] = make_uint4(0, 0, 0, 0);
            if (gi < groups) {
                raw[g] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(d.x) + row * d.ldx + gi * 8));
                if (RESID) res[g] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(d.residual) + row * d.ldr + gi * 8));
            }
        }
    };
    // the sum over a row's lanes; all of a row's warps come here the same number of times
    auto row_sum = [&](float v, float* slots) -> float {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (G > 1) {
            if (lane == 0) slots[warp] = v;
            asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + warp / G), "n"(32 * G) : "memory");
            v = slots[warp - w];
#pragma unroll
            for (int i = 1; i < G; ++i) v += slots[warp - w + i];
        }
        return v;
    };
    long long row = static_cast<long long>(blockIdx.x) * (8 / G) + warp / G;
    fetch(row);
    for (int i = threadIdx.x; i < NV * G * 256; i += 256) {
        const int g = i >> 8, r = i & 255, l = r >> 3, e = r & 7;
        const int at = (g * 2 + (e >> 2)) * 128 + l * 4 + (e & 3);   // conflict-free float4 per lane
        gb[at] = i < H ? __ldg(d.gamma + i) : 0.f;
        beta_s[at] = i < H ? __ldg(d.beta + i) : 0.f;
    }
    __syncthreads();
    const float inv_h = 1.0f / static_cast<float>(H);
    for (; row < d.rows; row += step) {
        float v[NV][8];
        float sum = 0.f;
#pragma unroll
        for (int g = 0; g < NV; ++g) {
            decode8(raw[g], DT, v[g]);
            if (RESID) {
                float r[8];
                decode8(res[g], DT, r);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[g][e] += r[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += v[g][e];
        }
        fetch(row + step);
        const float mean = row_sum(sum, part[0]) * inv_h;
        float sq = 0.f;
#pragma unroll
        for (int g = 0; g < NV; ++g)
            if ((g * G + w) * 32 + lane < groups) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[g][e] -= mean;
                    sq = fmaf(v[g][e], v[g][e], sq);
                }
            }
        const float rstd = 1.0f / sqrtf(fmaf(row_sum(sq, part[1]), inv_h, d.eps));
#pragma unroll
        for (int g = 0; g < NV; ++g) {
            const int ch = g * G + w, gi = ch * 32 + lane;
            uint32_t bits = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 gm = *reinterpret_cast<const float4*>(gb + (ch * 2 + h) * 128 + lane * 4);
                const float4 bt = *reinterpret_cast<const float4*>(beta_s + (ch * 2 + h) * 128 + lane * 4);
                v[g][h * 4 + 0] = fmaf(v[g][h * 4 + 0] * rstd, gm.x, bt.x);
                v[g][h * 4 + 1] = fmaf(v[g][h * 4 + 1] * rstd, gm.y, bt.y);
                v[g][h * 4 + 2] = fmaf(v[g][h * 4 + 2] * rstd, gm.z, bt.z);
                v[g][h * 4 + 3] = fmaf(v[g][h * 4 + 3] * rstd, gm.w, bt.w);
            }
            if (gi < groups) {
#pragma unroll
                for (int e = 0; e < 8; ++e) bits = max(bits, fp8::abs_bits(v[g][e]));
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
            if (gi < groups) {
                const float amax = fp8::amax_of_bits(bits);
                const float enc = fp8::encode_scale(amax);
                if (d.y) {
                    uint4 q;
                    q.x = pack2t<DT>(v[g][0], v[g][1]);
                    q.y = pack2t<DT>(v[g][2], v[g][3]);
                    q.z = pack2t<DT>(v[g][4], v[g][5]);
                    q.w = pack2t<DT>(v[g][6], v[g][7]);
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(d.y) + row * d.ldy + gi * 8) = q;
                }
                uint2 c;
                c.x = fp8::pack4(v[g][0] * enc, v[g][1] * enc, v[g][2] * enc, v[g][3] * enc);
                c.y = fp8::pack4(v[g][4] * enc, v[g][5] * enc, v[g][6] * enc, v[g][7] * enc);
                *reinterpret_cast<uint2*>(static_cast<uint8_t*>(d.q) + row * d.ldq + gi * 8) = c;
                if ((lane & 15) == 0) d.scale[(gi >> 4) * d.ld_scale + row] = fp8::decode_scale(amax);
            }
        }
    }
}

// ---------------------------------------------------------------- weight pre-pack
// fp32 w_kn[K, N] -> e4m3 w_nk[N, K] and one scale per 128 x 128 block.  A CTA per block; runs once, at load time: the
// block is read twice (its largest magnitude first), transposed through shared memory 32 columns of N at a time.
__global__ void __launch_bounds__(256) pack_weight_fp8_kernel(const float* src, long long K, long long N, long long ld_src,
                                                              uint8_t* dst, long long ld_dst, float* scale, int kblocks) {
    __shared__ uint32_t red[8];
    __shared__ float tile[128][33];
    const long long k0 = static_cast<long long>(blockIdx.x) * 128, n0 = static_cast<long long>(blockIdx.y) * 128;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    uint32_t bits = 0;
    for (int k = ty; k < 128 && k0 + k < K; k += 8)
        for (int n = tx; n < 128 && n0 + n < N; n += 32) bits = max(bits, fp8::abs_bits(src[(k0 + k) * ld_src + n0 + n]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    if (tx == 0) red[ty] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) bits = max(bits, red[w]);
    const float amax = fp8::amax_of_bits(bits);
    const float enc = fp8::encode_scale(amax);
    if (threadIdx.x == 0) scale[static_cast<long long>(blockIdx.y) * kblocks + blockIdx.x] = fp8::decode_scale(amax);
    for (int c = 0; c < 128; c += 32) {
        __syncthreads();
        for (int k = ty; k < 128; k += 8)
            tile[k][tx] = (k0 + k < K && n0 + c + tx < N) ? src[(k0 + k) * ld_src + n0 + c + tx] : 0.f;
        __syncthreads();
        for (int n = ty; n < 32 && n0 + c + n < N; n += 8)
            if (k0 + tx * 4 < K)   // K is a multiple of 16
                *reinterpret_cast<uint32_t*>(dst + (n0 + c + n) * ld_dst + k0 + tx * 4) =
                    fp8::pack4(tile[tx * 4][n] * enc, tile[tx * 4 + 1][n] * enc, tile[tx * 4 + 2][n] * enc, tile[tx * 4 + 3][n] * enc);
    }
}

constexpr int kQuantizeCtas = 3;   // resident CTAs per SM

template <int NV, int G, int DT, bool RESID>
int launch_layernorm_fp8(int sms, cudaStream_t stream, const B200LayerNormFp8Desc& d) {
    static PerDeviceOnce once;
    static std::atomic<int> resident[kMaxDevices];   // CTAs per SM: the grid is what runs at once, every warp walks rows
    const size_t smem = static_cast<size_t>(NV) * G * 256 * 2 * sizeof(float);
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return B200_ERR_LAUNCH;
    if (!once.ensure(dev, [&]() {
            int n = 0;
            if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, add_layernorm_fp8_kernel<NV, G, DT, RESID>, 256, smem) != cudaSuccess || n < 1)
                return false;
            resident[dev].store(n, std::memory_order_relaxed);
            return true;
        }))
        return B200_ERR_LAUNCH;
    const long long ctas = (d.rows * G + 7) / 8, most = static_cast<long long>(sms) * resident[dev].load(std::memory_order_relaxed);
    launch_kernel(add_layernorm_fp8_kernel<NV, G, DT, RESID>, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256), smem, stream, d);
    count_launch();
    return check_launch();
}

template <int DT, bool RESID>
int choose_layernorm_fp8(int sms, cudaStream_t stream, const B200LayerNormFp8Desc& d) {
    // As few warps per row as let a lane hold 24 values at most.  us for 25 million values, without | with a residual: 1024 columns
    // one warp 27.7 | 33.8, two 27.1 | 32.9; 2048 columns two warps 32.3 | 34.8, four 29.7 | 34.0; 4096 columns four warps
    // 36.2 | 39.1, eight 32.7 | 37.8; 768 columns one warp 25.5 | 31.4, two 31.2 | 35.2; 1536 two 27.4 | 38.9, four 33.1 | 40.3.
    // (One warp for every width: 1024 27.7 | 38.1, 2096 64 | 92, 4096 47 | 73.)
    int G = 1;
    while (d.H > 768 * G) G *= 2;
    const int nv = static_cast<int>((d.H + 256 * G - 1) / (256 * G));
    switch (G) {
        case 1: return nv <= 1 ? launch_layernorm_fp8<1, 1, DT, RESID>(sms, stream, d)
                               : (nv <= 2 ? launch_layernorm_fp8<2, 1, DT, RESID>(sms, stream, d) : launch_layernorm_fp8<3, 1, DT, RESID>(sms, stream, d));
        case 2: return nv <= 2 ? launch_layernorm_fp8<2, 2, DT, RESID>(sms, stream, d) : launch_layernorm_fp8<3, 2, DT, RESID>(sms, stream, d);
        case 4: return nv <= 2 ? launch_layernorm_fp8<2, 4, DT, RESID>(sms, stream, d) : launch_layernorm_fp8<3, 4, DT, RESID>(sms, stream, d);
        default: return launch_layernorm_fp8<2, 8, DT, RESID>(sms, stream, d);
    }
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_quantize_fp8(const B200QuantizeFp8Desc* d, b200_stream_t stream_) {
    using namespace b200;
    if (!d || !d->x || !d->q || !d->scale) return B200_ERR_PARAM;
    if (d->rows < 0 || d->K <= 0) return B200_ERR_PARAM;
    if (d->x_dtype != B200_F16 && d->x_dtype != B200_BF16 && d->x_dtype != B200_F32) return B200_ERR_PARAM;
    const int64_t per16 = d->x_dtype == B200_F32 ? 4 : 8;   // elements in 16 bytes
    if ((d->K % 16) || (d->ldx % per16) || (d->ldq % 16) || d->ldx < d->K || d->ldq < d->K || d->ld_scale < d->rows)
        return B200_ERR_PARAM;
    if (!aligned16(d->x) || !aligned16(d->q)) return B200_ERR_PARAM;
    if (d->rows > (1ll << 31) - 1 || d->K > (1ll << 24)) return B200_ERR_UNSUPPORTED;
    if (d->rows == 0) return B200_OK;
    const int sms = lin::device_sm_count();
    if (sms <= 0) return B200_ERR_NOT_SM100;
    const int blocks = static_cast<int>((d->K + fp8::kBlock - 1) / fp8::kBlock);
    const long long ctas = (d->rows * blocks + 31) / 32;
    const long long most = static_cast<long long>(sms) * kQuantizeCtas;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const dim3 grid(static_cast<unsigned>(ctas < most ? ctas : most));
    if (d->x_dtype == B200_F16) launch_kernel(quantize_fp8_kernel<B200_F16>, grid, dim3(256), 0, stream, *d, blocks);
    else if (d->x_dtype == B200_BF16) launch_kernel(quantize_fp8_kernel<B200_BF16>, grid, dim3(256), 0, stream, *d, blocks);
    else launch_kernel(quantize_fp8_kernel<B200_F32>, grid, dim3(256), 0, stream, *d, blocks);
    count_launch();
    return check_launch();
}

int b200_add_layernorm_fp8_fwd(const B200LayerNormFp8Desc* d, b200_stream_t stream_) {
    using namespace b200;
    if (!d || !d->x || !d->q || !d->scale || !d->gamma || !d->beta) return B200_ERR_PARAM;
    if (d->rows < 0 || d->H <= 0 || !is_half_dtype(d->dtype)) return B200_ERR_PARAM;
    if ((d->H % 16) || (d->ldx % 8) || (d->ldq % 16) || d->ldx < d->H || d->ldq < d->H || d->ld_scale < d->rows)
        return B200_ERR_PARAM;
    if (d->residual && ((d->ldr % 8) || d->ldr < d->H || !aligned16(d->residual))) return B200_ERR_PARAM;
    if (d->y && ((d->ldy % 8) || d->ldy < d->H || !aligned16(d->y))) return B200_ERR_PARAM;
    if (!aligned16(d->x) || !aligned16(d->q) || !aligned16(d->gamma) || !aligned16(d->beta)) return B200_ERR_PARAM;
    if (d->H > 4096 || d->rows > (1ll << 31) - 1) return B200_ERR_UNSUPPORTED;
    if (d->rows == 0) return B200_OK;
    const int sms = lin::device_sm_count();
    if (sms <= 0) return B200_ERR_NOT_SM100;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (d->dtype == B200_F16)
        return d->residual ? choose_layernorm_fp8<B200_F16, true>(sms, stream, *d) : choose_layernorm_fp8<B200_F16, false>(sms, stream, *d);
    return d->residual ? choose_layernorm_fp8<B200_BF16, true>(sms, stream, *d) : choose_layernorm_fp8<B200_BF16, false>(sms, stream, *d);
}

int b200_pack_weight_fp8(const float* w_kn, int64_t K, int64_t N, int64_t ld_src, void* w_nk, int64_t ld_dst, float* w_scale,
                         b200_stream_t stream_) {
    using namespace b200;
    if (!w_kn || !w_nk || !w_scale || K <= 0 || N <= 0 || ld_src < N || ld_dst < K || (K % 16) || (ld_dst % 16) || !aligned16(w_nk))
        return B200_ERR_PARAM;
    if (K > (1ll << 24) || N > 65535ll * 128) return B200_ERR_UNSUPPORTED;
    if (lin::device_sm_count() <= 0) return B200_ERR_NOT_SM100;
    const int kblocks = static_cast<int>((K + 127) / 128);
    const dim3 grid(static_cast<unsigned>(kblocks), static_cast<unsigned>((N + 127) / 128));
    pack_weight_fp8_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream_)>>>(w_kn, K, N, ld_src, static_cast<uint8_t*>(w_nk),
                                                                               ld_dst, w_scale, kblocks);
    count_launch();
    return check_launch();
}

}  // extern "C"
