// Projection / FFN GEMM on 8-bit operands with block scales:
//   y[m, n] = epilogue(sum_b xs[b, m] * ws[n / 128, b] * sum_{k in block b} x8[m, k] w8[n, k] + bias[n] (+ r[m, n])).
//
// The scales change every 128 values of K, so the tensor core may not add across blocks.  A k-block of a pipeline stage is
// exactly one scale block (128 e4m3 values = one 128-byte swizzled row): its four UMMAs (kind::f8f6f4, K = 32 each) start a
// fresh accumulator in a TMEM buffer, and the epilogue warps add scale * buffer to fp32 sums that stay in their registers for
// the whole tile (thread = row, COLS columns), while the tensor pipe fills the other buffers.  Products are exact in fp32; the
// sum inside a block is the tensor core's fp32 accumulation, the sum over blocks one fp32 FMA each, in ascending order whatever
// the tile, so among the tiles of this file a row's result depends on neither the batch nor the tile chosen (calls of up to 128
// rows may go to linear_fp8_rows.cu, which adds in another order).
//
// A tile is 128 x BN on one SM.
//   warp 0      : TMA producer
//   warp 1      : TMEM allocation, UMMA issue (one elected lane)
//   warps 2, 3  : scales, x_scale * w_scale per row, one warp per 128 columns
//   warps 4 ..  : EW epilogue warps: scale and add, then bias / activation / residual and the store
//
// What bounds it is the chain of a TMEM buffer: UMMAs, commit, reads, hand-back; the reads and the next k-block's accumulation
// share TMEM.  On 256 columns a k-block costs 0.48 us (its UMMAs alone 0.32), a tile 2.6 us beside its k-blocks.
// 16384 x 4096 x 4096 with an f16 result 277 to 300 us (1830 to 1980 TFLOP/s; 14 waves at those costs would take 252, but at K = 4096
// the clock gives way to the power limit), K = 1024 96 to 107 us, f32 108, e4m3 with GELU 121, 4096 -> 1024 with a residual 92.
// Pairs of CTAs on 256 x 256 and 256 x 128 tiles took 107 and 113 us at K = 1024.  Two CTAs per SM on 128 x 128 tiles, against this form
// then: bias 95 | 95, f32 106 | 111, e4m3 94 | 102, but GELU 157 | 128 and residual 160 | 124.
// ops.linear on half-precision operands is the faster one from 128 rows on at K = 768 and 1024 (16384 rows 1024 -> 4096 93 | 107 us); this
// one is for half the weight bytes, for a few rows (1.2 to 3 times) and for K of some thousands (16384 x 4096 x 4096 357 | 300).
// For up to 128 rows and few columns linear_fp8_rows.cu does the same without a pipeline.
#include "fp8.cuh"
#include "linear_common.cuh"
#include "linear_fp8.cuh"

namespace b200 {
namespace lin {

namespace {

enum { kOutHalf = 0, kOutF32 = 1, kOutF8 = 2 };

struct LinearFp8Params {
    const float* x_scale;
    const float* w_scale;
    const float* bias;
    float* y_scale;
    int M, N;
    int num_n_tiles, num_tiles, num_k_blocks, w_blocks;   // w_blocks = ceil(N / 128)
    int x_rows;                                           // rows of x in a load box
    int out_dtype, res_dtype, epilogue;
    long long ld_xs, ld_ys;
    uint32_t idesc;
    unsigned int* status;
};

template <int BN, int EW>
struct Fp8Cfg {
    static constexpr int THREADS = 128 + 32 * EW;        // a control warpgroup, EW / 4 epilogue warpgroups
    static constexpr int COLS = BN / (EW / 4);           // accumulator columns per epilogue warp
    static constexpr int NBUF = BN == 256 ? 2 : 4;       // TMEM buffers of BN columns
    static constexpr int TMEM_COLS = BN * NBUF;
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_BYTES = BN * 128;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STRIP_BYTES = 32 * 128;         // 32 rows of 128 bytes
    static constexpr int STRIPS = 2;                     // per epilogue warp: output staging, before that the residual
    static constexpr int BIAS_BYTES = EW * COLS * 4;
    static constexpr int GROUPS = BN == 256 ? 2 : 1;     // 128-column scale blocks of a tile, a scale warp each
    static constexpr int SCALE_BYTES = GROUPS * NBUF * 128 * 4;   // one per row, group and TMEM buffer
    static constexpr int TAIL_BYTES = EW * STRIPS * STRIP_BYTES + BIAS_BYTES + SCALE_BYTES + 512;
    static constexpr int FIT = (227 * 1024 - 1024 - TAIL_BYTES) / STAGE_BYTES;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int OUT_OFFSET = STAGES * STAGE_BYTES;
    static constexpr int BIAS_OFFSET = OUT_OFFSET + EW * STRIPS * STRIP_BYTES;
    static constexpr int SCALE_OFFSET = BIAS_OFFSET + BIAS_BYTES;
    static constexpr int BAR_OFFSET = SCALE_OFFSET + SCALE_BYTES;
    static constexpr int SMEM_BYTES = OUT_OFFSET + TAIL_BYTES + 1024;
    // 128 sums per thread and 32 values in flight do not fit the 168 registers that 384 threads get at launch (with them
    // spilled, a k-block's promotion took 0.9 us instead of 0.4): the control warpgroup hands most of its own over.
    static constexpr bool MOVE_REGS = EW == 8 && COLS == 128;
    static constexpr int REGS_CONTROL = 56, REGS_EPILOGUE = 224;
    static_assert(!MOVE_REGS || 128 * REGS_CONTROL + 256 * REGS_EPILOGUE <= THREADS * (65536 / THREADS / 8 * 8),
                  "setmaxnreg: the epilogue's registers must come out of the CTA's own pool");
    static_assert(STAGES >= 3 && TMEM_COLS <= 512 && COLS % 64 == 0, "tile does not fit");
};

template <int BN, int EW, int OUT>
__global__ void __launch_bounds__(128 + 32 * EW, 1)
linear_fp8_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_r, const LinearFp8Params p) {
    using C = Fp8Cfg<BN, EW>;
    constexpr int STAGES = C::STAGES, NBUF = C::NBUF, COLS = C::COLS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFFSET);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + NBUF;
    uint64_t* res_full = acc_empty + NBUF;              // [EW]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + EW);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    float* scale_s = reinterpret_cast<float*>(smem + C::SCALE_OFFSET);   // [NBUF][GROUPS][128]

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);    // the producer's expect_tx arrival
            mbar_init(&empty[s], 1);   // an epilogue warp, once the stage's UMMAs are done
        }
        for (int b = 0; b < NBUF; ++b) {
            mbar_init(&acc_full[b], 1 + C::GROUPS);   // the UMMAs' commit and the scale warps
            mbar_init(&acc_empty[b], EW);
        }
        for (int w = 0; w < EW; ++w) mbar_init(&res_full[w], 1);
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tm_x);
        prefetch_tmap(&tm_w);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        // The weights' way from HBM to L2 starts while the previous kernel of the stream drains (a hint, no data is taken).
        for (int b = blockIdx.x; b < p.num_k_blocks * p.num_n_tiles; b += gridDim.x)
            tma_prefetch_l2_2d(&tm_w, (b % p.num_k_blocks) * 64, (b / p.num_k_blocks) * BN);
    }
    pdl_wait();

    if (warp < 4) {
        if (C::MOVE_REGS) setmaxnreg_dec<C::REGS_CONTROL>();
        if (warp == 0) {
            // -------------------------------------------------------- TMA producer
            if (elect_one()) {
                uint32_t st = 0, ph = 0;
                bool ok = true;
                const uint32_t bytes = static_cast<uint32_t>(p.x_rows) * 128 + C::B_BYTES;
                for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x) {
                    const int x_row = tile / p.num_n_tiles * 128, w_row = tile % p.num_n_tiles * BN;
                    for (int kb = 0; kb < p.num_k_blocks; ++kb) {
                        if (!mbar_wait(&empty[st], ph ^ 1u, abort_flag)) { ok = false; break; }
                        uint8_t* a = smem + st * C::STAGE_BYTES;
                        mbar_expect_tx(&full[st], bytes);
                        // the maps count 16-bit units: a k-block is 64 of them
                        tma_load_2d(a, &tm_x, &full[st], kb * 64, x_row);
                        tma_load_2d(a + C::A_BYTES, &tm_w, &full[st], kb * 64, w_row);
                        if (++st == STAGES) { st = 0; ph ^= 1u; }
                    }
                }
            }
        } else if (warp == 1) {
            // -------------------------------------------------------- UMMA issuer
            if (elect_one()) {
                uint32_t st = 0, ph = 0, buf = 0, bph = 0;
                bool ok = true;
                const uint64_t a_desc0 = make_smem_desc_sw128(smem_u32(smem));
                const uint64_t b_desc0 = make_smem_desc_sw128(smem_u32(smem + C::A_BYTES));
                for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x) {
                    for (int kb = 0; kb < p.num_k_blocks; ++kb) {
                        if (!mbar_wait(&full[st], ph, abort_flag) || !mbar_wait(&acc_empty[buf], bph ^ 1u, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tcgen05_fence_after();
                        const uint32_t d_tmem = tmem_base + buf * BN;
                        const uint64_t a_desc = a_desc0 + static_cast<uint64_t>(st * (C::STAGE_BYTES >> 4));
                        const uint64_t b_desc = b_desc0 + static_cast<uint64_t>(st * (C::STAGE_BYTES >> 4));
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_f8_ss(d_tmem, a_desc + 2 * k, b_desc + 2 * k, p.idesc, k != 0 ? 1u : 0u);
                        // One commit a k-block (each costs the tensor pipe 30 to 60 clocks): the epilogue hands the stage back.
                        umma_f8_commit(&acc_full[buf]);
                        if (++st == STAGES) { st = 0; ph ^= 1u; }
                        if (++buf == NBUF) { buf = 0; bph ^= 1u; }
                    }
                }
            }
        } else if (warp - 2 < C::GROUPS) {
            // -------------------------------------------------------- scales: x_scale * w_scale of the rows and a column group
            // Loads U k-blocks ahead, over the end of a tile too: their way from L2 is longer than a k-block.  Slot u holds
            // k-blocks u, u + U, ... of a tile, then u of the next one.
            constexpr int U = 2;
            const int g = warp - 2;
            float x[U][4], w[U];
            const float *xs = nullptr, *ws = nullptr, *xs_next = nullptr, *ws_next = nullptr;
            int there = 0, there_next = 0;   // how many of this lane's four rows exist
            auto locate = [&](int tile) {
                const int r = tile / p.num_n_tiles * 128 + lane;
                const int b = (tile % p.num_n_tiles * BN + g * 128) / fp8::kBlock;
                xs_next = p.x_scale + r;
                ws_next = p.w_scale + static_cast<long long>(b < p.w_blocks ? b : p.w_blocks - 1) * p.num_k_blocks;
                there_next = (p.M - r + 31) >> 5;
            };
            auto fetch = [&](const float* px, const float* pw, int in, int kb, float (&xv)[4], float& wv) {
                wv = __ldg(pw + kb);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < in) xv[i] = __ldg(px + kb * p.ld_xs + 32 * i);
            };
            uint32_t buf = 0, bph = 0;
            bool ok = true;
            if (static_cast<int>(blockIdx.x) < p.num_tiles) locate(blockIdx.x);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                w[u] = x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
                if (static_cast<int>(blockIdx.x) < p.num_tiles && u < p.num_k_blocks) fetch(xs_next, ws_next, there_next, u, x[u], w[u]);
            }
            for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x) {
                xs = xs_next;
                ws = ws_next;
                there = there_next;
                const bool more = tile + static_cast<int>(gridDim.x) < p.num_tiles;
                if (more) locate(tile + gridDim.x);
                for (int kb0 = 0; ok && kb0 < p.num_k_blocks; kb0 += U) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int kb = kb0 + u;
                        if (kb >= p.num_k_blocks) break;
                        if (!mbar_wait(&acc_empty[buf], bph ^ 1u, abort_flag)) { ok = false; break; }
                        float* s = scale_s + (buf * C::GROUPS + g) * 128 + lane;
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[32 * i] = x[u][i] * w[u];
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_full[buf]);
                        if (kb + U < p.num_k_blocks) fetch(xs, ws, there, kb + U, x[u], w[u]);
                        else if (more) fetch(xs_next, ws_next, there_next, u, x[u], w[u]);
                        if (++buf == NBUF) { buf = 0; bph ^= 1u; }
                    }
                }
            }
        }
        __syncwarp();
    } else {
        if (C::MOVE_REGS) setmaxnreg_inc<C::REGS_EPILOGUE>();
        // ------------------------------------------------------------ scale, add, store (own 128 rows)
        const int ew = warp - 4;
        const int quarter = warp & 3;
        const int col_first = (ew >> 2) * COLS;
        uint8_t* strips = smem + C::OUT_OFFSET + ew * C::STRIPS * C::STRIP_BYTES;
        const int sw = lane & 7;            // 128-byte swizzle: 16-byte piece i of row r lies at i ^ (r & 7)
        float* bias_s = reinterpret_cast<float*>(smem + C::BIAS_OFFSET) + ew * COLS;
        const uint32_t tacc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + col_first;
        const bool res = p.epilogue == B200_EPI_BIAS_RESIDUAL;
        uint32_t buf = 0, bph = 0, st = 0, rph = 0, stored = 0;   // stored: strips sent off, the two in turn
        bool ok = true;
        const float* my_scale = scale_s + col_first / 128 * 128 + quarter * 32 + lane;
        const uint32_t first_lane = lane == 0;
        for (int tile = blockIdx.x; ok && tile < p.num_tiles; tile += gridDim.x) {
            const int row0 = tile / p.num_n_tiles * 128 + quarter * 32;
            const int n_first = tile % p.num_n_tiles * BN + col_first;
            // what this warp stores of the tile: 64-column pieces of its 32 rows (the store clips what lies outside y)
            const int pieces = row0 < p.M && n_first < p.N ? min(COLS / 64, (p.N - n_first + 63) / 64) : 0;
            __syncwarp();   // every lane has read the previous tile's bias
            if (p.bias != nullptr) {
#pragma unroll
                for (int i = 0; i < COLS / 32; ++i) {
                    const int n = n_first + i * 32 + lane;
                    bias_s[i * 32 + lane] = n < p.N ? __ldg(p.bias + n) : 0.f;
                }
            }
            uint64_t acc[COLS / 2];
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
            // 32 columns travel while the 32 before them are added, across k-blocks too: the chain of wait, load, release of one
            // warp is what bounds a k-block.
            uint32_t r[2][32];
            float scale = 0.f;
            auto open = [&]() -> bool {   // the next buffer: its first 32 columns and its scale
                if (!mbar_wait(&acc_full[buf], bph, abort_flag)) return false;
                __syncwarp();
                tcgen05_fence_after();
                tmem_ld_32x32b_x32(tacc + buf * BN, r[0]);
                scale = my_scale[buf * (C::GROUPS * 128)];
                return true;
            };
            ok = open();
#pragma unroll 1
            for (int kb = 0; ok && kb < p.num_k_blocks; ++kb) {
                const uint64_t s2 = pack_f32x2(scale, scale);
#pragma unroll
                for (int c = 0; c < COLS / 32; ++c) {
                    tmem_ld_wait(r[c & 1]);
                    if (c + 1 < COLS / 32) {
                        tmem_ld_32x32b_x32(tacc + buf * BN + (c + 1) * 32, r[(c + 1) & 1]);
                    } else {   // the buffer is in registers: hand it back, and the stage
                        tcgen05_fence_before();
                        __syncwarp();
                        mbar_arrive_if(&acc_empty[buf], first_lane);
                        mbar_arrive_if(&empty[st], first_lane & (ew == 0));
                        if (++st == STAGES) st = 0;
                        if (++buf == NBUF) { buf = 0; bph ^= 1u; }
                        if (kb + 1 < p.num_k_blocks) ok = open();
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        acc[c * 16 + j] = fma_f32x2(pack_f32x2(__uint_as_float(r[c & 1][2 * j]), __uint_as_float(r[c & 1][2 * j + 1])), s2,
                                                    acc[c * 16 + j]);
                }
                if (kb == 0 && res && pieces > 0 && lane == 0) {
                    // the residual of this tile into the strips, which the previous tile's stores have read by now
                    tma_store_wait_read<0>();
                    mbar_expect_tx(&res_full[ew], static_cast<uint32_t>(pieces) * C::STRIP_BYTES);
                    for (int i = 0; i < pieces; ++i)
                        tma_load_2d(strips + i * C::STRIP_BYTES, &tm_r, &res_full[ew], n_first + i * 64, row0);
                }
            }
            if (!ok) break;
            if (pieces == 0) continue;
            if (res) {
                if (!mbar_wait(&res_full[ew], rph, abort_flag)) { ok = false; break; }
                rph ^= 1u;
                __syncwarp();
            }

            // bias, activation, residual: 32 columns in place
            float top = 0.f;
            auto finish = [&](int c, float (&v)[32]) {
#pragma unroll
                for (int j = 0; j < 16; ++j) unpack_f32x2(acc[c * 16 + j], v[2 * j], v[2 * j + 1]);
                if (p.bias != nullptr) {
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        const float4 b = *reinterpret_cast<const float4*>(bias_s + c * 32 + g * 4);
                        unpack_f32x2(add_f32x2(pack_f32x2(v[g * 4 + 0], v[g * 4 + 1]), pack_f32x2(b.x, b.y)), v[g * 4 + 0], v[g * 4 + 1]);
                        unpack_f32x2(add_f32x2(pack_f32x2(v[g * 4 + 2], v[g * 4 + 3]), pack_f32x2(b.z, b.w)), v[g * 4 + 2], v[g * 4 + 3]);
                    }
                }
                if (p.epilogue == B200_EPI_BIAS_GELU) {
                    if (OUT == kOutF32) {   // nothing rounds the result: the library's erf
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0.5f * v[j] * (1.0f + erff(v[j] * 0.70710678118654752f));
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) gelu_tail_x2(v[j], v[j + 1]);
                    }
                } else if (p.epilogue == B200_EPI_BIAS_TANH) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        // (2^-11 relative: an error of the size of an f16 result's own rounding, less than bf16's and e4m3's; the
                        // epilogue's instructions are what a tile waits for.  linear_fp8_rows.cu, which waits for memory, calls tanhf.)
                        if (OUT == kOutF32) v[j] = tanhf(v[j]);
                        else asm("tanh.approx.f32 %0, %1;" : "=f"(v[j]) : "f"(v[j]));
                    }
                } else if (res && c / 2 < pieces) {
                    const uint8_t* srow = strips + (c / 2) * C::STRIP_BYTES + lane * 128;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const uint4 q = *reinterpret_cast<const uint4*>(srow + ((((c & 1) * 4 + g) ^ sw) << 4));
                        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = unpack2(w[e], p.res_dtype);
                            v[g * 8 + 2 * e] += f.x;
                            v[g * 8 + 2 * e + 1] += f.y;
                        }
                    }
                }
            };
            if (OUT == kOutHalf) {
                // a strip holds 64 columns; with a residual a thread replaces its own row's values in it
#pragma unroll
                for (int h = 0; h < COLS / 64; ++h) {
                    if (h >= pieces) break;
                    uint8_t* strip = strips + (res ? h : (stored++ & 1u)) * C::STRIP_BYTES;
                    uint8_t* srow = strip + lane * 128;
                    if (!res) {   // the store before the last one has read its strip
                        if (lane == 0) tma_store_wait_read<1>();
                        __syncwarp();
                    }
#pragma unroll
                    for (int cc = 0; cc < 2; ++cc) {
                        float v[32];
                        finish(h * 2 + cc, v);
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            uint4 q;
                            q.x = pack2(v[g * 8 + 0], v[g * 8 + 1], p.out_dtype);
                            q.y = pack2(v[g * 8 + 2], v[g * 8 + 3], p.out_dtype);
                            q.z = pack2(v[g * 8 + 4], v[g * 8 + 5], p.out_dtype);
                            q.w = pack2(v[g * 8 + 6], v[g * 8 + 7], p.out_dtype);
                            *reinterpret_cast<uint4*>(srow + (((cc * 4 + g) ^ sw) << 4)) = q;
                        }
                    }
                    fence_async_proxy_shared();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_y, strip, n_first + h * 64, row0);
                        tma_store_commit();
                    }
                }
            } else {
                if (OUT == kOutF8 || res) {   // everything but the store first: the strips' residual makes way for the output
#pragma unroll
                    for (int c = 0; c < COLS / 32; ++c) {
                        float v[32];
                        finish(c, v);
                        if (OUT == kOutF8) {
                            // columns at or beyond N are zeros (no weight, no bias, no residual): they do not move the maximum
#pragma unroll
                            for (int j = 0; j < 32; j += 2) top = fp8::amax3(top, v[j], v[j + 1]);
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[c * 16 + j] = pack_f32x2(v[2 * j], v[2 * j + 1]);
                    }
                    __syncwarp();
                }
                if (OUT == kOutF32) {
#pragma unroll
                    for (int c = 0; c < COLS / 32; ++c) {
                        if (n_first + c * 32 >= p.N) break;
                        uint8_t* strip = strips + (stored++ & 1u) * C::STRIP_BYTES;
                        uint8_t* srow = strip + lane * 128;
                        float v[32];
                        if (res) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) unpack_f32x2(acc[c * 16 + j], v[2 * j], v[2 * j + 1]);
                        } else {
                            finish(c, v);
                        }
                        if (lane == 0) tma_store_wait_read<1>();   // the store before the last one has read its strip
                        __syncwarp();
#pragma unroll
                        for (int g = 0; g < 8; ++g)
                            *reinterpret_cast<float4*>(srow + ((g ^ sw) << 4)) = make_float4(v[g * 4], v[g * 4 + 1], v[g * 4 + 2], v[g * 4 + 3]);
                        fence_async_proxy_shared();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&tm_y, strip, 2 * (n_first + c * 32), row0);
                            tma_store_commit();
                        }
                    }
                } else {
                    const float amax = fp8::amax_of_bits(fp8::abs_bits(top));
                    const float enc = fp8::encode_scale(amax);
                    const uint64_t enc2 = pack_f32x2(enc, enc);
                    uint8_t* srow = strips + lane * 128;
                    if (lane == 0) tma_store_wait_read<0>();
                    __syncwarp();
#pragma unroll
                    for (int g = 0; g < COLS / 16; ++g) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float a0, a1, a2, a3;
                            unpack_f32x2(mul_f32x2(acc[g * 8 + e * 2], enc2), a0, a1);
                            unpack_f32x2(mul_f32x2(acc[g * 8 + e * 2 + 1], enc2), a2, a3);
                            w[e] = fp8::pack4(a0, a1, a2, a3);
                        }
                        *reinterpret_cast<uint4*>(srow + ((g ^ sw) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (row0 + lane < p.M) p.y_scale[n_first / fp8::kBlock * p.ld_ys + row0 + lane] = fp8::decode_scale(amax);
                    fence_async_proxy_shared();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tm_y, strips, n_first / 2, row0);
                        tma_store_commit();
                    }
                }
            }
        }
        if (lane == 0) tma_store_wait_read<0>();
        __syncwarp();
    }

    // ---------------------------------------------------------------- teardown
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (*abort_flag != 0) let_copies_land();
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
    if (threadIdx.x == 0 && *abort_flag != 0 && p.status != nullptr) atomicOr(p.status, 1u);
}

template <int BN, int EW, int OUT>
int launch_linear_fp8(const B200LinearFp8Desc& d, cudaStream_t stream, int sms) {
    using C = Fp8Cfg<BN, EW>;
    static PerDeviceOnce once;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return B200_ERR_LAUNCH;
    if (!once.ensure(dev, []() {
            return cudaFuncSetAttribute(linear_fp8_kernel<BN, EW, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES) ==
                   cudaSuccess;
        }))
        return B200_ERR_LAUNCH;
    // Rows that do not exist are not fetched where all rows fit one box: what the stage holds there feeds no stored row.
    const int x_rows = d.M < 128 ? static_cast<int>((d.M + 7) / 8 * 8) : 128;
    CUtensorMap tx, tw, ty, tr;
    {   // two e4m3 values as one 16-bit element
        const uint64_t xd[2] = {static_cast<uint64_t>(d.K / 2), static_cast<uint64_t>(d.M)};
        const uint64_t xs[1] = {static_cast<uint64_t>(d.ldx)};
        const uint32_t xb[2] = {64, static_cast<uint32_t>(x_rows)};
        const uint64_t wd[2] = {static_cast<uint64_t>(d.K / 2), static_cast<uint64_t>(d.N)};
        const uint64_t ws[1] = {static_cast<uint64_t>(d.ldw)};
        const uint32_t wb[2] = {64, BN};
        const uint64_t cols = OUT == kOutF32 ? 2 * static_cast<uint64_t>(d.N) : (OUT == kOutF8 ? d.N / 2 : d.N);
        const uint64_t yd[2] = {cols, static_cast<uint64_t>(d.M)};
        const uint64_t ys[1] = {static_cast<uint64_t>(d.ldy) * (OUT == kOutF32 ? 4 : (OUT == kOutF8 ? 1 : 2))};
        const uint32_t yb[2] = {64, 32};
        if (!get_tensor_map(&tx, d.x, 2, xd, xs, xb) || !get_tensor_map(&tw, d.w_nk, 2, wd, ws, wb) ||
            !get_tensor_map(&ty, d.y, 2, yd, ys, yb))
            return B200_ERR_DRIVER;
        tr = ty;   // unused without a residual
        const uint64_t rd[2] = {static_cast<uint64_t>(d.N), static_cast<uint64_t>(d.M)};
        const uint64_t rs[1] = {static_cast<uint64_t>(d.ldr) * 2};
        if (d.epilogue == B200_EPI_BIAS_RESIDUAL && !get_tensor_map(&tr, d.residual, 2, rd, rs, yb)) return B200_ERR_DRIVER;
    }
    LinearFp8Params p;
    p.x_scale = d.x_scale;
    p.w_scale = d.w_scale;
    p.bias = d.bias;
    p.y_scale = d.y_scale;
    p.M = static_cast<int>(d.M);
    p.N = static_cast<int>(d.N);
    p.num_n_tiles = (p.N + BN - 1) / BN;
    const long long tiles = (d.M + 127) / 128 * p.num_n_tiles;
    if (tiles > 0x7fffffffll) return B200_ERR_UNSUPPORTED;
    p.num_tiles = static_cast<int>(tiles);
    p.num_k_blocks = static_cast<int>((d.K + 127) / 128);
    p.w_blocks = (p.N + 127) / 128;
    p.x_rows = x_rows;
    p.out_dtype = d.out_dtype;
    p.res_dtype = d.res_dtype;
    p.epilogue = d.epilogue;
    p.ld_xs = d.ld_x_scale;
    p.ld_ys = d.ld_y_scale;
    p.idesc = make_idesc_f16(128, BN, 0, 0, 0);   // format code 0 of kind::f8f6f4 = e4m3
    p.status = device_status_ptr();
    const dim3 grid(static_cast<unsigned>(p.num_tiles < sms ? p.num_tiles : sms));
    launch_kernel(linear_fp8_kernel<BN, EW, OUT>, grid, dim3(C::THREADS), C::SMEM_BYTES, stream, tx, tw, ty, tr, p);
    count_launch();
    return check_launch();
}

template <int BN>
int launch_by_output(const B200LinearFp8Desc& d, cudaStream_t stream, int sms) {
    // e4m3 output: a thread holds a whole scale block of its row, 128 columns
    constexpr int EW = BN == 64 ? 4 : 8, EW8 = BN == 256 ? 8 : 4;
    if (d.out_dtype == B200_E4M3) {
        if constexpr (BN >= 128) return launch_linear_fp8<BN, EW8, kOutF8>(d, stream, sms);
        else return B200_ERR_PARAM;
    }
    if (d.out_dtype == B200_F32) return launch_linear_fp8<BN, EW, kOutF32>(d, stream, sms);
    return launch_linear_fp8<BN, EW, kOutHalf>(d, stream, sms);
}

int validate_linear_fp8(const B200LinearFp8Desc* d) {
    if (!d || !d->x || !d->w_nk || !d->y || !d->x_scale || !d->w_scale) return B200_ERR_PARAM;
    if (d->M < 0 || d->N <= 0 || d->K <= 0) return B200_ERR_PARAM;
    if (d->M > (1ll << 30) || d->N > (1ll << 30) || d->K > (1ll << 24)) return B200_ERR_UNSUPPORTED;
    const bool f8 = d->out_dtype == B200_E4M3;
    if (!f8 && !is_half_dtype(d->out_dtype) && d->out_dtype != B200_F32) return B200_ERR_PARAM;
    if (d->epilogue < B200_EPI_BIAS || d->epilogue > B200_EPI_BIAS_TANH) return B200_ERR_PARAM;
    const int64_t per = f8 ? 16 : 8;
    if ((d->K % 16) || (d->N % per) || (d->ldx % 16) || (d->ldw % 16) || (d->ldy % per)) return B200_ERR_PARAM;
    if (d->ldx < d->K || d->ldw < d->K || d->ldy < d->N || d->ld_x_scale < d->M) return B200_ERR_PARAM;
    if (f8 && (!d->y_scale || d->ld_y_scale < d->M)) return B200_ERR_PARAM;
    if (!aligned16(d->x) || !aligned16(d->w_nk) || !aligned16(d->y) || (d->bias && !aligned16(d->bias))) return B200_ERR_PARAM;
    if (d->epilogue == B200_EPI_BIAS_RESIDUAL &&
        (!d->residual || !is_half_dtype(d->res_dtype) || (d->ldr % 8) || d->ldr < d->N || !aligned16(d->residual)))
        return B200_ERR_PARAM;
    if (d->block_n == -1 ? d->M > kFewRows : (d->block_n != 0 && d->block_n != 128 && d->block_n != 256 && (d->block_n != 64 || f8)))
        return B200_ERR_PARAM;
    return B200_OK;
}

// The tile of the smallest estimated time: waves of tiles over the SMs x (per tile + per k-block) + what the last tile's epilogue
// adds, in us, fitted to launches measured in a CUDA graph; over 60 drawn shapes the choice costs 0.2 % more than the best, over 42
// of six widths (K = 1024 to 4096) and 200 to 16384 rows 2.8 % at most.  (Many waves at K = 4096 take 10 to 19 % longer than estimated,
// on every width: the clock falls.)
// us per launch on 64 | 128 | 256 columns:  777 rows 768 -> 2304 7.5 | 6.0 | 8.0, 1024 -> 1024 5.6 | 6.4 | 8.8, 1024 -> 4096
// 13.7 | 10.5 | 9.5;  1300 rows 1024 -> 1024 8.2 | 6.6 | 8.9, 4096 -> 1024 22.1 | 15.2 | 21.2;  4096 rows 1024 -> 1024
// 14.4 | 10.8 | 9.4;  8192 rows 1024 -> 4096 81 | 57 | 49;  41339 rows 480 -> 832 59.8 | 39.9 | 45.2.
int choose_columns(const B200LinearFp8Desc& d, int sms) {
    const bool f8 = d.out_dtype == B200_E4M3;   // no 64-wide form; 128-wide tiles have half the epilogue warps
    const int columns[3] = {64, 128, 256};
    const double per_tile[3] = {0.73, f8 ? 1.8 : 1.25, 2.6}, per_block[3] = {0.29, f8 ? 0.335 : 0.31, 0.484}, last[3] = {0.0, f8 ? 0.6 : 0.4, 0.0};
    const double k_blocks = static_cast<double>((d.K + 127) / 128);
    int best = 256;
    double best_t = 1e300;
    for (int i = f8 ? 1 : 0; i < 3; ++i) {
        const int64_t tiles = (d.M + 127) / 128 * ((d.N + columns[i] - 1) / columns[i]);
        const double t = static_cast<double>((tiles + sms - 1) / sms) * (per_tile[i] + per_block[i] * k_blocks) + last[i];
        if (t < best_t) {
            best_t = t;
            best = columns[i];
        }
    }
    return best;
}

}  // namespace
}  // namespace lin
}  // namespace b200

extern "C" int b200_linear_fp8_fwd(const B200LinearFp8Desc* d, b200_stream_t stream_) {
    using namespace b200;
    using namespace b200::lin;
    const int valid = validate_linear_fp8(d);
    if (valid != B200_OK || d->M == 0) return valid;
    const int sms = device_sm_count();
    if (sms <= 0) return B200_ERR_NOT_SM100;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (d->block_n < 0 || (d->block_n == 0 && few_rows_pay(*d, sms))) return launch_linear_fp8_rows(*d, stream, sms);
    switch (d->block_n ? d->block_n : choose_columns(*d, sms)) {
        case 256: return launch_by_output<256>(*d, stream, sms);
        case 128: return launch_by_output<128>(*d, stream, sms);
        default: return launch_by_output<64>(*d, stream, sms);
    }
}
