// Window attention of a few query tokens against a long cache (head_dim 64): HBM-bound, every visible key and value once per block of
// up to 32 query rows (33 to 64 rows of a sequence stream them twice, the second time mostly from L2).
//
// The queries of one sequence whose heads share a key / value head (Sq x group rows) are one matrix, in blocks of MT x 16 rows.
// The visible keys, the first tokens and the window behind one another, are dealt in tiles of 32 to the warps of a cluster of
// up to eight CTAs; a warp streams its tiles through a private ring with cp.async (16-byte pieces, swizzled; rows that nobody
// may see arrive as zeros), multiplies with mma.sync m16n8k16 (a launch of few rows has no tile for the tcgen05 pipe, and this
// one waits for memory) and keeps its own running maximum, sum and output.  At the end the warps' results are joined in shared
// memory and the CTAs' through distributed shared memory: one launch, no workspace, a fixed order of summation.
// One token of each of 32 sequences of 2000 to 16384 keys, window 8192, 16 / 4 heads: 43 us, 0.80 of the measured copy rate (0.96 where
// all have 16384); about 5 us of it are launch, first loads and the join.
#include "window.cuh"
#include "ptx.cuh"

namespace b200 {
namespace win {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;                                  // keys per tile
constexpr int kStages = 3;
constexpr int kStageBytes = 2 * kTile * HD * 2;            // K and V
constexpr int kRingBytes = kStages * kStageBytes;          // one warp's
constexpr int kBlockRows = 32;                             // query rows per block at most
// Beyond this many rows (queries x heads of a group) the tile kernel takes over.  us, this kernel | tiles (one query tile of one head per
// CTA, keys not split), unlimited window, rows x keys:
//   1 sequence, 12 / 12 heads: 64 x 1024 9.8 | 14.4   72 x 1024 14.6 | 14.3   64 x 32768 52 | 315   128 x 32768 92 | 315   512 x 32768 268 | 354
//   1 sequence, 12 / 1 heads:  72 x 32768 36 | 314   192 x 32768 37 | 314
//   8 sequences, 16 / 4 heads: 64 x 8192 29 | 111   192 x 8192 84 | 111   512 x 8192 176 | 112
//   32 sequences, 16 / 4:      64 x 1024 17 | 36   128 x 1024 32 | 36   192 x 1024 47 | 37   192 x 8192 264 | 230   512 x 32768 2310 | 901
// So up to 64 rows this kernel is never behind; beyond, either may be, by up to nine times, depending on the number of sequences and
// the length of the cache.  The limit looks at the rows of a single sequence alone: with more than 64 of them a row's result depends
// neither on the batch nor on the length of the cache it lies in.
constexpr int kMaxRows = 64;

template <int MT>
constexpr int token_smem() { return kWarps * kRingBytes + (2 * kWarps + 2) * MT * 16 * 4; }
static_assert(kRingBytes >= kBlockRows * HD * 4, "a warp's result takes the place of its ring");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {   // the rest of 16 bytes as zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int DT>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (DT == B200_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// fp32 at this shared-memory address of the cluster's CTA `rank`
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 remote;\n\tmapa.shared::cluster.u32 remote, %1, %2;\n\tld.shared::cluster.f32 %0, [remote];\n\t}"
                 : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("{\n\t.reg .b32 remote;\n\tmapa.shared::cluster.u32 remote, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [remote];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}

template <int DT, int MT, bool MASKED>
__global__ void __launch_bounds__(32 * kWarps, 2) window_token_kernel(const WindowParams p, int ctas, int blocks) {
    constexpr int ROWS = MT * 16;
    static_assert(ROWS <= kBlockRows, "");
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = ctas > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int kv_heads = p.heads / p.group;
    const int unit = blockIdx.x / ctas;                    // one block of rows of one sequence's one key / value head
    const int r0 = unit % blocks * ROWS;
    const int kv_head = unit / blocks % kv_heads, b = unit / blocks / kv_heads;
    uint8_t* ring = smem + warp * kRingBytes;
    float* m_s = reinterpret_cast<float*>(smem + kWarps * kRingBytes);   // [kWarps + 1][ROWS] maxima, the CTA's last
    float* l_s = m_s + (kWarps + 1) * ROWS;                              // and sums
    pdl_launch_dependents();
    pdl_wait();   // q, k, v, kv_len and q_start come from earlier kernels; the output may still be read by one

    const int rows = min(ROWS, p.Sq * p.group - r0);       // row r = query (r0 + r) / group, head (r0 + r) % group
    const Window window = first_window(p, b);
    // keys that every row of the block sees: the window's between these
    const int all_lo = window.lo + (r0 + rows - 1) / p.group, all_hi = window.hi + r0 / p.group;
    const Runs runs = visible_runs(p, sequence_keys(p, b), window.lo + r0 / p.group, window.hi + (r0 + rows - 1) / p.group);
    const int n_a = runs.a_end, n = n_a + runs.b_hi - runs.b_lo;
    const int shift = runs.b_lo - n_a;                     // place in the list of visible keys -> key, from place n_a on
    const uint16_t* kp = static_cast<const uint16_t*>(p.k) + b * p.k_batch + kv_head * HD;
    const uint16_t* vp = static_cast<const uint16_t*>(p.v) + b * p.v_batch + kv_head * HD;
    const float* mask = MASKED ? p.mask_add + static_cast<long long>(b) * p.Sk : nullptr;
    const uint32_t ring_u = smem_u32(ring);

    const int tiles = (n + kTile - 1) / kTile;
    const int first = rank * kWarps + warp, step = ctas * kWarps;
    auto fetch = [&](int tile, int stage) {                // tile's keys and values; beyond the last tile an empty group
        if (tile < tiles) {
#pragma unroll
            for (int i = 0; i < kTile / 4; ++i) {
                const int r = (lane >> 3) + i * 4, piece = lane & 7;
                const int at = tile * kTile + r;
                const int key = at < n ? at + (at >= n_a ? shift : 0) : 0;
                const bool there = at < n && (!MASKED || mask[key] > p.mask_below);
                const uint32_t dst = ring_u + stage * kStageBytes + r * 128 + ((piece ^ (r & 7)) << 4);
                cp_async16(dst, kp + key * p.ldk + piece * 8, there ? 16u : 0u);
                cp_async16(dst + kTile * 128, vp + key * p.ldv + piece * 8, there ? 16u : 0u);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(first + i * step, i);

    // The rows of this thread: g and g + 8 of every m16 tile.
    const int g = lane >> 2, c2 = (lane & 3) * 2;
    uint32_t qf[MT][4][4];
    int lo[MT][2], hi[MT][2], first_keys[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = t * 16 + g + h * 8;
            const bool there = r < rows;
            const int i = there ? (r0 + r) / p.group : 0;
            lo[t][h] = there ? window.lo + i : 1;          // a row that does not exist sees nothing
            hi[t][h] = there ? window.hi + i : 0;
            first_keys[t][h] = there ? first_tokens(p, hi[t][h]) : 0;
            const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_batch + i * p.ldq + (kv_head * p.group + (there ? (r0 + r) % p.group : 0)) * HD;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                qf[t][k][h] = there ? *reinterpret_cast<const uint32_t*>(q + k * 16 + c2) : 0u;
                qf[t][k][2 + h] = there ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8 + c2) : 0u;
            }
        }
    float o[MT][8][4], m_run[MT][2], l_run[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][d][e] = 0.f;
        m_run[t][0] = m_run[t][1] = -INFINITY;
        l_run[t][0] = l_run[t][1] = 0.f;
    }

    int stage = 0;
    for (int tile = first; tile < tiles; tile += step) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        {   // the stage that the previous tile left
            int next = stage + kStages - 1;
            if (next >= kStages) next -= kStages;
            fetch(tile + (kStages - 1) * step, next);
        }
        const uint32_t ks = ring_u + stage * kStageBytes, vs = ks + kTile * 128;
        float s[MT][4][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][j][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {                      // 8 keys each
#pragma unroll
            for (int k = 0; k < 2; ++k) {                  // 32 dimensions each
                uint32_t bf[4];
                const int r = j * 8 + (lane & 7), piece = k * 4 + (lane >> 3);
                ldmatrix_x4(ks + r * 128 + ((piece ^ (r & 7)) << 4), bf);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    mma16816<DT>(s[t][j], qf[t][2 * k], bf[0], bf[1]);
                    mma16816<DT>(s[t][j], qf[t][2 * k + 1], bf[2], bf[3]);
                }
            }
        }
        // scale, mask, running maximum
        float alpha[MT][2];
        bool moved = false;
        const int at0 = tile * kTile;
        const bool plain = !MASKED && at0 >= n_a && at0 + kTile <= n && at0 + shift >= all_lo && at0 + shift + kTile - 1 <= all_hi;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float top[2] = {-INFINITY, -INFINITY};
            if (plain) {                                   // (a row that does not exist goes along: it is not stored)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[t][j][e] *= p.scale_log2;
                        top[e >> 1] = fmaxf(top[e >> 1], s[t][j][e]);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int at = at0 + j * 8 + c2 + e;
                        const int key = at + (at >= n_a ? shift : 0);
                        float mk = 0.f;
                        bool there = at < n;
                        if (MASKED) {
                            mk = there ? mask[key] : 0.f;
                            there = there && mk > p.mask_below;
                            mk *= kLog2e;
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const bool seen = there && ((key >= lo[t][h] && key <= hi[t][h]) || key < first_keys[t][h]);
                            const float x = seen ? fmaf(s[t][j][h * 2 + e], p.scale_log2, mk) : -INFINITY;
                            s[t][j][h * 2 + e] = x;
                            top[h] = fmaxf(top[h], x);
                        }
                    }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                const float m_new = fmaxf(m_run[t][h], top[h]);
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                alpha[t][h] = fast_exp2(m_run[t][h] - m_use);
                moved = moved || m_new != m_run[t][h];
                m_run[t][h] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = fast_exp2(s[t][j][h * 2 + e] - m_use);
                        s[t][j][h * 2 + e] = x;
                        sum += x;
                    }
                l_run[t][h] = l_run[t][h] * alpha[t][h] + sum;
            }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int d = 0; d < 8; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[t][d][e] *= alpha[t][e >> 1];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {                      // 16 keys each
            // The weights are rounded to the operands' type for this product, half a step of it each (2^-11, 2^-8) and independent
            // of one another: 2.2e-3 of the result's norm in bf16 where its own rounding is 1.7e-3.  Their sum is kept unrounded.
            uint32_t pf[MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                pf[t][0] = pack2t<DT>(s[t][2 * k][0], s[t][2 * k][1]);
                pf[t][1] = pack2t<DT>(s[t][2 * k][2], s[t][2 * k][3]);
                pf[t][2] = pack2t<DT>(s[t][2 * k + 1][0], s[t][2 * k + 1][1]);
                pf[t][3] = pack2t<DT>(s[t][2 * k + 1][2], s[t][2 * k + 1][3]);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {                  // 16 dimensions each
                uint32_t bf[4];
                const int r = k * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), piece = d * 2 + (lane >> 4);
                ldmatrix_x4_trans(vs + r * 128 + ((piece ^ (r & 7)) << 4), bf);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    mma16816<DT>(o[t][2 * d], pf[t], bf[0], bf[1]);
                    mma16816<DT>(o[t][2 * d + 1], pf[t], bf[2], bf[3]);
                }
            }
        }
        __syncwarp();                                      // the stage has been read
        if (++stage == kStages) stage = 0;
    }
    cp_async_wait<0>();
    __syncwarp();

    // the warp's result in the place of its ring
    float* ow = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float l = l_run[t][h];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            const int r = t * 16 + g + h * 8;
            if ((lane & 3) == 0) {
                m_s[warp * ROWS + r] = m_run[t][h];
                l_s[warp * ROWS + r] = l;
            }
#pragma unroll
            for (int d = 0; d < 8; ++d)
                *reinterpret_cast<float2*>(ow + r * HD + d * 8 + c2) = make_float2(o[t][d][h * 2], o[t][d][h * 2 + 1]);
        }
    __syncthreads();
    // the CTA's: sums over warps in place of warp 0's, its maximum and sum behind the warps'
    float* oc = reinterpret_cast<float*>(smem);
    for (int i = threadIdx.x; i < rows * (HD / 4); i += 32 * kWarps) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        float m = m_s[r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, m_s[w * ROWS + r]);
        const float m_use = m == -INFINITY ? 0.f : m;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = fast_exp2(m_s[w * ROWS + r] - m_use);
            const float4 x = *reinterpret_cast<const float4*>(smem + w * kRingBytes + (r * HD + d) * 4);
            acc.x = fmaf(x.x, f, acc.x);
            acc.y = fmaf(x.y, f, acc.y);
            acc.z = fmaf(x.z, f, acc.z);
            acc.w = fmaf(x.w, f, acc.w);
            l = fmaf(l_s[w * ROWS + r], f, l);
        }
        *reinterpret_cast<float4*>(oc + r * HD + d) = acc;
        if (d == 0) {
            m_s[kWarps * ROWS + r] = m;
            l_s[kWarps * ROWS + r] = l;
        }
    }
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    // the output: every CTA of the cluster a share of the rows' 8-column pieces
    const uint32_t oc_u = smem_u32(oc), m_u = smem_u32(m_s + kWarps * ROWS), l_u = smem_u32(l_s + kWarps * ROWS);
    for (int i = rank * 32 * kWarps + threadIdx.x; i < rows * (HD / 8); i += ctas * 32 * kWarps) {
        const int r = i / (HD / 8), d = i % (HD / 8) * 8;
        float m = -INFINITY;
        for (int c = 0; c < ctas; ++c) m = fmaxf(m, ld_cluster(m_u + r * 4, c));
        const float m_use = m == -INFINITY ? 0.f : m;
        float acc[8], l = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        for (int c = 0; c < ctas; ++c) {
            const float f = fast_exp2(ld_cluster(m_u + r * 4, c) - m_use);
            l = fmaf(ld_cluster(l_u + r * 4, c), f, l);
            const float4 x = ld_cluster4(oc_u + (r * HD + d) * 4, c), y = ld_cluster4(oc_u + (r * HD + d + 4) * 4, c);
            acc[0] = fmaf(x.x, f, acc[0]);
            acc[1] = fmaf(x.y, f, acc[1]);
            acc[2] = fmaf(x.z, f, acc[2]);
            acc[3] = fmaf(x.w, f, acc[3]);
            acc[4] = fmaf(y.x, f, acc[4]);
            acc[5] = fmaf(y.y, f, acc[5]);
            acc[6] = fmaf(y.z, f, acc[6]);
            acc[7] = fmaf(y.w, f, acc[7]);
        }
        uint4 w = make_uint4(0, 0, 0, 0);                  // a row that saw no key
        if (l != 0.f) {
            const float inv = 1.0f / l;
            w.x = pack2t<DT>(acc[0] * inv, acc[1] * inv);
            w.y = pack2t<DT>(acc[2] * inv, acc[3] * inv);
            w.z = pack2t<DT>(acc[4] * inv, acc[5] * inv);
            w.w = pack2t<DT>(acc[6] * inv, acc[7] * inv);
        }
        uint16_t* out = static_cast<uint16_t*>(p.out) + b * p.o_batch + ((r0 + r) / p.group) * p.ldo +
                        (kv_head * p.group + (r0 + r) % p.group) * HD + d;
        *reinterpret_cast<uint4*>(out) = w;
    }
    if (ctas > 1) cluster_sync();                          // nobody leaves while its results may be read
}

template <int DT, int MT, bool MASKED>
int launch_token(const WindowParams& p, int ctas, int blocks, cudaStream_t stream) {
    static PerDeviceOnce once;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return B200_ERR_LAUNCH;
    if (!once.ensure(dev, []() {
            return cudaFuncSetAttribute(window_token_kernel<DT, MT, MASKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, token_smem<MT>()) ==
                   cudaSuccess;
        }))
        return B200_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.B) * (p.heads / p.group) * blocks * ctas);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = token_smem<MT>();
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (ctas > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(ctas);
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = static_cast<unsigned>(n);
    cudaLaunchKernelEx(&cfg, window_token_kernel<DT, MT, MASKED>, p, ctas, blocks);
    count_launch();
    return check_launch();
}

template <int DT, bool MASKED>
int launch_rows(const WindowParams& p, int ctas, int blocks, cudaStream_t stream) {
    return p.Sq * p.group <= 16 ? launch_token<DT, 1, MASKED>(p, ctas, blocks, stream) : launch_token<DT, 2, MASKED>(p, ctas, blocks, stream);
}

}  // namespace

bool token_kernel_takes(const WindowParams& p) {
    return static_cast<long long>(p.Sq) * p.group <= kMaxRows && static_cast<long long>(p.B) * (p.heads / p.group) * 16 <= 0x7fffffffll;
}

int launch_window_token(const WindowParams& p, int dtype, int sms, cudaStream_t stream) {
    // The number of CTAs per key / value head with the smallest waves x (fixed cost + keys of a CTA), two CTAs per SM; a CTA's start
    // and join cost as much as some 600 keys (5.5 us).  us on 1 | 2 | 4 | 8: 32 sequences, 4 heads, window 8192 54.7 | 43.0 | 46.1 | 55.1;
    // 27 of 6088 keys, 12 heads 103 | 90 | 88 | 101; 60 of 5575, 4 heads, 5 tokens 64 | 71 | 84 | 111; 8 of 5711, 12 heads
    // 37.3 | 25.7 | 31.6 | 32.5; 4 of 4096, 8 heads 21.7 | 14.6 | 10.3 | 7.9.
    const int blocks = (p.Sq * p.group + kBlockRows - 1) / kBlockRows;
    const long long units = static_cast<long long>(p.B) * (p.heads / p.group) * blocks;
    const long long reach = p.left + p.right + p.Sq + p.sinks;
    const long long keys = p.Sk < reach ? p.Sk : reach;
    int ctas = 1;
    long long least = 0;
    for (int c = 1; c <= 8 && (c == 1 || keys >= static_cast<long long>(c) * kWarps * kTile); c *= 2) {   // a tile for every warp
        const long long t = (units * c + 2 * sms - 1) / (2 * sms) * (600 + keys / c);
        if (c == 1 || t < least) {
            least = t;
            ctas = c;
        }
    }
    if (p.mask_add != nullptr)
        return dtype == B200_F16 ? launch_rows<B200_F16, true>(p, ctas, blocks, stream) : launch_rows<B200_BF16, true>(p, ctas, blocks, stream);
    return dtype == B200_F16 ? launch_rows<B200_F16, false>(p, ctas, blocks, stream) : launch_rows<B200_BF16, false>(p, ctas, blocks, stream);
}

}  // namespace win
}  // namespace b200
