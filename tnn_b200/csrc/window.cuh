// What the two window-attention kernels share: the parameters and which keys a run of queries can see.
#pragma once
#include "common.cuh"

namespace b200 {
namespace win {

constexpr int HD = 64;                       // head dimension
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {   // one MUFU instruction, 0 below the normal range
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct WindowParams {
    const float* mask_add;
    const int* kv_len;
    const int* q_start;
    void* out;
    const void* q;
    const void* k;
    const void* v;
    int Sq, Sk, heads, group;           // group = heads / kv_heads
    long long ldq, ldk, ldv, ldo, q_batch, k_batch, v_batch, o_batch;
    long long left, right;              // >= 0, kUnlimited where there is no limit
    int sinks;
    int causal_sinks;                   // first tokens too are hidden from queries whose window ends before them
    float scale_log2, mask_below;
    int B;
    unsigned int* status;
};
constexpr float kLeastMask = -1.7014118e38f;  // -2^127: a mask at or below it is dropped whatever the threshold (x log2(e) it must stay finite)
constexpr long long kUnlimited = 1ll << 40;  // reaches every key from every 32-bit position

// The window of a sequence's first query, [lo, hi]; query i has [lo + i, hi + i].  The sums are taken in 64 bits and clamped to
// +-2^25, which changes nothing that is visible: keys and i are below 2^24, so beyond the clamp every key lies on the same side
// of the limit for every query.  (A clamped position with an unclamped width next to it would not do: position 2^27 and a window
// of 2^26 to the left see nothing.)
struct Window {
    int lo, hi;
};
__device__ __forceinline__ Window first_window(const WindowParams& p, int b) {
    const long long pos = p.q_start == nullptr ? 0 : p.q_start[b];
    constexpr long long kEnd = 1ll << 25;
    Window w;
    w.lo = static_cast<int>(min(max(pos - p.left, -kEnd), kEnd));
    w.hi = static_cast<int>(min(max(pos + p.right, -kEnd), kEnd));
    return w;
}

// How many first tokens a query sees whose window ends at `hi`.
__device__ __forceinline__ int first_tokens(const WindowParams& p, int hi) { return p.causal_sinks ? min(p.sinks, hi + 1) : p.sinks; }

// The keys that a run of queries of a sequence can see, as runs [0, a_end) and [b_lo, b_hi); `lo` is where the first one's window
// begins, `hi` where the last one's ends.
struct Runs {
    int a_end, b_lo, b_hi;
};
__device__ __forceinline__ Runs visible_runs(const WindowParams& p, int kv, int lo, int hi) {
    Runs r;
    r.a_end = min(p.sinks, kv);
    if (p.causal_sinks) r.a_end = max(0, min(r.a_end, hi + 1));
    r.b_lo = max(0, lo);
    r.b_hi = min(kv, hi + 1);
    if (r.b_hi <= r.b_lo) {                  // nothing but the first tokens
        r.b_lo = r.b_hi = 0;
    } else if (r.b_lo <= r.a_end) {          // the runs touch
        r.b_lo = 0;
        r.b_hi = max(r.b_hi, r.a_end);
        r.a_end = 0;
    }
    return r;
}
__device__ __forceinline__ int sequence_keys(const WindowParams& p, int b) {
    if (p.kv_len == nullptr) return p.Sk;
    return min(max(p.kv_len[b], 0), p.Sk);
}
// bits [0, n) of a word, n clamped to [0, 32]
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }

// A few queries against many keys (window_token.cu): whether it takes this call, and its launch.
bool token_kernel_takes(const WindowParams& p);
int launch_window_token(const WindowParams& p, int dtype, int sms, cudaStream_t stream);

}  // namespace win
}  // namespace b200
