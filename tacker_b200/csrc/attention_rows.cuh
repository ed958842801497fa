// Attention over packed sequences, one warp per query row and head.
//
//   out_t = sum_j p_tj v_j,  p_tj = exp(s_tj - lse_t),  s_tj = scale q_t . k_j,  lse_t = log sum_j exp(s_tj)
// over the keys j < k_len of the row's sequence, with `causal` over j <= t + k_len - q_len (the last query sees every
// key).  The keys are walked once with the running maximum m and sum l of the softmax; when m rises, what has been
// summed is multiplied by exp(m_old - m_new).  A row that sees no key gives zeros and lse = -infinity.
// This form takes every alignment, stride, scale and head size up to 256; it is bound by instruction issue (about 25 warp
// instructions per key and row, each key by itself: 1024 tokens x 16 heads x 256 take 3.1 ms, a token of 16 heads over 8192
// keys 12 ms) and serves the calls the other forms do not take.
#pragma once
#include "row_ops.cuh"

namespace tk {

struct AttnArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* lse;            // [total_q][heads] or null
    const int* q_start;    // [n_seqs + 1]
    const int* k_start;    // [n_seqs]
    const int* k_len;      // [n_seqs]
    long long ld_q, ld_k, ld_v, ld_out;
    int n_seqs, total_q, kv_rows, heads, kv_heads, dim, type, causal;
    float scale_log2;      // scale * log2(e): the softmax runs on powers of two
};

// One sequence of the call.  Whatever the arrays hold, the rows stay inside the tensors.
struct AttnSeq {
    int q0, q_len, k0, k_len;
    __device__ __forceinline__ void load(const AttnArgs& p, int i) {
        q0 = min(max(p.q_start[i], 0), p.total_q);
        q_len = min(max(p.q_start[i + 1], q0), p.total_q) - q0;
        k0 = p.k_start[i];
        k_len = p.k_len[i];
        if (k0 < 0 || k0 >= p.kv_rows) k0 = 0, k_len = 0;
        k_len = min(max(k_len, 0), p.kv_rows - k0);
    }
};

// the sequence that query row `row` belongs to, or -1: the last i with q_start[i] <= row (empty sequences share a start)
__device__ __forceinline__ int attn_seq_of(const AttnArgs& p, int row) {
    if (row < p.q_start[0] || row >= p.q_start[p.n_seqs]) return -1;
    int lo = 0, hi = p.n_seqs;  // q_start[lo] <= row < q_start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.q_start[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

// Weights that enter a product in fp16 are lifted by a power of two, which the division by their sum takes out again: at 1 for
// the largest weight, those below 2^-25 of it would be zeros, and 60000 keys of e^-17.5 each, 0.15 % of the sum, would be lost.
// Prompts keep a maximum that may lag behind by 2^8, so that 2^15 is the largest weight there too.
template <int TYPE>
constexpr float kPromptLift = TYPE == kF16 ? 7.0f : 0.0f;  // powers of two
template <int TYPE>
constexpr float kTokenLift = TYPE == kF16 ? 32768.0f : 1.0f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int E>  // elements of a head per lane: dim <= 32 E
__global__ void attention_rows_kernel(const AttnArgs p) {
    const int lane = threadIdx.x & 31;
    const long long item = (blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x) >> 5;
    if (item >= static_cast<long long>(p.total_q) * p.heads) return;
    const int row = static_cast<int>(item / p.heads), head = static_cast<int>(item % p.heads);
    const int i = attn_seq_of(p, row);
    if (i < 0) return;
    AttnSeq s;
    s.load(p, i);
    const int t = row - s.q0, kv = head / (p.heads / p.kv_heads);
    int keys = s.k_len;
    if (p.causal) keys = min(keys, max(0, t + 1 + s.k_len - s.q_len));
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = lane + 32 * e;
        q[e] = d < p.dim ? load1(p.q, p.type, row * p.ld_q + static_cast<long long>(head) * p.dim + d) * p.scale_log2 : 0.0f;
        o[e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < keys; ++j) {
        const long long kr = (s.k0 + static_cast<long long>(j)) * p.ld_k + static_cast<long long>(kv) * p.dim;
        const long long vr = (s.k0 + static_cast<long long>(j)) * p.ld_v + static_cast<long long>(kv) * p.dim;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < p.dim) x = fmaf(q[e], load1(p.k, p.type, kr + lane + 32 * e), x);
#pragma unroll
        for (int b = 16; b > 0; b >>= 1) x += __shfl_xor_sync(0xffffffffu, x, b);
        const float m_new = x > m || x != x ? x : m;
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        const float w = ex2(x - base), keep = ex2(m - base);
        l = fmaf(l, keep, w);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < p.dim) o[e] = fmaf(o[e], keep, w * load1(p.v, p.type, vr + lane + 32 * e));
        m = m_new;
    }
    const float inv = 1.0f / l;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 32 * e < p.dim)
            store1(p.out, p.type, row * p.ld_out + static_cast<long long>(head) * p.dim + lane + 32 * e,
                   l == 0.0f ? 0.0f : o[e] * inv);  // keys that score -infinity weigh zero, even where v is not finite
    if (p.lse && lane == 0)
        p.lse[static_cast<long long>(row) * p.heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace tk
