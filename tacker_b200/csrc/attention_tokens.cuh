// Attention over packed sequences for single tokens and a few tokens each (the definition is in attention_rows.cuh):
// the time is that of the keys and values coming from memory.
//
// The tokens and query heads that share a key head are rows, sixteen to a block (token after token).  A CTA takes one
// block of rows and one range of the key axis; its four warps take every fourth tile of 16 keys, each through a ring of
// its own that its first lane fills by TMA, and keep their own running maximum and sum: no barrier between warps until
// the end, where they meet in shared memory.  Scores and weighted values run on mma.sync 16 x 8 x 16 (a tcgen05 tile of
// 128 rows would be empty but for a few; the tensor pipe idles either way).  Weights enter as two 16-bit terms, p and
// what rounding p left over, so that their rounding does not add to that of the result.
// Two CTAs per SM keep 2 x 4 x (stages - 1) tiles of 8 KB in flight.  64 caches of 8192 keys, 8 key heads x 128: 320 us =
// 6.7 TB/s, a copy's rate; 64 of 1 to 4096 keys: 90 us = 5.6 TB/s; the second terms cost 3 % of that.
//
// Ranges of one row's key axis are joined by a second kernel from (maximum, sum, weighted values) in the workspace,
// started by programmatic launch while the first one drains.
#pragma once
#include "attention_prompt.cuh"

namespace tk {

constexpr int kTokKeys = 16;    // keys of a tile
constexpr int kTokWarps = 4;
constexpr int kTokRows = 16;    // rows of a block

template <int D>
struct TokSmem {
    static constexpr int kBoxBytes = kTokKeys * 128;
    static constexpr int kHalfBytes = (D / 64) * kBoxBytes;  // K or V of a tile
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kWarpBytes = kStages * 2 * kHalfBytes;
    static constexpr int kBarOffset = kTokWarps * kWarpBytes;
    static constexpr int kAbortOffset = kBarOffset + kTokWarps * kStages * 8;
    static constexpr int kBytes = kAbortOffset + 4;
    static_assert(kTokWarps * (kTokRows * D + 2 * kTokRows) * 4 <= kBarOffset, "the warps' results fit over the rings");
};

struct TokArgs {
    int group, row_blocks, splits;
    float* part_o;    // [splits][total_q * heads][dim]
    float2* part_ml;  // [splits][total_q * heads]: maximum (in units of log 2) and sum
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <int TYPE>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (TYPE == kBF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four weighted values over the sum of their weights.  Without a weight the result is zero whatever v holds: keys that the
// mask hides weigh zero, and zero times an infinity or a NaN among their values has made v NaN.
template <int TYPE>
__device__ __forceinline__ uint2 attn_result(const float4& v, float sum) {
    if (sum == 0.0f) return make_uint2(0u, 0u);
    const float inv = 1.0f / sum;
    return make_uint2(pack2(v.x * inv, v.y * inv, TYPE), pack2(v.z * inv, v.w * inv, TYPE));
}

template <int D, int TYPE>
__global__ void __launch_bounds__(kTokWarps * 32, 2)
attention_tokens_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                        const AttnArgs p, const TokArgs a, unsigned* status) {
    using L = TokSmem<D>;
    constexpr int ST = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_smem_1024(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem);
    const uint32_t ring = base + warp * L::kWarpBytes;
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbortOffset);
    auto full = [&](int s) { return base + L::kBarOffset + 8u * (warp * ST + s); };
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    int b = blockIdx.x;
    const int split = b % a.splits;
    b /= a.splits;
    const int rb0 = b % a.row_blocks;
    b /= a.row_blocks;
    const int kv = b % p.kv_heads;
    AttnSeq s;
    s.load(p, b / p.kv_heads);
    const int rows = s.q_len * a.group;
    if (rb0 * kTokRows >= rows) return;
    // this CTA's keys: equal ranges of whole rounds of tiles
    const int unit = kTokKeys * kTokWarps;
    const int per = ((s.k_len + unit - 1) / unit + a.splits - 1) / a.splits * unit;
    const int j0 = min(s.k_len, split * per), j1 = min(s.k_len, j0 + per);

    if (threadIdx.x == 0) *abort_flag = 0u;
    if (lane == 0) {
        for (int i = 0; i < ST; ++i) mbar_init(full(i), 1);
        fence_mbar_init();
    }
    __syncthreads();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;

    for (int rb = rb0; rb * kTokRows < rows; rb += a.row_blocks) {
        // the rows of this thread in the MMA: lane / 4 and that + 8
        const int gr = lane >> 2, gc = (lane & 3) * 2;
        int limit[2], t[2], head[2];
        bool live[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = rb * kTokRows + gr + 8 * i;
            live[i] = r < rows;
            t[i] = r / a.group;
            head[i] = kv * a.group + r % a.group;
            limit[i] = p.causal ? min(s.k_len, max(0, t[i] + 1 + s.k_len - s.q_len)) : s.k_len;
        }
        // tiles of this warp: j0 + 16 warp, + 64, ...
        const int first = j0 + warp * kTokKeys;
        const int tiles = first < j1 ? (j1 - first + unit - 1) / unit : 0;
        auto load = [&](int i, int st) {
            mbar_arrive_expect_tx(full(st), 2 * L::kHalfBytes);
            const uint32_t dst = ring + st * 2 * L::kHalfBytes;
            const int row = s.k0 + first + i * unit;
#pragma unroll
            for (int x = 0; x < D / 64; ++x) {
                tma_load_tile(dst + x * L::kBoxBytes, &tmap_k, full(st), 64 * x, kv, row);
                tma_load_tile(dst + L::kHalfBytes + x * L::kBoxBytes, &tmap_v, full(st), 64 * x, kv, row);
            }
        };
        if (lane == 0)
            for (int i = 0; i < ST - 1 && i < tiles; ++i) load(i, (stage + i) % ST);
        // Q as A fragments
        uint32_t q[D / 16][4];
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 16 * x + gc + 8 * (i >> 1), w = i & 1;
                q[x][i] = live[w] && d < p.dim
                              ? *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) +
                                                                   (s.q0 + static_cast<long long>(t[w])) * p.ld_q +
                                                                   static_cast<long long>(head[w]) * p.dim + d)
                              : 0u;
            }
        float o[D / 8][4];
#pragma unroll
        for (int x = 0; x < D / 8; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

        for (int i = 0; i < tiles; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait(full(stage), phase, abort_flag, status, DEV_TIMEOUT_FULL));
            if (!ok) break;
            const uint32_t ks = ring + stage * 2 * L::kHalfBytes, vs = ks + L::kHalfBytes;
            // the slot that the tile after next needs was read in the last step
            if (lane == 0 && i + ST - 1 < tiles) load(i + ST - 1, stage == 0 ? ST - 1 : stage - 1);
            const int j = first + i * unit, left = j1 - j;
            if (left < kTokKeys) {
                // values behind the range may be anything: zeros
                for (int e = lane; e < (kTokKeys - left) * 8 * (D / 64); e += 32) {
                    const int box = e / ((kTokKeys - left) * 8), r = e % ((kTokKeys - left) * 8);
                    *reinterpret_cast<uint4*>(smem + (vs - base) + box * L::kBoxBytes + (left + r / 8) * 128 + (r % 8) * 16) =
                        make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();  // the next tile in this slot is written by TMA
                __syncwarp();
            }
            float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            {
                const int key = ((lane >> 4) << 3) + (lane & 7), half = (lane >> 3) & 1;
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    uint32_t f[4];
                    const int chunk = 2 * (x & 3) + half;
                    ldmatrix_x4(ks + (x >> 2) * L::kBoxBytes + key * 128 + ((chunk ^ (key & 7)) << 4), f);
                    mma_16816<TYPE>(sc[0], q[x], f[0], f[1]);
                    mma_16816<TYPE>(sc[1], q[x], f[2], f[3]);
                }
            }
            // sc[n][2 w + e]: row lane / 4 + 8 w, key 8 n + gc + e
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int w = e >> 1, key = j + 8 * n + gc + (e & 1);
                    sc[n][e] = key < min(limit[w], j1) ? sc[n][e] * p.scale_log2 : -INFINITY;
                    top[w] = fmaxf(top[w], sc[n][e]);
                }
            float keep[2], off[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 1));
                top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], 2));
                const float up = fmaxf(m[w], top[w]);
                off[w] = up == -INFINITY ? 0.0f : up;
                keep[w] = ex2(m[w] - off[w]);
                m[w] = up;
                l[w] *= keep[w];
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const float a0 = ex2(sc[n][2 * w] - off[w]) * kTokenLift<TYPE>, a1 = ex2(sc[n][2 * w + 1] - off[w]) * kTokenLift<TYPE>;
                    l[w] += a0 + a1;
                    const uint32_t h = pack2(a0, a1, TYPE);
                    float h0, h1;
                    unpack2(h, TYPE, h0, h1);
                    hi[2 * n + w] = h;
                    lo[2 * n + w] = pack2(a0 - h0, a1 - h1, TYPE);
                }
            if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f)) {
#pragma unroll
                for (int x = 0; x < D / 8; ++x) {
                    o[x][0] *= keep[0], o[x][1] *= keep[0];
                    o[x][2] *= keep[1], o[x][3] *= keep[1];
                }
            }
            {
                const int key = lane & 15, half = lane >> 4;
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    uint32_t f[4];
                    const int chunk = 2 * (x & 3) + half;
                    ldmatrix_x4_trans(vs + (x >> 2) * L::kBoxBytes + key * 128 + ((chunk ^ (key & 7)) << 4), f);
                    mma_16816<TYPE>(o[2 * x], hi, f[0], f[1]);
                    mma_16816<TYPE>(o[2 * x + 1], hi, f[2], f[3]);
                    mma_16816<TYPE>(o[2 * x], lo, f[0], f[1]);
                    mma_16816<TYPE>(o[2 * x + 1], lo, f[2], f[3]);
                }
            }
            __syncwarp();
            if (++stage == ST) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // the warps' results meet over the rings, which are drained; after a wait that ran out nothing is to be joined
        if (!__syncthreads_and(ok)) break;
        float* acc = reinterpret_cast<float*>(smem);                            // [warp][16][D]
        float2* ml = reinterpret_cast<float2*>(acc + kTokWarps * kTokRows * D);  // [warp][16]
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
            l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
            const int r = warp * kTokRows + gr + 8 * w;
            if ((lane & 3) == 0) ml[r] = make_float2(m[w], l[w]);
#pragma unroll
            for (int x = 0; x < D / 8; ++x)
                *reinterpret_cast<float2*>(acc + r * D + 8 * x + gc) = make_float2(o[x][2 * w], o[x][2 * w + 1]);
        }
        __syncthreads();
        const int total_rows = p.total_q * p.heads;  // at most 2^31 (checked by the launcher)
        for (int e = threadIdx.x; e < kTokRows * (D / 4); e += kTokWarps * 32) {
            const int r = e / (D / 4), d = e % (D / 4) * 4, gi = rb * kTokRows + r;
            if (gi >= rows || d >= p.dim) continue;
            float mm = ml[r].x;
#pragma unroll
            for (int w = 1; w < kTokWarps; ++w) mm = fmaxf(mm, ml[w * kTokRows + r].x);
            // a NaN sum keeps its warp's weight NaN through the products below
            const float offm = mm == -INFINITY ? 0.0f : mm;
            float sum = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kTokWarps; ++w) {
                const float2 x = ml[w * kTokRows + r];
                const float f = ex2(x.x - offm);
                const float4 u = *reinterpret_cast<const float4*>(acc + (w * kTokRows + r) * D + d);
                sum = fmaf(x.y, f, sum);
                v.x = fmaf(u.x, f, v.x), v.y = fmaf(u.y, f, v.y), v.z = fmaf(u.z, f, v.z), v.w = fmaf(u.w, f, v.w);
            }
            const int tok = gi / a.group, hd = kv * a.group + gi % a.group;
            const long long row = s.q0 + static_cast<long long>(tok);
            if (a.splits > 1) {
                const long long slot = static_cast<long long>(split) * total_rows + row * p.heads + hd;
                *reinterpret_cast<float4*>(a.part_o + slot * p.dim + d) = v;
                if (d == 0) a.part_ml[slot] = make_float2(mm, sum);
            } else {
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * p.ld_out + static_cast<long long>(hd) * p.dim + d) =
                    attn_result<TYPE>(v, sum);
                if (d == 0 && p.lse) p.lse[row * p.heads + hd] = sum == 0.0f ? -INFINITY : (mm + log2f(sum * (1.0f / kTokenLift<TYPE>))) * kLn2;
            }
        }
        if (rb + a.row_blocks < static_cast<int>((rows + kTokRows - 1) / kTokRows)) {
            fence_proxy_async_smem();  // the rings are written by TMA again
            __syncthreads();
        }
    }
    if (*abort_flag) __nanosleep(1000000u);  // let bulk copies still in flight land before shared memory is released
}

// One block per query row and head: joins the ranges of its key axis.  Each warp takes every n-th range.
template <int TYPE>
__global__ void attention_join_kernel(const AttnArgs p, const TokArgs a) {
    __shared__ float4 acc[8][32];
    __shared__ float2 part[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const long long item = blockIdx.x;
    const long long row = item / p.heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row < p.q_start[0] || row >= p.q_start[p.n_seqs]) return;
    const long long stride = static_cast<long long>(p.total_q) * p.heads;
    float m = -INFINITY;
    for (int i = lane; i < a.splits; i += 32) m = fmaxf(m, a.part_ml[i * stride + item].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float off = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const int d = 4 * lane;
#pragma unroll 4
    for (int i = warp; i < a.splits; i += warps) {
        const long long slot = i * stride + item;
        const float2 x = a.part_ml[slot];
        const float f = ex2(x.x - off);
        sum = fmaf(x.y, f, sum);
        if (d < p.dim) {
            const float4 u = *reinterpret_cast<const float4*>(a.part_o + slot * p.dim + d);
            v.x = fmaf(u.x, f, v.x), v.y = fmaf(u.y, f, v.y), v.z = fmaf(u.z, f, v.z), v.w = fmaf(u.w, f, v.w);
        }
    }
    acc[warp][lane] = v;
    if (lane == 0) part[warp].x = sum;
    __syncthreads();
    if (warp != 0) return;
    for (int w = 1; w < warps; ++w) {
        const float4 u = acc[w][lane];
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        sum += part[w].x;
    }
    const int head = static_cast<int>(item - row * p.heads);
    if (d < p.dim)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * p.ld_out + static_cast<long long>(head) * p.dim + d) =
            attn_result<TYPE>(v, sum);
    if (lane == 0 && p.lse) p.lse[item] = sum == 0.0f ? -INFINITY : (m + log2f(sum * (1.0f / kTokenLift<TYPE>))) * kLn2;
}

}  // namespace tk
