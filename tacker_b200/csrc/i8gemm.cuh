// Product of 8-bit integers with a scale for each token and each output channel:
//   out[m][n] = (sum_k A[m][k] B[n][k]) * scale_a[m] * scale_b[n] + bias[n]
// The sums are exact: tcgen05.mma kind::i8 accumulates in 32-bit integers, and |sum| <= K 2^14 < 2^31 for K <= 131071.
// One rounding to fp32 follows, then the scales, then the rounding to the output's type.
//
// Operand tiles are 128 bytes (128 values of k) wide, K-major, 128-byte swizzled by TMA; rows and k beyond the matrices
// arrive as zeros and add nothing, so no size has to be a multiple of a tile.
#pragma once
#include "kernels.cuh"
#include "row_ops.cuh"

namespace tk {

// one lane of a full warp, always the same
__device__ __forceinline__ bool elect_lane() {
    uint32_t e;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(e));
    return e != 0;
}

struct I8Args {
    const float* scale_a;  // [M]
    const float* scale_b;  // [N]
    const float* bias;     // [N] or null
    void* out;
    long long ld_out;      // elements
    int M, N, K, out_type;
    int vec;               // 16-byte stores into out are aligned
    unsigned* status;
};

__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor, kind::i8: signed 8-bit A and B (both K-major), 32-bit integer accumulator.
__host__ __device__ constexpr uint32_t umma_idesc_i8_s32(uint32_t m, uint32_t n) {
    return (2u << 4)            // bits 4-5: accumulator format, 2 = s32
           | (1u << 7)          // bits 7-9: A format, 1 = signed 8-bit
           | (1u << 10)         // bits 10-12: B format
           | ((n >> 3) << 17)   // bits 17-22: N / 8
           | ((m >> 4) << 24);  // bits 24-28: M / 16
}

constexpr int kI8BK = 128;  // bytes of k per stage

// ---- output ----------------------------------------------------------------------------------------------------
constexpr int kI8OutPitch = 36;                       // floats per staged row: conflict-free by rows and by columns
constexpr int kI8OutBytes = 32 * kI8OutPitch * 4;     // one warp's staging
constexpr int kI8PartPitch = 132;                     // integers per row of 128 partial sums

// Scales and biases of the columns a lane stores of a chunk of 32: eight neighbours, or one where rows are not aligned or
// the chunk is cut off by the matrix's edge.  Fetched before the sums are waited for.
struct I8Cols {
    float sc[8], b[8];
};
__device__ __forceinline__ bool i8_wide(const I8Args& p, int col0) { return p.vec && col0 + 32 <= p.N; }
__device__ __forceinline__ void i8_columns(const I8Args& p, int col0, int lane, I8Cols& k) {
    const bool wide = i8_wide(p, col0);
    const int c = wide ? col0 + (lane & 3) * 8 : min(col0 + lane, p.N - 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        k.sc[i] = wide || i == 0 ? __ldg(p.scale_b + c + i) : 0.0f;
        k.b[i] = p.bias && (wide || i == 0) ? __ldg(p.bias + c + i) : 0.0f;
    }
}

// 32 x 32 sums of a warp (one row per lane) on their way to out rows row0 .., columns col0 ..: times the row's scale into
// shared memory, then times the column's scale and stored with neighbouring lanes on neighbouring columns.  A row per lane
// and store would touch 32 lines with every instruction.
__device__ __forceinline__ void i8_store_chunk(const I8Args& p, float* stage, const uint32_t (&v)[32], float row_scale,
                                               const I8Cols& k, int row0, int col0, int lane) {
    float4* mine = reinterpret_cast<float4*>(stage + lane * kI8OutPitch);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        mine[i] = make_float4(static_cast<float>(static_cast<int>(v[4 * i])) * row_scale,
                              static_cast<float>(static_cast<int>(v[4 * i + 1])) * row_scale,
                              static_cast<float>(static_cast<int>(v[4 * i + 2])) * row_scale,
                              static_cast<float>(static_cast<int>(v[4 * i + 3])) * row_scale);
    __syncwarp();
    if (i8_wide(p, col0)) {
        // eight columns per lane: four lanes per row, eight rows at a time
        const long long at = (row0 + (lane >> 2)) * p.ld_out + col0 + (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 8 * i + (lane >> 2);
            const float4* src = reinterpret_cast<const float4*>(stage + r * kI8OutPitch + (lane & 3) * 8);
            const float4 x = src[0], y = src[1];
            const float o[8] = {x.x * k.sc[0] + k.b[0], x.y * k.sc[1] + k.b[1], x.z * k.sc[2] + k.b[2], x.w * k.sc[3] + k.b[3],
                                y.x * k.sc[4] + k.b[4], y.y * k.sc[5] + k.b[5], y.z * k.sc[6] + k.b[6], y.w * k.sc[7] + k.b[7]};
            if (row0 + r < p.M) store8(p.out, p.out_type, at + 8 * i * p.ld_out, o);
        }
    } else if (col0 + lane < p.N) {
        const int n = min(32, p.M - row0);
#pragma unroll 8
        for (int r = 0; r < n; ++r)
            store1(p.out, p.out_type, (row0 + r) * p.ld_out + col0 + lane, stage[r * kI8OutPitch + lane] * k.sc[0] + k.b[0]);
    }
    __syncwarp();
}

template <int BN, int STAGES>
struct I8Smem {
    static constexpr int kABytes = 128 * kI8BK;
    static constexpr int kBBytes = BN * kI8BK;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kPartBytes = 128 * kI8PartPitch * 4;  // partial sums of a range of k, over the drained stages
    static constexpr int kRing = STAGES * kStageBytes;
    static constexpr int kBarOffset = ((kRing > kPartBytes ? kRing : kPartBytes) + 7) / 8 * 8;
    static_assert(4 * kI8OutBytes <= kRing, "the output warps' staging fits over the drained stages");
    static constexpr int kTmemSlotOffset = kBarOffset + (2 * STAGES + 1) * 8;
    static constexpr int kAbortOffset = kTmemSlotOffset + 4;
    static constexpr int kBytes = kAbortOffset + 4;
};

__device__ __forceinline__ int4 ld_shared_cluster_v4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// One output tile per cluster.  The 128 rows of the MMA are tokens and its BN columns output channels, or with SWAP the
// other way round: with few tokens the weights are the long operand, they fill the 128 rows, and the tokens are the
// columns, so that neither tensor-core time nor shared memory goes to rows that do not exist and a warp's stores run
// along the output row.  The CTAs of a cluster take equal ranges of k; their integer partial sums meet in shared memory
// and every CTA finishes an equal share of the tile's columns: no scratch in global memory, no atomics, the same sums in
// every split.
//   warp 0 TMA producer, warp 1 MMA issuer, warps 2..5 epilogue
template <int BN, int STAGES, bool SWAP>
__global__ void __launch_bounds__(192)
i8gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const I8Args p,
              const int split, const int tiles_b) {
    using L = I8Smem<BN, STAGES>;
    constexpr uint32_t kTmemCols = BN < 32 ? 32 : BN;
    constexpr uint32_t kIdesc = umma_idesc_i8_s32(128, BN);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_smem_1024(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem_base = smem_u32(smem);
    auto full_bar = [&](int s) { return smem_base + L::kBarOffset + 8u * s; };
    auto empty_bar = [&](int s) { return smem_base + L::kBarOffset + 8u * (STAGES + s); };
    const uint32_t done_bar = smem_base + L::kBarOffset + 8u * (2 * STAGES);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kTmemSlotOffset);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbortOffset);

    const int tile = blockIdx.x / split, rank = blockIdx.x % split;
    const int row_a = tile / tiles_b * 128, row_b = tile % tiles_b * BN;
    const int kblocks = (p.K + kI8BK - 1) / kI8BK;
    const int kb0 = static_cast<int>(static_cast<long long>(kblocks) * rank / split);
    const int kb1 = static_cast<int>(static_cast<long long>(kblocks) * (rank + 1) / split);

    if (warp == 0 && lane == 0) {
        *abort_flag = 0u;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            auto advance = [&]() {
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                mbar_arrive_expect_tx(full_bar(stage), L::kStageBytes);
                const uint32_t dst = smem_base + stage * L::kStageBytes;
                tma_load_2d(dst, &tmap_a, full_bar(stage), kb * kI8BK, row_a);
                tma_load_2d(dst + L::kABytes, &tmap_b, full_bar(stage), kb * kI8BK, row_b);
                advance();
            }
            // the last commits arrive on the empty barriers asynchronously, and nothing orders them before the one on done_bar:
            // the CTA must not retire before they have landed
            for (int s = 0; s < STAGES && ok; ++s, advance())
                ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_EMPTY);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, DEV_TIMEOUT_FULL);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t src = smem_base + stage * L::kStageBytes;
                const uint64_t a_desc = umma_smem_desc_sw128(src), b_desc = umma_smem_desc_sw128(src + L::kABytes);
#pragma unroll
                for (int k = 0; k < kI8BK / 32; ++k)  // 32 values of k = 32 bytes along the swizzled row
                    umma_i8(tmem, a_desc + 2u * k, b_desc + 2u * k, kIdesc, (kb > kb0 || k != 0) ? 1u : 0u);
                umma_commit(empty_bar(stage));
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok) umma_commit(done_bar);
        }
    }
    // the accumulator is complete, so all loads have landed
    __syncwarp();
    const bool good = mbar_wait(done_bar, 0, abort_flag, p.status, DEV_TIMEOUT_TMEM_FULL);
    tc_fence_after_sync();

    const int q = warp & 3;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const int r = row_a + q * 32 + lane;  // this thread's row of the MMA
    if (split > 1) {
        // partial sums as rows of 128 consecutive outputs of one token: with SWAP those run along the rows of the MMA
        static_assert(SWAP || BN == 128, "128 outputs per row");
        constexpr int kTokens = SWAP ? BN : 128;
        const int token0 = SWAP ? row_b : row_a, col0 = SWAP ? row_a : row_b;
        int* part = reinterpret_cast<int*>(smem);
        if (warp >= 2 && good) {
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                uint32_t v[32];
                tmem_ld_32x32(t_lane + c, v);
                tmem_ld_wait();
                if (SWAP) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (c + j < BN) part[(c + j) * kI8PartPitch + q * 32 + lane] = static_cast<int>(v[j]);
                } else {
                    uint4* dst = reinterpret_cast<uint4*>(part + (q * 32 + lane) * kI8PartPitch + c);
#pragma unroll
                    for (int j = 0; j < 8; ++j) dst[j] = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2 && good) {
            // each CTA finishes an equal share of the tokens, each lane four neighbouring outputs
            const int col = col0 + 4 * lane, share = kTokens / split;
            float sc[4], b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sc[j] = col + j < p.N ? __ldg(p.scale_b + col + j) : 0.0f;
                b[j] = p.bias && col + j < p.N ? __ldg(p.bias + col + j) : 0.0f;
            }
#pragma unroll 2
            for (int i = rank * share + q; i < (rank + 1) * share; i += 4) {
                const int token = token0 + i;
                if (token >= p.M) break;
                const uint32_t at = smem_base + 4u * (i * kI8PartPitch + 4 * lane);
                int4 x[8];
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    if (s < split) x[s] = ld_shared_cluster_v4(mapa_shared(at, s));
                int4 sum = x[0];
#pragma unroll
                for (int s = 1; s < 8; ++s)
                    if (s < split) sum.x += x[s].x, sum.y += x[s].y, sum.z += x[s].z, sum.w += x[s].w;
                const float sa = __ldg(p.scale_a + token);
                const float o[4] = {static_cast<float>(sum.x) * sa * sc[0] + b[0], static_cast<float>(sum.y) * sa * sc[1] + b[1],
                                    static_cast<float>(sum.z) * sa * sc[2] + b[2], static_cast<float>(sum.w) * sa * sc[3] + b[3]};
                const long long to = token * p.ld_out + col;
                if (p.vec && col + 4 <= p.N) {
                    if (p.out_type == kF32)
                        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + to) = make_float4(o[0], o[1], o[2], o[3]);
                    else
                        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + to) =
                            make_uint2(pack2(o[0], o[1], p.out_type), pack2(o[2], o[3], p.out_type));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col + j < p.N) store1(p.out, p.out_type, to + j, o[j]);
                }
            }
        }
        __syncwarp();
        cluster_arrive();  // no CTA leaves while another may still read its partial sums
        cluster_wait();
    } else if (warp >= 2 && good) {
        if (SWAP) {
            const float sr = r < p.N ? p.scale_b[r] : 0.0f, b = p.bias && r < p.N ? p.bias[r] : 0.0f;
#pragma unroll 1
            for (int c = 0; c < BN && row_b + c < p.M; c += 32) {
                uint32_t v[32];
                __syncwarp();
                tmem_ld_32x32(t_lane + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const int token = row_b + c + j;
                    if (c + j >= BN || token >= p.M) break;
                    if (r < p.N)
                        store1(p.out, p.out_type, token * p.ld_out + r,
                               static_cast<float>(static_cast<int>(v[j])) * p.scale_a[token] * sr + b);
                }
            }
        } else {
            const float sa = r < p.M ? p.scale_a[r] : 0.0f;
#pragma unroll 1
            for (int c = 0; c < BN && row_b + c < p.N; c += 32) {
                uint32_t v[32];
                I8Cols k;
                __syncwarp();
                tmem_ld_32x32(t_lane + c, v);
                i8_columns(p, row_b + c, lane, k);
                tmem_ld_wait();
                i8_store_chunk(p, reinterpret_cast<float*>(smem + q * kI8OutBytes), v, sa, k, row_a + q * 32, row_b + c, lane);
            }
        }
    }
    __syncwarp();
    if (*abort_flag) __nanosleep(1000000u);  // let bulk copies still in flight land before shared memory is released
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// ---- the product on CTA pairs ------------------------------------------------------------------------------------
// Large products: 256 x 256 tiles on clusters of two CTAs (tcgen05.mma.cta_group::2), one persistent pair per two SMs.  Each
// CTA loads its own 128 rows of A and one half of the tile's rows of B, so that a stage of 128 k costs it 32 KB for 128 x 256
// results instead of the 48 KB of a tile of its own: at 512 cycles a stage, 64 bytes a cycle from L2.  The roles and signals
// are those of the fp16 role (gemm_role2.cuh): full barriers in the leader, empty barriers in both CTAs, two accumulators of
// 256 columns so that a tile is written while the next one is summed.  8192 x 8192 x 4096: 170 us = 3.2 POP/s at full clock, where
// twice the measured bf16 rate would be 163 us; sustained it runs at 1.55 GHz under the power limit.
__device__ __forceinline__ void umma_i8_pair_x4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, t;\n"
        ".reg .b64 a, b;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.eq.b32 t, 0, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
        "add.s64 a, %1, 2;\n"
        "add.s64 b, %2, 2;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, t;\n"
        "add.s64 a, %1, 4;\n"
        "add.s64 b, %2, 4;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, t;\n"
        "add.s64 a, %1, 6;\n"
        "add.s64 b, %2, 6;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, t;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst_smem, const void* tmap, uint32_t bar_cluster_addr, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar_cluster_addr), "r"(x), "r"(y)
        : "memory");
}

struct I8PairSmem {
    static constexpr int kStages = 5;
    static constexpr int kOutWarps = 8;
    static constexpr int kTileBytes = 128 * kI8BK;
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr int kOutOffset = kStages * kStageBytes;
    static constexpr int kBarOffset = kOutOffset + kOutWarps * kI8OutBytes;
    static constexpr int kNumBars = 2 * kStages + 4;
    static constexpr int kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr int kAbortOffset = kTmemSlotOffset + 4;
    static constexpr int kBytes = kAbortOffset + 4;
};

constexpr int kI8PairThreads = 64 + 32 * I8PairSmem::kOutWarps;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kI8PairThreads, 1)
i8gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const I8Args p) {
    using L = I8PairSmem;
    constexpr int ST = L::kStages;
    constexpr uint32_t kIdesc = umma_idesc_i8_s32(256, 256);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_smem_1024(smem_raw);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader_cta = rank == 0;
    const uint32_t base = smem_u32(smem), bars = base + L::kBarOffset;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (ST + s); };
    auto tfull_bar = [&](int a) { return bars + 8u * (2 * ST + a); };
    auto tempty_bar = [&](int a) { return bars + 8u * (2 * ST + 2 + a); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kTmemSlotOffset);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbortOffset);
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int tiles_m = (p.M + 255) / 256, tiles_n = (p.N + 255) / 256, kblocks = (p.K + kI8BK - 1) / kI8BK;
    // up to 2^22 tiles a side (M, N <= 2^30): the launcher keeps their product below 2^31
    const int tiles = tiles_m * tiles_n;

    if (warp == 0 && lane == 0) {
        *abort_flag = 0u;
        for (int s = 0; s < ST; ++s) {
            mbar_init(full_bar(s), 1);   // used in the leader only
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 2 * L::kOutWarps);  // used in the leader only: the output warps of both CTAs
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
    }
    __syncwarp();
    cluster_arrive();  // publishes the barrier initialisation to the peer
    cluster_wait();
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (lane == 0) {
            int stage = 0, waits = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint32_t empty_peer0 = mapa_shared(empty_bar(0), 1u);
            // wait number i of the leader sees the commit of K-block i - ST; every one after the first ST, which pass without
            // an arrival in both CTAs, is passed on to the peer
            auto wait_empty = [&]() {
                ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_EMPTY);
                if (ok && leader_cta && waits >= ST) mbar_arrive_cluster_relaxed(empty_peer0 + 8u * stage);
                ++waits;
                return ok;
            };
            auto advance = [&]() {
                if (++stage == ST) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            for (int tile = pair; ok && tile < tiles; tile += npairs) {
                const int row_a = tile % tiles_m * 256 + static_cast<int>(rank) * 128;
                const int row_b = tile / tiles_m * 256 + static_cast<int>(rank) * 128;
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!wait_empty()) break;
                    if (leader_cta) mbar_arrive_expect_tx(full_bar(stage), 2u * L::kStageBytes);
                    const uint32_t full_leader = mapa_shared(full_bar(stage), 0u);
                    const uint32_t dst = base + stage * L::kStageBytes;
                    tma_load_2d_pair(dst, &tmap_a, full_leader, kb * kI8BK, row_a);
                    tma_load_2d_pair(dst + L::kTileBytes, &tmap_b, full_leader, kb * kI8BK, row_b);
                    advance();
                }
            }
            // the last commits arrive on the empty barriers asynchronously: no CTA retires before they have landed
            for (int s = 0; s < ST && ok; ++s) {
                wait_empty();
                advance();
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader only) ----------------
        if (leader_cta) {
            const bool issuer = elect_lane();
            int stage = 0;
            uint32_t phase = 0, it = 0;
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity, unsigned code) {
                return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, code)) != 0;
            };
            for (int tile = pair; ok && tile < tiles; tile += npairs, ++it) {
                const uint32_t as = it & 1u;
                ok = wait(tempty_bar(as), ((it >> 1) & 1u) ^ 1u, DEV_TIMEOUT_TMEM_EMPTY);
                if (!ok) break;
                tc_fence_after_sync();
                for (int kb = 0; kb < kblocks; ++kb) {
                    ok = wait(full_bar(stage), phase, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t src = base + stage * L::kStageBytes;
                    const uint64_t a_desc = umma_smem_desc_sw128(src), b_desc = umma_smem_desc_sw128(src + L::kTileBytes);
                    if (issuer) {
                        umma_i8_pair_x4(tmem + as * 256, a_desc, b_desc, kIdesc, kb != 0);
                        umma_commit_pair(empty_bar(stage));
                    }
                    __syncwarp();
                    if (++stage == ST) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok && issuer) {
                    umma_commit_pair(tfull_bar(as));
                    umma_commit_pair(mapa_shared(tfull_bar(as), 1u));
                }
                __syncwarp();
            }
            // the peer's output warps arrive on this CTA's barriers: wait until both accumulators have been given back
            for (int j = 0; j < 2 && ok; ++j, ++it)
                ok = wait(tempty_bar(it & 1u), ((it >> 1) & 1u) ^ 1u, DEV_TIMEOUT_TMEM_EMPTY);
        }
    } else {
        // ---------------- output (both CTAs) ----------------
        // two warps for each 32 rows, half of the columns each: four warps took 12,000 cycles for a tile, more than the MMAs
        // of K = 2048 take
        const int q = warp & 3, first = (warp - 2) / 4 * 128;
        const uint32_t tempty_leader0 = mapa_shared(tempty_bar(0), 0u);
        float* stage = reinterpret_cast<float*>(smem + L::kOutOffset + (warp - 2) * kI8OutBytes);
        uint32_t it = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < tiles; tile += npairs, ++it) {
            const uint32_t as = it & 1u;
            ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(as), (it >> 1) & 1u, abort_flag, p.status, DEV_TIMEOUT_TMEM_FULL)) != 0;
            if (!ok) break;
            tc_fence_after_sync();
            const int row0 = tile % tiles_m * 256 + static_cast<int>(rank) * 128 + q * 32, col0 = tile / tiles_m * 256;
            const float sa = row0 + lane < p.M ? __ldg(p.scale_a + row0 + lane) : 0.0f;
            const uint32_t t_lane = tmem + (static_cast<uint32_t>(q * 32) << 16) + as * 256;
#pragma unroll 1
            for (int c = first; c < first + 128 && col0 + c < p.N && row0 < p.M; c += 64) {
                // two chunks on their way at once
                uint32_t v[32], w[32];
                I8Cols k, m;
                tmem_ld_32x32(t_lane + c, v);
                tmem_ld_32x32(t_lane + c + 32, w);
                i8_columns(p, col0 + c, lane, k);
                i8_columns(p, min(col0 + c + 32, p.N - 1), lane, m);
                tmem_ld_wait();
                i8_store_chunk(p, stage, v, sa, k, row0, col0 + c, lane);
                if (col0 + c + 32 < p.N) i8_store_chunk(p, stage, w, sa, m, row0, col0 + c + 32, lane);
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(tempty_leader0 + 8u * as);
        }
    }
    __syncwarp();
    if (*abort_flag) __nanosleep(1000000u);  // let bulk copies still in flight land before shared memory is released
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

}  // namespace tk
