// Product of 8-bit integers with a scale for each token and each output channel:
//   out[m][n] = (sum_k A[m][k] B[n][k]) * scale_a[m] * scale_b[n] + bias[n]
// The sums are exact: tcgen05.mma kind::i8 accumulates in 32-bit integers, and |sum| <= K 2^14 < 2^31 for K <= 131071.
// One rounding to fp32 follows, then the scales, then the rounding to the output's type.
//
// Operand tiles are 128 bytes (128 values of k) wide, K-major, 128-byte swizzled by TMA; rows and k beyond the matrices
// arrive as zeros and add nothing, so no size has to be a multiple of a tile.
#pragma once
#include "gemm_role2.cuh"
#include "row_ops.cuh"

namespace tk {

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

template <int BN, int STAGES>
struct I8Smem {
    static constexpr int kABytes = 128 * kI8BK;
    static constexpr int kBBytes = BN * kI8BK;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kPartBytes = 128 * BN * 4;  // partial sums of a K range, over the drained stages
    static constexpr int kRing = STAGES * kStageBytes;
    static constexpr int kBarOffset = kRing > kPartBytes ? kRing : kPartBytes;
    static constexpr int kTmemSlotOffset = kBarOffset + (2 * STAGES + 1) * 8;
    static constexpr int kAbortOffset = kTmemSlotOffset + 4;
    static constexpr int kBytes = kAbortOffset + 4;
};

__device__ __forceinline__ int ld_shared_cluster_s32(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
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
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_EMPTY)) break;
                mbar_arrive_expect_tx(full_bar(stage), L::kStageBytes);
                const uint32_t dst = smem_base + stage * L::kStageBytes;
                tma_load_2d(dst, &tmap_a, full_bar(stage), kb * kI8BK, row_a);
                tma_load_2d(dst + L::kABytes, &tmap_b, full_bar(stage), kb * kI8BK, row_b);
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
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
    // the accumulator is complete: so have all loads landed and all commits before this one been signalled
    __syncwarp();
    const bool good = mbar_wait(done_bar, 0, abort_flag, p.status, DEV_TIMEOUT_TMEM_FULL);
    tc_fence_after_sync();

    const int q = warp & 3;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const int r = row_a + q * 32 + lane;  // this thread's row of the MMA
    if (split > 1) {
        int* part = reinterpret_cast<int*>(smem);  // [BN][128]
        if (warp >= 2 && good) {
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                uint32_t v[32];
                tmem_ld_32x32(t_lane + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c + j < BN) part[(c + j) * 128 + q * 32 + lane] = static_cast<int>(v[j]);
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2 && good) {
            const int share = BN / split, c0 = rank * share;
            const int rows = SWAP ? p.N : p.M, cols = SWAP ? p.M : p.N;
            const float sr = r < rows ? (SWAP ? p.scale_b[r] : p.scale_a[r]) : 0.0f;
            const float bias_r = SWAP && p.bias && r < rows ? p.bias[r] : 0.0f;
            const uint32_t mine = smem_base + 4u * (q * 32 + lane);
#pragma unroll 4
            for (int c = c0; c < c0 + share; ++c) {
                const int cg = row_b + c;
                if (cg >= cols) break;
                int sum = 0;
                for (int s = 0; s < split; ++s) sum += ld_shared_cluster_s32(mapa_shared(mine + 512u * c, s));
                const float sc = SWAP ? p.scale_a[cg] : p.scale_b[cg];
                float v = static_cast<float>(sum) * (SWAP ? sc : sr) * (SWAP ? sr : sc);
                v += SWAP ? bias_r : (p.bias ? p.bias[cg] : 0.0f);
                if (r < rows)
                    store1(p.out, p.out_type, SWAP ? cg * p.ld_out + r : r * p.ld_out + cg, v);
            }
        }
        __syncwarp();
        cluster_arrive();  // no CTA leaves while another may still read its partial sums
        cluster_wait();
    } else if (warp >= 2 && good) {
        const int rows = SWAP ? p.N : p.M, cols = SWAP ? p.M : p.N;
        const float sr = r < rows ? (SWAP ? p.scale_b[r] : p.scale_a[r]) : 0.0f;
        const float bias_r = SWAP && p.bias && r < rows ? p.bias[r] : 0.0f;
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
            if (row_b + c >= cols) break;
            uint32_t v[32];
            __syncwarp();
            tmem_ld_32x32(t_lane + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
                const int cg = row_b + c + j;
                if (r >= rows || c + j >= BN || cg >= cols) break;
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int ci = min(cg + i, cols - 1);
                    const float sc = __ldg((SWAP ? p.scale_a : p.scale_b) + ci);
                    o[i] = static_cast<float>(static_cast<int>(v[j + i])) * (SWAP ? sc : sr) * (SWAP ? sr : sc);
                    o[i] += SWAP ? bias_r : (p.bias ? __ldg(p.bias + ci) : 0.0f);
                }
                if (!SWAP && p.vec && cg + 8 <= cols) {
                    store8(p.out, p.out_type, r * p.ld_out + cg, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (cg + i < cols)
                            store1(p.out, p.out_type, SWAP ? (cg + i) * p.ld_out + r : r * p.ld_out + cg + i, o[i]);
                }
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

}  // namespace tk
