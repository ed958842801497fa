// Attention over packed sequences on the tensor cores: prompts and chunks of prompts (the definition is in
// attention_rows.cuh).
//
// Rows.  The query heads that share a key head are rows of one tile: a tile has 128 / group tokens x group heads, token
// after token, so that a key tile fetched once serves the whole group and short sequences still fill rows.  One work item
// is two tiles (256 rows) of one sequence and key head; one persistent CTA per SM walks the items.
//
//   warps 0..3, 4..7  softmax of tile 0 and of tile 1, one row per thread; at the end of an item they write its rows
//   warp 8            issues the MMAs of both tiles:  S = Q K^T (128 x 128, fp32, TMEM),  O += P V  with P read from TMEM
//   warp 9            TMA: Q tiles, then K and V tiles of 128 keys through a ring
//
// While the softmax of one tile runs, the tensor cores work for the other one.  P overwrites the columns of its S.
// The running maximum is raised (and O multiplied by what that costs, in TMEM) only when the new one exceeds it by more
// than 2^8: weights stay below 2^8, well inside the 16-bit types, the sums are fp32, and the final division makes it
// exact; after the first tiles almost no item pays for a rescale.  P is rounded to the type of V because the tensor
// cores take two operands of one type; the row sum is taken before that rounding.
//
// Masks.  Keys beyond a row's limit get -infinity whatever their score is.  Weights of hidden keys are exact zeros, and
// the values behind the sequence's last key within the last 16 that an MMA reads are zeroed in shared memory, so that
// nothing they hold (NaN included) can enter.
//
// Bound: per key tile and SM the two tiles take 2 x 2 x 512 cycles of the tensor pipe (head size 128) and 32768 powers of
// two = 2048 cycles of the special-function units; both run at the same time.
#pragma once
#include <cuda.h>

#include "attention_rows.cuh"
#include "gemm_role2.cuh"

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

// The MMAs of a tile are issued back to back from one block of instructions: with N = 128 each takes 64 cycles of the
// tensor pipe, and a loop that rebuilds its operands for each (138 cycles per MMA as measured) leaves the pipe idle.
// Four k-steps of S = Q K^T: 16 elements = 32 bytes further along both swizzled rows
__device__ __forceinline__ void umma_scores_x4(uint32_t d_tmem, uint64_t q_desc, uint64_t k_desc, uint32_t idesc,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, t;\n"
        ".reg .b64 a, b;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.eq.b32 t, 0, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "add.s64 a, %1, 2;\n"
        "add.s64 b, %2, 2;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
        "add.s64 a, %1, 4;\n"
        "add.s64 b, %2, 4;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
        "add.s64 a, %1, 6;\n"
        "add.s64 b, %2, 6;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
        "}\n" ::"r"(d_tmem),
        "l"(q_desc), "l"(k_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Four k-steps of O += P V, P in tensor memory: 16 keys = 8 columns of P and 2048 bytes of V
__device__ __forceinline__ void umma_values_x4(uint32_t d_tmem, uint32_t p_tmem, uint64_t v_desc, uint32_t idesc,
                                               uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, t;\n"
        ".reg .b64 b;\n"
        ".reg .b32 a;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.eq.b32 t, 0, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "add.s32 a, %1, 8;\n"
        "add.s64 b, %2, 128;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n"
        "add.s32 a, %1, 16;\n"
        "add.s64 b, %2, 256;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n"
        "add.s32 a, %1, 24;\n"
        "add.s64 b, %2, 384;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n"
        "}\n" ::"r"(d_tmem),
        "r"(p_tmem), "l"(v_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// one k-step of O += P V
__device__ __forceinline__ void umma_values(uint32_t d_tmem, uint32_t p_tmem, uint64_t v_desc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(p_tmem), "l"(v_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// V as the B operand of P V: its rows are keys (the k of the product), 64 head elements = 128 bytes contiguous, written
// by TMA with the 128-byte swizzle.  The operand is therefore "MN-major": eight keys apart is the stride byte offset,
// 64 head elements apart (the next box) the leading byte offset.
__device__ __forceinline__ uint64_t umma_smem_desc_sw128_mn(uint32_t smem_addr, uint32_t box_bytes) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(box_bytes >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= 1ull << 46;
    d |= 2ull << 61;
    return d;
}

constexpr int kAttnThreads = 384;  // the last two warps only give their registers away
constexpr int kAttnKeys = 128;  // keys of a tile

// Registers: launched with 168 a thread (3 warps per scheduler); the softmax warps take 208, the others keep 88:
// 2 x 128 x 208 + 128 x 88 = 384 x 168.
constexpr int kAttnSoftmaxRegs = 208, kAttnOtherRegs = 88;
static_assert(256 * kAttnSoftmaxRegs + 128 * kAttnOtherRegs <= kAttnThreads * 168, "registers of the block");
template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// two fp32 operations per instruction
__device__ __forceinline__ void fma2(float& x, float& y, float sx, float sy, float ax, float ay) {
    asm("{\n"
        ".reg .b64 v, w, c;\n"
        "mov.b64 v, {%0, %1};\n"
        "mov.b64 w, {%2, %3};\n"
        "mov.b64 c, {%4, %5};\n"
        "fma.rn.f32x2 v, v, w, c;\n"
        "mov.b64 {%0, %1}, v;\n"
        "}\n"
        : "+f"(x), "+f"(y)
        : "f"(sx), "f"(sy), "f"(ax), "f"(ay));
}
__device__ __forceinline__ void add2(float& x, float& y, float ax, float ay) {
    asm("{\n"
        ".reg .b64 v, w;\n"
        "mov.b64 v, {%0, %1};\n"
        "mov.b64 w, {%2, %3};\n"
        "add.rn.f32x2 v, v, w;\n"
        "mov.b64 {%0, %1}, v;\n"
        "}\n"
        : "+f"(x), "+f"(y)
        : "f"(ax), "f"(ay));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ float max_of(const uint32_t (&s)[32]) {
    float m0 = __uint_as_float(s[0]), m1 = __uint_as_float(s[1]);
#pragma unroll
    for (int i = 2; i < 30; i += 4) {
        m0 = max3(m0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        m1 = max3(m1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
    }
    return max3(max3(m0, __uint_as_float(s[30]), __uint_as_float(s[31])), m1, m1);
}
__device__ __forceinline__ void hide_from(uint32_t (&s)[32], int limit) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (i >= limit) s[i] = 0xff800000u;  // -infinity
}
// 32 weights 2^(scale s + off) of a row: their sums by fours and, rounded to the type, their pairs from w[at] on
template <int TYPE>
__device__ __forceinline__ void weights(const uint32_t (&s)[32], float scale, float off, float (&sum)[4], uint32_t (&w)[32],
                                        const int at) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        float x = __uint_as_float(s[i]), y = __uint_as_float(s[i + 1]);
        fma2(x, y, scale, scale, off, off);
        x = ex2(x), y = ex2(y);
        if (i & 2) add2(sum[2], sum[3], x, y);
        else add2(sum[0], sum[1], x, y);
        w[at + i / 2] = pack2(x, y, TYPE);
    }
}

template <int D>
struct AttnSmem {
    static constexpr int kBoxBytes = 128 * 128;  // 128 rows x 64 elements
    static constexpr int kTileBytes = (D / 64) * kBoxBytes;
    static constexpr int kStages = D == 128 ? 5 : 10;
    static constexpr int kKvOffset = 2 * kTileBytes;
    static constexpr int kBarOffset = kKvOffset + kStages * kTileBytes;
    // barriers: ring full / empty, Q full / empty per tile, S full, P full, O full per tile
    static constexpr int kNumBars = 2 * kStages + 10;
    static constexpr int kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr int kAbortOffset = kTmemSlotOffset + 4;
    static constexpr int kBytes = kAbortOffset + 4;
};

// One work item: two tiles of query rows of one sequence and key head.
struct AttnItem {
    AttnSeq s;
    int kv;    // key head
    int t0;    // first token of tile 0
    int n[2];  // key tiles that some row of the tile sees
};

// Finds work items by index, in ascending order of calls.  Items of a sequence run from its last tokens (which see the
// most keys) to its first, key heads innermost.  All lanes of a warp call it together.
struct AttnWalk {
    int base;         // first sequence of the window of 32 that the search stands at
    long long before; // items of the sequences before it
    __device__ __forceinline__ void init() { base = 0, before = 0; }

    __device__ __forceinline__ bool find(const AttnArgs& p, long long index, int tile_tokens, int lane, AttnItem& it) {
        const int pair_tokens = 2 * tile_tokens;
        while (base < p.n_seqs) {
            AttnSeq s;
            s.q_len = 0, s.q0 = 0, s.k0 = 0, s.k_len = 0;
            if (base + lane < p.n_seqs) s.load(p, base + lane);
            const long long mine = static_cast<long long>((s.q_len + pair_tokens - 1) / pair_tokens) * p.kv_heads;
            long long upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += u;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > index);
            if (hit) {
                const int l = __ffs(hit) - 1;
                it.s.q0 = __shfl_sync(0xffffffffu, s.q0, l);
                it.s.q_len = __shfl_sync(0xffffffffu, s.q_len, l);
                it.s.k0 = __shfl_sync(0xffffffffu, s.k0, l);
                it.s.k_len = __shfl_sync(0xffffffffu, s.k_len, l);
                const long long of = __shfl_sync(0xffffffffu, mine, l);
                const long long at = index - before - (__shfl_sync(0xffffffffu, upto, l) - of);
                it.kv = static_cast<int>(at % p.kv_heads);
                it.t0 = static_cast<int>((of - 1 - at) / p.kv_heads) * pair_tokens;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int first = it.t0 + h * tile_tokens;
                    const int last = min(first + tile_tokens, it.s.q_len) - 1;
                    int keys = it.s.k_len;
                    if (p.causal) keys = min(keys, max(0, last + 1 + it.s.k_len - it.s.q_len));
                    it.n[h] = last < first ? 0 : (keys + kAttnKeys - 1) / kAttnKeys;
                }
                return true;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
            base += 32;
        }
        return false;
    }
};

// item of CTA c in round r: every other round runs backwards, so that long and short items even out
__device__ __forceinline__ long long attn_index(int round) {
    const long long g = gridDim.x;
    return round * g + ((round & 1) ? g - 1 - blockIdx.x : static_cast<long long>(blockIdx.x));
}

template <int D, int TYPE>
__global__ void __launch_bounds__(kAttnThreads, 1)
attention_prompt_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                        const __grid_constant__ CUtensorMap tmap_v, const AttnArgs p, const int group,
                        unsigned* status) {
    using L = AttnSmem<D>;
    constexpr int ST = L::kStages;
    constexpr uint32_t kO = 256;  // TMEM: S / P of tile 0 at column 0, of tile 1 at 128, O of the tiles at 256 and 384
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_smem_1024(smem_raw);
    // values that are the same in a whole warp are taken from lane 0, so that the compiler knows it
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem);
    const uint32_t bars = base + L::kBarOffset;
    auto kv_full = [&](int s) { return bars + 8u * s; };
    auto kv_empty = [&](int s) { return bars + 8u * (ST + s); };
    auto q_full = [&](int h) { return bars + 8u * (2 * ST + h); };
    auto q_empty = [&](int h) { return bars + 8u * (2 * ST + 2 + h); };
    auto s_full = [&](int h) { return bars + 8u * (2 * ST + 4 + h); };
    auto p_full = [&](int h) { return bars + 8u * (2 * ST + 6 + h); };
    auto o_full = [&](int h) { return bars + 8u * (2 * ST + 8 + h); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kTmemSlotOffset);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbortOffset);

    if (warp == 8) {
        if (lane == 0) {
            *abort_flag = 0u;
            for (int s = 0; s < ST; ++s) {
                mbar_init(kv_full(s), 1);
                mbar_init(kv_empty(s), 1);
            }
            for (int h = 0; h < 2; ++h) {
                mbar_init(q_full(h), 1);
                mbar_init(q_empty(h), 1);
                mbar_init(s_full(h), 1);
                mbar_init(p_full(h), 4);  // one arrival per softmax warp
                mbar_init(o_full(h), 1);
            }
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish();
    }
    if (warp == 9 && lane == 0) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int tile_tokens = 128 / group;

    AttnWalk walk;
    walk.init();
    AttnItem it;
    // a wait of a whole warp: one verdict for all lanes
    auto wait = [&](uint32_t bar, uint32_t parity, unsigned code) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code)) != 0;
    };

    if (warp >= 8) {
      fewer_registers<kAttnOtherRegs>();
      if (warp == 9) {
        // ---------------- TMA producer ----------------
        int stage = 0;
        uint32_t phase = 0, q_phase[2] = {0, 0};
        bool ok = true;
        const uint32_t q_bytes = static_cast<uint32_t>((D / 64) * tile_tokens * group * 128);
        for (int round = 0; ok && walk.find(p, attn_index(round), tile_tokens, lane, it); ++round) {
            if (lane == 0) {
                const int n = max(it.n[0], it.n[1]);
                auto load_q = [&](int h) {
                    if (it.n[h] == 0) return true;
                    if (!mbar_wait(q_empty(h), q_phase[h] ^ 1u, abort_flag, status, DEV_TIMEOUT_EMPTY)) return false;
                    q_phase[h] ^= 1u;
                    mbar_arrive_expect_tx(q_full(h), q_bytes);
#pragma unroll
                    for (int x = 0; x < D; x += 64)
                        tma_load_tile(base + h * L::kTileBytes + (x / 64) * L::kBoxBytes, &tmap_q, q_full(h), x,
                                      it.kv * group, it.s.q0 + it.t0 + h * tile_tokens);
                    return true;
                };
                auto load_kv = [&](const CUtensorMap* map, int j) {
                    if (!mbar_wait(kv_empty(stage), phase ^ 1u, abort_flag, status, DEV_TIMEOUT_EMPTY)) return false;
                    mbar_arrive_expect_tx(kv_full(stage), L::kTileBytes);
#pragma unroll
                    for (int x = 0; x < D; x += 64)
                        tma_load_tile(base + L::kKvOffset + stage * L::kTileBytes + (x / 64) * L::kBoxBytes, map,
                                      kv_full(stage), x, it.kv, it.s.k0 + j * kAttnKeys);
                    if (++stage == ST) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    return true;
                };
                ok = load_q(0);
                for (int j = 0; ok && j < n; ++j) {
                    ok = load_kv(&tmap_k, j);
                    if (ok && j == 0) ok = load_q(1);
                    ok = ok && load_kv(&tmap_v, j);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        }
        // the last commits arrive on the empty barriers asynchronously: the CTA must not retire before they have landed
        if (lane == 0) {
            for (int s = 0; s < ST && ok; ++s) {
                ok = mbar_wait(kv_empty(stage), phase ^ 1u, abort_flag, status, DEV_TIMEOUT_EMPTY);
                if (++stage == ST) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
                ok = ok && mbar_wait(q_empty(h), q_phase[h] ^ 1u, abort_flag, status, DEV_TIMEOUT_EMPTY);
        }
      } else if (warp == 8) {
        // ---------------- MMA issuer ----------------
        const uint32_t fmt = TYPE == kBF16 ? (1u << 7) | (1u << 10) : 0u;  // A and B format: 0 = fp16, 1 = bf16
        const uint32_t idesc_s = umma_idesc_f16_f32(128, kAttnKeys) | fmt;
        const uint32_t idesc_o = umma_idesc_f16_f32(128, D) | fmt | (1u << 16);  // B = V is MN-major
        int stage = 0;  // ring position: K_0 V_0 K_1 V_1 ... of one item after another
        uint32_t phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
        bool ok = true;
        auto advance = [&](int& st, uint32_t& ph) {
            if (++st == ST) {
                st = 0;
                ph ^= 1u;
            }
        };
        const bool leader = elect_lane();
        auto scores = [&](int h, int st) {
            const uint64_t q_desc = umma_smem_desc_sw128(base + h * L::kTileBytes);
            const uint64_t k_desc = umma_smem_desc_sw128(base + L::kKvOffset + st * L::kTileBytes);
            if (leader) {
#pragma unroll
                for (int x = 0; x < D / 64; ++x)
                    umma_scores_x4(tmem + h * 128, q_desc + x * (L::kBoxBytes >> 4), k_desc + x * (L::kBoxBytes >> 4),
                                   idesc_s, x != 0);
                umma_commit(s_full(h));
            }
        };
        for (int round = 0; ok && walk.find(p, attn_index(round), tile_tokens, lane, it); ++round) {
            const int n = max(it.n[0], it.n[1]);
            if (n == 0) continue;
            // the first scores of both tiles
            ok = wait(kv_full(stage), phase, DEV_TIMEOUT_FULL);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!ok || it.n[h] == 0) continue;
                ok = wait(q_full(h), q_phase[h], DEV_TIMEOUT_FULL);
                q_phase[h] ^= 1u;
                if (!ok) continue;
                tc_fence_after_sync();
                scores(h, stage);
                if (it.n[h] == 1 && leader) umma_commit(q_empty(h));
            }
            if (!ok) break;
            if (leader) umma_commit(kv_empty(stage));
            __syncwarp();
            advance(stage, phase);
            for (int j = 0; ok && j < n; ++j) {
                const int v_stage = stage;
                const uint32_t v_phase = phase;
                advance(stage, phase);
                const int k_stage = stage;
                const uint32_t k_phase = phase;
                ok = wait(kv_full(v_stage), v_phase, DEV_TIMEOUT_FULL);
                if (!ok) break;
                const uint32_t v = base + L::kKvOffset + v_stage * L::kTileBytes;
                const int left = it.s.k_len - j * kAttnKeys;  // keys of the sequence from this tile on
                if (left < kAttnKeys && (left & 15)) {
                    // rows behind the last key, up to the next 16: zeros (16 bytes per lane and step)
                    const int rows = 16 - (left & 15);
                    for (int e = lane; e < rows * 8 * (D / 64); e += 32) {
                        const int box = e / (rows * 8), r = e % (rows * 8);
                        *reinterpret_cast<uint4*>(smem + (v - base) + box * L::kBoxBytes + (left + r / 8) * 128 + (r % 8) * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                const bool more = j + 1 < n;
                if (more) ok = wait(kv_full(k_stage), k_phase, DEV_TIMEOUT_FULL);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!ok || j >= it.n[h]) continue;
                    ok = wait(p_full(h), p_phase[h], DEV_TIMEOUT_TMEM_EMPTY);
                    p_phase[h] ^= 1u;
                    if (!ok) continue;
                    tc_fence_after_sync();
                    // weights behind the tile's last visible key are zeros: those k-steps are left out
                    int keys = left;
                    if (p.causal) {
                        const int last = min(it.t0 + (h + 1) * tile_tokens, it.s.q_len);
                        keys = min(keys, last + it.s.k_len - it.s.q_len - j * kAttnKeys);
                    }
                    const uint64_t v_desc = umma_smem_desc_sw128_mn(v, L::kBoxBytes);
                    const uint32_t o_tmem = tmem + kO + h * 128, p_tmem = tmem + h * 128;
                    const int steps = (keys + 15) / 16;
                    if (leader) {
                        if (steps >= kAttnKeys / 16) {
                            umma_values_x4(o_tmem, p_tmem, v_desc, idesc_o, j != 0);
                            umma_values_x4(o_tmem, p_tmem + 32, v_desc + 512, idesc_o, 1);
                        } else {
                            for (int x = 0; x < steps; ++x)
                                umma_values(o_tmem, p_tmem + 8 * x, v_desc + 128 * x, idesc_o, j != 0 || x != 0);
                        }
                        if (j == it.n[h] - 1) umma_commit(o_full(h));
                    }
                    if (j + 1 < it.n[h]) {
                        scores(h, k_stage);
                        if (j + 2 == it.n[h] && leader) umma_commit(q_empty(h));
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (leader) {
                    umma_commit(kv_empty(v_stage));
                    if (more) umma_commit(kv_empty(k_stage));
                }
                __syncwarp();
                if (more) advance(stage, phase);
            }
        }
      }
    } else {
        // ---------------- softmax ----------------
        more_registers<kAttnSoftmaxRegs>();
        const int h = warp >> 2, r = threadIdx.x & 127;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_s = t_lane + h * 128, t_o = t_lane + kO + h * 128;
        const int token = r / group, head_in = r - token * group;
        uint32_t s_phase = 0, o_phase = 0;
        bool ok = true;
        for (int round = 0; ok && walk.find(p, attn_index(round), tile_tokens, lane, it); ++round) {
            const int first = it.t0 + h * tile_tokens;
            if (first >= it.s.q_len) continue;  // this tile has no rows
            const int t = first + token;
            const bool live = token < tile_tokens && t < it.s.q_len;
            int limit = it.s.k_len, tile_limit = it.s.k_len;  // keys this row sees; keys every row of the tile sees
            if (p.causal) {
                limit = min(limit, max(0, t + 1 + it.s.k_len - it.s.q_len));
                tile_limit = min(tile_limit, max(0, first + 1 + it.s.k_len - it.s.q_len));
            }
            const int n = h ? it.n[1] : it.n[0];
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < n; ++j) {
                ok = wait(s_full(h), s_phase, DEV_TIMEOUT_TMEM_FULL);
                s_phase ^= 1u;
                if (!ok) break;
                tc_fence_after_sync();
                uint32_t s0[32], s1[32], s2[32], s3[32];  // 128 scores of the row
                float top;
                tmem_ld_32x32(t_s, s0);
                tmem_ld_32x32(t_s + 32, s1);
                tmem_ld_wait();
                tmem_ld_32x32(t_s + 64, s2);
                tmem_ld_32x32(t_s + 96, s3);
                if ((j + 1) * kAttnKeys > tile_limit) {
                    const int lim = limit - j * kAttnKeys;
                    tmem_ld_wait();
                    hide_from(s0, lim);
                    hide_from(s1, lim - 32);
                    hide_from(s2, lim - 64);
                    hide_from(s3, lim - 96);
                    top = fmaxf(fmaxf(max_of(s0), max_of(s1)), fmaxf(max_of(s2), max_of(s3)));
                } else {
                    top = fmaxf(max_of(s0), max_of(s1));
                    tmem_ld_wait();
                    top = max3(top, max_of(s2), max_of(s3));
                }
                if (j == 0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, (top - m) * p.scale_log2 > 8.0f || (m == -INFINITY && top > m))) {
                    // the scores of this tile follow the product that last added to O: O is at rest
                    const float up = fmaxf(m, top);
                    const float keep = m == -INFINITY ? 0.0f : ex2((m - up) * p.scale_log2);
                    m = up;
                    l *= keep;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32(t_o + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                        tmem_st_32x32(t_o + c, o);
                    }
                }
                const float off = m == -INFINITY ? 0.0f : -m * p.scale_log2;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                {
                    uint32_t w[32];
                    weights<TYPE>(s0, p.scale_log2, off, sum, w, 0);
                    weights<TYPE>(s1, p.scale_log2, off, sum, w, 16);
                    tmem_st_32x32(t_s, w);
                }
                {
                    uint32_t w[32];
                    weights<TYPE>(s2, p.scale_log2, off, sum, w, 0);
                    weights<TYPE>(s3, p.scale_log2, off, sum, w, 16);
                    tmem_st_32x32(t_s + 32, w);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st_wait();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(h));
            }
            if (ok && n > 0) {
                ok = wait(o_full(h), o_phase, DEV_TIMEOUT_TMEM_FULL);
                o_phase ^= 1u;
                tc_fence_after_sync();
            }
            if (!ok) break;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const long long row = it.s.q0 + static_cast<long long>(t);
            const int head = it.kv * group + head_in;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                __syncwarp();
                if (n > 0) {
                    tmem_ld_32x32(t_o + c, o);
                    tmem_ld_wait();
                }
                if (!live || c >= p.dim) continue;
                uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + row * p.ld_out + static_cast<long long>(head) * p.dim + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (c + 8 * i >= p.dim) break;
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = l == 0.0f ? 0u
                                         : pack2(__uint_as_float(o[8 * i + 2 * e]) * inv,
                                                 __uint_as_float(o[8 * i + 2 * e + 1]) * inv, TYPE);
                    dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            if (live && p.lse)
                p.lse[row * p.heads + head] = l == 0.0f ? -INFINITY : (m * p.scale_log2 + log2f(l)) * kLn2;
            tc_fence_before_sync();  // O has been read: the weights of the next item may follow
        }
    }

    __syncwarp();
    if (*abort_flag) __nanosleep(1000000u);  // let bulk copies still in flight land before shared memory is released
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 8) tmem_dealloc(tmem, 512);
}

}  // namespace tk
