// Attention over packed sequences on the tensor cores: prompts and chunks of prompts (the definition is in
// attention_rows.cuh).
//
// Rows.  The query heads that share a key head are rows of one tile: a tile has 128 / group tokens x group heads, token
// after token, so that a key tile fetched once serves the whole group and short sequences still fill rows.  One work item
// is two tiles (256 rows) of one sequence and key head; one persistent CTA per SM takes items until none is left.
//
//   warps 0..3, 4..7  softmax of tile 0 and of tile 1, one row per thread
//   warps 8..11       write the rows of finished tiles
//   warp 12           issues the MMAs of both tiles:  S = Q K^T (128 x 128, fp32, TMEM),  O += P V  with P read from TMEM
//   warp 13           TMA: Q tiles, then K and V tiles of 128 keys through a ring
//   warp 14           finds the next item and hands it to the others
//
// The grid has a block for every item there can be; a CTA that is done takes over a block that has not started yet
// (cluster launch control), so that items of different lengths even out without a counter in memory.
//
// While the softmax of one tile runs, the tensor cores work for the other one.  P overwrites the columns of its S.
// The running maximum is raised (and O multiplied by what that costs, in TMEM) only when the new one exceeds it by more
// than 2^8: weights stay below 2^8 (2^15 with the lift that fp16 gets), inside the 16-bit types, the sums are fp32, and the
// final division makes it exact; after the first tiles almost no item pays for a rescale.  P is rounded to the type of V
// because the tensor cores take two operands of one type: half a step on each value, error against binary64 1.2 to 1.3
// times that of rounding the result alone.  The row sum is taken before that rounding.
//
// Masks.  Keys beyond a row's limit get -infinity whatever their score is.  Weights of hidden keys are exact zeros, and
// the values behind the sequence's last key within the last 16 that an MMA reads are zeroed in shared memory, so that
// nothing they hold (NaN included) can enter.
//
// Bound: per key tile and SM the two tiles take 2 x 2 x 512 cycles of the tensor pipe (head size 128) and 32768 powers of
// two = 2048 cycles of the special-function units, both at the same time; measured are about 3100 cycles, 1930 of them the softmax
// of a tile (scores from tensor memory and their maximum 370, powers 1460) and 1000 from its weights to its next scores.
// 8192 tokens x 16 heads x 128, causal: 231 us = 1190 TFLOP/s of visible products; sixteen packed prompts 91 us.
#pragma once
#include <cuda.h>

#include "attention_rows.cuh"
#include "i8gemm.cuh"

namespace tk {

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

constexpr int kAttnThreads = 512;
constexpr int kAttnKeys = 128;  // keys of a tile

// Registers: launched with 128 a thread; the softmax warps keep a row of scores each.
constexpr int kAttnSoftmaxRegs = 192, kAttnOutRegs = 72, kAttnOtherRegs = 56;
static_assert(256 * kAttnSoftmaxRegs + 128 * kAttnOutRegs + 128 * kAttnOtherRegs <= kAttnThreads * 128,
              "registers of the block");
template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// maxima that are NaN where an operand is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max2(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
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
// scores from `limit` on become -infinity
__device__ __forceinline__ void hide_from(uint32_t (&s)[32], int limit) {
    const uint32_t seen = limit >= 32 ? 0xffffffffu : limit <= 0 ? 0u : (1u << limit) - 1u;
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (!(seen & (1u << i))) s[i] = 0xff800000u;
}

__device__ __forceinline__ void less(uint32_t (&s)[32], float x) {
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) - x);
}

// 32 weights 2^(scale s + off) of a row: their sums by fours and, rounded to the type, their pairs from w[at] on.  (A share
// of the powers as polynomials on the multiply-add pipes, 1/8 to 3/8 of them, gained nothing: the tiles take turns on the
// special-function units, and at full load the clock is set by the power limit.)
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
    static constexpr int kStages = D == 128 ? 4 : 8;
    static constexpr int kKvOffset = 2 * kTileBytes;
    static constexpr int kOutOffset = kKvOffset + kStages * kTileBytes;
    static constexpr int kOutWarpBytes = 32 * D * 2;  // 32 rows of the output on their way out
    static constexpr int kStatOffset = kOutOffset + 4 * kOutWarpBytes;  // maximum and sum of each row of both tiles
    static constexpr int kItemOffset = kStatOffset + 2 * 128 * 8;
    static constexpr int kClaimOffset = kItemOffset + 32;
    static constexpr int kBarOffset = kClaimOffset + 16;
    // barriers: ring full / empty; per tile Q full / empty, S full, first half of P, all of P, O full, statistics full,
    // O and statistics empty; item full / empty; claim
    static constexpr int kNumBars = 2 * kStages + 16 + 3;
    static constexpr int kTmemSlotOffset = kBarOffset + kNumBars * 8;
    static constexpr int kAbortOffset = kTmemSlotOffset + 4;
    static constexpr int kProgressOffset = kAbortOffset + 4;
    static constexpr int kBytes = kProgressOffset + 4;
};

// One work item: two tiles of query rows of one sequence and key head.
struct AttnItem {
    AttnSeq s;
    int kv;    // key head
    int t0;    // first token of tile 0
    int n[2];  // key tiles that some row of the tile sees
};

// The search for a work item by its number.  Sequences are looked through in windows of 32, forward from where the last
// search ended and from the start again for a number that lies before; the end is remembered.  `Window` holds the sequences
// of one window: load(base) reads them, items() counts their items.
struct AttnSeek {
    int base = 0;             // first sequence of the window
    long long before = 0;     // items of the sequences before it
    long long total = 0x7fffffffffffffffll;  // all items, once a search has come to the end

    // (host and device windows both: the compiler's check of where a template argument's functions may run is off)
#pragma nv_exec_check_disable
    template <class Window>
    __host__ __device__ __forceinline__ bool find(long long index, int n_seqs, Window& w) {
        if (index >= total) return false;
        if (index < before) {
            base = 0, before = 0;
            w.load(base);
        }
        for (long long n; index >= before + (n = w.items());) {
            before += n;
            base += 32;
            if (base >= n_seqs) {
                total = before;
                return false;
            }
            w.load(base);
        }
        return true;
    }
};

// The course of one CTA: its own block's number, then those of the blocks it takes over, until all have started.  Blocks
// are given out in no order that could be relied on, so each number is looked up, also after one that lies behind the last
// item.  hand(index) does with an item what is to be done, take(index) asks for the next number (-1: none left); both are
// false after a wait that ran out.
#pragma nv_exec_check_disable
template <class Find, class Hand, class Take>
__host__ __device__ __forceinline__ bool attn_items(int index, Find find, Hand hand, Take take) {
    while (index >= 0) {
        if (find(index) && !hand()) return false;
        if (!take(index)) return false;
    }
    return true;
}

// Place of item `at` of a sequence that has `of`: items run from its last tokens (which see the most keys) to its first, key
// heads innermost.
__host__ __device__ __forceinline__ void attn_item_place(int at, long long of, int kv_heads, int tile_tokens, int& kv, int& t0) {
    kv = at % kv_heads;
    t0 = (static_cast<int>(of) - 1 - at) / kv_heads * 2 * tile_tokens;
}
__host__ __device__ __forceinline__ long long attn_items_of(int q_len, int kv_heads, int tile_tokens) {
    return static_cast<long long>((q_len + 2 * tile_tokens - 1) / (2 * tile_tokens)) * kv_heads;
}

// A window of the search in the registers of a warp, a sequence per lane; all lanes call together.
struct AttnWindow {
    const AttnArgs& p;
    const int tile_tokens, lane;
    uint32_t* progress;
    AttnSeq s;
    long long mine, upto;  // items of this lane's sequence, and of the window up to and with it

    __device__ __forceinline__ void load(int base) {
        if (lane == 0) atomicAdd(progress, 1u);
        s.q_len = 0, s.q0 = 0, s.k0 = 0, s.k_len = 0;
        if (base + lane < p.n_seqs) s.load(p, base + lane);
        mine = attn_items_of(s.q_len, p.kv_heads, tile_tokens);
        upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
    }
    __device__ __forceinline__ long long items() const { return __shfl_sync(0xffffffffu, upto, 31); }
    // item number `index` of the window
    __device__ __forceinline__ void item(long long index, AttnItem& it) const {
        const int l = __ffs(__ballot_sync(0xffffffffu, upto > index)) - 1;
        it.s.q0 = __shfl_sync(0xffffffffu, s.q0, l);
        it.s.q_len = __shfl_sync(0xffffffffu, s.q_len, l);
        it.s.k0 = __shfl_sync(0xffffffffu, s.k0, l);
        it.s.k_len = __shfl_sync(0xffffffffu, s.k_len, l);
        const long long of = __shfl_sync(0xffffffffu, mine, l);
        attn_item_place(static_cast<int>(index - (__shfl_sync(0xffffffffu, upto, l) - of)), of, p.kv_heads, tile_tokens, it.kv,
                        it.t0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int first = it.t0 + h * tile_tokens;
            const int last = min(first + tile_tokens, it.s.q_len) - 1;
            int keys = it.s.k_len;
            if (p.causal) keys = min(keys, max(0, last + 1 + it.s.k_len - it.s.q_len));
            it.n[h] = last < first ? 0 : (keys + kAttnKeys - 1) / kAttnKeys;
        }
    }
};

// ---- cluster launch control: take over a block of this grid that has not started -------------------------------------
__device__ __forceinline__ void claim_request(uint32_t result_smem, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     result_smem),
                 "r"(bar)
                 : "memory");
}
// the block taken over, or -1 when all have started
__device__ __forceinline__ int claim_result(uint32_t result_smem) {
    int x;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        ".reg .b128 r;\n"
        ".reg .b32 y, z, w;\n"
        "ld.shared.b128 r, [%1];\n"
        "mov.s32 %0, -1;\n"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, r;\n"
        "}\n"
        : "=r"(x)
        : "r"(result_smem)
        : "memory");
    return x;
}

template <int D, int TYPE>
__global__ void __launch_bounds__(kAttnThreads, 1)
attention_prompt_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                        const __grid_constant__ CUtensorMap tmap_v, const AttnArgs p, const int group,
                        unsigned* status) {
    using L = AttnSmem<D>;
    constexpr int ST = L::kStages;
    constexpr float kUnlift = 1.0f / (1 << static_cast<int>(kPromptLift<TYPE>));
    constexpr uint32_t kO = 256;  // TMEM: S / P of tile 0 at column 0, of tile 1 at 128, O of the tiles at 256 and 384
    extern __shared__ __align__(1024) uint8_t attn_smem[];  // tiles need it; there is no room to align by hand
    uint8_t* smem = attn_smem;
    // values that are the same in a whole warp are taken from lane 0, so that the compiler knows it
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem);
    const uint32_t bars = base + L::kBarOffset;
    auto kv_full = [&](int s) { return bars + 8u * s; };
    auto kv_empty = [&](int s) { return bars + 8u * (ST + s); };
    auto q_full = [&](int h) { return bars + 8u * (2 * ST + h); };
    auto q_empty = [&](int h) { return bars + 8u * (2 * ST + 2 + h); };
    auto s_full = [&](int h) { return bars + 8u * (2 * ST + 4 + h); };
    auto p_half = [&](int h) { return bars + 8u * (2 * ST + 6 + h); };
    auto p_full = [&](int h) { return bars + 8u * (2 * ST + 8 + h); };
    auto o_full = [&](int h) { return bars + 8u * (2 * ST + 10 + h); };
    auto stat_full = [&](int h) { return bars + 8u * (2 * ST + 12 + h); };
    auto o_empty = [&](int h) { return bars + 8u * (2 * ST + 14 + h); };
    const uint32_t item_full = bars + 8u * (2 * ST + 16), item_empty = item_full + 8, claim_bar = item_full + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kTmemSlotOffset);
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbortOffset);
    // steps of the producer (tiles asked for) and of the search for items (blocks taken over, windows looked through)
    uint32_t* progress = reinterpret_cast<uint32_t*>(smem + L::kProgressOffset);

    if (warp == 12) {
        if (lane == 0) {
            *abort_flag = 0u;
            *progress = 0u;
            for (int s = 0; s < ST; ++s) {
                mbar_init(kv_full(s), 1);
                mbar_init(kv_empty(s), 1);
            }
            for (int h = 0; h < 2; ++h) {
                mbar_init(q_full(h), 1);
                mbar_init(q_empty(h), 1);
                mbar_init(s_full(h), 1);
                mbar_init(p_half(h), 4);  // one arrival per softmax warp of the tile
                mbar_init(p_full(h), 4);
                mbar_init(o_full(h), 1);
                mbar_init(stat_full(h), 4);
                mbar_init(o_empty(h), 4);  // one per output warp
            }
            mbar_init(item_full, 1);
            mbar_init(item_empty, 14);  // every warp that works on items
            mbar_init(claim_bar, 1);
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish();
    }
    if (warp == 13 && lane == 0) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int tile_tokens = 128 / group;

    // a wait of a whole warp: one verdict for all lanes
    auto wait = [&](uint32_t bar, uint32_t parity, unsigned code) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code)) != 0;
    };
    // a wait that spans an item or the search for the next one, which have no bound: their steps keep it alive
    auto wait_item = [&](uint32_t bar, uint32_t parity, unsigned code) {
        return __all_sync(0xffffffffu, mbar_wait_progress(bar, parity, abort_flag, status, code, progress)) != 0;
    };
    // the next item, for the warps that work on items; false at the end
    uint32_t item_phase = 0;
    AttnItem it;
    auto next_item = [&](bool release) {
        if (!wait_item(item_full, item_phase, DEV_TIMEOUT_FULL)) return false;
        const int4* src = reinterpret_cast<const int4*>(smem + L::kItemOffset);
        const int4 a = src[0], b = src[1];
        it.s.q0 = __shfl_sync(0xffffffffu, a.x, 0), it.s.q_len = __shfl_sync(0xffffffffu, a.y, 0);
        it.s.k0 = __shfl_sync(0xffffffffu, a.z, 0), it.s.k_len = __shfl_sync(0xffffffffu, a.w, 0);
        it.kv = __shfl_sync(0xffffffffu, b.x, 0), it.t0 = __shfl_sync(0xffffffffu, b.y, 0);
        it.n[0] = __shfl_sync(0xffffffffu, b.z, 0), it.n[1] = __shfl_sync(0xffffffffu, b.w, 0);
        __syncwarp();
        if (release && lane == 0) mbar_arrive(item_empty);
        item_phase ^= 1u;
        return it.t0 >= 0;
    };

    if (warp >= 12) {
      fewer_registers<kAttnOtherRegs>();
      if (warp == 14) {
        // ---------------- items ----------------
        AttnWindow window = {p, tile_tokens, lane, progress};
        window.load(0);
        AttnSeek seek;
        uint32_t claim_phase = 0;
        auto publish = [&](int t0) {
            if (lane == 0) {
                int4* dst = reinterpret_cast<int4*>(smem + L::kItemOffset);
                dst[0] = make_int4(it.s.q0, it.s.q_len, it.s.k0, it.s.k_len);
                dst[1] = make_int4(it.kv, t0, it.n[0], it.n[1]);
                mbar_arrive(item_full);
            }
            __syncwarp();
        };
        auto find = [&](int index) {
            if (!seek.find(index, p.n_seqs, window)) return false;
            window.item(index - seek.before, it);
            return true;
        };
        // the next one is claimed when the loads of this one are on their way and everyone has read it: earlier, and a CTA
        // that is at a long item would hold another that nobody else can take
        auto hand = [&]() {
            publish(it.t0);
            const bool read = wait_item(item_empty, item_phase, DEV_TIMEOUT_EMPTY);
            item_phase ^= 1u;
            return read;
        };
        auto take = [&](int& index) {
            if (lane == 0) {
                atomicAdd(progress, 1u);
                fence_proxy_async_smem();  // the last result has been read
                mbar_arrive_expect_tx(claim_bar, 16);
                claim_request(base + L::kClaimOffset, claim_bar);
            }
            __syncwarp();
            if (!wait(claim_bar, claim_phase, DEV_TIMEOUT_FULL)) return false;
            claim_phase ^= 1u;
            index = claim_result(base + L::kClaimOffset);
            __syncwarp();
            return true;
        };
        it.s.q0 = it.s.q_len = it.s.k0 = it.s.k_len = it.kv = it.n[0] = it.n[1] = 0;
        if (attn_items(blockIdx.x, find, hand, take)) publish(-1);  // the end
      } else if (warp == 13) {
        // ---------------- TMA producer ----------------
        int stage = 0;
        uint32_t phase = 0, q_phase0 = 0, q_phase1 = 0;
        bool ok = true;
        const uint32_t q_bytes = static_cast<uint32_t>((D / 64) * tile_tokens * group * 128);
        while (ok && next_item(false)) {
            if (lane == 0) {
                const int n = max(it.n[0], it.n[1]);
                auto load_q = [&](int h, uint32_t& q_phase) {
                    if (!mbar_wait(q_empty(h), q_phase ^ 1u, abort_flag, status, DEV_TIMEOUT_EMPTY)) return false;
                    q_phase ^= 1u;
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
                    atomicAdd(progress, 1u);
                    if (++stage == ST) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    return true;
                };
                if (it.n[0] > 0) ok = load_q(0, q_phase0);
                for (int j = 0; ok && j < n; ++j) {
                    ok = load_kv(&tmap_k, j);
                    if (ok && j == 0 && it.n[1] > 0) ok = load_q(1, q_phase1);
                    ok = ok && load_kv(&tmap_v, j);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
            if (lane == 0) mbar_arrive(item_empty);
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
            ok = ok && mbar_wait(q_empty(0), q_phase0 ^ 1u, abort_flag, status, DEV_TIMEOUT_EMPTY);
            ok = ok && mbar_wait(q_empty(1), q_phase1 ^ 1u, abort_flag, status, DEV_TIMEOUT_EMPTY);
        }
      } else if (warp == 12) {
        // ---------------- MMA issuer ----------------
        // Tile 0 and tile 1 strictly in turn: their softmaxes then run half a period apart, one on the special-function
        // units while the other waits for its products (two independent issuers let them fall into step, where the powers
        // of both take 2048 cycles at a time: 275 instead of 235 us for the long prompt).
        const uint32_t fmt = TYPE == kBF16 ? (1u << 7) | (1u << 10) : 0u;  // A and B format: 0 = fp16, 1 = bf16
        const uint32_t idesc_s = umma_idesc_f16_f32(128, kAttnKeys) | fmt;
        const uint32_t idesc_o = umma_idesc_f16_f32(128, D) | fmt | (1u << 16);  // B = V is MN-major
        const bool leader = elect_lane();
        int stage = 0;  // ring position: K_0 V_0 K_1 V_1 ... of one item after another
        uint32_t phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
        bool ok = true;
        auto advance = [&](int& st, uint32_t& ph) {
            if (++st == ST) {
                st = 0;
                ph ^= 1u;
            }
        };
        // S = Q K^T of tile h with the keys at ring position st; P lies over S and has been read when S overwrites it: MMAs
        // of one thread run in order
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
        while (ok && next_item(true)) {
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
                const uint64_t v_desc = umma_smem_desc_sw128_mn(v, L::kBoxBytes);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!ok || j >= it.n[h]) continue;
                    // weights behind the tile's last visible key are zeros: those k-steps are left out
                    int keys = left;
                    if (p.causal) {
                        const int last = min(it.t0 + (h + 1) * tile_tokens, it.s.q_len);
                        keys = min(keys, last + it.s.k_len - it.s.q_len - j * kAttnKeys);
                    }
                    const int steps = (keys + 15) / 16;
                    const uint32_t o_tmem = tmem + kO + h * 128, p_tmem = tmem + h * 128;
                    ok = wait(p_half(h), p_phase[h], DEV_TIMEOUT_TMEM_EMPTY);
                    if (!ok) continue;
                    tc_fence_after_sync();
                    if (leader) {
                        if (steps >= kAttnKeys / 32) {
                            umma_values_x4(o_tmem, p_tmem, v_desc, idesc_o, j != 0);
                        } else {
                            for (int x = 0; x < steps; ++x)
                                umma_values(o_tmem, p_tmem + 8 * x, v_desc + 128 * x, idesc_o, j != 0 || x != 0);
                        }
                    }
                    ok = wait(p_full(h), p_phase[h], DEV_TIMEOUT_TMEM_EMPTY);
                    p_phase[h] ^= 1u;
                    if (!ok) continue;
                    tc_fence_after_sync();
                    if (leader) {
                        if (steps >= kAttnKeys / 16) {
                            umma_values_x4(o_tmem, p_tmem + 32, v_desc + 512, idesc_o, 1);
                        } else {
                            for (int x = kAttnKeys / 32; x < steps; ++x)
                                umma_values(o_tmem, p_tmem + 8 * x, v_desc + 128 * x, idesc_o, 1);
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
    } else if (warp >= 8) {
        // ---------------- output ----------------
        fewer_registers<kAttnOutRegs>();
        const int w32 = (warp & 3) * 32, r = w32 + lane;  // this thread's row of a tile
        uint8_t* stage = smem + L::kOutOffset + (warp & 3) * L::kOutWarpBytes;
        const uint32_t by_group = (65536u + group - 1) / group;  // r / group = r * by_group >> 16 for r < 128
        uint32_t o_phase[2] = {0, 0}, stat_phase[2] = {0, 0};
        bool ok = true;
        while (ok && next_item(true)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int first = it.t0 + h * tile_tokens;
                if (!ok || first >= it.s.q_len) continue;  // the tile has no rows
                const int n = it.n[h];
                ok = wait_item(stat_full(h), stat_phase[h], DEV_TIMEOUT_TMEM_FULL);
                stat_phase[h] ^= 1u;
                if (!ok) continue;
                if (n > 0) {
                    ok = wait(o_full(h), o_phase[h], DEV_TIMEOUT_TMEM_FULL);
                    o_phase[h] ^= 1u;
                    if (!ok) continue;
                    tc_fence_after_sync();
                }
                const float2 ml = *reinterpret_cast<const float2*>(smem + L::kStatOffset + (h * 128 + r) * 8);
                const float inv = ml.y == 0.0f ? 0.0f : kUnlift / ml.y;
                // through shared memory, so that the bytes of a row are written by neighbouring lanes: a row per lane and
                // store touches 32 lines with each instruction
                const uint32_t t_o = tmem + (static_cast<uint32_t>(w32) << 16) + kO + h * 128;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    if (n > 0) {
                        tmem_ld_32x32(t_o + c, o);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = ml.y == 0.0f ? 0u
                                                : pack2(__uint_as_float(o[8 * i + 2 * e]) * inv,
                                                        __uint_as_float(o[8 * i + 2 * e + 1]) * inv, TYPE);
                        *reinterpret_cast<uint4*>(stage + lane * (D * 2) + (((c / 8 + i) ^ (lane & 7)) << 4)) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                const int token = static_cast<int>(r * by_group >> 16);
                if (p.lse && token < tile_tokens && first + token < it.s.q_len)
                    p.lse[(it.s.q0 + static_cast<long long>(first + token)) * p.heads + it.kv * group + r - token * group] =
                        ml.y == 0.0f ? -INFINITY : (ml.x * p.scale_log2 + log2f(ml.y)) * kLn2;
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_empty(h));  // O and the statistics have been read
                // D / 8 lanes per row
                constexpr int kLanes = D / 8, kRows = 32 / kLanes;
                const int chunk = lane % kLanes;
                if (chunk * 8 < p.dim) {
                    uint16_t* out = static_cast<uint16_t*>(p.out) + (it.s.q0 + static_cast<long long>(first)) * p.ld_out +
                                    static_cast<long long>(it.kv) * group * p.dim + chunk * 8;
#pragma unroll 4
                    for (int i = 0; i < 32 / kRows; ++i) {
                        const int rr = i * kRows + lane / kLanes;
                        const int tr = static_cast<int>((w32 + rr) * by_group >> 16);
                        if (tr < tile_tokens && first + tr < it.s.q_len)
                            *reinterpret_cast<uint4*>(out + tr * p.ld_out + (w32 + rr - tr * group) * p.dim) =
                                *reinterpret_cast<const uint4*>(stage + rr * (D * 2) + ((chunk ^ (rr & 7)) << 4));
                    }
                }
                __syncwarp();
            }
        }
    } else {
        // ---------------- softmax ----------------
        more_registers<kAttnSoftmaxRegs>();
        const int h = warp >> 2, r = threadIdx.x & 127;
        const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_s = t_lane + h * 128, t_o = t_lane + kO + h * 128;
        const int token = r / group;
        uint32_t s_phase = 0, o_phase = 0;
        bool ok = true;
        while (ok && next_item(true)) {
            const int first = it.t0 + h * tile_tokens;
            if (first >= it.s.q_len) continue;  // this tile has no rows
            int limit = it.s.k_len, tile_limit = it.s.k_len;  // keys this row sees; keys every row of the tile sees
            if (p.causal) {
                limit = min(limit, max(0, first + token + 1 + it.s.k_len - it.s.q_len));
                tile_limit = min(tile_limit, max(0, first + 1 + it.s.k_len - it.s.q_len));
            }
            const bool stored = token < tile_tokens && first + token < it.s.q_len;
            const int n = h ? it.n[1] : it.n[0];
            float m = -INFINITY, l = 0.0f, off = 0.0f;
            bool far = false;
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
                    top = max2(max2(max_of(s0), max_of(s1)), max2(max_of(s2), max_of(s3)));
                } else {
                    top = max2(max_of(s0), max_of(s1));
                    tmem_ld_wait();
                    top = max3(top, max_of(s2), max_of(s3));
                }
                bool moved = true;  // the maximum of some row of the warp
                if (j == 0) {
                    m = top;
                } else {
                    // a row's own scores decide, so that its result does not depend on its neighbours'; true from -infinity
                    // and for NaN as well.  Rows that are not stored have no say: what lies there (of other sequences,
                    // behind them, or in shared memory where no box reaches) may hold NaN, and would have its warp rescale
                    // for every key tile (16384 keys, 65 tokens and NaN behind them: 233 us instead of 206).  Rows with scores
                    // so far from zero that they need what follows below come here for every tile, so that others do not
                    // pass by it
                    const bool raise = stored && (far || !((top - m) * p.scale_log2 <= 8.0f));
                    moved = __any_sync(0xffffffffu, raise);
                    if (moved) {
                        // the scores of this tile follow the product that last added to O: O is at rest
                        const float up = raise ? max2(m, top) : m;
                        const float keep = !raise ? 1.0f : m == -INFINITY ? 0.0f : ex2((m - up) * p.scale_log2);
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
                }
                if (moved) {
                    // a maximum of +infinity or NaN makes every weight of the row NaN, as the definition does
                    off = m == -INFINITY ? 0.0f : m == INFINITY ? NAN : fmaf(-m, p.scale_log2, kPromptLift<TYPE>);
                    // scale s + off rounds off to its last place: from scores of 2^16 on, where that is more than 2^-8, the
                    // maximum is taken from the scores first, which is exact near it
                    far = stored && fabsf(off) > 65536.0f;
                    if (__any_sync(0xffffffffu, far)) {
                        const float from = far ? m : 0.0f;
                        less(s0, from), less(s1, from), less(s2, from), less(s3, from);
                        if (far) off = kPromptLift<TYPE>;
                    }
                }
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                {
                    uint32_t w[32];
                    weights<TYPE>(s0, p.scale_log2, off, sum, w, 0);
                    weights<TYPE>(s1, p.scale_log2, off, sum, w, 16);
                    tmem_st_32x32(t_s, w);
                }
                if (j == 0) {  // the item before has left O
                    ok = wait(o_empty(h), o_phase ^ 1u, DEV_TIMEOUT_TMEM_EMPTY);
                    if (!ok) break;
                    tc_fence_after_sync();
                }
                tmem_st_wait();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half(h));  // the product with the first 64 values may start
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
            if (ok && n == 0) ok = wait(o_empty(h), o_phase ^ 1u, DEV_TIMEOUT_TMEM_EMPTY);
            if (!ok) break;
            o_phase ^= 1u;
            if (m == -INFINITY) l = 0.0f;  // every key of the row scored -infinity
            // the sum without the lift: the product takes the lift out of O
            *reinterpret_cast<float2*>(smem + L::kStatOffset + (h * 128 + r) * 8) = make_float2(m, l * kUnlift);
            __syncwarp();
            if (lane == 0) mbar_arrive(stat_full(h));
        }
    }

    __syncwarp();
    if (*abort_flag) __nanosleep(1000000u);  // let bulk copies still in flight land before shared memory is released
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

}  // namespace tk
