// C-ABI entry points of the decoder-block operators (the contracts are in include/tacker_b200.h).  Part of
// tacker_b200.cu: uses its launch helpers and device state.
#pragma once
#include "attention_prompt.cuh"
#include "attention_rows.cuh"
#include "attention_tokens.cuh"
#include "i8gemm.cuh"
#include "row_ops.cuh"

namespace tk {

static int type_bytes(int type) { return type == kF32 ? 4 : 2; }
static bool type_ok(int type) { return type == kF32 || type == kF16 || type == kBF16; }
static bool aligned16(std::initializer_list<const void*> ps) {
    uintptr_t u = 0;
    for (const void* p : ps) u |= reinterpret_cast<uintptr_t>(p);
    return (u & 15u) == 0;
}
static bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Buffers of another GPU than the current one are refused (machines with one GPU skip the look-up).  Memory that CUDA
// does not know is refused as well; managed memory belongs everywhere.
static int on_this_device(std::initializer_list<const void*> ps) {
    static const int devices = [] {
        int n = 1;
        return cudaGetDeviceCount(&n) == cudaSuccess ? n : 1;
    }();
    if (devices < 2) return TK_OK;
    int dev = 0;
    TK_CUDA(cudaGetDevice(&dev));
    for (const void* p : ps) {
        if (!p) continue;
        cudaPointerAttributes a;
        TK_CUDA(cudaPointerGetAttributes(&a, p));
        if (a.type == cudaMemoryTypeManaged || a.type == cudaMemoryTypeHost) continue;
        if (a.type != cudaMemoryTypeDevice || a.device != dev) {
            t_last_error = "a buffer does not belong to the current device";
            return TK_ERR_ARGS;
        }
    }
    return TK_OK;
}

// The opt-in to large shared memory, once per kernel and device (the call takes 1.5 us; devices beyond 64 pay it each time).
template <auto KERNEL>
static int enable_smem_once(int bytes) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    TK_CUDA(cudaGetDevice(&dev));
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
    if (done.load(std::memory_order_acquire) & bit) return TK_OK;
    TK_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
    return TK_OK;
}

static int pow2_at_least(long long n, int lo, int hi) {
    int p = lo;
    while (p < n && p < hi) p <<= 1;
    return p;
}

constexpr long long kMaxGridX = 0x7fffffffll;
constexpr int kMaxCols = 1 << 30;  // of a row: column numbers and their steps of a block's threads stay in 32 bits

// threads per row of the row kernels (sixteen columns each), threads and blocks of the launch
struct RowShape {
    int tpr, block;
    long long blocks;
};
static RowShape row_shape(long long rows, int cols) {
    RowShape s;
    s.tpr = pow2_at_least((cols + 15) / 16, 32, 1024);
    s.block = s.tpr < 128 ? 128 : s.tpr;
    const long long per = s.block / s.tpr;
    s.blocks = (rows + per - 1) / per;
    return s;
}

// a runtime element type as a template argument
template <typename F>
static int with_type(int type, F f) {
    if (type == kF32) return f(std::integral_constant<int, kF32>());
    if (type == kF16) return f(std::integral_constant<int, kF16>());
    return f(std::integral_constant<int, kBF16>());
}

// Tensor maps with 128-byte swizzle and zero fill.  Encoding one takes the driver about 1.5 us, as much as a launch, and a
// serving loop asks for the same shapes again and again: each host thread keeps the last eight shapes it encoded and only
// puts the buffer's address in.
typedef CUresult (*ReplaceAddressFn)(CUtensorMap*, void*);
struct TmapShape {
    cuuint64_t dims[3], strides[2];
    cuuint32_t box[3];
    int type, rank;
};
static int make_tmap_cached(CUtensorMap* m, const void* base, const TmapShape& shape) {
    static thread_local struct {
        TmapShape shape[8];
        CUtensorMap map[8];
        int n = 0, next = 0;
    } kept;
    static const ReplaceAddressFn replace = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapReplaceAddress", &fn, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<ReplaceAddressFn>(fn) : nullptr;
    }();
    for (int i = 0; replace && i < kept.n; ++i) {
        if (std::memcmp(&kept.shape[i], &shape, sizeof(shape)) != 0) continue;
        *m = kept.map[i];
        if (replace(m, const_cast<void*>(base)) == CUDA_SUCCESS) return TK_OK;
    }
    int rc = get_encoder();
    if (rc != TK_OK) return rc;
    const cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = g_encode(m, static_cast<CUtensorMapDataType>(shape.type), static_cast<cuuint32_t>(shape.rank),
                          const_cast<void*>(base), shape.dims, shape.strides, shape.box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        t_last_error = "cuTensorMapEncodeTiled failed with CUresult " + std::to_string(static_cast<int>(r));
        return TK_ERR_CUDA;
    }
    kept.shape[kept.next] = shape;
    kept.map[kept.next] = *m;
    kept.next = (kept.next + 1) % 8;
    kept.n = std::min(8, kept.n + 1);
    return TK_OK;
}

// 8-bit matrix [rows][k], k contiguous, leading dimension ld bytes; box = 128 bytes x box_rows
static int make_tmap_i8(CUtensorMap* m, const void* base, int rows, int k, long long ld, int box_rows) {
    TmapShape s = {};
    s.dims[0] = static_cast<cuuint64_t>(k), s.dims[1] = static_cast<cuuint64_t>(rows);
    s.strides[0] = static_cast<cuuint64_t>(ld);
    s.box[0] = kI8BK, s.box[1] = static_cast<cuuint32_t>(box_rows);
    s.type = CU_TENSOR_MAP_DATA_TYPE_UINT8, s.rank = 2;
    return make_tmap_cached(m, base, s);
}

// 16-bit tensor [rows][heads][dim] with rows `ld` elements apart; box = 64 elements x box_heads x box_rows; elements behind
// dim and rows behind the last arrive as zeros
static int make_tmap_heads(CUtensorMap* m, const void* base, int type, int rows, int heads, int dim, long long ld,
                           int box_heads, int box_rows) {
    TmapShape s = {};
    s.dims[0] = static_cast<cuuint64_t>(dim), s.dims[1] = static_cast<cuuint64_t>(heads), s.dims[2] = static_cast<cuuint64_t>(rows);
    s.strides[0] = static_cast<cuuint64_t>(dim) * 2, s.strides[1] = static_cast<cuuint64_t>(ld) * 2;
    s.box[0] = 64, s.box[1] = static_cast<cuuint32_t>(box_heads), s.box[2] = static_cast<cuuint32_t>(box_rows);
    s.type = type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, s.rank = 3;
    return make_tmap_cached(m, base, s);
}

template <int BN, int STAGES, bool SWAP>
static int launch_i8gemm(const void* A, long long lda, const void* B, long long ldb, const I8Args& p, int split,
                         cudaStream_t st) {
    constexpr auto kernel = i8gemm_kernel<BN, STAGES, SWAP>;
    constexpr int smem = I8Smem<BN, STAGES>::kBytes + 1024;
    int rc = enable_smem_once<kernel>(smem);
    if (rc != TK_OK) return rc;
    const int rows_a = SWAP ? p.N : p.M, rows_b = SWAP ? p.M : p.N;
    CUtensorMap ta, tb;
    if ((rc = make_tmap_i8(&ta, SWAP ? B : A, rows_a, p.K, SWAP ? ldb : lda, 128)) != TK_OK) return rc;
    if ((rc = make_tmap_i8(&tb, SWAP ? A : B, rows_b, p.K, SWAP ? lda : ldb, BN)) != TK_OK) return rc;
    const int tiles_b = (rows_b + BN - 1) / BN;
    const long long ctas = static_cast<long long>((rows_a + 127) / 128) * tiles_b * split;
    if (ctas > kMaxGridX) return TK_ERR_SHAPE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
    cfg.blockDim = dim3(192, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    TK_CUDA(cudaLaunchKernelEx(&cfg, kernel, ta, tb, p, split, tiles_b));
    return TK_OK;
}

static int launch_i8gemm_pair(const void* A, long long lda, const void* B, long long ldb, const I8Args& p, DeviceInfo* d,
                              cudaStream_t st) {
    constexpr auto kernel = i8gemm_pair_kernel;
    constexpr int smem = I8PairSmem::kBytes + 1024;
    static_assert(smem <= kMaxDynSmem, "shared memory of a CTA");
    int rc = enable_smem_once<kernel>(smem);
    if (rc != TK_OK) return rc;
    CUtensorMap ta, tb;
    if ((rc = make_tmap_i8(&ta, A, p.M, p.K, lda, 128)) != TK_OK) return rc;
    if ((rc = make_tmap_i8(&tb, B, p.N, p.K, ldb, 128)) != TK_OK) return rc;
    const long long tiles = (p.M + 255ll) / 256 * ((p.N + 255ll) / 256);
    if (tiles > kMaxGridX) return TK_ERR_SHAPE;
    const long long pairs = std::min(tiles, static_cast<long long>(d->sm_count / 2));
    kernel<<<static_cast<unsigned>(2 * pairs), kI8PairThreads, smem, st>>>(ta, tb, p);
    return launch_error("i8gemm_pair_kernel launch");
}

// how many ranges of k, at most 8 (a cluster): while the launch has no more CTAs than `slots` and a range no fewer than
// `least` stages
static int i8_split(long long tiles, int kblocks, int slots, int least) {
    int s = 1;
    while (s < 8 && tiles * s * 2 <= slots && kblocks / (2 * s) >= least) s *= 2;
    return s;
}

constexpr int kTokenRows = 64;  // most rows (tokens x heads of a group) of a sequence for the token form
// query rows of a call: row numbers of the last block of rows, and of the block behind it that the token form's loop looks at,
// stay in 32 bits
constexpr long long kMaxTokenHeads = 0x7fffffffll - kTokenRows;

template <int D, int TYPE>
static int launch_attention_prompt(const AttnArgs& p, DeviceInfo* d, cudaStream_t st) {
    constexpr auto kernel = attention_prompt_kernel<D, TYPE>;
    constexpr int smem = AttnSmem<D>::kBytes;
    static_assert(smem <= kMaxDynSmem, "shared memory of a CTA");
    int rc = enable_smem_once<kernel>(smem);
    if (rc != TK_OK) return rc;
    const int group = p.heads / p.kv_heads, tile_tokens = 128 / group;
    CUtensorMap tq, tk_, tv;
    if ((rc = make_tmap_heads(&tq, p.q, p.type, p.total_q, p.heads, p.dim, p.ld_q, group, tile_tokens)) != TK_OK) return rc;
    if ((rc = make_tmap_heads(&tk_, p.k, p.type, p.kv_rows, p.kv_heads, p.dim, p.ld_k, 1, kAttnKeys)) != TK_OK) return rc;
    if ((rc = make_tmap_heads(&tv, p.v, p.type, p.kv_rows, p.kv_heads, p.dim, p.ld_v, 1, kAttnKeys)) != TK_OK) return rc;
    // no more items than this, whatever the lengths are
    const long long items = (p.total_q / (2ll * tile_tokens) + p.n_seqs) * p.kv_heads;
    if (items > kMaxGridX) return TK_ERR_SHAPE;
    kernel<<<static_cast<unsigned>(items), kAttnThreads, smem, st>>>(tq, tk_, tv, p, group, d->status_ptr);
    return launch_error("attention_prompt_kernel launch");
}

// ranges of the key axis for the token form: a full device of CTAs (two per SM), or several rounds of them where the
// lengths may differ; no range shorter than 256 keys; what the workspace holds
static int token_splits(long long base, int max_k, int slots, size_t row_bytes, size_t workspace_bytes) {
    long long s = base >= slots ? (4ll * slots + base - 1) / base : slots / base;
    s = std::min(s, (static_cast<long long>(max_k) + 255) / 256);
    s = std::min(s, static_cast<long long>(workspace_bytes / row_bytes));
    return static_cast<int>(std::max(1ll, std::min(s, 1024ll)));
}

template <int D, int TYPE>
static int launch_attention_tokens(const AttnArgs& p, DeviceInfo* d, int max_q, int max_k, void* workspace,
                                   size_t workspace_bytes, cudaStream_t st) {
    constexpr auto kernel = attention_tokens_kernel<D, TYPE>;
    constexpr int smem = TokSmem<D>::kBytes + 1024;
    static_assert(2 * (smem + 1024) <= kMaxDynSmem + 1024, "two CTAs per SM");
    int rc = enable_smem_once<kernel>(smem);
    if (rc != TK_OK) return rc;
    CUtensorMap tk_, tv;
    if ((rc = make_tmap_heads(&tk_, p.k, p.type, p.kv_rows, p.kv_heads, p.dim, p.ld_k, 1, kTokKeys)) != TK_OK) return rc;
    if ((rc = make_tmap_heads(&tv, p.v, p.type, p.kv_rows, p.kv_heads, p.dim, p.ld_v, 1, kTokKeys)) != TK_OK) return rc;
    TokArgs a;
    a.group = p.heads / p.kv_heads;
    a.row_blocks = std::max(1, (std::min(max_q, p.total_q) * a.group + kTokRows - 1) / kTokRows);
    const long long base = static_cast<long long>(p.n_seqs) * p.kv_heads * a.row_blocks;
    const long long rows = static_cast<long long>(p.total_q) * p.heads;
    const size_t row_bytes = static_cast<size_t>(rows) * (p.dim * sizeof(float) + sizeof(float2));
    a.splits = token_splits(base, max_k, 2 * d->sm_count, row_bytes, workspace ? workspace_bytes : 0);
    a.part_ml = static_cast<float2*>(workspace);
    // the sums first: their size is a multiple of 8 bytes, rounded up to 16 for the vectors behind
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + (static_cast<size_t>(rows) * a.splits * 8 + 15) / 16 * 16);
    while (a.splits > 1 && static_cast<size_t>(reinterpret_cast<char*>(a.part_o) - static_cast<char*>(workspace)) +
                                   static_cast<size_t>(rows) * a.splits * p.dim * 4 > workspace_bytes) {
        --a.splits;
        a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + (static_cast<size_t>(rows) * a.splits * 8 + 15) / 16 * 16);
    }
    if (base * a.splits > kMaxGridX) return TK_ERR_SHAPE;
    kernel<<<static_cast<unsigned>(base * a.splits), kTokWarps * 32, smem, st>>>(tk_, tv, p, a, d->status_ptr);
    if (a.splits == 1) return launch_error("attention_tokens_kernel launch");
    if ((rc = launch_error("attention_tokens_kernel launch")) != TK_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows), 1, 1);
    cfg.blockDim = dim3(32 * std::min(8, (a.splits + 3) / 4), 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TK_CUDA(cudaLaunchKernelEx(&cfg, attention_join_kernel<TYPE>, p, a));
    return TK_OK;
}

}  // namespace tk

TK_API int tk_norm_residual_rows(const void* a, int a_type, long long ld_a, int post, const float* post_gamma,
                                 const float* post_beta, const float* gate, long long ld_gate, long long gate_rows,
                                 float scale, const void* x, long long ld_x, void* y, long long ld_y, int x_type,
                                 const float* pre_gamma, const float* pre_beta, void* h, long long ld_h, int h_type,
                                 int layer, float eps, long long rows, int cols, void* stream) {
    if (rows < 0 || cols <= 0 || !type_ok(a_type) || !type_ok(x_type) || !type_ok(h_type) || !(eps >= 0.0f)) return TK_ERR_ARGS;
    if (post < 0 || post > 1 || layer < 0 || layer > 1) return TK_ERR_ARGS;
    if (rows == 0) return TK_OK;
    if (!a || (!y && !h) || ld_a < cols || (x && ld_x < cols) || (y && ld_y < cols) || (h && ld_h < cols)) return TK_ERR_ARGS;
    if (gate && (ld_gate < cols || gate_rows < 1)) return TK_ERR_ARGS;
    if (rows > kMaxGridX || cols > kMaxCols) return TK_ERR_SHAPE;
    if (!aligned_to(a, type_bytes(a_type)) || !aligned_to(x, type_bytes(x_type)) || !aligned_to(y, type_bytes(x_type)) ||
        !aligned_to(h, type_bytes(h_type)))
        return TK_ERR_ALIGN;
    for (const float* f : {post_gamma, post_beta, gate, pre_gamma, pre_beta})
        if (!aligned_to(f, 4)) return TK_ERR_ALIGN;
    // in place: each element is read and written by one thread, so the elements have to lie the same way
    struct Rows {
        const void* at;
        long long ld;
        int bytes;
    };
    const Rows in[2] = {{a, ld_a, type_bytes(a_type)}, {x, ld_x, type_bytes(x_type)}};
    for (const Rows& o : {Rows{y, ld_y, type_bytes(x_type)}, Rows{h, ld_h, type_bytes(h_type)}})
        for (const Rows& i : in)
            if (o.at && o.at == i.at && (o.bytes != i.bytes || (rows > 1 && o.ld != i.ld))) return TK_ERR_ARGS;
    if (y && y == h) return TK_ERR_ARGS;
    int rc = on_this_device({a, x, y, h, gate, post_gamma, post_beta, pre_gamma, pre_beta});
    if (rc != TK_OK) return rc;
    NormArgs p;
    p.a = a, p.x = x, p.y = y, p.h = h;
    p.post_gamma = post_gamma, p.post_beta = post_beta, p.pre_gamma = pre_gamma, p.pre_beta = pre_beta;
    p.gate = gate;
    p.ld_a = ld_a, p.ld_x = ld_x, p.ld_y = ld_y, p.ld_h = ld_h, p.ld_gate = ld_gate;
    p.gate_rows = gate ? static_cast<uint32_t>(std::min(gate_rows, rows)) : 1u;
    p.rows = rows;
    p.a_type = a_type, p.x_type = x_type, p.h_type = h_type, p.cols = cols, p.post = post, p.layer = layer;
    p.scale = scale, p.eps = eps;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool vec = cols % 8 == 0 && cols <= kNormCols && ld_a % 8 == 0 && (!x || ld_x % 8 == 0) &&
                     (!y || ld_y % 8 == 0) && (!h || ld_h % 8 == 0) && (!gate || ld_gate % 4 == 0) &&
                     aligned16({a, x, y, h, gate, post_gamma, post_beta, pre_gamma, pre_beta});
    if (!vec) {
        norm_residual_any_kernel<<<static_cast<unsigned>(rows), 256, 0, st>>>(p);
        return launch_error("norm_residual_any_kernel launch");
    }
    DeviceInfo* d = nullptr;
    if ((rc = device_info(&d)) != TK_OK) return rc;
    const RowShape s = row_shape(rows, cols);
    // 64 registers a thread: 1024 threads per SM
    const unsigned grid = static_cast<unsigned>(std::min(s.blocks, static_cast<long long>(d->sm_count) * (1024 / s.block)));
    return with_type(a_type, [&](auto at) {
        return with_type(x_type, [&](auto xt) {
            return with_type(h_type, [&](auto ht) {
                norm_residual_kernel<at.value, xt.value, ht.value><<<grid, s.block, 0, st>>>(p, s.tpr);
                return launch_error("norm_residual_kernel launch");
            });
        });
    });
}

TK_API int tk_quantize_rows_i8(const void* x, int x_type, long long ld_x, void* codes, long long ld_codes, float* scales,
                               long long rows, int cols, void* stream) {
    if (rows < 0 || cols <= 0 || !type_ok(x_type)) return TK_ERR_ARGS;
    if (rows == 0) return TK_OK;
    if (!x || !codes || !scales || ld_x < cols || ld_codes < cols) return TK_ERR_ARGS;
    if (rows > kMaxGridX || cols > kMaxCols) return TK_ERR_SHAPE;
    if (!aligned_to(x, type_bytes(x_type)) || !aligned_to(scales, 4)) return TK_ERR_ALIGN;
    int rc = on_this_device({x, codes, scales});
    if (rc != TK_OK) return rc;
    QuantArgs p;
    p.x = x, p.codes = static_cast<int8_t*>(codes), p.scales = scales;
    p.ld_x = ld_x, p.ld_codes = ld_codes, p.rows = rows, p.type = x_type, p.cols = cols;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cols % 8 || cols > kQuantCols || ld_x % 8 || ld_codes % 8 || !aligned16({x}) || !aligned_to(codes, 8)) {
        quantize_rows_any_kernel<<<static_cast<unsigned>(rows), 256, 0, st>>>(p);
        return launch_error("quantize_rows_any_kernel launch");
    }
    const RowShape s = row_shape(rows, cols);
    const unsigned grid = static_cast<unsigned>(s.blocks);
    return with_type(x_type, [&](auto xt) {
        if (cols <= kNormCols) quantize_rows_kernel<2, xt.value><<<grid, s.block, 0, st>>>(p, s.tpr);
        else quantize_rows_kernel<4, xt.value><<<grid, s.block, 0, st>>>(p, s.tpr);
        return launch_error("quantize_rows_kernel launch");
    });
}

TK_API int tk_i8gemm(const void* A, long long lda, const float* scale_a, const void* B, long long ldb,
                     const float* scale_b, const float* bias, void* out, long long ld_out, int out_type, int M, int N,
                     int K, void* stream) {
    if (M < 0 || N < 0 || K <= 0 || !type_ok(out_type)) return TK_ERR_ARGS;
    if (M == 0 || N == 0) return TK_OK;
    if (!A || !B || !scale_a || !scale_b || !out || lda < K || ldb < K || ld_out < N) return TK_ERR_ARGS;
    if (K > 131071 || M > (1 << 30) || N > (1 << 30)) return TK_ERR_SHAPE;  // 131071 * 2^14 is the largest sum that fits 32 bits
    if (lda % 16 || ldb % 16 || !aligned16({A, B}) || !aligned_to(scale_a, 4) || !aligned_to(scale_b, 4) ||
        !aligned_to(bias, 4) || !aligned_to(out, type_bytes(out_type)))
        return TK_ERR_ALIGN;
    int rc = on_this_device({A, B, scale_a, scale_b, bias, out});
    if (rc != TK_OK) return rc;
    DeviceInfo* d = nullptr;
    if ((rc = device_info(&d)) != TK_OK) return rc;
    I8Args p;
    p.scale_a = scale_a, p.scale_b = scale_b, p.bias = bias, p.out = out, p.ld_out = ld_out;
    p.M = M, p.N = N, p.K = K, p.out_type = out_type;
    p.vec = aligned16({out}) && ld_out * type_bytes(out_type) % 16 == 0;
    p.status = d->status_ptr;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int kblocks = (K + kI8BK - 1) / kI8BK;
    const long long tn = (N + 127) / 128;
    // Few tokens: the weights' bytes are the time.  Two CTAs per SM, ranges of at least eight stages (16 x 8192 x 4096: 12.0 us
    // unsplit, 8.7 / 8.0 / 13.0 with 2 / 4 / 8 ranges; 1 x 4096 x 4096: 11.2, then 8.2 / 6.4 / 7.1).
    if (M <= 64) {
        const int split = i8_split(tn, kblocks, 2 * d->sm_count, 8);
        if (M <= 16) return launch_i8gemm<16, 5, true>(A, lda, B, ldb, p, split, st);
        if (M <= 32) return launch_i8gemm<32, 5, true>(A, lda, B, ldb, p, split, st);
        return launch_i8gemm<64, 4, true>(A, lda, B, ldb, p, split, st);
    }
    // Large products on CTA pairs: when their 256 x 256 tiles give half of the pairs of SMs something to do (64 tiles: 512 x 8192
    // x 4096 16.4 us, 19.0 in smaller tiles; 32 tiles: 300 x 4096 x 4096 15.4 us against 14.6)
    if ((M + 255ll) / 256 * ((N + 255ll) / 256) >= d->sm_count / 4) return launch_i8gemm_pair(A, lda, B, ldb, p, d, st);
    // In between 128 x 128 tiles, fewer than the device has SMs (256 x 256 tiles that reach here are less than a quarter of
    // that, each four of these), in a deep ring.  Joining ranges of k pays while the device is not full (257 x 512 x 1024:
    // 7.7 us, with eight ranges 6.8) and costs more than it gains once it is (300 x 4096 x 4096: 14.4 us, 15.1 with two).
    const long long tiles = (M + 127ll) / 128 * tn;
    return launch_i8gemm<128, 6, false>(A, lda, B, ldb, p, i8_split(tiles, kblocks, d->sm_count, 1), st);
}

// pair i of a rotary head turns by pos * turns[i] full turns
TK_API int tk_rope_turns(int rot_dim, double base, int scaling, double factor, double trained_len, double fast,
                         double slow, double* turns, float* magnitude) {
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > kRopeMaxDim || !(base > 0.0) || !(factor >= 1.0) || !turns || !magnitude)
        return TK_ERR_ARGS;
    if (scaling < TK_ROPE_PLAIN || scaling > TK_ROPE_RAMP) return TK_ERR_ARGS;
    if (scaling == TK_ROPE_RAMP && !(base > 1.0 && trained_len > 0.0 && fast > slow && slow > 0.0)) return TK_ERR_ARGS;
    if (scaling == TK_ROPE_BASE && rot_dim < 4) return TK_ERR_SHAPE;
    const double two_pi = 6.283185307179586476925;
    if (scaling == TK_ROPE_BASE) base *= std::pow(factor, static_cast<double>(rot_dim) / (rot_dim - 2));
    double lo = 0.0, hi = 0.0;
    if (scaling == TK_ROPE_RAMP) {
        // the pair that turns `over` times in the trained length; lo and hi: where the mixture begins and ends
        auto pair_of = [&](double over) {
            return rot_dim * std::log(trained_len / (over * two_pi)) / (2.0 * std::log(base));
        };
        lo = std::fmax(std::floor(pair_of(fast)), 0.0);
        hi = std::fmin(std::ceil(pair_of(slow)), rot_dim - 1.0);
    }
    *magnitude = 1.0f;
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim) / two_pi;
        if (scaling == TK_ROPE_LINEAR) f /= factor;
        if (scaling == TK_ROPE_RAMP) {
            const double share = hi > lo ? std::fmin(std::fmax((i - lo) / (hi - lo), 0.0), 1.0) : (i > lo ? 1.0 : 0.0);
            f = f * (1.0 - share) + f / factor * share;
        }
        turns[i] = f;
    }
    if (scaling == TK_ROPE_RAMP && factor > 1.0) *magnitude = static_cast<float>(0.1 * std::log(factor) + 1.0);
    return TK_OK;
}

TK_API int tk_rope_qkv(const void* x, int x_type, long long ld_x, const float* bias, const int* positions,
                       const double* turns, int rot_dim, int interleaved, float magnitude, long long tokens, int heads,
                       int kv_heads, int dim, void* q, long long ld_q, void* k, long long ld_k, void* v, long long ld_v,
                       int out_type, const long long* slots, long long n_slots, void* stream) {
    if (tokens < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || !type_ok(x_type) || !type_ok(out_type)) return TK_ERR_ARGS;
    if (rot_dim < 0 || rot_dim % 2 || rot_dim > dim || interleaved < 0 || interleaved > 1 || (slots && n_slots < 0))
        return TK_ERR_ARGS;
    if (tokens == 0) return TK_OK;
    const long long width = (static_cast<long long>(heads) + 2ll * kv_heads) * dim;
    if (dim > kRopeMaxDim || width > (1ll << 30) || tokens > kMaxGridX) return TK_ERR_SHAPE;
    if (!x || !q || !k || !v || (rot_dim && (!positions || !turns))) return TK_ERR_ARGS;
    if (ld_x < width || ld_q < static_cast<long long>(heads) * dim || ld_k < static_cast<long long>(kv_heads) * dim ||
        ld_v < static_cast<long long>(kv_heads) * dim)
        return TK_ERR_ARGS;
    const int eb = type_bytes(out_type);
    if (!aligned_to(x, type_bytes(x_type)) || !aligned_to(bias, 4) || !aligned_to(positions, 4) || !aligned_to(turns, 8) ||
        !aligned_to(q, eb) || !aligned_to(k, eb) || !aligned_to(v, eb) || !aligned_to(slots, 8))
        return TK_ERR_ALIGN;
    int rc = on_this_device({x, bias, positions, turns, q, k, v, slots});
    if (rc != TK_OK) return rc;
    RopeArgs p;
    p.x = x, p.bias = bias, p.pos = positions, p.turns = turns, p.slots = slots, p.q = q, p.k = k, p.v = v;
    p.ld_x = ld_x, p.ld_q = ld_q, p.ld_k = ld_k, p.ld_v = ld_v, p.n_slots = n_slots;
    p.x_type = x_type, p.out_type = out_type, p.heads = heads, p.kv_heads = kv_heads, p.dim = dim, p.rot = rot_dim;
    p.interleaved = interleaved, p.magnitude = magnitude;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool vec = dim % 16 == 0 && rot_dim % 16 == 0 && ld_x % 8 == 0 && ld_q % 8 == 0 && ld_k % 8 == 0 &&
                     ld_v % 8 == 0 && aligned16({x, bias, q, k, v});
    if (!vec) {
        rope_qkv_any_kernel<<<static_cast<unsigned>(tokens), 128, 0, st>>>(p);
        return launch_error("rope_qkv_any_kernel launch");
    }
    return with_type(x_type, [&](auto xt) {
        return with_type(out_type, [&](auto ot) {
            rope_qkv_vec_kernel<xt.value, ot.value><<<static_cast<unsigned>(tokens), 128, 0, st>>>(p);
            return launch_error("rope_qkv_vec_kernel launch");
        });
    });
}

TK_API int tk_attention_packed(const void* q, long long ld_q, const void* k, long long ld_k, const void* v, long long ld_v,
                               void* out, long long ld_out, float* lse, int type, const int* q_start, const int* k_start,
                               const int* k_len, int n_seqs, int total_q, int kv_rows, int max_q, int max_k, int heads,
                               int kv_heads, int dim, float scale, int causal, void* workspace, size_t workspace_bytes,
                               void* stream) {
    if (n_seqs < 0 || total_q < 0 || kv_rows < 0 || max_q < 0 || max_k < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 ||
        causal < 0 || causal > 1 || (type != kF16 && type != kBF16))
        return TK_ERR_ARGS;
    if (heads % kv_heads) return TK_ERR_ARGS;
    if (n_seqs == 0 || total_q == 0) return TK_OK;
    if (dim > 256 || static_cast<long long>(total_q) * heads > kMaxTokenHeads || total_q > (1 << 30) || kv_rows > (1 << 30))
        return TK_ERR_SHAPE;
    if (!q || !out || !q_start || !k_start || !k_len || (kv_rows > 0 && (!k || !v))) return TK_ERR_ARGS;
    if (ld_q < static_cast<long long>(heads) * dim || ld_out < static_cast<long long>(heads) * dim ||
        ld_k < static_cast<long long>(kv_heads) * dim || ld_v < static_cast<long long>(kv_heads) * dim)
        return TK_ERR_ARGS;
    if (!aligned_to(q, 2) || !aligned_to(k, 2) || !aligned_to(v, 2) || !aligned_to(out, 2) || !aligned_to(lse, 4) ||
        !aligned_to(q_start, 4) || !aligned_to(k_start, 4) || !aligned_to(k_len, 4) || !aligned16({workspace}))
        return TK_ERR_ALIGN;
    int rc = on_this_device({q, k, v, out, lse, q_start, k_start, k_len, workspace});
    if (rc != TK_OK) return rc;
    AttnArgs p;
    p.q = q, p.k = k, p.v = v, p.out = out, p.lse = lse, p.q_start = q_start, p.k_start = k_start, p.k_len = k_len;
    p.ld_q = ld_q, p.ld_k = ld_k, p.ld_v = ld_v, p.ld_out = ld_out;
    p.n_seqs = n_seqs, p.total_q = total_q, p.kv_rows = kv_rows, p.heads = heads, p.kv_heads = kv_heads, p.dim = dim;
    p.type = type, p.causal = causal, p.scale_log2 = scale * kLog2e;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int group = heads / kv_heads;
    // what the tensor maps take: 16-byte rows of whole heads, a group within one tile, at least one key row
    const bool tiles = dim % 8 == 0 && dim <= 128 && group <= 128 && kv_rows > 0 && ld_q % 8 == 0 && ld_k % 8 == 0 &&
                       ld_v % 8 == 0 && ld_out % 8 == 0 && aligned16({q, k, v, out}) && p.scale_log2 > 1e-30f &&
                       p.scale_log2 < 1e30f;
    if (tiles) {
        DeviceInfo* d = nullptr;
        if ((rc = device_info(&d)) != TK_OK) return rc;
        // few rows per sequence: the time is that of reading the keys and values
        if (static_cast<long long>(max_q) * group <= kTokenRows) {
            if (dim <= 64)
                return type == kF16 ? launch_attention_tokens<64, kF16>(p, d, max_q, max_k, workspace, workspace_bytes, st)
                                    : launch_attention_tokens<64, kBF16>(p, d, max_q, max_k, workspace, workspace_bytes, st);
            return type == kF16 ? launch_attention_tokens<128, kF16>(p, d, max_q, max_k, workspace, workspace_bytes, st)
                                : launch_attention_tokens<128, kBF16>(p, d, max_q, max_k, workspace, workspace_bytes, st);
        }
        if (dim <= 64)
            return type == kF16 ? launch_attention_prompt<64, kF16>(p, d, st) : launch_attention_prompt<64, kBF16>(p, d, st);
        return type == kF16 ? launch_attention_prompt<128, kF16>(p, d, st) : launch_attention_prompt<128, kBF16>(p, d, st);
    }
    const long long blocks = (static_cast<long long>(total_q) * heads + 3) / 4;
    if (blocks > kMaxGridX) return TK_ERR_SHAPE;
    if (dim <= 128)
        attention_rows_kernel<4><<<static_cast<unsigned>(blocks), 128, 0, st>>>(p);
    else
        attention_rows_kernel<8><<<static_cast<unsigned>(blocks), 128, 0, st>>>(p);
    return launch_error("attention_rows_kernel launch");
}
