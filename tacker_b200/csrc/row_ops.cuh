// Row kernels of a decoder block over packed tokens: element types chosen at run time, the residual stream between
// two blocks (norm behind a block, gate, residual scale, norm before the next), rows rounded to 8-bit integers, and
// the split of a fused projection into rotary query / key / value heads.
// All of them are bound by memory traffic: every operand is read once and every result written once, 16 bytes per
// access where the addresses allow it, with the row held in registers between the passes over it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tk {

// element types of the C ABI (tk_type)
constexpr int kF32 = 0, kF16 = 1, kBF16 = 2;

__device__ __forceinline__ float load1(const void* p, int type, long long i) {
    if (type == kF32) return static_cast<const float*>(p)[i];
    if (type == kF16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store1(void* p, int type, long long i, float v) {
    if (type == kF32)
        static_cast<float*>(p)[i] = v;
    else if (type == kF16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// eight consecutive elements as they lie in memory: 16 bytes of a 16-bit type, 32 bytes of fp32 (16-byte aligned)
struct Raw8 {
    uint4 lo, hi;
};
__device__ __forceinline__ Raw8 load_raw8(const void* p, int type, long long i) {
    Raw8 r;
    if (type == kF32) {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
        r.lo = s[0];
        r.hi = s[1];
    } else {
        r.lo = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
        r.hi = make_uint4(0u, 0u, 0u, 0u);
    }
    return r;
}
__device__ __forceinline__ void unpack2(uint32_t w, int type, float& a, float& b) {
    if (type == kF16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a = f.x, b = f.y;
    } else {  // bf16 is the upper half of an fp32
        a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack8(const Raw8& r, int type, float (&v)[8]) {
    if (type == kF32) {
        v[0] = __uint_as_float(r.lo.x), v[1] = __uint_as_float(r.lo.y), v[2] = __uint_as_float(r.lo.z);
        v[3] = __uint_as_float(r.lo.w), v[4] = __uint_as_float(r.hi.x), v[5] = __uint_as_float(r.hi.y);
        v[6] = __uint_as_float(r.hi.z), v[7] = __uint_as_float(r.hi.w);
    } else {
        unpack2(r.lo.x, type, v[0], v[1]);
        unpack2(r.lo.y, type, v[2], v[3]);
        unpack2(r.lo.z, type, v[4], v[5]);
        unpack2(r.lo.w, type, v[6], v[7]);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int type) {
    if (type == kF16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store8(void* p, int type, long long i, const float (&v)[8]) {
    if (type == kF32) {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        d[0] = make_float4(v[0], v[1], v[2], v[3]);
        d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(
            pack2(v[0], v[1], type), pack2(v[2], v[3], type), pack2(v[4], v[5], type), pack2(v[6], v[7], type));
    }
}
__device__ __forceinline__ void load8f(const float* p, int i, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p + i)), b = __ldg(reinterpret_cast<const float4*>(p + i) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
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
__device__ __forceinline__ void mul2(float& x, float& y, float sx, float sy) {
    asm("{\n"
        ".reg .b64 v, w;\n"
        "mov.b64 v, {%0, %1};\n"
        "mov.b64 w, {%2, %3};\n"
        "mul.rn.f32x2 v, v, w;\n"
        "mov.b64 {%0, %1}, v;\n"
        "}\n"
        : "+f"(x), "+f"(y)
        : "f"(sx), "f"(sy));
}

// Sum over the `tpr` threads of a row (a power of two, at least a warp).  `slots` is a shared array of 2 x 32 floats, used in
// turn so that one barrier per sum is enough; `turn` counts the sums.  Every thread of the block calls it, the same number
// of times.
__device__ __forceinline__ float row_sum(float v, int tpr, float* slots, int& turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5, first = warp & -per, lane = threadIdx.x & 31;  // powers of two
    float* slot = slots + 32 * (turn++ & 1);
    if (lane == 0) slot[warp] = v;
    __syncthreads();
    // at most 32 warps share a row: one more butterfly over their partial sums, the same order in every warp
    float s = lane < per ? slot[first + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// ---- the residual stream between two blocks ------------------------------------------------------------------------
//   y = x + scale * gate * post(a),   h = pre(y)
// post and pre are root-mean-square or layer norms over the row (or absent).  Statistics are fp32 sums of fp32 values;
// the layer norm takes the mean first and the squares of the differences after it.  h is made from y before y is
// rounded to its type: one rounding for each result.
struct NormArgs {
    const void* a;
    const void* x;      // may be null (no residual stream) and may be y
    void* y;            // may be null
    void* h;            // may be null (no norm behind)
    const float* post_gamma;
    const float* post_beta;
    const float* pre_gamma;
    const float* pre_beta;
    const float* gate;  // rows r of a share gate row r / gate_rows; null = 1
    long long ld_a, ld_x, ld_y, ld_h, ld_gate, rows;
    uint32_t gate_rows;  // 32 bits: a 64-bit division is a hundred instructions per thread and row
    int a_type, x_type, h_type, cols, post, layer;
    float scale, eps;
};

// One row per `tpr` threads, two groups of eight columns per thread in registers; the blocks stay and walk over the rows,
// with the next row's a and x on their way while this one is summed up.  The types are compile-time constants: chosen at
// run time, the conversions were most of 54 instructions per element (80 us at 8191 x 4096 bf16 with both norms and a gate;
// now 52 us = 5.1 TB/s, 41 us at the rate of a copy).  Groups of four columns, whose fp32 weights would come without gaps
// between the lanes, cost 8 us more: more accesses.
constexpr int kNormCols = 1024 * 2 * 8;  // widest row
template <int AT, int XT, int HT>
__global__ void __launch_bounds__(1024) norm_residual_kernel(const NormArgs p, const int tpr) {
    __shared__ float slots[64];
    const int t = threadIdx.x & (tpr - 1), c0 = t * 8, c1 = (t + tpr) * 8;
    const uint32_t rows = static_cast<uint32_t>(p.rows), per_block = blockDim.x >> (31 - __clz(tpr));
    const uint32_t step = gridDim.x * per_block;
    const bool in0 = c0 < p.cols, in1 = c1 < p.cols;
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    int turn = 0;
    Raw8 a0, a1, x0, x1;
    uint32_t row = blockIdx.x * per_block + (threadIdx.x >> (31 - __clz(tpr)));
    // this thread's first group of the row at hand in each array
    long long at_a = row * p.ld_a + c0, at_x = row * p.ld_x + c0, at_y = row * p.ld_y + c0, at_h = row * p.ld_h + c0;
    const int apart = tpr * 8;
    const bool has_x = p.x != nullptr;
    if (row < rows && in0) a0 = load_raw8(p.a, AT, at_a);
    if (row < rows && in1) a1 = load_raw8(p.a, AT, at_a + apart);
    if (has_x && row < rows && in0) x0 = load_raw8(p.x, XT, at_x);
    if (has_x && row < rows && in1) x1 = load_raw8(p.x, XT, at_x + apart);
    // all threads of a block make the same number of rounds, for the barriers in the sums
    for (uint32_t base = blockIdx.x * per_block; base < rows; base += step) {
        const bool live0 = row < rows && in0, live1 = row < rows && in1;
        const uint32_t next = row + step;
        float v[8], w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = w[j] = 0.0f;
        if (live0) unpack8(a0, AT, v);
        if (live1) unpack8(a1, AT, w);
        at_a += step * p.ld_a;
        if (next < rows && in0) a0 = load_raw8(p.a, AT, at_a);
        if (next < rows && in1) a1 = load_raw8(p.a, AT, at_a + apart);
        // (v, w) <- ((v, w) - mean) * rstd over the columns of the row; groups that do not exist stay zero
        auto normalise = [&]() {
            if (p.layer) {
                float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j += 2) add2(s0, s1, v[j], v[j + 1]), add2(s0, s1, w[j], w[j + 1]);
                const float mean = row_sum(s0 + s1, tpr, slots, turn) * inv_cols;
                const float m0 = in0 ? -mean : 0.0f, m1 = in1 ? -mean : 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j += 2) add2(v[j], v[j + 1], m0, m0), add2(w[j], w[j + 1], m1, m1);
            }
            float q0 = 0.0f, q1 = 0.0f, r0 = 0.0f, r1 = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float sx = v[j], sy = v[j + 1], ux = w[j], uy = w[j + 1];
                fma2(sx, sy, sx, sy, q0, q1);
                fma2(ux, uy, ux, uy, r0, r1);
                q0 = sx, q1 = sy, r0 = ux, r1 = uy;
            }
            const float rstd = rsqrtf(row_sum((q0 + q1) + (r0 + r1), tpr, slots, turn) * inv_cols + p.eps);
#pragma unroll
            for (int j = 0; j < 8; j += 2) mul2(v[j], v[j + 1], rstd, rstd), mul2(w[j], w[j + 1], rstd, rstd);
        };
        auto times = [&](const float* g) {
            float u[8];
            if (live0) {
                load8f(g, c0, u);
#pragma unroll
                for (int j = 0; j < 8; j += 2) mul2(v[j], v[j + 1], u[j], u[j + 1]);
            }
            if (live1) {
                load8f(g, c1, u);
#pragma unroll
                for (int j = 0; j < 8; j += 2) mul2(w[j], w[j + 1], u[j], u[j + 1]);
            }
        };
        auto plus = [&](const float* g) {
            float u[8];
            if (live0) {
                load8f(g, c0, u);
#pragma unroll
                for (int j = 0; j < 8; j += 2) add2(v[j], v[j + 1], u[j], u[j + 1]);
            }
            if (live1) {
                load8f(g, c1, u);
#pragma unroll
                for (int j = 0; j < 8; j += 2) add2(w[j], w[j + 1], u[j], u[j + 1]);
            }
        };
        if (p.post) {
            normalise();
            if (p.post_gamma) times(p.post_gamma);
            if (p.post_beta) plus(p.post_beta);
        }
        if (p.gate) times(p.gate + (row < rows ? row / p.gate_rows * p.ld_gate : 0));
        {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.0f;
            if (has_x && live0) unpack8(x0, XT, x);
#pragma unroll
            for (int j = 0; j < 8; j += 2) fma2(v[j], v[j + 1], p.scale, p.scale, x[j], x[j + 1]);
            if (has_x && live1) unpack8(x1, XT, x);
#pragma unroll
            for (int j = 0; j < 8; j += 2) fma2(w[j], w[j + 1], p.scale, p.scale, x[j], x[j + 1]);
            if (!in1) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = 0.0f;  // x of the first group went into one that does not exist
            }
        }
        if (p.y && live0) store8(p.y, XT, at_y, v);
        if (p.y && live1) store8(p.y, XT, at_y + apart, w);
        at_x += step * p.ld_x;
        if (has_x && next < rows && in0) x0 = load_raw8(p.x, XT, at_x);
        if (has_x && next < rows && in1) x1 = load_raw8(p.x, XT, at_x + apart);
        if (p.h) {
            normalise();
            if (p.pre_gamma) times(p.pre_gamma);
            if (p.pre_beta) plus(p.pre_beta);
            if (live0) store8(p.h, HT, at_h, v);
            if (live1) store8(p.h, HT, at_h + apart, w);
        }
        row = next;
        at_y += step * p.ld_y;
        at_h += step * p.ld_h;
    }
}

// Any width, stride and alignment: one block per row, each pass reads the row again (from L2 after the first).  y is
// written in the last pass only, so that it may be x.
__global__ void norm_residual_any_kernel(const NormArgs p) {
    __shared__ float slots[64];
    int turn = 0;
    const int tpr = blockDim.x;
    const long long row = blockIdx.x;
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    const float* gate = p.gate ? p.gate + static_cast<uint32_t>(row) / p.gate_rows * p.ld_gate : nullptr;
    auto stats = [&](auto value, float& mean, float& rstd) {
        mean = 0.0f;
        if (p.layer) {
            float s = 0.0f;
            for (int c = threadIdx.x; c < p.cols; c += tpr) s += value(c);
            mean = row_sum(s, tpr, slots, turn) * inv_cols;
        }
        float q = 0.0f;
        for (int c = threadIdx.x; c < p.cols; c += tpr) {
            const float d = value(c) - mean;
            q = fmaf(d, d, q);
        }
        rstd = rsqrtf(row_sum(q, tpr, slots, turn) * inv_cols + p.eps);
    };
    float m1 = 0.0f, r1 = 1.0f, m2 = 0.0f, r2 = 1.0f;
    if (p.post) stats([&](int c) { return load1(p.a, p.a_type, row * p.ld_a + c); }, m1, r1);
    auto stream = [&](int c) {
        float v = load1(p.a, p.a_type, row * p.ld_a + c);
        if (p.post) {
            v = (v - m1) * r1;
            if (p.post_gamma) v *= p.post_gamma[c];
            if (p.post_beta) v += p.post_beta[c];
        }
        if (gate) v *= gate[c];
        return fmaf(p.scale, v, p.x ? load1(p.x, p.x_type, row * p.ld_x + c) : 0.0f);
    };
    if (p.h) stats(stream, m2, r2);
    for (int c = threadIdx.x; c < p.cols; c += tpr) {
        const float y = stream(c);
        if (p.y) store1(p.y, p.x_type, row * p.ld_y + c, y);
        if (p.h) {
            float h = (y - m2) * r2;
            if (p.pre_gamma) h *= p.pre_gamma[c];
            if (p.pre_beta) h += p.pre_beta[c];
            store1(p.h, p.h_type, row * p.ld_h + c, h);
        }
    }
}

// ---- rows to 8-bit integers ----------------------------------------------------------------------------------------
//   scale_r = max_c |x_rc| / 127 (fp32),   code_rc = x_rc / scale_r rounded to the nearest integer, halves to even
// The rounding is that of the exact quotient: an fp32 quotient can be rounded onto a half that the exact one misses (the
// half of the largest value is such a place), so the candidate is put right by the remainder x - k s, which one fma
// gives without rounding: it is a multiple of the last place of s (or of x) below 2^24 such places.
// 8192 x 4096 bf16 take about 20 us (100 MB, 15 us at the rate of a copy); a few rows 2.5 us, a launch.
// Rows whose scale is no normal number (all zero, or below 127 * 2^-126) get scale 0 and codes 0; a row with a NaN or an
// infinity gets that as its scale and codes 0, so that products with it are NaN.
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
    const float amax = __uint_as_float(amax_bits);
    if (amax_bits >= 0x7f800000u) return amax;
    const float s = __fdiv_rn(amax, 127.0f);
    return s < 1.17549435e-38f ? 0.0f : s;
}
__device__ __forceinline__ int row_code(float x, float s, float inv) {
    float k = rintf(x * inv);
    const float r2 = 2.0f * fmaf(-k, s, x);
    const bool odd = (static_cast<int>(k) & 1) != 0;
    if (r2 > s || (r2 == s && odd)) k += 1.0f;
    if (r2 < -s || (r2 == -s && odd)) k -= 1.0f;
    return static_cast<int>(fminf(fmaxf(k, -127.0f), 127.0f));
}
// |x| as its bits: as unsigned numbers they are ordered like the values, with NaN above everything
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t row_umax(uint32_t v, int tpr, uint32_t* slot) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (tpr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tpr >> 5, first = warp & -per, lane = threadIdx.x & 31;
    if (lane == 0) slot[warp] = v;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < per ? slot[first + lane] : 0u);
}

constexpr int kQuantCols = 1024 * 4 * 8;  // widest row that is held in registers

struct QuantArgs {
    const void* x;
    int8_t* codes;
    float* scales;
    long long ld_x, ld_codes, rows;
    int type, cols;
};

template <int NV, int TYPE>
__global__ void quantize_rows_kernel(const QuantArgs p, const int tpr) {
    __shared__ uint32_t slot[32];
    const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
    const int t = threadIdx.x & (tpr - 1);
    const bool live = row < p.rows;
    float v[NV][8];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * tpr) * 8;
        if (live && c < p.cols) {
            unpack8(load_raw8(p.x, TYPE, row * p.ld_x + c), TYPE, v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i][j]));
        }
    }
    m = row_umax(m, tpr, slot);
    if (!live) return;
    const float s = row_scale(m);
    const bool usable = s > 0.0f && m < 0x7f800000u;
    const float inv = usable ? 1.0f / s : 0.0f;
    if (t == 0) p.scales[row] = s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * tpr) * 8;
        if (c >= p.cols) continue;
        uint32_t w[2] = {0u, 0u};
        if (usable) {
            // x / s to the nearest integer by adding 1.5 * 2^23, whose last bits then are the integer; the largest
            // remainder of the eight says whether any lies so near a border that the exact rule has to decide
            const float magic = 12582912.0f;
            float far = 0.0f;
            uint32_t bits[8];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float kx = v[i][j], ky = v[i][j + 1];
                fma2(kx, ky, inv, inv, magic, magic);
                bits[j] = __float_as_uint(kx), bits[j + 1] = __float_as_uint(ky);
                add2(kx, ky, -magic, -magic);
                fma2(kx, ky, -s, -s, v[i][j], v[i][j + 1]);
                far = fmaxf(far, fmaxf(fabsf(kx), fabsf(ky)));
            }
            if (2.0f * far >= s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) bits[j] = static_cast<uint32_t>(row_code(v[i][j], s, inv));
            }
#pragma unroll
            for (int j = 0; j < 8; j += 4)
                w[j >> 2] = __byte_perm(__byte_perm(bits[j], bits[j + 1], 0x0040), __byte_perm(bits[j + 2], bits[j + 3], 0x0040), 0x5410);
        }
        *reinterpret_cast<uint2*>(p.codes + row * p.ld_codes + c) = make_uint2(w[0], w[1]);
    }
}

__global__ void quantize_rows_any_kernel(const QuantArgs p) {
    __shared__ uint32_t slot[32];
    const long long row = blockIdx.x;
    uint32_t m = 0u;
    for (int c = threadIdx.x; c < p.cols; c += blockDim.x) m = max(m, abs_bits(load1(p.x, p.type, row * p.ld_x + c)));
    m = row_umax(m, blockDim.x, slot);
    const float s = row_scale(m);
    const bool usable = s > 0.0f && m < 0x7f800000u;
    const float inv = usable ? 1.0f / s : 0.0f;
    if (threadIdx.x == 0) p.scales[row] = s;
    for (int c = threadIdx.x; c < p.cols; c += blockDim.x)
        p.codes[row * p.ld_codes + c] =
            usable ? static_cast<int8_t>(row_code(load1(p.x, p.type, row * p.ld_x + c), s, inv)) : static_cast<int8_t>(0);
}

// ---- rotary head split ---------------------------------------------------------------------------------------------
// One token per block.  Row t of x holds heads query heads, kv_heads key heads and kv_heads value heads side by side;
// pair i of a query or key head is turned by 2 pi pos_t turns_i.  The product is taken in binary64 and reduced to a
// fraction of a turn there: an fp32 angle at position 10^6 is off by 0.06.  What is left in [-1/2, 1/2] loses nothing
// in fp32.  The angles of a token serve all its heads and are computed once, into shared memory.
struct RopeArgs {
    const void* x;
    const float* bias;          // [(heads + 2 kv_heads) dim] or null
    const int* pos;
    const double* turns;        // [rot / 2]
    const long long* slots;     // row of k and v for each token (negative or >= n_slots: none), or null = the token
    void* q;
    void* k;
    void* v;
    long long ld_x, ld_q, ld_k, ld_v, n_slots;
    int x_type, out_type, heads, kv_heads, dim, rot, interleaved;
    float magnitude;
};
constexpr int kRopeMaxDim = 512;
// shared-memory place of angle i: two more after every eight, so that threads which read eight each hit different banks
__device__ __forceinline__ int rope_at(int i) { return i + 2 * (i >> 3); }
constexpr int kRopeAngles = kRopeMaxDim / 2 + kRopeMaxDim / 8;

__device__ __forceinline__ void rope_angles(const RopeArgs& p, long long token, float2* cs) {
    for (int i = threadIdx.x; i < p.rot / 2; i += blockDim.x) {
        double a = static_cast<double>(p.pos[token]) * p.turns[i];
        a -= rint(a);
        float s, c;
        sincospif(2.0f * static_cast<float>(a), &s, &c);
        cs[rope_at(i)] = make_float2(c * p.magnitude, s * p.magnitude);
    }
}

// where head `head` of the row goes: q, or the slot's row of k or v; null = nowhere
__device__ __forceinline__ void* rope_dest(const RopeArgs& p, long long token, long long slot, int head, long long& at) {
    if (head < p.heads) {
        at = token * p.ld_q + static_cast<long long>(head) * p.dim;
        return p.q;
    }
    if (slot < 0) return nullptr;
    head -= p.heads;
    if (head < p.kv_heads) {
        at = slot * p.ld_k + static_cast<long long>(head) * p.dim;
        return p.k;
    }
    at = slot * p.ld_v + static_cast<long long>(head - p.kv_heads) * p.dim;
    return p.v;
}
__device__ __forceinline__ long long rope_slot(const RopeArgs& p, long long token) {
    if (!p.slots) return token;
    const long long s = p.slots[token];
    return s < p.n_slots ? s : -1;
}

__global__ void rope_qkv_any_kernel(const RopeArgs p) {
    __shared__ __align__(16) float2 cs[kRopeAngles];
    const long long token = blockIdx.x;
    rope_angles(p, token, cs);
    __syncthreads();
    const long long slot = rope_slot(p, token);
    const int total = (p.heads + 2 * p.kv_heads) * p.dim;
    auto value = [&](int e) { return load1(p.x, p.x_type, token * p.ld_x + e) + (p.bias ? p.bias[e] : 0.0f); };
    for (int e = threadIdx.x; e < total; e += blockDim.x) {
        const int head = e / p.dim, d = e - head * p.dim;
        long long at;
        void* dst = rope_dest(p, token, slot, head, at);
        if (!dst) continue;
        float o = value(e);
        if (head < p.heads + p.kv_heads && d < p.rot) {
            const int half = p.rot / 2;
            const int pair = p.interleaved ? d >> 1 : (d < half ? d : d - half);
            const bool second = p.interleaved ? (d & 1) != 0 : d >= half;
            const int apart = p.interleaved ? 1 : half;
            const float other = value(second ? e - apart : e + apart);
            const float2 w = cs[rope_at(pair)];
            o = second ? o * w.x + other * w.y : o * w.x - other * w.y;
        }
        store1(dst, p.out_type, at + d, o);
    }
}

// Bound by memory: 49 us for 8191 tokens of 48 heads x 128, fp32 to bf16 = 6.1 TB/s (57 us before the angles were padded).
// The same, sixteen elements per step: the two groups of eight whose pairs lie half the rotary part apart, or sixteen
// neighbours (pairs side by side, elements behind the rotary part, values).  dim and rot are multiples of 16.  The
// first step's loads are issued before the angles are computed.
template <int XT, int OT>
__global__ void rope_qkv_vec_kernel(const RopeArgs p) {
    __shared__ __align__(16) float2 cs[kRopeAngles];
    const long long token = blockIdx.x;
    const int per = p.dim / 16, nrot = p.rot / 16, units = (p.heads + 2 * p.kv_heads) * per;
    auto place = [&](int u, int& head, int& d0, int& d1) {
        head = u / per;
        const int c = u - head * per;
        const bool apart = !p.interleaved && c < nrot && head < p.heads + p.kv_heads;
        d0 = apart ? 8 * c : 16 * c;
        d1 = apart ? p.rot / 2 + 8 * c : 16 * c + 8;
        return c;
    };
    int u = threadIdx.x, head = 0, d0 = 0, d1 = 0, c = 0;
    Raw8 r0, r1;
    if (u < units) {
        c = place(u, head, d0, d1);
        r0 = load_raw8(p.x, XT, token * p.ld_x + head * p.dim + d0);
        r1 = load_raw8(p.x, XT, token * p.ld_x + head * p.dim + d1);
    }
    const long long slot = rope_slot(p, token);
    rope_angles(p, token, cs);
    __syncthreads();
    while (u < units) {
        float a[8], b[8];
        unpack8(r0, XT, a);
        unpack8(r1, XT, b);
        const int head_now = head, d0_now = d0, d1_now = d1, c_now = c;
        u += blockDim.x;
        if (u < units) {
            c = place(u, head, d0, d1);
            r0 = load_raw8(p.x, XT, token * p.ld_x + head * p.dim + d0);
            r1 = load_raw8(p.x, XT, token * p.ld_x + head * p.dim + d1);
        }
        long long at;
        void* dst = rope_dest(p, token, slot, head_now, at);
        if (!dst) continue;
        if (p.bias) {
            float w[8];
            load8f(p.bias, head_now * p.dim + d0_now, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] += w[j];
            load8f(p.bias, head_now * p.dim + d1_now, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] += w[j];
        }
        if (head_now < p.heads + p.kv_heads && c_now < nrot) {
            if (p.interleaved) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 wa = cs[rope_at(8 * c_now) + j], wb = cs[rope_at(8 * c_now) + 4 + j];
                    const float a0 = a[2 * j], a1 = a[2 * j + 1], b0 = b[2 * j], b1 = b[2 * j + 1];
                    a[2 * j] = a0 * wa.x - a1 * wa.y;
                    a[2 * j + 1] = a1 * wa.x + a0 * wa.y;
                    b[2 * j] = b0 * wb.x - b1 * wb.y;
                    b[2 * j + 1] = b1 * wb.x + b0 * wb.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 w = cs[rope_at(8 * c_now) + j];
                    const float a0 = a[j];
                    a[j] = a0 * w.x - b[j] * w.y;
                    b[j] = b[j] * w.x + a0 * w.y;
                }
            }
        }
        store8(dst, OT, at + d0_now, a);
        store8(dst, OT, at + d1_now, b);
    }
}

}  // namespace tk
