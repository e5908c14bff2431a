// The kernels of MXFP4 dense layers for gfx950 and their launches: products with a packed matrix,
// the gated feed-forward projection and its backward pass, dense and of a mixture's experts
// (include/kadan_amd.h; entry points in mxfp4_dense.hip and mxfp4_linear.hip).  The reference
// multiplies MXFP4 rows on the host only (IW/src/weights/quantization.cpp:207-247; IW =
// services/hikari/inference_worker).
//
//   pack_kernel        rows -> the packed form every product reads
//   pack_t_kernel      rows -> the form the backward pass reads (summed over the rows)
//   decode_kernel      a few rows of x: one workgroup per 16 or 32 matrix rows, K over its
//                      wavefronts, the weights read once
//   decode_t_kernel    the same for the backward pass, over 32 columns
//   gemm_kernel        more rows: 256 matrix rows x 32..256 rows of x a workgroup
//   reduce_kernel      K slices of gemm_kernel summed in slice order, then its epilogue
//   gate_grad_kernel   dg, du from dh and the kept pre-activations
//   act_grad_kernel    the gradient of a product's activation
//
// The products come in three families: plain ones, those with an epilogue (bias, activation,
// residual) and those of a mixture's experts, where every row has a matrix of its own.
//
// mxfp4_plan.hpp chooses among them.  Times below are of single MI355X cards, up to 20 % apart
// where the matrix cores are the bound; one's 1 GB copy runs at 5.2 TB/s and its library 8192^3
// bf16 product at 1.25 PFLOP/s.
#pragma once
#include "kdq_common.hpp"
#include "mxfp4_plan.hpp"

#include <algorithm>
#include <atomic>
#include <utility>

namespace kdq {
namespace {

using namespace mxfp4;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ packed forms
//
// Packed (kdq_mxfp4_pack): per group of 32 rows and step of 64 values one 1 KB block of
// codes, lane i + 32h holding the 16 bytes of values 64q + 32h .. +31 of row 32g + i; then
// per group and 4 steps one 256-byte block of scales, byte j of lane i + 32h's dword the
// scale of step 4p + j.  Rows and values past the matrix are zero codes with scale 0.
//
// Transposed (kdq_mxfp4_pack_transposed), for sums over the rows: per group of 64 columns
// and step of 64 rows one 2 KB block of codes in two 1 KB pieces, lane c + 32h of piece p
// holding for rows 64q + 32h + 16p .. +15 the byte that holds columns 64g + 2c (low nibble)
// and 64g + 2c + 1; then per group and step 128 bytes of scales, byte b of run 2h + e the
// scale of row 64q + 32h + b for columns 64g + 32e .. +31.

struct Form {
    size_t groups, steps, code_bytes, scale_bytes;
};

__host__ __device__ inline Form packed_form(size_t rows, size_t cols) {
    Form f;
    f.groups = ceil_div(rows, 32);
    f.steps = ceil_div(cols, 64);
    f.code_bytes = f.groups * f.steps * 1024;
    f.scale_bytes = f.groups * ceil_div(f.steps, 4) * 256;
    return f;
}

__host__ __device__ inline Form transposed_form(size_t rows, size_t cols) {
    Form f;
    f.groups = ceil_div(cols, 64);
    f.steps = ceil_div(rows, 64);
    f.code_bytes = f.groups * f.steps * 2048;
    f.scale_bytes = f.groups * f.steps * 128;
    return f;
}

// Stacks of matrices (the experts'): workgroups of blockIdx.y pack matrix blockIdx.y.  The codes of
// all lie before the scales of all, as kdq_moe_mxfp4_pack lays them.
struct Packed {
    uint8_t *codes, *scales;
    __device__ __forceinline__ Packed(const Form& f, uint8_t* out)
        : codes(out + blockIdx.y * f.code_bytes),
          scales(out + gridDim.y * f.code_bytes + blockIdx.y * f.scale_bytes) {}
};

// A copy in another order, once per weight: whole 16 bytes of 32 rows a half wavefront, so a
// row's lines are shared by the steps of four wavefronts side by side.  14336 x 4096: 14 us,
// 62 MB read and written at 4.5 TB/s.
__global__ __launch_bounds__(256) void pack_kernel(const uint8_t* __restrict__ blocks,
                                                   const uint8_t* __restrict__ scales,
                                                   size_t rows, size_t cols, Form f,
                                                   uint8_t* __restrict__ out) {
    blocks += blockIdx.y * (rows * (cols / 2));
    scales += blockIdx.y * (rows * (cols / 32));
    const Packed to(f, out);
    const size_t u = size_t(blockIdx.x) * 256 + threadIdx.x;
    const size_t units = f.code_bytes / 16;
    if (u < units) {  // 16 bytes of codes
        const unsigned l = unsigned(u % 64);
        const size_t q = u / 64 % f.steps, row = u / 64 / f.steps * 32 + l % 32;
        const size_t at = q * 32 + 16 * (l / 32);
        u32x4 v{0, 0, 0, 0};
        if (row < rows && at < cols / 2)
            v = load16(blocks + row * (cols / 2) + at);
        *reinterpret_cast<u32x4*>(to.codes + u * 16) = v;
    } else if (u - units < f.scale_bytes / 4) {  // a dword of scales
        const size_t w = u - units, sg = ceil_div(f.steps, 4);
        const unsigned l = unsigned(w % 64);
        const size_t p = w / 64 % sg, row = w / 64 / sg * 32 + l % 32;
        unsigned word = 0;
        for (unsigned j = 0; j < 4; ++j) {
            const size_t b = 2 * (4 * p + j) + l / 32;  // the row's 32-value block
            if (row < rows && b < cols / 32)
                word |= unsigned(scales[row * (cols / 32) + b]) << (8 * j);
        }
        reinterpret_cast<unsigned*>(to.scales)[w] = word;
    }
}

// Bytes, not lines, are gathered: 32 lanes read 32 bytes of a row, 16 rows in turn.  14336 x
// 4096: 25-35 us, 2.5 TB/s at best (pack_kernel's rate would be 14; once per weight it was left so).
__global__ __launch_bounds__(256) void pack_t_kernel(const uint8_t* __restrict__ blocks,
                                                     const uint8_t* __restrict__ scales,
                                                     size_t rows, size_t cols, Form f,
                                                     uint8_t* __restrict__ out) {
    blocks += blockIdx.y * (rows * (cols / 2));
    scales += blockIdx.y * (rows * (cols / 32));
    const Packed to(f, out);
    const size_t u = size_t(blockIdx.x) * 256 + threadIdx.x;
    const size_t units = f.code_bytes / 16, width = cols / 2;
    if (u < units) {  // one column byte of 16 rows
        const unsigned l = unsigned(u % 64), piece = unsigned(u / 64 % 2);
        const size_t q = u / 128 % f.steps, g = u / 128 / f.steps;
        const size_t byte = 32 * g + l % 32, row = 64 * q + 32 * (l / 32) + 16 * piece;
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (unsigned b = 0; b < 16; ++b)
            if (row + b < rows && byte < width)
                w[b / 4] |= unsigned(blocks[(row + b) * width + byte]) << (8 * (b % 4));
        *reinterpret_cast<u32x4*>(to.codes + u * 16) = u32x4{w[0], w[1], w[2], w[3]};
    } else if (u - units < f.scale_bytes / 4) {
        const size_t w = u - units, within = w % 32;  // 32 dwords per group and step
        const size_t q = w / 32 % f.steps, g = w / 32 / f.steps;
        const size_t run = within / 8, row = 64 * q + 32 * (run / 2) + 4 * (within % 8);
        const size_t block = 2 * g + run % 2;
        unsigned word = 0;
        for (unsigned b = 0; b < 4; ++b)
            if (row + b < rows && block < cols / 32)
                word |= unsigned(scales[(row + b) * (cols / 32) + block]) << (8 * b);
        reinterpret_cast<unsigned*>(to.scales)[w] = word;
    }
}

// ------------------------------------------------------------------ decoding

// Byte j of a dword of E8M0 scales as the fp32 operand of the conversions, which take its
// exponent field and nothing else (checked on the device for every scale byte, with other
// bits set as well): a rotation puts the byte there.
__device__ __forceinline__ float scale_of(unsigned word, unsigned j) {
    return __uint_as_float(__builtin_amdgcn_alignbit(word, word, 9 + 8 * j));
}

__device__ __forceinline__ unsigned bits(bf16x2 v) {
    return __builtin_bit_cast(unsigned, v);
}

// Eight E2M1 codes times their scale as bf16, which holds every such value (scale bytes up
// to 252; past that the largest codes are infinite, as in fp32; 255 gives NaN).
__device__ __forceinline__ bf16x8 decode8(unsigned codes, float scale) {
    const u4 v{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
               bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
               bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
               bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
    return __builtin_bit_cast(bf16x8, v);
}

// The transposed form: byte j of `codes` is row j's pair of columns, byte j of `scales` its
// scale.  Eight rows as the operands of the even columns and of the odd ones.
__device__ __forceinline__ void decode8_pair(const unsigned (&codes)[2],
                                             const unsigned (&scales)[2], bf16x8& even,
                                             bf16x8& odd) {
    unsigned e[4], o[4];
#pragma unroll
    for (int d = 0; d < 2; ++d) {
        const unsigned v0 = bits(
            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[d], scale_of(scales[d], 0), 0));
        const unsigned v1 = bits(
            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[d], scale_of(scales[d], 1), 1));
        const unsigned v2 = bits(
            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[d], scale_of(scales[d], 2), 2));
        const unsigned v3 = bits(
            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[d], scale_of(scales[d], 3), 3));
        e[2 * d] = __builtin_amdgcn_perm(v1, v0, 0x05040100);
        o[2 * d] = __builtin_amdgcn_perm(v1, v0, 0x07060302);
        e[2 * d + 1] = __builtin_amdgcn_perm(v3, v2, 0x05040100);
        o[2 * d + 1] = __builtin_amdgcn_perm(v3, v2, 0x07060302);
    }
    even = __builtin_bit_cast(bf16x8, u4{e[0], e[1], e[2], e[3]});
    odd = __builtin_bit_cast(bf16x8, u4{o[0], o[1], o[2], o[3]});
}

// ------------------------------------------------------------------ outputs

// Of the experts' (rows sorted by expert, a stack of matrices): _experts.  kOutLinear: with bias,
// activation and residual; kOutOneBackward: a product of gradients with one matrix, where
// kOutBackward has two.
enum Out {
    kOutF32,
    kOutBf16,
    kOutGated,
    kOutBackward,
    kOutLinear,
    kOutExpertsLinear,
    kOutExpertsGated,
    kOutOneBackward,
    kOutExpertsOneBackward,
    kOutExpertsBackward
};

constexpr bool of_experts(int out) {
    return out == kOutExpertsLinear || out == kOutExpertsGated || out == kOutExpertsOneBackward ||
           out == kOutExpertsBackward;
}
constexpr bool of_linear(int out) {
    return out == kOutLinear || out == kOutExpertsLinear;
}
constexpr bool of_gated(int out) {
    return out == kOutGated || out == kOutExpertsGated;
}
constexpr bool of_one_backward(int out) {
    return out == kOutOneBackward || out == kOutExpertsOneBackward;
}
constexpr bool of_backward(int out) {
    return out == kOutBackward || out == kOutExpertsBackward || of_one_backward(out);
}

// What an epilogue does to the sums of a product: y = residual + act(sum + bias), and of the
// experts' gated projection: h = act(g + bias, u + bias_up).  Biases: fp32 [n], the experts'
// [experts][n]; null where there is none.
struct Epilogue {
    const float *bias, *bias_up;
    const void* residual;  // of y's type
    size_t residual_stride;
    int act;
    bool f32;              // the type of y
};

// A stack of matrices in a packed form: codes of every expert, then scales of every expert.
// Expert e has rows offsets[e] .. offsets[e + 1] - 1 of x.
struct Stack {
    const int32_t* offsets;
    unsigned experts;
    size_t code_bytes, scale_bytes;  // of one expert
};

// Where results go.  Products: y [m][n].  Gated: y = h bf16 [m][n], and the kept
// pre-activations if asked for: bf16 [m][2n] (gates, then ups), or int8 [m][2n] with an
// fp32 scale per 32.  Backward: y = dx bf16 [m][n].
struct Target {
    void* y;
    size_t stride;  // values per row of y
    unsigned m, n;
    uint16_t* kept;
    int8_t* kept_q;
    float* kept_d;
    Epilogue e;
};

__device__ __forceinline__ unsigned bf16_pair(float a, float b) {
    const bf16x2 v{__bf16(a), __bf16(b)};  // round to nearest even
    return bits(v);
}

// silu(g) * u with the hardware exp2 and reciprocal (2^-21 (1 + |g|) relative; h leaves as bf16)
__device__ __forceinline__ float gate_value(float g, float u) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * g);
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

typedef unsigned pair_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned quad_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float quadf_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Four values of consecutive columns c .. c+3 of row `row` as bf16 / fp32 (those below n).
__device__ __forceinline__ void store4_bf16(uint16_t* y, size_t stride, unsigned n,
                                            unsigned row, unsigned c, f32x4 v) {
    uint16_t* at = y + size_t(row) * stride + c;
    const unsigned lo = bf16_pair(v.x, v.y), hi = bf16_pair(v.z, v.w);
    if (c + 3 < n) {
        *reinterpret_cast<pair_a2*>(at) = pair_a2{lo, hi};
    } else {
        if (c < n)
            at[0] = uint16_t(lo);
        if (c + 1 < n)
            at[1] = uint16_t(lo >> 16);
        if (c + 2 < n)
            at[2] = uint16_t(hi);
    }
}

__device__ __forceinline__ void store4_f32(float* y, size_t stride, unsigned n, unsigned row,
                                           unsigned c, f32x4 v) {
    float* at = y + size_t(row) * stride + c;
    if (c + 3 < n) {
        *reinterpret_cast<quadf_a4*>(at) = quadf_a4{v.x, v.y, v.z, v.w};
    } else {
        if (c < n)
            at[0] = v.x;
        if (c + 1 < n)
            at[1] = v.y;
        if (c + 2 < n)
            at[2] = v.z;
    }
}

// sigmoid, by the hardware exp2 and reciprocal: each is within 2^-22, and the argument, rounded to
// fp32 twice, adds 2^-21 |z| (all relative); below about -88 the result is 0.
__device__ __forceinline__ float sigmoid_value(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z));
}

// v sigmoid(z): silu has z = v; gelu's tanh form, 0.5 v (1 + tanh(z / 2)), has
// z = 2 sqrt(2 / pi) (v + 0.044715 v^3).
constexpr float kGelu1 = 1.59576912f, kGelu3 = 0.0713548163f;

__device__ __forceinline__ float act_value(float v, int act) {
    if (act == KDQ_ACT_NONE)
        return v;
    return v * sigmoid_value(act == KDQ_ACT_SILU ? v : v * fmaf(kGelu3, v * v, kGelu1));
}

// its derivative: s + v s (1 - s) z' (far out, where z or z' is past fp32, s is 0 or 1 and the
// second term 0)
__device__ __forceinline__ float act_slope(float v, int act) {
    if (act == KDQ_ACT_NONE)
        return 1.0f;
    const float q = v * v;
    const float z = act == KDQ_ACT_SILU ? v : v * fmaf(kGelu3, q, kGelu1);
    const float dz = act == KDQ_ACT_SILU ? 1.0f : fmaf(3.0f * kGelu3, q, kGelu1);
    const float s = sigmoid_value(z), rest = s * (1.0f - s);
    return rest == 0.0f ? s : fmaf(v * rest, dz, s);
}

// The clamped gate: with g' = min(g, 7) and u' = u between -7 and 7, g' sigmoid(1.702 g') (u' + 1)
constexpr float kClamp = 7.0f, kSharp = 1.702f;

// (comparisons, so that NaN stays NaN)
__device__ __forceinline__ float clamp_above(float v) {
    return v > kClamp ? kClamp : v;
}
__device__ __forceinline__ float clamp_both(float v) {
    return v > kClamp ? kClamp : v < -kClamp ? -kClamp : v;
}

__device__ __forceinline__ float gate_value(float g, float u, int act) {
    if (act == KDQ_ACT_SILU)
        return gate_value(g, u);
    const float c = clamp_above(g);
    return c * sigmoid_value(kSharp * c) * (clamp_both(u) + 1.0f);
}

// N values from column c on, of which those past n read as zeros and are not written.
template <int N>
__device__ __forceinline__ void load_f32(const float* p, unsigned c, unsigned n, float (&f)[N]) {
    if (c + N <= n) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const quadf_a4 v = *reinterpret_cast<const quadf_a4*>(p + c + 4 * i);
            f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            f[i] = c + i < n ? p[c + i] : 0.f;
    }
}

template <int N>
__device__ __forceinline__ void load_bf16(const uint16_t* p, unsigned c, unsigned n,
                                          float (&f)[N]) {
    if (c + N <= n) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const pair_a2 v = *reinterpret_cast<const pair_a2*>(p + c + 4 * i);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f[4 * i + 2 * j] = __uint_as_float(v[j] << 16);
                f[4 * i + 2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            f[i] = c + i < n ? __uint_as_float(unsigned(p[c + i]) << 16) : 0.f;
    }
}

template <int N>
__device__ __forceinline__ void store_bf16(uint16_t* p, unsigned c, unsigned n,
                                           const float (&f)[N]) {
    unsigned w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
        w[i] = bf16_pair(f[2 * i], f[2 * i + 1]);
    if (c + N <= n) {
        if constexpr (N == 8)
            *reinterpret_cast<quad_a2*>(p + c) = quad_a2{w[0], w[1], w[2], w[3]};
        else
            *reinterpret_cast<pair_a2*>(p + c) = pair_a2{w[0], w[1]};
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < n)
                p[c + i] = uint16_t(w[i / 2] >> (16 * (i % 2)));
    }
}

template <int N>
__device__ __forceinline__ void store_f32(float* p, unsigned c, unsigned n, const float (&f)[N]) {
    if (c + N <= n) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
            *reinterpret_cast<quadf_a4*>(p + c + 4 * i) =
                quadf_a4{f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < n)
                p[c + i] = f[i];
    }
}

// What an epilogue adds to N values of a row from column c on.  It is asked for ahead of the sums
// it is added to, so that its way from memory is not waited for behind theirs.
template <int N> struct Added {
    float bias[N], residual[N];
};

template <int N>
__device__ __forceinline__ void bias_of(const float* bias, unsigned c, unsigned n,
                                        float (&b)[N]) {
    if (bias)
        load_f32(bias, c, n, b);
    else
#pragma unroll
        for (int i = 0; i < N; ++i)
            b[i] = 0.f;
}

template <int N>
__device__ __forceinline__ void residual_of(const Target& t, unsigned row, unsigned c,
                                            float (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        r[i] = 0.f;
    if (!t.e.residual || row >= t.m)
        return;
    const size_t at = size_t(row) * t.e.residual_stride;
    if (t.e.f32)
        load_f32(static_cast<const float*>(t.e.residual) + at, c, t.n, r);
    else
        load_bf16(static_cast<const uint16_t*>(t.e.residual) + at, c, t.n, r);
}

// N sums of a row from column c on, to y; kept: the pre-activations as bf16 [m][n].
template <int N>
__device__ __forceinline__ void finish(const Target& t, unsigned row, unsigned c, float (&v)[N],
                                       const float (&bias)[N], const float (&residual)[N]) {
    if (row >= t.m || c >= t.n)
        return;
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] += bias[i];
    if (t.kept)
        store_bf16(t.kept + size_t(row) * t.n, c, t.n, v);
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = act_value(v[i], t.e.act) + residual[i];
    if (t.e.f32)
        store_f32(static_cast<float*>(t.y) + size_t(row) * t.stride, c, t.n, v);
    else
        store_bf16(static_cast<uint16_t*>(t.y) + size_t(row) * t.stride, c, t.n, v);
}

__device__ __forceinline__ Added<4> added4(const Target& t, unsigned row, unsigned c) {
    Added<4> a;
    bias_of(t.e.bias, c, t.n, a.bias);
    residual_of(t, row, c, a.residual);
    return a;
}

__device__ __forceinline__ void finish4(const Target& t, unsigned row, unsigned c, f32x4 v,
                                        const Added<4>& a) {
    float f[4] = {v.x, v.y, v.z, v.w};
    finish(t, row, c, f, a.bias, a.residual);
}

// Quad j of a wavefront's two 32 x 32 result tiles (group G, row `token` of x, lane half
// h): values 8j + 4h .. +3 of the tiles' matrix rows.  Products: the tiles are rows 64G and
// 64G + 32; gated: gate and up rows 32G; backward: columns 64G + 2i and 64G + 2i + 1.
template <int OUT>
__device__ __forceinline__ void store_quad(const Target& t, unsigned G, unsigned token,
                                           unsigned h, unsigned j, f32x4 v0, f32x4 v1) {
    if (token >= t.m)
        return;
    const unsigned r = 8 * j + 4 * h;
    if constexpr (OUT == kOutF32) {
        store4_f32(static_cast<float*>(t.y), t.stride, t.n, token, 64 * G + r, v0);
        store4_f32(static_cast<float*>(t.y), t.stride, t.n, token, 64 * G + 32 + r, v1);
    } else if constexpr (OUT == kOutBf16) {
        store4_bf16(static_cast<uint16_t*>(t.y), t.stride, t.n, token, 64 * G + r, v0);
        store4_bf16(static_cast<uint16_t*>(t.y), t.stride, t.n, token, 64 * G + 32 + r, v1);
    } else if constexpr (of_gated(OUT)) {
        const unsigned c = 32 * G + r;
        const auto gate = [&](float g, float u) {
            if constexpr (OUT == kOutExpertsGated)
                return gate_value(g, u, t.e.act);
            else
                return gate_value(g, u);
        };
        const f32x4 hv{gate(v0.x, v1.x), gate(v0.y, v1.y), gate(v0.z, v1.z), gate(v0.w, v1.w)};
        store4_bf16(static_cast<uint16_t*>(t.y), t.stride, t.n, token, c, hv);
        if (t.kept && c < t.n) {  // (n % 32 == 0)
            store4_bf16(t.kept, 2 * size_t(t.n), 2 * t.n, token, c, v0);
            store4_bf16(t.kept, 2 * size_t(t.n), 2 * t.n, token, t.n + c, v1);
        }
    } else {
        const unsigned c = 64 * G + 2 * r;  // (n % 32 == 0: all eight or none)
        if (c < t.n)
            *reinterpret_cast<quad_a2*>(static_cast<uint16_t*>(t.y) + size_t(token) * t.stride +
                                        c) =
                quad_a2{bf16_pair(v0.x, v1.x), bf16_pair(v0.y, v1.y), bf16_pair(v0.z, v1.z),
                        bf16_pair(v0.w, v1.w)};
    }
}

// One row's 32 pre-activations (a lane holds 16 of them, lane ^ 32 the others) as int8
// codes with scale amax / 127, codes round-half-even(v * 127 / amax): kdq_quantize_q8's
// format.  A block with a value that is not finite keeps a NaN scale; one whose largest
// magnitude is below 2^-120 is kept as zeros (127 / amax would overflow).
struct Q8 {
    unsigned codes[4];
    float scale;
};

__device__ __forceinline__ Q8 q8_of(const f32x4 (&v)[4]) {
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
    top = max(top, unsigned(__shfl_xor(int(top), 32, 64)));
    const bool finite = top < 0x7f800000u;
    const float amax = __uint_as_float(top);
    const bool some = finite && amax >= 0x1p-120f;
    const float inv = some ? 127.0f / amax : 0.f;
    Q8 q;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q.codes[j] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int code = some ? int(rintf(v[j][i] * inv)) : 0;
            q.codes[j] |= (unsigned(code) & 255u) << (8 * i);
        }
    }
    q.scale = !finite ? __uint_as_float(0x7fc00000u) : some ? amax / 127.0f : 0.f;
    return q;
}

__device__ __forceinline__ void keep_q8(const Target& t, unsigned column, unsigned token,
                                        unsigned h, const f32x4 (&v)[4]) {
    const Q8 q = q8_of(v);
    if (token >= t.m || column >= 2 * t.n)
        return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<unsigned*>(t.kept_q + size_t(token) * 2 * t.n + column + 8 * j + 4 * h) =
            q.codes[j];
    if (h == 0)
        t.kept_d[size_t(token) * (2 * t.n / 32) + column / 32] = q.scale;
}

__device__ __forceinline__ f32x4 quad_of(const f32x16& a, int j) {
    return f32x4{a[4 * j], a[4 * j + 1], a[4 * j + 2], a[4 * j + 3]};
}

// 32 rows of 128 bytes, a wavefront's own in LDS, to rows `first` .. of y (their bytes from
// byte column `c` on, those below `bytes`): whole lines in 16-byte pieces, where a lane's own
// values would be 8- or 16-byte pieces of 32 rows (each a request of its own to the L2: 3.7
// million of 10 million for 2048 x 14336 bf16 results).
constexpr unsigned kPatchBytes = 4096;

__device__ __forceinline__ unsigned patch_at(unsigned row, unsigned piece) {
    return row * 128 + (piece ^ (row / 2 % 8)) * 16;
}

__device__ __forceinline__ void store_patch(const uint8_t* patch, uint8_t* y, size_t row_bytes,
                                            unsigned first, unsigned m, size_t c, size_t bytes) {
    const unsigned lane = threadIdx.x % 64, piece = lane % 8;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    u4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = *reinterpret_cast<const u4*>(patch + patch_at(8 * i + lane / 8, piece));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned row = first + 8 * i + lane / 8;
        const size_t at = c + 16 * piece;
        if (row >= m || at >= bytes)
            continue;
        uint8_t* to = y + size_t(row) * row_bytes + at;
        if (at + 16 <= bytes) {
            *reinterpret_cast<quad_a2*>(to) = quad_a2{v[i].x, v[i].y, v[i].z, v[i].w};
        } else {
#pragma unroll
            for (unsigned e = 0; e < 7; ++e)  // (values are 2 or 4 bytes)
                if (at + 2 * e < bytes)
                    *reinterpret_cast<uint16_t*>(to + 2 * e) =
                        uint16_t(v[i][e / 2] >> (16 * (e % 2)));
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Two tiles of 32 columns as bf16, side by side in the patch.
__device__ __forceinline__ void patch_pair(uint8_t* patch, unsigned token, unsigned h,
                                           const f32x16& a0, const f32x16& a1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x4 v0 = quad_of(a0, j), v1 = quad_of(a1, j);
        *reinterpret_cast<uint2*>(patch + patch_at(token, j) + 8 * h) =
            make_uint2(bf16_pair(v0.x, v0.y), bf16_pair(v0.z, v0.w));
        *reinterpret_cast<uint2*>(patch + patch_at(token, 4 + j) + 8 * h) =
            make_uint2(bf16_pair(v1.x, v1.y), bf16_pair(v1.z, v1.w));
    }
}

// Two tiles of 32 columns as fp32, side by side in 8 KB of LDS that are the wavefront's own, so
// that bias, residual and results move in whole lines: a lane takes eight columns of a row.
// (256 bytes are all the banks, so rows are told apart by their place of 16 bytes.)
constexpr unsigned kWidePatchBytes = 8192;

__device__ __forceinline__ unsigned wide_at(unsigned row, unsigned piece) {
    return row * 256 + (piece ^ row % 16) * 16;
}

__device__ __forceinline__ void spread_wide(uint8_t* patch, const f32x16& a0, const f32x16& a1) {
    const unsigned row = threadIdx.x % 32, h = threadIdx.x % 64 / 32;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<f32x4*>(patch + wide_at(row, 2 * j + h)) = quad_of(a0, j);
        *reinterpret_cast<f32x4*>(patch + wide_at(row, 8 + 2 * j + h)) = quad_of(a1, j);
    }
}

// ROWS of the tiles' 32 rows from `from` on, out of a patch, or of two whose sum they are.
template <int ROWS, int PATCHES>
__device__ __forceinline__ void store_wide(const Target& t, unsigned G, unsigned T, unsigned from,
                                           const uint8_t* patch, const uint8_t* second,
                                           const float (&bias)[8],
                                           const float (&residual)[ROWS / 8][8]) {
    const unsigned lane = threadIdx.x % 64, eighth = lane % 8, c = 64 * G + 8 * eighth;
#pragma unroll
    for (int i = 0; i < ROWS / 8; ++i) {
        const unsigned row = from + 8 * i + lane / 8;
        f32x4 lo = *reinterpret_cast<const f32x4*>(patch + wide_at(row, 2 * eighth));
        f32x4 hi = *reinterpret_cast<const f32x4*>(patch + wide_at(row, 2 * eighth + 1));
        if constexpr (PATCHES == 2) {
            lo += *reinterpret_cast<const f32x4*>(second + wide_at(row, 2 * eighth));
            hi += *reinterpret_cast<const f32x4*>(second + wide_at(row, 2 * eighth + 1));
        }
        float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        finish(t, T * 32 + row, c, v, bias, residual[i]);
    }
}

template <int ROWS>
__device__ __forceinline__ void ask_for(const Target& t, unsigned G, unsigned T, unsigned from,
                                        float (&bias)[8], float (&residual)[ROWS / 8][8]) {
    const unsigned lane = threadIdx.x % 64, c = 64 * G + 8 * (lane % 8);
    bias_of(t.e.bias, c, t.n, bias);
#pragma unroll
    for (int i = 0; i < ROWS / 8; ++i)
        residual_of(t, T * 32 + from + 8 * i + lane / 8, c, residual[i]);
}

__device__ __forceinline__ void store_linear(const Target& t, unsigned G, unsigned T,
                                             uint8_t* patch, const f32x16& a0, const f32x16& a1) {
    float bias[8], residual[4][8];
    ask_for<32>(t, G, T, 0, bias, residual);
    spread_wide(patch, a0, a1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    store_wide<32, 1>(t, G, T, 0, patch, nullptr, bias, residual);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wavefront's two 32 x 32 result tiles (group G, rows 32T .. of x), but for the gated
// projection's: as store_quad, through `patch`, kPatchBytes of LDS that are the wavefront's own.
template <int OUT>
__device__ __forceinline__ void store_tiles(const Target& t, unsigned G, unsigned T,
                                            uint8_t* patch, const f32x16& a0, const f32x16& a1) {
    const unsigned lane = threadIdx.x % 64, row = lane % 32, h = lane / 32;
    auto* y = static_cast<uint8_t*>(t.y);
    if constexpr (OUT == kOutF32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4*>(patch + patch_at(row, 2 * j + h)) =
                    quad_of(i ? a1 : a0, j);
            store_patch(patch, y, t.stride * 4, T * 32, t.m, (size_t(64) * G + 32 * i) * 4,
                        size_t(t.n) * 4);
        }
    } else if constexpr (OUT == kOutBf16) {
        patch_pair(patch, row, h, a0, a1);
        store_patch(patch, y, t.stride * 2, T * 32, t.m, size_t(64) * G * 2, size_t(t.n) * 2);
    } else if constexpr (of_linear(OUT)) {
        store_linear(t, G, T, patch, a0, a1);
    } else {
        static_assert(of_backward(OUT));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 v0 = quad_of(a0, j), v1 = quad_of(a1, j);
            *reinterpret_cast<u4*>(patch + patch_at(row, 2 * j + h)) =
                u4{bf16_pair(v0.x, v1.x), bf16_pair(v0.y, v1.y), bf16_pair(v0.z, v1.z),
                   bf16_pair(v0.w, v1.w)};
        }
        store_patch(patch, y, t.stride * 2, T * 32, t.m, size_t(64) * G * 2, size_t(t.n) * 2);
    }
}

// The gated projection's results of four wavefronts (32 features each, side by side) and 32
// rows meet in LDS, so that they leave in whole lines: h and kept bf16 values 256 bytes a
// row, kept codes 128.  (Each wavefront by itself: pieces of 8 bytes for h, of 4 for codes;
// 2048 x 4096 -> 14336 with kept codes 445 us against 387 with nothing kept.)
constexpr unsigned kWidePitch = 272, kCodePitch = 144;
constexpr unsigned kGatedPatch = 32 * 3 * kWidePitch;  // h, g, u; or h, codes and scales

template <int OUT>
__device__ __forceinline__ void gather_gated(const Target& t, uint8_t* patch, unsigned rg,
                                             unsigned row, unsigned h, const f32x16& a0,
                                             const f32x16& a1) {
    const auto gate = [&](float g, float u) {
        if constexpr (OUT == kOutExpertsGated)
            return gate_value(g, u, t.e.act);
        else
            return gate_value(g, u);
    };
    uint8_t* kept = patch + 32 * kWidePitch;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x4 g = quad_of(a0, j), u = quad_of(a1, j);
        const unsigned at = row * kWidePitch + (32 * rg + 8 * j + 4 * h) * 2;
        *reinterpret_cast<uint2*>(patch + at) = make_uint2(
            bf16_pair(gate(g.x, u.x), gate(g.y, u.y)), bf16_pair(gate(g.z, u.z), gate(g.w, u.w)));
        if (t.kept) {
            *reinterpret_cast<uint2*>(kept + at) =
                make_uint2(bf16_pair(g.x, g.y), bf16_pair(g.z, g.w));
            *reinterpret_cast<uint2*>(kept + 32 * kWidePitch + at) =
                make_uint2(bf16_pair(u.x, u.y), bf16_pair(u.z, u.w));
        }
    }
    if (!t.kept_q)
        return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x16& a = i ? a1 : a0;
        const f32x4 v[4] = {quad_of(a, 0), quad_of(a, 1), quad_of(a, 2), quad_of(a, 3)};
        const Q8 q = q8_of(v);
        uint8_t* codes = kept + i * 32 * kCodePitch + row * kCodePitch;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<unsigned*>(codes + 32 * rg + 8 * j + 4 * h) = q.codes[j];
        if (h == 0)  // (the pitch's last 16 bytes: the four wavefronts' scales)
            *reinterpret_cast<float*>(codes + 128 + 4 * rg) = q.scale;
    }
}

// Thread `i` of 256; features first .. first + 127, rows of x from 32T on.
__device__ __forceinline__ void store_gated(const Target& t, const uint8_t* patch, unsigned i,
                                            unsigned first, unsigned T) {
    const uint8_t* kept = patch + 32 * kWidePitch;
    auto wide = [&](const uint8_t* from, uint16_t* to, size_t stride) {  // 512 pieces
#pragma unroll
        for (unsigned e = 0; e < 2; ++e) {
            const unsigned row = 16 * e + i / 16, c = i % 16 * 8;
            const u4 v = *reinterpret_cast<const u4*>(from + row * kWidePitch + c * 2);
            if (32 * T + row < t.m && first + c < t.n)  // (n % 32 == 0)
                *reinterpret_cast<quad_a2*>(to + size_t(32 * T + row) * stride + first + c) =
                    quad_a2{v.x, v.y, v.z, v.w};
        }
    };
    wide(patch, static_cast<uint16_t*>(t.y), t.stride);
    if (t.kept) {
        wide(kept, t.kept, 2 * size_t(t.n));
        wide(kept + 32 * kWidePitch, t.kept + t.n, 2 * size_t(t.n));
    }
    if (!t.kept_q)
        return;
    const unsigned row = i / 8, c = i % 8 * 16, token = 32 * T + row;
#pragma unroll
    for (unsigned e = 0; e < 2; ++e) {
        const uint8_t* codes = kept + (e * 32 + row) * kCodePitch;
        const u4 v = *reinterpret_cast<const u4*>(codes + c);
        if (token < t.m && first + c < t.n)
            *reinterpret_cast<quad_a2*>(t.kept_q + size_t(token) * 2 * t.n + e * t.n + first + c) =
                quad_a2{v.x, v.y, v.z, v.w};
        // four of the eight threads of a row: a scale each
        if (token < t.m && i % 8 < 4 && first + 32 * (i % 8) < t.n)
            t.kept_d[size_t(token) * (t.n / 16) + e * (t.n / 32) + first / 32 + i % 8] =
                *reinterpret_cast<const float*>(codes + 128 + 4 * (i % 8));
    }
}

// ------------------------------------------------------------------ a few rows of x
//
// One workgroup takes R tiles of 16 matrix rows (of both matrices for the gated projection)
// and all of K, a run of 128-value units to each wavefront.  Per unit a lane holds 32 values
// of one matrix row (lane r + 16q: row r, values 128t + 32q ..) and of one row of x, so four
// v_mfma_f32_16x16x32_bf16 multiply the unit without moving a value between lanes: the sum
// over K may run in any order.  Weights are read once, whole lines (R == 2: whole 1 KB
// blocks), and not kept in the caches.
//
// STAGED: x, up to kStagedBytes, passes through LDS, requested before the weights (a compute
// unit's loads return in order); otherwise every wavefront reads its operands of x itself.
// (With that, runs of K to a wavefront in place of interleaved units, and whole blocks, 1 row
// of 4096 -> 14336 went from 9.1 to 7.8 us, its gated projection from 18.6 to 13.6.)
//
// Bound by reading the weights: 31 MB in 8 us (3.9 TB/s; 6.0 us at the copy rate, the rest is
// the launch and its first loads), the gated projection's 62 MB in 13.2 us (4.7 TB/s); eight
// MXFP4 rows 8.5 us.

struct Decode {
    const uint8_t *w0, *w1;
    const uint8_t* x;         // bf16 rows, or MXFP4 blocks
    const uint8_t* x_scales;  // MXFP4 scales
    unsigned x_stride;        // bytes
    unsigned k, steps, groups, units;  // units of a wavefront
    Target out;
    Stack stack;
};

// ------------------------------------------------------------------ experts
//
// The rows of x are sorted by expert, and only the device knows where each expert's begin, so a
// launch has as many workgroups as any sizes could need and each finds its own: every wavefront
// reads all the offsets (a quad of experts a lane), counts the tiles of `rows_of_tile` rows and
// adds up the counts along the lanes.  That takes 0.6 to 0.8 us ahead of the first load of
// weights, 0.9 to 1.1 where the offsets come out of memory (32 to 256 experts); a launch that wrote
// a list of tiles first would take several.

__device__ __forceinline__ unsigned uniform(unsigned v) {
    return unsigned(__builtin_amdgcn_readfirstlane(int(v)));
}

template <int CTRL, int ROWS> __device__ __forceinline__ unsigned shifted(unsigned v) {
    return unsigned(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xf, false));
}

// The sum of the lanes up to and with this one (all 64 active).
__device__ __forceinline__ unsigned lanes_up_to(unsigned v) {
    v += shifted<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += shifted<0x112, 0xf>(v);
    v += shifted<0x114, 0xf>(v);
    v += shifted<0x118, 0xf>(v);
    v += shifted<0x142, 0xa>(v);  // row_bcast:15 -> rows 1 and 3
    v += shifted<0x143, 0xc>(v);  // row_bcast:31 -> rows 2 and 3
    return v;
}

constexpr unsigned kMaxExperts = 256;

// A quad of experts of each lane: their rows, and how many tiles of `rows` they make: in the low
// half of a word, and in the high half those whose last tile has at most half the rows (where
// HALVES tells them apart: it is then in no low half).
template <unsigned ROWS, bool HALVES> struct Tiles {
    unsigned first[4], end[4], tiles[4], before, total;

    // Offsets are taken as they are, but for those outside of the rows (m of them).
    __device__ __forceinline__ Tiles(const Stack& s, unsigned m) {
        const unsigned lane = threadIdx.x % 64;
        unsigned at[5], sum = 0;
#pragma unroll
        for (unsigned j = 0; j < 5; ++j)
            at[j] = unsigned(min(max(s.offsets[min(4 * lane + j, s.experts)], 0), int(m)));
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {  // (past the last expert: no rows)
            first[j] = at[j];
            end[j] = max(at[j], at[j + 1]);
            tiles[j] = tiles_of(end[j] - first[j], ROWS, HALVES);
            sum += tiles[j];
        }
        const unsigned through = lanes_up_to(sum);
        before = through - sum;
        total = unsigned(__builtin_amdgcn_readlane(int(through), 63));
    }

    __device__ __forceinline__ unsigned whole() const {
        return total & 0xffffu;
    }
    __device__ __forceinline__ unsigned halves() const {
        return total >> 16;
    }

    struct Place {
        // rows of the expert from its first such tile on; such tiles before the expert's, and its
        unsigned expert, first, end, before, tiles;
    };

    // The expert whose whole tiles (or halves) number `t` is among; no tiles where there is none,
    // as offsets that decrease might have it.
    __device__ __forceinline__ Place of(unsigned t, bool half) const {
        const unsigned shift = half ? 16 : 0;
        unsigned from = before >> shift & 0xffffu, e = 0, lo = 0, hi = 0, b = 0, n = 0;
        bool mine = false;
#pragma unroll
        for (unsigned j = 0; j < 4; ++j) {
            const unsigned count = tiles[j] >> shift & 0xffffu;
            if (t >= from && t < from + count) {
                mine = true;
                e = 4 * (threadIdx.x % 64) + j;
                lo = first[j] + (half ? (tiles[j] & 0xffffu) * ROWS : 0);
                hi = end[j], b = from, n = count;
            }
            from += count;
        }
        const uint64_t who = __builtin_amdgcn_ballot_w64(mine);
        const int lane = who ? int(__builtin_ctzll(who)) : 0;
        const auto read = [&](unsigned v) {
            return unsigned(__builtin_amdgcn_readlane(int(v), lane));
        };
        return {read(e), read(lo), read(hi), read(b), read(n)};
    }
};

// The call's pointers moved on to an expert and its rows from `first` on, as if `rows` were all.
template <int OUT>
__device__ __forceinline__ void move_to(Target& t, unsigned expert, unsigned first,
                                        unsigned rows) {
    const size_t size = of_linear(OUT) && t.e.f32 ? 4 : 2;
    t.y = static_cast<uint8_t*>(t.y) + size_t(first) * t.stride * size;
    if (t.e.residual)
        t.e.residual = static_cast<const uint8_t*>(t.e.residual) +
                       size_t(first) * t.e.residual_stride * size;
    if (t.e.bias)
        t.e.bias += size_t(expert) * t.n;
    if (t.e.bias_up)
        t.e.bias_up += size_t(expert) * t.n;
    const size_t width = of_gated(OUT) ? 2 * size_t(t.n) : t.n;
    if (t.kept)
        t.kept += first * width;
    if (t.kept_q) {
        t.kept_q += first * width;
        t.kept_d += first * (width / 32);
    }
    t.m = rows;
}

constexpr int kOutside = 0x7ffffff0;  // past any buffer's range: such loads return zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const uint8_t* p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, int(bytes), 0x00027000);
}

template <int POLICY = 0>
__device__ __forceinline__ u4 load_b128(const __amdgpu_buffer_rsrc_t& r, int at) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, POLICY);
    return u4{unsigned(v[0]), unsigned(v[1]), unsigned(v[2]), unsigned(v[3])};
}

template <int R, int TB, bool GATED, bool FP4, bool STAGED, int OUT>
__global__ __launch_bounds__(1024) void decode_kernel(Decode a) {
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr int kNt = 2;  // cache policy of loads that nothing reads again
    constexpr int TILES = GATED ? 2 * R : R;
    constexpr int kBatch = TB == 1 ? 4 : TB == 2 ? 2 : 1;
    constexpr int kScales = (kBatch + 1) / 2;  // dwords of scales
    constexpr int kX = FP4 ? 1 : 4;
    const unsigned lane = threadIdx.x % 64, waves = blockDim.x / 64;
    const unsigned wave = unsigned(__builtin_amdgcn_readfirstlane(int(threadIdx.x / 64)));
    const unsigned r = lane % 16, q = lane / 16;
    unsigned first_row = blockIdx.y * (16 * TB);
    size_t expert = 0;
    if constexpr (of_experts(OUT)) {
        const Tiles<16 * TB, false> list(a.stack, a.out.m);
        const auto p = list.of(blockIdx.y, false);
        if (!p.tiles)
            return;
        first_row = p.first + (blockIdx.y - p.before) * (16 * TB);
        move_to<OUT>(a.out, p.expert, first_row, min(p.end - first_row, 16u * TB));
        a.x += size_t(first_row) * a.x_stride;
        expert = p.expert;
        first_row = 0;
    }
    const unsigned rows = min(a.out.m - first_row, 16u * TB);
    const unsigned row_bytes = FP4 ? a.k / 2 : a.k * 2;
    const auto xs = buffer(a.x + size_t(first_row) * a.x_stride,
                           (rows - 1) * a.x_stride + row_bytes);
    const auto xscales = buffer(a.x_scales + size_t(first_row) * (a.k / 32),
                                FP4 ? rows * (a.k / 32) : 0);

    constexpr unsigned kPieces = kStagedBytes / 16 / 256;  // of a thread, at 256 threads
    u4 piece[STAGED ? kPieces : 1];
    const unsigned row_pieces = row_bytes / 16, pieces = rows * row_pieces;
    if constexpr (STAGED) {
#pragma unroll
        for (unsigned j = 0; j < kPieces; ++j) {
            const unsigned i = j * blockDim.x + threadIdx.x;
            if (j * blockDim.x < pieces)
                piece[j] = load_b128(
                    xs, i < pieces ? int(i / row_pieces * a.x_stride + i % row_pieces * 16)
                                   : kOutside);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }

    // tile i: rows 16 (R * blockIdx.x + i % R) .. of matrix i / R
    const unsigned scale_groups = (a.steps + 3) / 4;
    __amdgpu_buffer_rsrc_t codes[GATED ? 2 : 1], scales[GATED ? 2 : 1];
    const unsigned group = R == 2 ? blockIdx.x : blockIdx.x / 2;
#pragma unroll
    for (int i = 0; i < (GATED ? 2 : 1); ++i) {
        const uint8_t* w = i ? a.w1 : a.w0;
        const uint8_t* s = w + size_t(a.groups) * a.steps * 1024;
        if constexpr (of_experts(OUT)) {
            s = w + a.stack.experts * a.stack.code_bytes + expert * a.stack.scale_bytes;
            w += expert * a.stack.code_bytes;
        }
        codes[i] = buffer(w + size_t(group) * a.steps * 1024, a.steps * 1024);
        scales[i] = buffer(s + size_t(group) * scale_groups * 256, scale_groups * 256);
    }
    const unsigned block_row = 16 * (R == 2 ? 0 : blockIdx.x % 2) + r + 32 * (q % 2);
    const unsigned lane_codes = (q / 2) * 1024 + block_row * 16, lane_scales = block_row * 4;
    // (an even number of units: a dword of scales is two)
    const unsigned begin = wave * a.units, end = begin + a.units;
    // x ends with the run as well: a batch past it would multiply the zeros that stand for its
    // weights by the next wavefront's x, which may be infinite
    const unsigned limit = min(a.k, end * 128);
    u4 c[kBatch][TILES];
    unsigned s[kScales][TILES];
    auto load = [&](unsigned t0) {  // units past K, or past the wavefront's run, are zeros
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                c[b][i] = load_b128<kNt>(
                    codes[i / R],
                    t0 + b < end ? int((t0 + b) * 2048 + lane_codes + i % R * 256) : kOutside);
#pragma unroll
            for (int b = 0; b < kScales; ++b)
                s[b][i] = __builtin_amdgcn_raw_buffer_load_b32(
                    scales[i / R], int((t0 / 2 + b) * 256 + lane_scales + i % R * 64), 0, kNt);
        }
    };
    load(begin);
    const unsigned pitch = staged_pitch(row_bytes);
    if constexpr (STAGED) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (unsigned j = 0; j < kPieces; ++j) {
            const unsigned i = j * blockDim.x + threadIdx.x;
            if (i < pieces)
                *reinterpret_cast<u4*>(lds + i / row_pieces * pitch + i % row_pieces * 16) =
                    piece[j];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the weights stay in flight)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    f32x4 acc[TILES][TB] = {};
    const unsigned staged_row = min(r, rows - 1) * pitch;  // (others' results are not stored)
    for (unsigned t0 = begin; t0 < end; t0 += kBatch) {
        if (t0 != begin)
            load(t0);
        u4 x[kBatch][TB][kX];
        unsigned xb[kBatch][TB];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const unsigned t = t0 + b;
            const bool inside = 128 * t + 32 * q < limit;
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const unsigned token = r + 16 * i;
                const bool there = token < rows && inside;
                if constexpr (FP4)
                    xb[b][i] = __builtin_amdgcn_raw_buffer_load_b8(
                        xscales, there ? int(token * (a.k / 32) + 4 * t + q) : kOutside, 0, 0);
                if constexpr (STAGED) {
#pragma unroll
                    for (int d = 0; d < kX; ++d) {
                        const unsigned at =
                            FP4 ? (4 * t + q) * 16 : (128 * t + 32 * q + 8 * d) * 2;
                        const u4 v = *reinterpret_cast<const u4*>(
                            lds + staged_row + (inside ? at : 0));
                        x[b][i][d] = inside ? v : u4{0, 0, 0, 0};
                    }
                } else if constexpr (FP4) {
                    x[b][i][0] =
                        load_b128(xs, there ? int(token * a.x_stride + (4 * t + q) * 16) : kOutside);
                } else {
                    const int at = there ? int(token * a.x_stride + (128 * t + 32 * q) * 2)
                                         : kOutside - 64;
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        x[b][i][d] = load_b128(xs, at + 16 * d);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            float ws[TILES];
#pragma unroll
            for (int i = 0; i < TILES; ++i)  // (t0 is even, but for batches of one)
                ws[i] = scale_of(s[b / 2][i], 2 * (kBatch == 1 ? t0 % 2 : b % 2) + q / 2);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                bf16x8 xv[TB];
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    if constexpr (FP4)
                        xv[i] = decode8(x[b][i][0][d], scale_of(xb[b][i], 0));
                    else
                        xv[i] = __builtin_bit_cast(bf16x8, x[b][i][d]);
                }
#pragma unroll
                for (int j = 0; j < TILES; ++j) {
                    const bf16x8 wv = decode8(c[b][j][d], ws[j]);
#pragma unroll
                    for (int i = 0; i < TB; ++i)
                        acc[j][i] =
                            __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[i], acc[j][i], 0, 0, 0);
                }
            }
        }
    }
    // the wavefronts' sums meet in wavefront order
    Added<4> added;  // of the first tile that the wavefront finishes
    if constexpr (of_linear(OUT))
        if (wave < R * TB)
            added = added4(a.out, first_row + 16 * (wave % TB) + r,
                           (blockIdx.x * R + wave / TB) * 16 + 4 * q);
    if constexpr (STAGED)
        __syncthreads();
    auto* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int j = 0; j < TILES; ++j)
#pragma unroll
        for (int i = 0; i < TB; ++i)
            red[((wave * TILES + j) * TB + i) * 64 + lane] = acc[j][i];
    __syncthreads();
    auto total = [&](unsigned j, unsigned tb) {
        f32x4 sum = red[(j * TB + tb) * 64 + lane];
        for (unsigned i = 1; i < waves; ++i)
            sum += red[((i * TILES + j) * TB + tb) * 64 + lane];
        return sum;
    };
    for (unsigned i = wave; i < R * TB; i += waves) {
        const unsigned tile = i / TB, tb = i % TB;
        const unsigned token = first_row + 16 * tb + r, at = (blockIdx.x * R + tile) * 16 + 4 * q;
        if (token >= a.out.m)
            continue;
        f32x4 v = total(tile, tb);
        if constexpr (OUT == kOutExpertsGated) {
            const f32x4 u = total(R + tile, tb);
            float bg[4], bu[4];
            bias_of(a.out.e.bias, at, a.out.n, bg);
            bias_of(a.out.e.bias_up, at, a.out.n, bu);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = gate_value(v[j] + bg[j], u[j] + bu[j], a.out.e.act);
        } else if constexpr (GATED) {
            const f32x4 u = total(R + tile, tb);
            v = f32x4{gate_value(v.x, u.x), gate_value(v.y, u.y), gate_value(v.z, u.z),
                      gate_value(v.w, u.w)};
        }
        if constexpr (of_linear(OUT))
            finish4(a.out, token, at, v, i == wave ? added : added4(a.out, token, at));
        else if constexpr (OUT == kOutF32)
            store4_f32(static_cast<float*>(a.out.y), a.out.stride, a.out.n, token, at, v);
        else
            store4_bf16(static_cast<uint16_t*>(a.out.y), a.out.stride, a.out.n, token, at, v);
    }
}

// The backward pass's product for a few rows: x = [dg | du], the matrices in the transposed
// form.  A workgroup takes 32 columns (16 byte lanes e = blockIdx.x % 2 of a group, as a tile
// of even and a tile of odd columns), half its wavefronts the gate's rows and half the up's,
// in units of 128 rows: lane r + 16q holds byte lane r's rows 128t + 32q .. +31.  Bound by
// decoding, which sorts every converted pair of columns into two operands: 1 row of 2880 ->
// 2880 10.3 us (gemm_kernel 13.0), of 1024 -> 8192 6.6 (11.6).
template <int TB>
__global__ __launch_bounds__(1024) void decode_t_kernel(Decode a) {
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr int kNt = 2;
    constexpr int kBatch = TB == 1 ? 2 : 1;
    const unsigned lane = threadIdx.x % 64, waves = blockDim.x / 64, share = waves / 2;
    const unsigned wave = unsigned(__builtin_amdgcn_readfirstlane(int(threadIdx.x / 64)));
    const unsigned r = lane % 16, q = lane / 16;
    const unsigned group = blockIdx.x / 2, e = blockIdx.x % 2, matrix = wave / share;
    const uint8_t* w = matrix ? a.w1 : a.w0;
    const auto codes = buffer(w + size_t(group) * a.steps * 2048, a.steps * 2048);
    const auto scales = buffer(w + size_t(a.groups) * a.steps * 2048 +
                                   size_t(group) * a.steps * 128,
                               a.steps * 128);
    const unsigned first_row = blockIdx.y * (16 * TB), rows = min(a.out.m - first_row, 16u * TB);
    const auto xs = buffer(a.x + size_t(first_row) * a.x_stride + matrix * (a.k * 2),
                           (rows - 1) * a.x_stride + a.k * 2);
    const unsigned lane_codes = (q / 2) * 2048 + (16 * e + r + 32 * (q % 2)) * 16;
    const unsigned lane_scales = (q / 2) * 128 + (2 * (q % 2) + e) * 32;
    const unsigned begin = wave % share * a.units, end = begin + a.units;
    const unsigned limit = min(a.k, end * 128);  // x ends with the run, as decode_kernel's
    f32x4 acc[2][TB] = {};
    struct Batch {
        u4 c[kBatch][2], s[kBatch][2];
    };
    auto load = [&](unsigned t0, Batch& v) {  // units past the wavefront's run are zeros
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const unsigned t = t0 + b;
                v.c[b][p] = load_b128<kNt>(
                    codes, t < end ? int(t * 4096 + p * 1024 + lane_codes) : kOutside);
                v.s[b][p] = load_b128(scales, int(t * 256 + lane_scales + 16 * p));
            }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // a batch's x is requested before the next batch's weights, which then stream while it is
    // multiplied (loads return in order)
    auto multiply = [&](unsigned t0, const Batch& now, Batch& next) {
        u4 x[kBatch][TB][4];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const unsigned from = 128 * (t0 + b) + 32 * q;
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const unsigned token = r + 16 * i;
                const int at = token < rows && from < limit ? int(token * a.x_stride + from * 2)
                                                          : kOutside - 64;
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    x[b][i][d] = load_b128(xs, at + 16 * d);
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        load(t0 + kBatch, next);
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const unsigned cw[2] = {now.c[b][d / 2][2 * (d % 2)],
                                        now.c[b][d / 2][2 * (d % 2) + 1]};
                const unsigned sw[2] = {now.s[b][d / 2][2 * (d % 2)],
                                        now.s[b][d / 2][2 * (d % 2) + 1]};
                bf16x8 even, odd;
                decode8_pair(cw, sw, even, odd);
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    const bf16x8 xv = __builtin_bit_cast(bf16x8, x[b][i][d]);
                    acc[0][i] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, xv, acc[0][i], 0, 0, 0);
                    acc[1][i] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, xv, acc[1][i], 0, 0, 0);
                }
            }
    };
    Batch first, second;
    load(begin, first);
    for (unsigned t0 = begin; t0 < end; t0 += 2 * kBatch) {
        multiply(t0, first, second);
        multiply(t0 + kBatch, second, first);
    }
    auto* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < TB; ++i)
            red[((wave * 2 + j) * TB + i) * 64 + lane] = acc[j][i];
    __syncthreads();
    const unsigned col = blockIdx.x * 32 + 8 * q;  // (n % 32 == 0)
    for (unsigned tb = wave; tb < TB; tb += waves) {
        const unsigned token = first_row + 16 * tb + r;
        if (token >= a.out.m)
            continue;
        f32x4 v[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            v[j] = red[(j * TB + tb) * 64 + lane];
            for (unsigned i = 1; i < waves; ++i)
                v[j] += red[((i * 2 + j) * TB + tb) * 64 + lane];
        }
        *reinterpret_cast<quad_a2*>(static_cast<uint16_t*>(a.out.y) +
                                    size_t(token) * a.out.stride + col) =
            quad_a2{bf16_pair(v[0].x, v[1].x), bf16_pair(v[0].y, v[1].y),
                    bf16_pair(v[0].z, v[1].z), bf16_pair(v[0].w, v[1].w)};
    }
}

// ------------------------------------------------------------------ more rows of x
//
// A workgroup of eight wavefronts takes 256 matrix rows (four row groups of two 32-row
// tiles) and, as two wavefront groups, either two parts of K of the same TT * 32 rows of x
// (SPLIT; the groups' sums meet in LDS at the end) or two sets of TT * 32 rows.  x passes
// through LDS in chunks of 128 bytes a row (64 bf16 values, or 256 MXFP4 values), copied
// by DMA three chunks ahead into four buffers, eight rows to an instruction; a row's
// 16-byte segments lie in it by (segment ^ row / 2 % 8): the copies read whole lines, and
// operands of 16 neighbouring rows lie in all 64 banks (two neighbouring rows are 256 bytes,
// all the banks, so it is pairs of rows that have to be told apart; by row % 8 an eighth of
// the LDS cycles were conflicts).  Weights go from memory to registers, every one read and
// decoded by one wavefront (two where the groups share rows).
//
// Operands: bf16 x (v_mfma_f32_32x32x16_bf16, weights decoded to bf16, exact), MXFP4 x
// (v_mfma_scale_f32_32x32x64_f8f6f4 over both codes as they lie, so that 6 at scale byte 254 is
// its value, where decode_kernel's bf16 weight is infinite), and the backward pass's
// transposed weights under bf16 gradients (their scales lie along the columns, which are not
// summed over, so the scaled MFMA cannot take them).
//
// bf16, 512 x 4096 -> 14336: 49-59 us, 1.0-1.2 PFLOP/s; gated projection 2048 x 4096 ->
// 14336 387 us, 1.24, with codes kept 409-426, 1.13-1.18, with bf16 values kept 430, 1.12; backward
// of that 397-412 us, 1.17-1.21.  Bound by the matrix cores' clock under load: products of random
// values alone, with nothing to load, decode or wait for, run at 1.68 PFLOP/s here.  MXFP4, 2048 x
// 4096 -> 14336: 73-84 us, 2.9-3.3 PFLOP/s of 6.4 by that measure, 38 us of products: 448 tiles of
// 256 x 256 are 1.75 rounds of the compute units, which take as long as two (43 us); the rest are
// waits for operands and the results' way out.  (By count, at the products' own pace, operands would take a third of the
// LDS's 128 bytes a cycle and weights and x about 30 bytes a cycle of a compute unit's loads.)
// (Four wavefronts of 64 x 256 in place of eight took 74-96 us.)
//
// Tiles of 32 and, but for MXFP4 x (whose scales need the registers), 64 rows of x fit two
// workgroups to a compute unit, which hide each other's waits: 333 x 2880 -> 2880 gated 24.4 ->
// 13.6 us, 77 x 14336 -> 4096 22.1 -> 17.5.  There the launch, the first loads and the slices'
// sum are the larger part.

struct Gemm {
    const uint8_t *w0, *w1;   // the matrices of the wavefront's two tiles; backward: of the groups
    const uint8_t* x;
    const uint8_t* x_scales;  // kFp4
    unsigned x_stride;        // bytes
    unsigned x_second;        // kTransposed: bytes to the second matrix's values in a row
    unsigned segments;        // 16-byte segments of a row of x (of one matrix's part)
    unsigned groups, steps;   // of the packed form
    unsigned chunks, part;    // chunks of K, and how many a part has (kFp4: any number; else a
                              // multiple of 4, the loop's turn)
    unsigned tiles_n, tiles_m;
    Target out;
    float* partial;           // K slices: results go here
    unsigned slices;
    Stack stack;
};

constexpr int kStages = 4;

__device__ __forceinline__ void issue_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
    [&]<int... I>(std::integer_sequence<int, I...>) {
        (f.template operator()<I>(), ...);
    }(std::make_integer_sequence<int, N>{});
}

__device__ __forceinline__ i32x8 fp4_operand(const u4& c) {
    const i32x4 v{int(c.x), int(c.y), int(c.z), int(c.w)};
    return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}

// Tiles small enough for two workgroups to a compute unit (128 registers).
template <int TT, int OPS> constexpr bool shares_unit = TT == 1 || (TT == 2 && OPS != kFp4);

// Tiles of 32 rows whose epilogue takes both wavefront groups' sums out of LDS at once, 64 KB.
template <int TT, int OUT> constexpr bool whole_epilogue = TT == 1 && of_linear(OUT);

template <int TT, bool SPLIT, int OPS, int OUT>
__global__ __launch_bounds__(512, (shares_unit<TT, OPS> ? 4 : 2)) void gemm_kernel(Gemm a) {
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr int GROUPS = 2, kWaves = 4 * GROUPS, kStageBytes = TT * 8192;
    const unsigned lane = threadIdx.x % 64, h = lane / 32;
    const unsigned wave = uniform(threadIdx.x / 64);
    const unsigned rg = wave % 4, kg = wave / 4;

    // neighbouring tiles on one XCD (workgroups go round the eight of them), its matrix rows'
    // tiles over all rows of x in turn
    // (the experts': in turn, each its tiles over all of its rows, on the same terms)
    constexpr unsigned kRows = SPLIT ? TT * 32 : TT * 64;
    unsigned tiles = a.tiles_n * a.tiles_m;
    const unsigned xcd = blockIdx.x % 8;
    size_t expert = 0;
    unsigned tile_m, tile_n, slice = blockIdx.y;
    unsigned spot = 0;  // the experts' tile among all of them
    if constexpr (of_experts(OUT)) {
        // (whole tiles first, then the halves, so that what is left at a launch's end is small: an
        // XCD has its share of either: 2048 rows of 32 experts of 2880 x 2880 gated 91 us against
        // 97, 4096 rows 146 against 156; all K slices before the workgroups that have no tile, or
        // two share a compute unit while others are idle: gated backward of 40 rows of 8 experts,
        // 5888 -> 1120 in six slices 22 us against 28)
        const Tiles<kRows, (TT > 1)> list(a.stack, a.out.m);
        const ExpertsItem item =
            experts_item(blockIdx.x, list.whole(), list.halves(), a.tiles_n, a.slices);
        const auto p = list.of(item.tile / a.tiles_n, item.half);
        if (!item.there || !p.tiles) [[unlikely]]
            return;
        slice = item.slice;
        const unsigned within = item.tile - p.before * a.tiles_n;
        const unsigned first = p.first + within % p.tiles * kRows;
        spot = (item.half ? list.whole() : 0) + p.before + within % p.tiles;
        if (a.slices > 1 && !has_partials(spot, a.tiles_m)) [[unlikely]]
            return;  // (offsets that decrease, which no call may have)
        tile_m = 0;
        tile_n = within / p.tiles;
        move_to<OUT>(a.out, p.expert, first, min(p.end - first, kRows));
        a.x += size_t(first) * a.x_stride;
        expert = p.expert;
    } else {
        const unsigned tile = xcd * (tiles / 8) + min(xcd, tiles % 8) + blockIdx.x / 8;
        tile_m = tile % a.tiles_m, tile_n = tile / a.tiles_m;
    }
    const unsigned G = tile_n * 4 + rg;  // the wavefront's pair of tiles

    // this wavefront group's part of K, in chunks
    // (the experts' products with an epilogue take parts of whole half turns, two chunks: K of 768
    // is 6 + 6 chunks in place of 8 + 4, 4096 rows over 128 experts of 768 -> 2048 160 -> 145 us;
    // the others' longer turns gain less than the branch costs them, 3 to 15 %)
    constexpr bool kHalfTurns = OUT == kOutExpertsLinear;
    constexpr bool kTwoParts = SPLIT && (OPS != kTransposed || of_one_backward(OUT));
    const auto part_of = [&](unsigned set) {
        return kTwoParts ? slice * 2 + set : slice;
    };
    const unsigned begin = min(a.chunks, part_of(kg) * a.part);
    const unsigned end = min(a.chunks, begin + a.part);

    // x: rows past the last are the last one again (such rows' results are not stored);
    // segments past the part's end, or the row's, read as zeros
    const unsigned first_row = tile_m * kRows;
    const unsigned rows = min(kRows, a.out.m - first_row);
    // (a tile of the experts' that holds one of its two halves multiplies one)
    const bool both = rows > 32;
    const auto xs = buffer(a.x + size_t(first_row) * a.x_stride,
                           (rows - 1) * a.x_stride + a.x_second * (OPS == kTransposed) +
                               a.segments * 16);
    int x_at[TT];            // this lane's offset in chunk 0 of its part
    unsigned x_limit[TT];    // chunks * 8 it may read, counted from its segment
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        const unsigned u = j * kWaves + wave;  // this instruction's eight rows
        const unsigned set = SPLIT ? u / (4 * TT) : 0;
        const unsigned place = (SPLIT ? u % (4 * TT) : u) * 8 + lane / 8;
        const unsigned row = min(place, rows - 1);
        const unsigned seg = (lane % 8) ^ (place / 2 % 8);
        const unsigned b = min(a.chunks, part_of(set) * a.part);
        const unsigned e = min(a.segments, min(a.chunks, b + a.part) * 8);
        const unsigned from = b * 8 + seg;
        x_at[j] = int(row * a.x_stride + from * 16 +
                      (OPS == kTransposed && set ? a.x_second : 0));
        // (the experts' tiles are seldom full: rows past the last are zeros)
        x_limit[j] = e > from && (!of_experts(OUT) || place < rows) ? e - from : 0;
    }
    // kFp4: the scales of four chunks are 32 bytes of a row, copied as the nine dwords that
    // hold them (a row's bytes start anywhere; the buffer ends with the dword of the last one)
    // into 40 bytes of LDS: read by single chunks, each row's line would come four times
    constexpr int kScaleRows = GROUPS * TT * 32;
    constexpr int kScaleBytes = OPS == kFp4 ? kScaleRows * 40 : 0;
    constexpr int kScaleCopies = (kScaleBytes / 256 + kWaves - 1) / kWaves;
    const unsigned x_blocks = a.segments;  // scale bytes of a row: a segment is 32 values
    const size_t scales_from = size_t(first_row) * x_blocks;
    const unsigned odd = unsigned(scales_from % 4);
    const auto xscales = buffer(a.x_scales + (scales_from - odd),
                                OPS == kFp4 ? (odd + rows * x_blocks + 3) / 4 * 4 : 0);
    int scale_at[kScaleCopies + 1];
    unsigned scale_to[kScaleCopies + 1];
#pragma unroll
    for (int j = 0; j < kScaleCopies; ++j) {
        // (the last round's spare wavefronts repeat its last copy)
        const unsigned copy = min(j * kWaves + wave, unsigned(kScaleBytes / 256 - 1));
        const unsigned place = (copy * 64 + lane) / 10, dword = (copy * 64 + lane) % 10;
        const unsigned set = SPLIT ? place / (TT * 32) : 0;
        const unsigned row = min(SPLIT ? place % (TT * 32) : place, rows - 1);
        const unsigned from = odd + row * x_blocks + min(a.chunks, part_of(set) * a.part) * 8;
        scale_at[j] = int(from / 4 * 4 + dword * 4);
        scale_to[j] = uniform(kStages * kStageBytes + copy * 256);
    }
    auto stage_scales = [&](unsigned chunk, unsigned slot) {  // of the four chunks from `chunk`
#pragma unroll
        for (int j = 0; j < kScaleCopies; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                xscales,
                (__attribute__((address_space(3))) void*)(lds + scale_to[j] + slot * kScaleBytes),
                4, scale_at[j] + int(chunk * 8), 0, 0, 0);
        issue_order();
    };
    auto stage = [&](unsigned chunk, unsigned slot) {  // chunk of the part
        uint8_t* to = lds + slot * kStageBytes;
#pragma unroll
        for (int j = 0; j < TT; ++j) {
            const int at = chunk * 8 < x_limit[j] ? x_at[j] + int(chunk * 128) : kOutside;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                xs, (__attribute__((address_space(3))) void*)(to + (j * kWaves + wave) * 1024),
                16, at, 0, 0, 0);
        }
        issue_order();
    };

    // weights: buffers that end with the part, so that steps past it are zero codes
    constexpr unsigned kStepsPerChunk = OPS == kFp4 ? 4 : 1;
    constexpr unsigned kStepBytes = OPS == kTransposed ? 2048 : 1024;
    // (in scalar registers, or every load would loop over its buffer's possible values)
    const unsigned end_step = uniform(min(a.steps, end * kStepsPerChunk));
    const unsigned begin_step = uniform(begin * kStepsPerChunk);
    // (a part of nothing begins where K ends, within four steps' scales: zero codes times another
    // row's scale there would be NaN where that is)
    const bool some = begin_step < end_step;
    const unsigned scale_groups = (a.steps + 3) / 4;
    __amdgpu_buffer_rsrc_t codes_buf[2], scales_buf[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const bool second =
            of_one_backward(OUT) ? false : OPS == kTransposed ? kg != 0 : t != 0;
        const uint8_t* w = second ? a.w1 : a.w0;
        const unsigned group = OPS == kTransposed || of_gated(OUT) ? G : 2 * G + t;
        const bool there = group < a.groups;
        const size_t g = there ? group : 0;
        const uint8_t* s = w + size_t(a.groups) * a.steps * kStepBytes;
        if constexpr (of_experts(OUT)) {
            s = w + a.stack.experts * a.stack.code_bytes + expert * a.stack.scale_bytes;
            w += expert * a.stack.code_bytes;
        }
        codes_buf[t] = buffer(w + g * a.steps * kStepBytes, there ? end_step * kStepBytes : 0);
        if constexpr (OPS == kTransposed)
            scales_buf[t] = buffer(s + g * a.steps * 128, there ? end_step * 128 : 0);
        else
            scales_buf[t] =
                buffer(s + g * scale_groups * 256, there && some ? scale_groups * 256 : 0);
    }
    // steps (registers for two are left, or several workgroups share a compute unit)
    constexpr int kAhead =
        OPS == kFp4 ? 4 : OPS == kTransposed || shares_unit<TT, OPS> ? 2 : 4;
    struct Codes {
        u4 w[2];
        u4 s[OPS == kTransposed ? 2 : 1];
    };
    auto load_codes = [&](unsigned step, Codes& c) {
        if constexpr (OPS == kTransposed) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                c.w[t] = load_b128(codes_buf[0], int(step * 2048 + t * 1024 + lane * 16));
#pragma unroll
            for (int t = 0; t < 2; ++t)
                c.s[t] = load_b128(scales_buf[0],
                                   int(step * 128 + (2 * h + (lane % 32) / 16) * 32 + 16 * t));
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                c.w[t] = load_b128(codes_buf[t], int(step * 1024 + lane * 16));
        }
        issue_order();
    };
    struct Scales {
        unsigned w[2];
    };
    // Scales of the four steps from `step` (a multiple of 4).
    auto load_scales = [&](unsigned step, Scales& s) {
        if constexpr (OPS != kTransposed) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                s.w[t] = __builtin_amdgcn_raw_buffer_load_b32(
                    scales_buf[t], int(step * 64 + lane * 4), 0, 0);
        }
        issue_order();
    };

    f32x16 acc[2][TT];
#pragma unroll
    for (int t = 0; t < TT; ++t)
        acc[0][t] = acc[1][t] = f32x16{};

    // A wavefront's loads return in order.  Chunk c's copies were issued three chunks ago; the
    // copies of the two chunks after it, the weights of three chunks and their scales were
    // issued behind them, so a wait for all but that many is a wait for the chunk, and the
    // barrier makes it everyone's.  The first three chunks' copies are issued before the loop,
    // and only kAhead steps of weights behind them: kBehindFirst loads lie behind chunk 0's.
    constexpr int kStepLoads = OPS == kTransposed ? 4 : 2;
    constexpr int kCodeLoads = kStepLoads * int(kStepsPerChunk);
    constexpr int kScaleLoads = OPS == kTransposed ? 0 : 2;  // of four steps
    constexpr int kBehindFirst = 2 * TT + kScaleLoads + kAhead * kStepLoads;
    auto arrive = [&]<int BEHIND>() {
        static_assert(BEHIND < 64, "vmcnt holds six bits");
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(BEHIND) : "memory");
        __builtin_amdgcn_s_barrier();
        issue_order();
    };
    const uint8_t* x_lane = lds + kg * (TT * 4096) + (lane % 32) * 128;
    auto x_operand = [&](const uint8_t* buf, int t, unsigned seg) {
        return *reinterpret_cast<const u4*>(buf + t * 4096 + ((seg ^ (lane / 2 % 8)) * 16));
    };

    // operands are read (and weights decoded) a step ahead of their products where one
    // workgroup has the compute unit, at their step where two share it
    constexpr int kBuffers = shares_unit<TT, OPS> ? 1 : 2;
    Codes codes[kAhead];
    Scales scales, next;
    // (parts that are no whole turns may begin within a dword's four steps: two dwords give one)
    const unsigned shift = kHalfTurns ? begin_step % 4 : 0, scale_step = begin_step - shift;
    Scales after, shifted;
    // the x operands of a chunk's step S, and (bf16) the chunk's weights of it
    auto read_x = [&]<int S>(const uint8_t* buf, u4 (&v)[TT]) {
#pragma unroll
        for (int t = 0; t < TT; ++t)
            v[t] = x_operand(buf, t, OPS == kFp4 ? 2 * S + h : 4 * h + S);
    };
    auto decode_w = [&]<int C, int S>(bf16x8 (&v)[2]) {
        if constexpr (OPS == kTransposed) {
            const unsigned cw[2] = {codes[C % kAhead].w[S / 2][2 * (S % 2)],
                                    codes[C % kAhead].w[S / 2][2 * (S % 2) + 1]};
            const unsigned sw[2] = {codes[C % kAhead].s[S / 2][2 * (S % 2)],
                                    codes[C % kAhead].s[S / 2][2 * (S % 2) + 1]};
            decode8_pair(cw, sw, v[0], v[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                v[i] = decode8(codes[C % kAhead].w[i][S],
                               scale_of(kHalfTurns ? shifted.w[i] : scales.w[i], C));
        }
    };
    issue_order();
    if constexpr (OPS == kFp4)
        stage_scales(0, 0);
    stage(0, 0);
    stage(1, 1);
    stage(2, 2);
    load_scales(scale_step, scales);
    if constexpr (kHalfTurns)
        load_scales(scale_step + 4, after);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        load_codes(begin_step + i, codes[i]);

    if constexpr (OPS == kFp4) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the first turn's loads are fewer)
        // (32 rows on, a row's bytes start the same)
        const unsigned scale_shift = (odd + lane % 32 * x_blocks) % 4;
        for (unsigned c0 = 0; c0 < a.part; c0 += 4) {
            static_for<4>([&]<int C>() {
                // (the next four chunks' scales go out ahead of chunk 0 of them)
                constexpr int kScalesBehind = C == 2 || C == 3 ? kScaleCopies : 0;
                arrive.template operator()<2 * TT + kScalesBehind + 3 * kCodeLoads + 4>();
                const uint8_t* buf = x_lane + C * kStageBytes;
                Scales& now = C % 2 ? next : scales;
                load_scales(begin_step + 4 * (c0 + C + 1), C % 2 ? scales : next);
                const unsigned group = c0 / 4 % 2;
                if constexpr (C == 1)
                    stage_scales(c0 + 4, 1 - group);
                stage(c0 + C + 3, (C + 3) % kStages);
                // (chunks past the part's end multiply nothing, but every load is issued)
                const bool active = c0 + C < a.part;
                // a row's eight scales, those past its end (the next row's, or none) as zero;
                // the lane's half has every other one
                const unsigned block = (begin + c0 + C) * 8;
                const unsigned there = x_blocks - min(x_blocks, block);
                unsigned xs_now[TT];
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const auto* at = reinterpret_cast<const unsigned*>(
                        lds + kStages * kStageBytes + group * kScaleBytes +
                        (kg * (TT * 32) + t * 32 + lane % 32) * 40 + C * 8);
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    uint64_t bytes =
                        uint64_t(__builtin_amdgcn_alignbyte(at[2], v.y, scale_shift)) << 32 |
                        __builtin_amdgcn_alignbyte(v.y, v.x, scale_shift);
                    if (there < 8)
                        bytes &= (uint64_t(1) << (8 * there)) - 1;
                    xs_now[t] = __builtin_amdgcn_perm(unsigned(bytes >> 32), unsigned(bytes),
                                                      h ? 0x07050301u : 0x06040200u);
                }
                u4 xv[kBuffers][TT];
                if constexpr (kBuffers == 2)
                    read_x.template operator()<0>(buf, xv[0]);
                static_for<4>([&]<int S>() {
                    if (active) {
                        if constexpr (S + kBuffers < 5)
                            read_x.template operator()<S + kBuffers - 1>(
                                buf, xv[(S + kBuffers - 1) % kBuffers]);
                        if constexpr (kBuffers == 2)
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int t = 0; t < TT; ++t)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                acc[i][t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                                    fp4_operand(codes[S].w[i]), fp4_operand(xv[S % kBuffers][t]),
                                    acc[i][t], 4, 4, S, int(now.w[i]), S, int(xs_now[t]));
                    }
                    issue_order();
                    load_codes(begin_step + 4 * (c0 + C + 1) + S, codes[S]);
                });
            });
        }
    } else {
        // scales are loaded in chunk 0 of four, which is one of the three behind the others
        constexpr int kBehind = 2 * TT + 3 * kCodeLoads;
        // (the first turn's chunks 1 and 2: what the loop issued for the chunks before them too)
        static_assert(kBehindFirst + kCodeLoads + kScaleLoads >= kBehind + kScaleLoads &&
                          kBehindFirst + 2 * kCodeLoads + kScaleLoads >= kBehind + kScaleLoads,
                      "a wait of the first turn counts loads that were not issued");
        if constexpr (kBehindFirst < kBehind)  // (kTransposed: 8 loads of weights, not 12)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kBehindFirst) : "memory");
        for (unsigned c0 = 0; c0 < a.part; c0 += 4) {
            static_for<4>([&]<int C>() {
                if constexpr (kHalfTurns && C >= 2)
                    if (c0 + 2 >= a.part) [[unlikely]]
                        return;
                arrive.template operator()<kBehind + (C == 0 ? 0 : kScaleLoads)>();
                const uint8_t* buf = x_lane + C * kStageBytes;
                stage(c0 + C + 3, (C + 3) % kStages);
                if constexpr (C == 0)
                    load_scales(scale_step + c0 + (kHalfTurns ? 8 : 4), next);
                if constexpr (C == 0 && kHalfTurns)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        shifted.w[i] = __builtin_amdgcn_alignbyte(after.w[i], scales.w[i], shift);
                u4 xv[kBuffers][TT];
                bf16x8 wv[kBuffers][2];
                if constexpr (kBuffers == 2) {
                    read_x.template operator()<0>(buf, xv[0]);
                    decode_w.template operator()<C, 0>(wv[0]);
                }
                static_for<4>([&]<int S>() {
                    if constexpr (S + kBuffers < 5)
                        read_x.template operator()<S + kBuffers - 1>(
                            buf, xv[(S + kBuffers - 1) % kBuffers]);
                    if constexpr (kBuffers == 2)
                        __builtin_amdgcn_sched_barrier(0);
                    if constexpr (S + kBuffers < 5)
                        decode_w.template operator()<C, S + kBuffers - 1>(
                            wv[(S + kBuffers - 1) % kBuffers]);
#pragma unroll
                    for (int t = 0; t < TT; ++t) {
                        if (of_experts(OUT) && t > 0 && !both)
                            continue;
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            acc[i][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                                wv[S % kBuffers][i],
                                __builtin_bit_cast(bf16x8, xv[S % kBuffers][t]),
                                acc[i][t], 0, 0, 0);
                    }
                });
                issue_order();
                load_codes(begin_step + c0 + C + kAhead, codes[C % kAhead]);
            });
            scales = kHalfTurns ? after : next;
            after = next;
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no copy outlives the loop
    __syncthreads();

    // one tile of rows: both groups' sums meet in LDS as they leave, and each takes half the rows
    // (as below, the first group would do all of it: 333 rows of 2880 -> 2880 with bias, GELU and
    // residual 16.5 us against 14.1; the backward pass's, which only rounds, lost 4 %)
    if constexpr (whole_epilogue<TT, OUT>) {
        if (!a.partial) {
            const unsigned T = first_row / 32;
            float bias[8], residual[2][8];
            ask_for<16>(a.out, G, T, 16 * kg, bias, residual);
            uint8_t* patch = lds + rg * (2 * kWidePatchBytes);
            spread_wide(patch + kg * kWidePatchBytes, acc[0][0], acc[1][0]);
            __syncthreads();
            store_wide<16, 2>(a.out, G, T, 16 * kg, patch, patch + kWidePatchBytes, bias,
                              residual);
            return;
        }
    }

    // SPLIT: the first group finishes the first kOwn tiles and is handed the second one's sums
    // of them, and the other way round
    constexpr int kOwn = SPLIT ? (TT + 1) / 2 : TT, kOther = TT - kOwn;
    if constexpr (SPLIT) {
        auto* meet = reinterpret_cast<f32x4*>(lds) + rg * (TT * 512) + lane;
        auto hand = [&]<int FROM, int COUNT>() {
#pragma unroll
            for (int t = FROM; t < FROM + COUNT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        meet[((t * 2 + i) * 4 + j) * 64] = quad_of(acc[i][t], j);
        };
        auto add = [&]<int FROM, int COUNT>() {  // (kept from place 0 on)
#pragma unroll
            for (int t = 0; t < COUNT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f32x4 v = meet[(((FROM + t) * 2 + i) * 4 + j) * 64];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[i][t][4 * j + e] = acc[i][FROM + t][4 * j + e] + v[e];
                    }
        };
        if (kg)
            hand.template operator()<0, kOwn>();
        else
            hand.template operator()<kOwn, kOther>();
        __syncthreads();
        if (kg)
            add.template operator()<kOwn, kOther>();
        else
            add.template operator()<0, kOwn>();
    }
    // (SPLIT: LDS that only this wavefront read from)
    uint8_t* patch = lds + (SPLIT ? (rg * TT + (kg ? kOwn : 0)) * 8192 : wave * kPatchBytes);
    const unsigned own = SPLIT && kg ? kOther : kOwn;
    if constexpr (OUT == kOutExpertsGated) {  // (n % 32 == 0)
        const unsigned c = 32 * G + 4 * h;
        if (a.out.e.bias && !a.partial && 32 * G < a.out.n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float bg[4], bu[4];
                load_f32(a.out.e.bias, c + 8 * j, a.out.n, bg);
                load_f32(a.out.e.bias_up, c + 8 * j, a.out.n, bu);
#pragma unroll
                for (int t = 0; t < kOwn; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[0][t][4 * j + e] += bg[e];
                        acc[1][t][4 * j + e] += bu[e];
                    }
            }
        }
    }
    if constexpr (of_gated(OUT)) {
        if (!a.partial) {
            uint8_t* shared = lds + kg * kGatedPatch;
            const unsigned from = first_row / 32 + kg * (SPLIT ? kOwn : TT);
            __syncthreads();
#pragma unroll
            for (int t = 0; t < kOwn; ++t) {
                const bool mine = t < int(own) && (from + t) * 32 < a.out.m;
                if (mine)
                    gather_gated<OUT>(a.out, shared, rg, lane % 32, h, acc[0][t], acc[1][t]);
                __syncthreads();
                if (mine)
                    store_gated(a.out, shared, rg * 64 + lane, tile_n * 128, from + t);
                __syncthreads();
            }
            return;
        }
    }
    const unsigned first_tile =
        (first_row / 32) + kg * (SPLIT ? kOwn : TT);  // of 32 rows of x, the wavefront's first
#pragma unroll
    for (int t = 0; t < kOwn; ++t) {
        if (t >= int(own))
            break;
        const unsigned T = first_tile + t;
        if (a.partial) {
            if (T < (a.out.m + 31) / 32) {
                auto* to = reinterpret_cast<f32x4*>(
                               a.partial + (of_experts(OUT)
                                                ? partial_tile(slice, G, spot, T, a.tiles_n, TT,
                                                               a.tiles_m)
                                                : (size_t(slice) * (a.tiles_n * 4) + G) *
                                                          ((a.out.m + 31) / 32) + T) *
                                               kTileFloats) +
                           lane;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        to[(i * 4 + j) * 64] = quad_of(acc[i][t], j);
            }
        } else if constexpr (!of_gated(OUT)) {
            store_tiles<OUT>(a.out, G, T, patch, acc[0][t], acc[1][t]);
        }
    }
}

// The K slices' partial results of one pair of tiles, summed in slice order: a wavefront
// takes one quad of rows (four of them all of a pair's; kept pre-activations in 8 bits
// need a row's 32 values together, so there one wavefront takes all).  Bound by reading the
// slices, which mostly lie in the caches: 5 slices of 96 x 4096 3.4 us, 2 of 1024 x 4096 7.2 us
// (42 MB in all, 5.8 TB/s).  (A last workgroup that sums in place of this launch has to make
// the others' partial results visible first: backward of 1024 rows 225 -> 299 us.)
template <int OUT, bool WHOLE>
__device__ __forceinline__ void finish_slices(const float* partial, unsigned slices, size_t pairs,
                                              size_t pair, unsigned G, unsigned T, unsigned j0,
                                              const Target& out) {
    const unsigned lane = threadIdx.x % 64;
    const auto* from = reinterpret_cast<const f32x4*>(partial + pair * kTileFloats) + lane;
    const size_t step = pairs * (kTileFloats / 4);
    constexpr int kQuads = WHOLE ? 4 : 1;
    const unsigned token = T * 32 + lane % 32, h = lane / 32;
    Added<4> added[2];
    if constexpr (of_linear(OUT))
#pragma unroll
        for (int i = 0; i < 2; ++i)
            added[i] = added4(out, token, 64 * G + 32 * i + 8 * j0 + 4 * h);
    f32x4 v[2][kQuads];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
            v[i][j] = from[(i * 4 + j0 + j) * 64];
#pragma unroll 4
    for (unsigned s = 1; s < slices; ++s)  // (loads of four slices in flight)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
                v[i][j] += from[s * step + (i * 4 + j0 + j) * 64];
    if constexpr (OUT == kOutExpertsGated) {
        if (out.e.bias && 32 * G < out.n) {  // (n % 32 == 0)
#pragma unroll
            for (int j = 0; j < kQuads; ++j) {
                const unsigned c = 32 * G + 8 * (j0 + j) + 4 * h;
                float bg[4], bu[4];
                load_f32(out.e.bias, c, out.n, bg);
                load_f32(out.e.bias_up, c, out.n, bu);
                v[0][j] += f32x4{bg[0], bg[1], bg[2], bg[3]};
                v[1][j] += f32x4{bu[0], bu[1], bu[2], bu[3]};
            }
        }
    }
    if constexpr (of_linear(OUT)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            finish4(out, token, 64 * G + 32 * i + 8 * j0 + 4 * h, v[i][0], added[i]);
    } else {
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
            store_quad<OUT>(out, G, token, h, j0 + j, v[0][j], v[1][j]);
    }
    if constexpr (WHOLE) {
        if (32 * G < out.n) {
            keep_q8(out, 32 * G, token, h, v[0]);
            keep_q8(out, out.n + 32 * G, token, h, v[1]);
        }
    }
}

template <int OUT, bool WHOLE>
__global__ __launch_bounds__(256) void reduce_kernel(const float* __restrict__ partial,
                                                     unsigned slices, size_t pairs,
                                                     unsigned row_tiles, Target out) {
    const size_t w = size_t(blockIdx.x) * 4 + threadIdx.x / 64;
    const size_t pair = WHOLE ? w : w / 4;
    if (pair >= pairs)
        return;
    finish_slices<OUT, WHOLE>(partial, slices, pairs, pair, unsigned(pair / row_tiles),
                              unsigned(pair % row_tiles), WHOLE ? 0 : unsigned(w % 4), out);
}

// The same for the experts' tiles of TT * 32 rows, of which there may be fewer than `spots`.
template <int TT, int OUT, bool WHOLE>
__global__ __launch_bounds__(256) void experts_reduce_kernel(const float* __restrict__ partial,
                                                             unsigned slices, size_t pairs,
                                                             unsigned spots, Stack stack,
                                                             Target out) {
    const size_t w = size_t(blockIdx.x) * 4 + threadIdx.x / 64;
    const size_t pair = WHOLE ? w : w / 4;
    if (pair >= pairs)
        return;
    const unsigned row_tile = uniform(unsigned(pair % (spots * TT)));
    const unsigned spot = row_tile / TT, T = row_tile % TT;
    const Tiles<TT * 32, (TT > 1)> list(stack, out.m);
    const bool half = spot >= list.whole();
    const unsigned number = half ? spot - list.whole() : spot;
    const auto p = list.of(number, half);
    const unsigned first = p.first + (number - p.before) * (half ? 0 : TT * 32);
    if (!p.tiles || first + T * 32 >= p.end)
        return;
    move_to<OUT>(out, p.expert, first, min(p.end - first, TT * 32u));
    finish_slices<OUT, WHOLE>(partial, slices, pairs, pair, unsigned(pair / (spots * TT)), T,
                              WHOLE ? 0 : unsigned(w % 4), out);
}

// ------------------------------------------------------------------ dg and du
//
// s = sigmoid(g): dg = dh * u * s * (1 + g * (1 - s)), du = dh * g * s.  One lane takes
// eight columns; the traffic is dh, the kept g and u, and the two results, each once.
// g and u come as bf16 [m][2n] or as 8-bit codes with a scale per 32.  dg and du leave as bf16,
// the operands of the product with the weights and what a framework's gradients of bf16
// activations are: dx is off by 2.3e-3 of its root mean square for it, 1.7e-3 being its own
// rounding.  (What the rounding leaves over, as a second bf16 operand, would double the matrix
// products, which are nine tenths of the pass: 207 us of 1024 rows to about 400.)  Bound by
// memory: 2048 x 14336 from codes 37 us (242 MB, 6.5 TB/s), 1024 rows from bf16 25 us (147 MB,
// 5.9 TB/s).

// CLAMPED: the clamped gate's: with c = min(g, 7), v = u between -7 and 7 and s = sigmoid(1.702 c),
// dg = dh (v + 1) s (1 + 1.702 c (1 - s)) where g is at most 7, du = dh c s where |u| is.

template <bool Q8, bool CLAMPED>
__global__ __launch_bounds__(256) void gate_grad_kernel(const uint16_t* __restrict__ dh,
                                                        size_t dh_stride, unsigned m, unsigned n,
                                                        const uint16_t* __restrict__ kept,
                                                        const int8_t* __restrict__ kept_q,
                                                        const float* __restrict__ kept_d,
                                                        uint16_t* __restrict__ dgu) {
    const unsigned eighths = n / 8;
    const size_t u = size_t(blockIdx.x) * 256 + threadIdx.x;
    if (u >= size_t(m) * eighths)
        return;
    const unsigned row = unsigned(u / eighths), c = unsigned(u % eighths) * 8;
    const u32x4 dv = load16(reinterpret_cast<const uint8_t*>(dh + size_t(row) * dh_stride + c));
    float g[8], up[8];
    const size_t at = size_t(row) * 2 * n + c;
    if constexpr (Q8) {
        const float dg = kept_d[at / 32], du = kept_d[(at + n) / 32];
        const uint2 gq = *reinterpret_cast<const uint2*>(kept_q + at);
        const uint2 uq = *reinterpret_cast<const uint2*>(kept_q + at + n);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            g[i] = float(int8_t((i < 4 ? gq.x : gq.y) >> (8 * (i % 4)))) * dg;
            up[i] = float(int8_t((i < 4 ? uq.x : uq.y) >> (8 * (i % 4)))) * du;
        }
    } else {
        const u32x4 gv = load16(reinterpret_cast<const uint8_t*>(kept + at));
        const u32x4 uv = load16(reinterpret_cast<const uint8_t*>(kept + at + n));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            g[2 * i] = __uint_as_float(gv[i] << 16);
            g[2 * i + 1] = __uint_as_float(gv[i] & 0xffff0000u);
            up[2 * i] = __uint_as_float(uv[i] << 16);
            up[2 * i + 1] = __uint_as_float(uv[i] & 0xffff0000u);
        }
    }
    float rg[8], ru[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float d = __uint_as_float(i % 2 ? dv[i / 2] & 0xffff0000u : dv[i / 2] << 16);
        if constexpr (CLAMPED) {
            const float c = clamp_above(g[i]), s = sigmoid_value(kSharp * c);
            rg[i] = g[i] > kClamp ? 0.f
                                  : d * (clamp_both(up[i]) + 1.0f) *
                                        (s * (1.0f + kSharp * c * (1.0f - s)));
            ru[i] = fabsf(up[i]) > kClamp ? 0.f : d * (c * s);
        } else {
            const float s =
                __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g[i]));
            rg[i] = d * up[i] * (s * (1.0f + g[i] * (1.0f - s)));
            ru[i] = d * (g[i] * s);
        }
    }
    *reinterpret_cast<u32x4*>(dgu + at) = u32x4{bf16_pair(rg[0], rg[1]), bf16_pair(rg[2], rg[3]),
                                                bf16_pair(rg[4], rg[5]), bf16_pair(rg[6], rg[7])};
    *reinterpret_cast<u32x4*>(dgu + at + n) =
        u32x4{bf16_pair(ru[0], ru[1]), bf16_pair(ru[2], ru[3]), bf16_pair(ru[4], ru[5]),
              bf16_pair(ru[6], ru[7])};
}

// dpre = dy act'(pre) of a product's activation, eight columns a lane (n % 8 == 0).  It leaves as
// bf16 for dg's and du's reasons (above): dx is off by 2.3e-3 of its root mean square, 1.7e-3 being
// its own rounding.  Bound by memory: 1024 x 14336 17 us (88 MB, 5.2 TB/s).
__global__ __launch_bounds__(256) void act_grad_kernel(const uint16_t* __restrict__ dy,
                                                       size_t dy_stride, unsigned m, unsigned n,
                                                       const uint16_t* __restrict__ kept, int act,
                                                       uint16_t* __restrict__ dpre) {
    const unsigned eighths = n / 8;
    const size_t u = size_t(blockIdx.x) * 256 + threadIdx.x;
    if (u >= size_t(m) * eighths)
        return;
    const unsigned row = unsigned(u / eighths), c = unsigned(u % eighths) * 8;
    float d[8], v[8];
    load_bf16(dy + size_t(row) * dy_stride, c, n, d);
    load_bf16(kept + size_t(row) * n, c, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        d[i] *= act_slope(v[i], act);
    store_bf16(dpre + size_t(row) * n, c, n, d);
}

// ------------------------------------------------------------------ launches

constexpr size_t kMaxRows = size_t(1) << 20, kMaxK = size_t(1) << 20, kMaxN = size_t(1) << 24;

template <int TT, bool SPLIT, int OPS, int OUT>
int launch_gemm(const Gemm& a, const Plan& p, hipStream_t st) {
    const auto f = gemm_kernel<TT, SPLIT, OPS, OUT>;
    constexpr int kLds =
        whole_epilogue<TT, OUT> ? 8 * kWidePatchBytes
                                : kStages * TT * 8192 + (OPS == kFp4 ? 2 * TT * 64 * 40 : 0);
    if constexpr (kLds > 64 * 1024) {
        static std::atomic<uint64_t> configured{0};  // devices whose attribute is set
        int device = 0;
        KDQ_HIP(hipGetDevice(&device));
        const uint64_t bit = uint64_t(1) << (device % 64);
        if (device >= 64 || !(configured.load(std::memory_order_relaxed) & bit)) {
            KDQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(f),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
            configured.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    // (the experts': p.tiles_m is the most that they may have, and eight XCDs' shares of two kinds
    // are rounded up)
    const dim3 grid = of_experts(OUT) ? dim3(p.tiles_n * p.tiles_m * p.slices + 16)
                                      : dim3(p.tiles_n * p.tiles_m, p.slices);
    hipLaunchKernelGGL(f, grid, dim3(512), kLds, st, a);
    KDQ_HIP(hipGetLastError());
    return KDQ_OK;
}

template <int TT, int OUT>
int run_experts_reduce(const Gemm& a, const Plan& p, hipStream_t st) {
    const size_t pairs = size_t(p.tiles_n) * 4 * p.tiles_m * TT;
    const auto launch = [&](auto kernel, size_t blocks) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, st, a.partial, p.slices,
                           pairs, p.tiles_m, a.stack, a.out);
        KDQ_HIP(hipGetLastError());
        return int(KDQ_OK);
    };
    if constexpr (OUT == kOutExpertsGated)
        if (a.out.kept_q)
            return launch(experts_reduce_kernel<TT, OUT, true>, ceil_div(pairs, 4));
    return launch(experts_reduce_kernel<TT, OUT, false>, pairs);
}

template <int OPS, int OUT> int launch_tall(const Gemm& a, const Plan& p, hipStream_t st) {
    if constexpr (of_experts(OUT))  // (no plan of theirs has such tiles)
        return KDQ_ERR_UNSUPPORTED;
    else
        return p.tt == 3 ? launch_gemm<3, true, OPS, OUT>(a, p, st)
                         : launch_gemm<4, true, OPS, OUT>(a, p, st);
}

template <int OUT> int run_reduce(const Gemm& a, const Plan& p, hipStream_t st) {
    const unsigned row_tiles = unsigned(ceil_div(a.out.m, 32));
    const size_t pairs = size_t(p.tiles_n) * 4 * row_tiles;
    bool whole = false;
    if constexpr (OUT == kOutGated)
        whole = a.out.kept_q != nullptr;
    if (whole) {
        if constexpr (OUT == kOutGated)
            hipLaunchKernelGGL((reduce_kernel<OUT, true>), dim3(unsigned(ceil_div(pairs, 4))),
                               dim3(256), 0, st, a.partial, p.slices, pairs, row_tiles, a.out);
    } else {
        hipLaunchKernelGGL((reduce_kernel<OUT, false>), dim3(unsigned(pairs)), dim3(256), 0, st,
                           a.partial, p.slices, pairs, row_tiles, a.out);
    }
    KDQ_HIP(hipGetLastError());
    return KDQ_OK;
}

template <int OPS, int OUT> int run_gemm(Gemm a, const Plan& p, void* workspace, hipStream_t st) {
    a.chunks = p.chunks;
    a.part = p.part;
    a.tiles_n = p.tiles_n;
    a.tiles_m = p.tiles_m;
    a.slices = p.slices;
    a.partial = p.slices > 1 ? static_cast<float*>(workspace) : nullptr;
    int rc;
    if (!p.split) {
        if constexpr (OPS == kFp4)
            rc = launch_gemm<4, false, OPS, OUT>(a, p, st);
        else
            return KDQ_ERR_UNSUPPORTED;
    } else {
        rc = p.tt == 1   ? launch_gemm<1, true, OPS, OUT>(a, p, st)
             : p.tt == 2 ? launch_gemm<2, true, OPS, OUT>(a, p, st)
                         : launch_tall<OPS, OUT>(a, p, st);
    }
    if (!rc && p.slices > 1) {
        if constexpr (of_experts(OUT))
            rc = p.tt == 1 ? run_experts_reduce<1, OUT>(a, p, st)
                           : run_experts_reduce<2, OUT>(a, p, st);
        else
            rc = run_reduce<OUT>(a, p, st);
    }
    return rc;
}

template <int R, int TB, bool GATED, bool FP4, bool STAGED, int OUT>
int launch_decode(Decode a, unsigned waves, hipStream_t st) {
    const unsigned tiles = GATED ? 2 * R : R;
    const unsigned row_bytes = FP4 ? a.k / 2 : a.k * 2;
    unsigned bytes = waves * tiles * TB * 1024;
    if (STAGED)
        bytes = std::max(bytes, std::min(a.out.m, 16u * TB) * staged_pitch(row_bytes));
    hipLaunchKernelGGL((decode_kernel<R, TB, GATED, FP4, STAGED, OUT>),
                       dim3(unsigned(ceil_div(a.out.n, 16 * R)),
                            unsigned(of_experts(OUT)
                                         ? most_tiles(a.out.m, a.stack.experts, 16 * TB)
                                         : ceil_div(a.out.m, 16 * TB))),
                       dim3(waves * 64), bytes, st, a);
    KDQ_HIP(hipGetLastError());
    return KDQ_OK;
}

// (x is read by every wavefront: through LDS a token's projections took as long)
template <bool GATED, int OUT>
int run_experts_decode(Decode a, const DecodeShape& s, hipStream_t st) {
    a.units = s.units;
    if constexpr (!GATED)
        if (s.wide)
            return launch_decode<2, 1, GATED, false, false, OUT>(a, s.waves, st);
    return launch_decode<1, 1, GATED, false, false, OUT>(a, s.waves, st);
}

template <int OPS, int OUT>
int run_experts_gemm(Gemm a, const ExpertsPlan& e, void* workspace, hipStream_t st) {
    Plan p{};
    p.split = true;
    p.tt = e.tt;
    p.tiles_n = unsigned(e.tiles_n);
    p.tiles_m = unsigned(e.most);
    p.slices = e.slices;
    p.chunks = e.chunks;
    p.part = e.part;
    return run_gemm<OPS, OUT>(a, p, workspace, st);
}

template <bool GATED, bool FP4, int OUT> int run_decode(Decode a, hipStream_t st) {
    const DecodeShape s = decode_shape(a.out.m, a.out.n, a.k, GATED, FP4, compute_units());
    a.units = s.units;
    if constexpr (FP4)
        if (s.tb == 4)
            return launch_decode<1, 4, GATED, FP4, false, OUT>(a, s.waves, st);
    if (s.tb == 2)
        return s.wide ? launch_decode<2, 2, GATED, FP4, false, OUT>(a, s.waves, st)
                      : launch_decode<1, 2, GATED, FP4, false, OUT>(a, s.waves, st);
    if (s.staged)
        return s.wide ? launch_decode<2, 1, GATED, FP4, true, OUT>(a, s.waves, st)
                      : launch_decode<1, 1, GATED, FP4, true, OUT>(a, s.waves, st);
    return s.wide ? launch_decode<2, 1, GATED, FP4, false, OUT>(a, s.waves, st)
                  : launch_decode<1, 1, GATED, FP4, false, OUT>(a, s.waves, st);
}

template <int TB> int launch_decode_t(const Decode& a, unsigned waves, hipStream_t st) {
    hipLaunchKernelGGL((decode_t_kernel<TB>),
                       dim3(a.out.n / 32, unsigned(ceil_div(a.out.m, 16 * TB))),
                       dim3(waves * 64), waves * 2 * TB * 1024, st, a);
    KDQ_HIP(hipGetLastError());
    return KDQ_OK;
}

int run_decode_t(Decode a, hipStream_t st) {
    const unsigned units = (a.k + 127) / 128;  // of each matrix
    const unsigned waves = 2 * (units <= 4 ? 1 : units <= 8 ? 2 : units <= 16 ? 4 : 8);
    a.units = unsigned(ceil_div(units, waves / 2));
    return a.out.m <= 16 ? launch_decode_t<1>(a, waves, st) : launch_decode_t<2>(a, waves, st);
}

// (a packing launch counts its threads, one per 16 bytes of codes or 4 of scales, in 32 bits)
constexpr size_t kMaxCodes = size_t(1) << 35;

bool packs(size_t rows, size_t cols) {
    return rows && cols && cols % 32 == 0 && rows <= kMaxN && cols <= kMaxK &&
           packed_form(rows, cols).code_bytes <= kMaxCodes;
}

bool packs_transposed(size_t rows, size_t cols) {
    return rows && cols && cols % 32 == 0 && rows <= kMaxK && cols <= kMaxK &&
           transposed_form(rows, cols).code_bytes <= kMaxCodes;
}

bool sizes_ok(size_t m, size_t n, size_t k) {
    return m <= kMaxRows && packs(n, k);
}

bool backward_sizes_ok(size_t m, size_t n, size_t k) {
    return m <= kMaxRows && n % 32 == 0 && n <= kMaxK / 2 && packs_transposed(n, k);
}

// Bytes of `rows` rows `stride` values apart, `cols` values of `size` bytes each.
size_t extent(size_t rows, size_t stride, size_t cols, size_t size) {
    return ((rows - 1) * stride + cols) * size;
}

constexpr size_t kMaxStride = size_t(1) << 21;  // 256 rows stay within a buffer's range

int check_workspace(size_t need, const void* workspace, size_t bytes) {
    if (!need)
        return KDQ_OK;
    if (!workspace || bytes < need)
        return KDQ_ERR_SCRATCH;
    return misaligned(workspace, 16) ? KDQ_ERR_ALIGNMENT : KDQ_OK;
}

int check_form(const Form& f, const void* blocks, const void* scales, const void* packed,
               size_t rows, size_t cols, size_t matrices = 1) {
    if (misaligned(blocks, 16) || misaligned(packed, 16))
        return KDQ_ERR_ALIGNMENT;
    const size_t bytes = matrices * (f.code_bytes + f.scale_bytes);
    if (overlaps(packed, bytes, blocks, matrices * rows * (cols / 2)) ||
        overlaps(packed, bytes, scales, matrices * rows * (cols / 32)))
        return KDQ_ERR_ALIAS;
    return KDQ_OK;
}

template <class K>
int launch_pack(K kernel, const Form& f, const uint8_t* blocks, const uint8_t* scales,
                size_t rows, size_t cols, uint8_t* packed, void* stream, size_t matrices = 1) {
    const size_t units = f.code_bytes / 16 + f.scale_bytes / 4;
    hipLaunchKernelGGL(kernel, dim3(unsigned(ceil_div(units, 256)), unsigned(matrices)),
                       dim3(256), 0, static_cast<hipStream_t>(stream), blocks, scales, rows, cols, f, packed);
    KDQ_HIP(hipGetLastError());
    return KDQ_OK;
}

int check_output(int type, const void* y, size_t y_stride, size_t m, size_t n) {
    if (type != KDQ_F32 && type != KDQ_BF16)
        return KDQ_ERR_UNSUPPORTED;
    if (y_stride < n || y_stride > (SIZE_MAX >> 4) / m)
        return KDQ_ERR_SHAPE;
    return misaligned(y, type == KDQ_F32 ? 4 : 2) ? KDQ_ERR_ALIGNMENT : KDQ_OK;
}
}  // namespace
}  // namespace kdq
