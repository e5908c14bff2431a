// MXFP4 quantisation and decoding of rows (include/kadan_amd.h).  The reference only
// decodes the format (IW/src/weights/quantization.cpp:79-99,193-205; IW =
// services/hikari/inference_worker).
#include "kdq_common.hpp"

namespace kdq {
namespace {

// Eight consecutive values as fp32 (exact); 16-byte aligned.
template <int TYPE> __device__ __forceinline__ void load8(const void* x, size_t at, float (&v)[8]) {
    if constexpr (TYPE == KDQ_F32) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(x) + at + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const u32x4 w = load16(reinterpret_cast<const uint8_t*>(x) + at * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned half = i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
            v[i] = TYPE == KDQ_BF16 ? __uint_as_float(half << 16) : half_hw(half);
        }
    }
}

__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = max(v, unsigned(quad_xor1(int(v))));
    return max(v, unsigned(quad_xor2(int(v))));
}

// Four lanes take the 32 values of a block, eight each, so that the reads and the code
// writes of a wavefront are whole lines.  The scale byte is the exponent field of the
// block's largest magnitude less 2 (E2M1's largest exponent), at least 0; the conversion
// rounds value / 2^(byte - 127) to the nearest code, ties to the even one, past 6 to 6
// (checked on the device around every tie, for the smallest and largest scales too).
// Bound by memory: 14336 x 4096 fp32 58 us (235 MB read, 31 written, 4.6 TB/s); a few rows by
// the launch (4 x 2880 2 us).
template <int TYPE, bool DENSE>
__global__ __launch_bounds__(256) void quantize_kernel(const void* __restrict__ x, size_t stride,
                                                       size_t eighths, unsigned per_row,
                                                       uint8_t* __restrict__ blocks,
                                                       uint8_t* __restrict__ scales,
                                                       unsigned* __restrict__ status) {
    const size_t u = size_t(blockIdx.x) * 256 + threadIdx.x;
    const bool there = u < eighths;  // (a block's four lanes together)
    float v[8] = {};
    if (there) {
        size_t at = u * 8;
        if constexpr (!DENSE)
            at = u / per_row * stride + u % per_row * 8;
        load8<TYPE>(x, at, v);
    }
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = quad_max(top);
    const unsigned field = top >> 23;
    const bool finite = field < 255;
    const unsigned byte = finite ? (field > 2 ? field - 2 : 0) : 255;
    const float scale = __uint_as_float(byte << 23);
    unsigned codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], scale, 3);
    if (!there)
        return;
    reinterpret_cast<unsigned*>(blocks)[u] = finite ? codes : 0u;
    if (u % 4 == 0)
        scales[u / 4] = uint8_t(byte);
    if (status && !finite)
        atomicOr(status, 1u);
}

template <int TYPE>
int launch_quantize(const void* x, size_t stride, size_t rows, size_t cols, uint8_t* blocks,
                    uint8_t* scales, unsigned* status, hipStream_t st) {
    const size_t eighths = rows * (cols / 8);
    const dim3 grid(unsigned((eighths + 255) / 256));
    if (stride == cols || rows == 1)
        hipLaunchKernelGGL((quantize_kernel<TYPE, true>), grid, dim3(256), 0, st, x, stride,
                           eighths, unsigned(cols / 8), blocks, scales, status);
    else
        hipLaunchKernelGGL((quantize_kernel<TYPE, false>), grid, dim3(256), 0, st, x, stride,
                           eighths, unsigned(cols / 8), blocks, scales, status);
    KDQ_HIP(hipGetLastError());
    return KDQ_OK;
}
}  // namespace
}  // namespace kdq

extern "C" int kdq_mxfp4_quantize(int type, const void* x, size_t x_stride, size_t rows,
                                  size_t cols, uint8_t* blocks, uint8_t* scales,
                                  unsigned* status, void* stream) {
    using namespace kdq;
    if (!x || !blocks || !scales || !rows || !cols)
        return KDQ_ERR_ARGUMENT;
    const size_t size = type == KDQ_F32 ? 4 : 2;
    if (type != KDQ_F32 && type != KDQ_F16 && type != KDQ_BF16)
        return KDQ_ERR_UNSUPPORTED;
    if (cols % 32 || cols > (size_t(1) << 31) || x_stride < cols || x_stride % 8 ||
        x_stride > (SIZE_MAX >> 4) / rows || rows * (cols / 8) > UINT32_MAX - 255)
        return KDQ_ERR_SHAPE;
    if (misaligned(x, 16) || misaligned(blocks, 4))
        return KDQ_ERR_ALIGNMENT;
    const size_t x_bytes = ((rows - 1) * x_stride + cols) * size;
    const size_t code_bytes = rows * (cols / 2), scale_bytes = rows * (cols / 32);
    if (overlaps(blocks, code_bytes, x, x_bytes) || overlaps(scales, scale_bytes, x, x_bytes) ||
        overlaps(blocks, code_bytes, scales, scale_bytes))
        return KDQ_ERR_ALIAS;
    const auto st = static_cast<hipStream_t>(stream);
    return type == KDQ_F32
               ? launch_quantize<KDQ_F32>(x, x_stride, rows, cols, blocks, scales, status, st)
           : type == KDQ_F16
               ? launch_quantize<KDQ_F16>(x, x_stride, rows, cols, blocks, scales, status, st)
               : launch_quantize<KDQ_BF16>(x, x_stride, rows, cols, blocks, scales, status, st);
}
