// Entry points of the MXFP4 dense layers (include/kadan_amd.h): argument checks, the choice of
// kernel (mxfp4_plan.hpp) and the launches of mxfp4_kernels.hpp.
#include "mxfp4_kernels.hpp"

using namespace kdq;

extern "C" size_t kdq_mxfp4_packed_bytes(size_t rows, size_t cols) {
    if (!packs(rows, cols))
        return 0;
    const Form f = packed_form(rows, cols);
    return f.code_bytes + f.scale_bytes;
}

extern "C" int kdq_mxfp4_pack(const uint8_t* blocks, const uint8_t* scales, size_t rows,
                              size_t cols, uint8_t* packed, void* stream) {
    if (!blocks || !scales || !packed || !rows || !cols)
        return KDQ_ERR_ARGUMENT;
    if (!kdq_mxfp4_packed_bytes(rows, cols))
        return KDQ_ERR_SHAPE;
    const Form f = packed_form(rows, cols);
    if (const int rc = check_form(f, blocks, scales, packed, rows, cols))
        return rc;
    return launch_pack(pack_kernel, f, blocks, scales, rows, cols, packed, stream);
}

extern "C" size_t kdq_mxfp4_packed_transposed_bytes(size_t rows, size_t cols) {
    if (!packs_transposed(rows, cols))
        return 0;
    const Form f = transposed_form(rows, cols);
    return f.code_bytes + f.scale_bytes;
}

extern "C" int kdq_mxfp4_pack_transposed(const uint8_t* blocks, const uint8_t* scales,
                                         size_t rows, size_t cols, uint8_t* packed,
                                         void* stream) {
    if (!blocks || !scales || !packed || !rows || !cols)
        return KDQ_ERR_ARGUMENT;
    if (!kdq_mxfp4_packed_transposed_bytes(rows, cols))
        return KDQ_ERR_SHAPE;
    const Form f = transposed_form(rows, cols);
    if (const int rc = check_form(f, blocks, scales, packed, rows, cols))
        return rc;
    return launch_pack(pack_t_kernel, f, blocks, scales, rows, cols, packed, stream);
}

extern "C" size_t kdq_mxfp4_product_workspace(size_t m, size_t n, size_t k, int quantized) {
    if (!m || !n || !k || !sizes_ok(m, n, k))
        return 0;
    return partial_bytes(plan_product(m, n, k, quantized != 0, compute_units()), m);
}

extern "C" size_t kdq_mxfp4_gated_workspace(size_t m, size_t n, size_t k, int kept) {
    if (!m || !n || !k || !sizes_ok(m, n, k) || n % 32)
        return 0;
    return partial_bytes(plan_gated(m, n, k, kept != 0, compute_units()), m);
}

extern "C" size_t kdq_mxfp4_gated_backward_workspace(size_t m, size_t n, size_t k) {
    if (!m || !n || !k || !backward_sizes_ok(m, n, k))
        return 0;
    return partial_bytes(plan_backward(m, n, k, compute_units()), m);
}

namespace kdq {
namespace {
template <int OPS> int product(Gemm g, const Plan& p, int type, void* workspace, hipStream_t st) {
    if (p.decode) {
        Decode d{g.w0, nullptr, g.x, g.x_scales, g.x_stride,
                 unsigned(OPS == kFp4 ? g.segments * 32 : g.segments * 8), g.steps, g.groups,
                 0, g.out};
        constexpr bool kQ = OPS == kFp4;
        return type == KDQ_F32 ? run_decode<false, kQ, kOutF32>(d, st)
                               : run_decode<false, kQ, kOutBf16>(d, st);
    }
    return type == KDQ_F32 ? run_gemm<OPS, kOutF32>(g, p, workspace, st)
                           : run_gemm<OPS, kOutBf16>(g, p, workspace, st);
}
}  // namespace
}  // namespace kdq

extern "C" int kdq_mxfp4_product(const uint16_t* x_bf16, size_t x_stride, size_t m,
                                 const uint8_t* packed, size_t n, size_t k, int type, void* y,
                                 size_t y_stride, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    if (!x_bf16 || !packed || !y || !m || !n || !k)
        return KDQ_ERR_ARGUMENT;
    if (!sizes_ok(m, n, k) || x_stride < k || x_stride % 8 || x_stride > kMaxStride)
        return KDQ_ERR_SHAPE;
    if (const int rc = check_output(type, y, y_stride, m, n))
        return rc;
    if (misaligned(x_bf16, 16) || misaligned(packed, 16))
        return KDQ_ERR_ALIGNMENT;
    const Range out[] = {{y, extent(m, y_stride, n, type == KDQ_F32 ? 4 : 2)},
                         {workspace, workspace_bytes}},
                in[] = {{x_bf16, extent(m, x_stride, k, 2)},
                        {packed, kdq_mxfp4_packed_bytes(n, k)}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    const Plan p = plan_product(m, n, k, false, compute_units());
    if (const int rc = check_workspace(partial_bytes(p, m), workspace, workspace_bytes))
        return rc;
    const Form f = packed_form(n, k);
    Gemm g{};
    g.w0 = g.w1 = packed;
    g.x = reinterpret_cast<const uint8_t*>(x_bf16);
    g.x_stride = unsigned(x_stride * 2);
    g.segments = unsigned(k / 8);
    g.groups = unsigned(f.groups);
    g.steps = unsigned(f.steps);
    g.out = {y, y_stride, unsigned(m), unsigned(n), nullptr, nullptr, nullptr};
    return product<kBf16>(g, p, type, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int kdq_mxfp4_product_quantized(const uint8_t* x_blocks, const uint8_t* x_scales,
                                           size_t m, const uint8_t* packed, size_t n, size_t k,
                                           int type, void* y, size_t y_stride, void* workspace,
                                           size_t workspace_bytes, void* stream) {
    if (!x_blocks || !x_scales || !packed || !y || !m || !n || !k)
        return KDQ_ERR_ARGUMENT;
    if (!sizes_ok(m, n, k))
        return KDQ_ERR_SHAPE;
    if (const int rc = check_output(type, y, y_stride, m, n))
        return rc;
    if (misaligned(x_blocks, 16) || misaligned(x_scales, 4) || misaligned(packed, 16))
        return KDQ_ERR_ALIGNMENT;
    const Range out[] = {{y, extent(m, y_stride, n, type == KDQ_F32 ? 4 : 2)},
                         {workspace, workspace_bytes}},
                in[] = {{x_blocks, m * (k / 2)},
                        {x_scales, m * (k / 32)},
                        {packed, kdq_mxfp4_packed_bytes(n, k)}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    const Plan p = plan_product(m, n, k, true, compute_units());
    if (const int rc = check_workspace(partial_bytes(p, m), workspace, workspace_bytes))
        return rc;
    const Form f = packed_form(n, k);
    Gemm g{};
    g.w0 = g.w1 = packed;
    g.x = x_blocks;
    g.x_scales = x_scales;
    g.x_stride = unsigned(k / 2);
    g.segments = unsigned(k / 32);
    g.groups = unsigned(f.groups);
    g.steps = unsigned(f.steps);
    g.out = {y, y_stride, unsigned(m), unsigned(n), nullptr, nullptr, nullptr};
    return product<kFp4>(g, p, type, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int kdq_mxfp4_gated(const uint16_t* x_bf16, size_t x_stride, size_t m,
                               const uint8_t* gate_packed, const uint8_t* up_packed, size_t n,
                               size_t k, uint16_t* h_bf16, size_t h_stride,
                               uint16_t* kept_bf16, int8_t* kept_q8, float* kept_scales,
                               void* workspace, size_t workspace_bytes, void* stream) {
    if (!x_bf16 || !gate_packed || !up_packed || !h_bf16 || !m || !n || !k ||
        (kept_bf16 && kept_q8) || !kept_q8 != !kept_scales)
        return KDQ_ERR_ARGUMENT;
    if (!sizes_ok(m, n, k) || n % 32 || x_stride < k || x_stride % 8 || x_stride > kMaxStride)
        return KDQ_ERR_SHAPE;
    if (const int rc = check_output(KDQ_BF16, h_bf16, h_stride, m, n))
        return rc;
    if (misaligned(x_bf16, 16) || misaligned(gate_packed, 16) || misaligned(up_packed, 16) ||
        misaligned(kept_bf16, 16) || misaligned(kept_q8, 16) || misaligned(kept_scales, 4))
        return KDQ_ERR_ALIGNMENT;
    const Range out[] = {{h_bf16, extent(m, h_stride, n, 2)},
                         {kept_bf16, 4 * m * n},
                         {kept_q8, 2 * m * n},
                         {kept_scales, m * n / 4},
                         {workspace, workspace_bytes}},
                in[] = {{x_bf16, extent(m, x_stride, k, 2)},
                        {gate_packed, kdq_mxfp4_packed_bytes(n, k)},
                        {up_packed, kdq_mxfp4_packed_bytes(n, k)}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    const Plan p = plan_gated(m, n, k, kept_bf16 || kept_q8, compute_units());
    if (const int rc = check_workspace(partial_bytes(p, m), workspace, workspace_bytes))
        return rc;
    const Form f = packed_form(n, k);
    const auto st = static_cast<hipStream_t>(stream);
    const Target t{h_bf16, h_stride, unsigned(m), unsigned(n), kept_bf16, kept_q8, kept_scales};
    if (p.decode)
        return run_decode<true, false, kOutBf16>(
            {gate_packed, up_packed, reinterpret_cast<const uint8_t*>(x_bf16), nullptr,
             unsigned(x_stride * 2), unsigned(k), unsigned(f.steps), unsigned(f.groups), 0, t},
            st);
    Gemm g{};
    g.w0 = gate_packed;
    g.w1 = up_packed;
    g.x = reinterpret_cast<const uint8_t*>(x_bf16);
    g.x_stride = unsigned(x_stride * 2);
    g.segments = unsigned(k / 8);
    g.groups = unsigned(f.groups);
    g.steps = unsigned(f.steps);
    g.out = t;
    return run_gemm<kBf16, kOutGated>(g, p, workspace, st);
}

extern "C" int kdq_mxfp4_gated_backward(const uint16_t* dh_bf16, size_t dh_stride, size_t m,
                                        const uint16_t* kept_bf16, const int8_t* kept_q8,
                                        const float* kept_scales, const uint8_t* gate_transposed,
                                        const uint8_t* up_transposed, size_t n, size_t k,
                                        uint16_t* dgu_bf16, uint16_t* dx_bf16, size_t dx_stride,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    if (!dh_bf16 || !gate_transposed || !up_transposed || !dgu_bf16 || !dx_bf16 || !m || !n ||
        !k || !kept_bf16 == !kept_q8 || !kept_q8 != !kept_scales)
        return KDQ_ERR_ARGUMENT;
    if (!backward_sizes_ok(m, n, k) || dh_stride < n || dh_stride % 8 ||
        dh_stride > kMaxStride || m * (n / 8) > UINT32_MAX - 255)
        return KDQ_ERR_SHAPE;
    if (const int rc = check_output(KDQ_BF16, dx_bf16, dx_stride, m, k))
        return rc;
    if (misaligned(dh_bf16, 16) || misaligned(gate_transposed, 16) ||
        misaligned(up_transposed, 16) || misaligned(kept_bf16, 16) || misaligned(kept_q8, 16) ||
        misaligned(kept_scales, 4) || misaligned(dgu_bf16, 16))
        return KDQ_ERR_ALIGNMENT;
    const size_t w_bytes = kdq_mxfp4_packed_transposed_bytes(n, k);
    const Range out[] = {{dgu_bf16, 4 * m * n},
                         {dx_bf16, extent(m, dx_stride, k, 2)},
                         {workspace, workspace_bytes}},
                in[] = {{dh_bf16, extent(m, dh_stride, n, 2)}, {kept_bf16, 4 * m * n},
                        {kept_q8, 2 * m * n},                  {kept_scales, m * n / 4},
                        {gate_transposed, w_bytes},            {up_transposed, w_bytes}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    const Plan p = plan_backward(m, n, k, compute_units());
    if (const int rc = check_workspace(partial_bytes(p, m), workspace, workspace_bytes))
        return rc;
    const auto st = static_cast<hipStream_t>(stream);
    const dim3 grid(unsigned(ceil_div(m * (n / 8), 256)));
    const auto kernel = kept_q8 ? gate_grad_kernel<true, false> : gate_grad_kernel<false, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, dh_bf16, dh_stride, unsigned(m), unsigned(n),
                       kept_bf16, kept_q8, kept_scales, dgu_bf16);
    KDQ_HIP(hipGetLastError());
    const Form f = transposed_form(n, k);
    const Target t{dx_bf16, dx_stride, unsigned(m), unsigned(k), nullptr, nullptr, nullptr};
    if (p.decode)
        return run_decode_t({gate_transposed, up_transposed,
                             reinterpret_cast<const uint8_t*>(dgu_bf16), nullptr,
                             unsigned(n * 4), unsigned(n), unsigned(f.steps), unsigned(f.groups),
                             0, t},
                            st);
    Gemm g{};
    g.w0 = gate_transposed;
    g.w1 = up_transposed;
    g.x = reinterpret_cast<const uint8_t*>(dgu_bf16);
    g.x_stride = unsigned(n * 4);
    g.x_second = unsigned(n * 2);
    g.segments = unsigned(n / 8);
    g.groups = unsigned(f.groups);
    g.steps = unsigned(f.steps);
    g.out = t;
    return run_gemm<kTransposed, kOutBackward>(g, p, workspace, st);
}
