// Entry points of the MXFP4 products with an epilogue, dense or of a mixture's experts, and of the
// experts' gated projection, with their backward passes (include/kadan_amd.h): argument checks,
// the choice of kernel (mxfp4_plan.hpp) and the launches of mxfp4_kernels.hpp.
#include "mxfp4_kernels.hpp"

using namespace kdq;

namespace kdq {
namespace {

bool experts_pack(size_t experts, size_t rows, size_t cols) {
    return experts && experts <= kMaxExperts && packs(rows, cols);
}

bool experts_pack_transposed(size_t experts, size_t rows, size_t cols) {
    return experts && experts <= kMaxExperts && packs_transposed(rows, cols);
}

size_t bytes_of(const Form& f, size_t matrices) {
    return matrices * (f.code_bytes + f.scale_bytes);
}

// Dense calls have no offsets and one matrix.
int check_experts(const int32_t* offsets, size_t experts) {
    if (!experts || (!offsets && experts != 1))
        return KDQ_ERR_ARGUMENT;
    if (experts > kMaxExperts)
        return KDQ_ERR_SHAPE;
    return misaligned(offsets, 4) ? KDQ_ERR_ALIGNMENT : KDQ_OK;
}

// Strides and alignment of bf16 inputs of m rows.
int check_input(const void* x, size_t stride, size_t cols) {
    if (stride < cols || stride % 8 || stride > kMaxStride)
        return KDQ_ERR_SHAPE;
    return misaligned(x, 16) ? KDQ_ERR_ALIGNMENT : KDQ_OK;
}

Stack stack_of(const int32_t* offsets, size_t experts, const Form& f) {
    return {offsets, unsigned(experts), f.code_bytes, f.scale_bytes};
}

size_t offset_bytes(const int32_t* offsets, size_t experts) {
    return offsets ? (experts + 1) * 4 : 0;
}

// (a launch's threads are counted in 32 bits)
bool launches(const ExpertsPlan& p) {
    return p.decode ? p.most <= 65535
                    : p.most * p.tiles_n * p.slices + 16 <= UINT32_MAX / 512 &&
                          (p.slices == 1 || p.tiles_n * 4 * p.most * p.tt <= UINT32_MAX / 256);
}

Gemm gemm_of(const uint8_t* w0, const uint8_t* w1, const uint16_t* x, size_t x_stride,
             size_t x_cols, const Form& f, const Target& out) {
    Gemm g{};
    g.w0 = w0;
    g.w1 = w1;
    g.x = reinterpret_cast<const uint8_t*>(x);
    g.x_stride = unsigned(x_stride * 2);
    g.segments = unsigned(x_cols / 8);
    g.groups = unsigned(f.groups);
    g.steps = unsigned(f.steps);
    g.out = out;
    return g;
}

Decode decode_of(const Gemm& g, size_t k) {
    return {g.w0,    g.w1,     g.x, nullptr, g.x_stride, unsigned(k), g.steps,
            g.groups, 0, g.out, g.stack};
}
}  // namespace
}  // namespace kdq

extern "C" size_t kdq_mxfp4_experts_packed_bytes(size_t experts, size_t rows, size_t cols) {
    return experts_pack(experts, rows, cols) ? bytes_of(packed_form(rows, cols), experts) : 0;
}

extern "C" int kdq_mxfp4_experts_pack(const uint8_t* blocks, const uint8_t* scales,
                                      size_t experts, size_t rows, size_t cols, uint8_t* packed,
                                      void* stream) {
    if (!blocks || !scales || !packed || !experts || !rows || !cols)
        return KDQ_ERR_ARGUMENT;
    if (!experts_pack(experts, rows, cols))
        return KDQ_ERR_SHAPE;
    const Form f = packed_form(rows, cols);
    if (const int rc = check_form(f, blocks, scales, packed, rows, cols, experts))
        return rc;
    return launch_pack(pack_kernel, f, blocks, scales, rows, cols, packed, stream, experts);
}

extern "C" size_t kdq_mxfp4_experts_packed_transposed_bytes(size_t experts, size_t rows,
                                                            size_t cols) {
    return experts_pack_transposed(experts, rows, cols)
               ? bytes_of(transposed_form(rows, cols), experts)
               : 0;
}

extern "C" int kdq_mxfp4_experts_pack_transposed(const uint8_t* blocks, const uint8_t* scales,
                                                 size_t experts, size_t rows, size_t cols,
                                                 uint8_t* packed, void* stream) {
    if (!blocks || !scales || !packed || !experts || !rows || !cols)
        return KDQ_ERR_ARGUMENT;
    if (!experts_pack_transposed(experts, rows, cols))
        return KDQ_ERR_SHAPE;
    const Form f = transposed_form(rows, cols);
    if (const int rc = check_form(f, blocks, scales, packed, rows, cols, experts))
        return rc;
    return launch_pack(pack_t_kernel, f, blocks, scales, rows, cols, packed, stream, experts);
}

extern "C" size_t kdq_mxfp4_linear_workspace(size_t m, size_t experts, size_t n, size_t k) {
    if (!experts)
        return kdq_mxfp4_product_workspace(m, n, k, 0);
    if (!m || !n || !k || experts > kMaxExperts || !sizes_ok(m, n, k))
        return 0;
    return partial_bytes(plan_experts(m, experts, n, k, false, false, compute_units()));
}

extern "C" int kdq_mxfp4_linear(const uint16_t* x_bf16, size_t x_stride, size_t m,
                                const int32_t* offsets, size_t experts, const uint8_t* packed,
                                size_t n, size_t k, const float* bias, int activation,
                                const void* residual, size_t residual_stride, int type, void* y,
                                size_t y_stride, uint16_t* kept_bf16, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (!x_bf16 || !packed || !y || !m || !n || !k)
        return KDQ_ERR_ARGUMENT;
    if (const int rc = check_experts(offsets, experts))
        return rc;
    if (!sizes_ok(m, n, k))
        return KDQ_ERR_SHAPE;
    if (activation < KDQ_ACT_NONE || activation > KDQ_ACT_GELU)
        return KDQ_ERR_UNSUPPORTED;
    if (const int rc = check_output(type, y, y_stride, m, n))
        return rc;
    if (residual)
        if (const int rc = check_output(type, residual, residual_stride, m, n))
            return rc;
    if (const int rc = check_input(x_bf16, x_stride, k))
        return rc;
    if (misaligned(packed, 16) || misaligned(bias, 4) || misaligned(kept_bf16, 2))
        return KDQ_ERR_ALIGNMENT;
    const Form f = packed_form(n, k);
    const size_t size = type == KDQ_F32 ? 4 : 2;
    // (y may be the residual itself: a lane reads what it then writes)
    const bool in_place = residual == y && residual_stride == y_stride;
    const Range out[] = {{y, extent(m, y_stride, n, size)},
                         {kept_bf16, 2 * m * n},
                         {workspace, workspace_bytes}},
                in[] = {{x_bf16, extent(m, x_stride, k, 2)},
                        {packed, bytes_of(f, experts)},
                        {bias, experts * n * 4},
                        {offsets, offset_bytes(offsets, experts)},
                        {in_place ? nullptr : residual, extent(m, residual_stride, n, size)}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    const auto st = static_cast<hipStream_t>(stream);
    Target t{y, y_stride, unsigned(m), unsigned(n), kept_bf16, nullptr, nullptr};
    t.e = {bias, nullptr, residual, residual_stride, activation, type == KDQ_F32};
    Gemm g = gemm_of(packed, packed, x_bf16, x_stride, k, f, t);
    if (offsets) {
        const ExpertsPlan p = plan_experts(m, experts, n, k, false, false, compute_units());
        if (!launches(p))
            return KDQ_ERR_SHAPE;
        if (const int rc = check_workspace(partial_bytes(p), workspace, workspace_bytes))
            return rc;
        g.stack = stack_of(offsets, experts, f);
        return p.decode
                   ? run_experts_decode<false, kOutExpertsLinear>(decode_of(g, k), p.shape, st)
                   : run_experts_gemm<kBf16, kOutExpertsLinear>(g, p, workspace, st);
    }
    const Plan p = plan_product(m, n, k, false, compute_units());
    if (const int rc = check_workspace(partial_bytes(p, m), workspace, workspace_bytes))
        return rc;
    return p.decode ? run_decode<false, false, kOutLinear>(decode_of(g, k), st)
                    : run_gemm<kBf16, kOutLinear>(g, p, workspace, st);
}

extern "C" size_t kdq_mxfp4_linear_backward_workspace(size_t m, size_t experts, size_t n,
                                                      size_t k) {
    if (!m || !n || !k || m > kMaxRows || experts > kMaxExperts || !packs_transposed(n, k))
        return 0;
    const size_t cus = compute_units();
    return experts ? partial_bytes(plan_experts_backward(m, experts, n, k, false, cus))
                   : partial_bytes(plan_one_backward(m, n, k, cus), m);
}

extern "C" int kdq_mxfp4_linear_backward(const uint16_t* dy_bf16, size_t dy_stride, size_t m,
                                         const int32_t* offsets, size_t experts,
                                         const uint16_t* kept_bf16, int activation,
                                         const uint8_t* transposed, size_t n, size_t k,
                                         uint16_t* dpre_bf16, uint16_t* dx_bf16, size_t dx_stride,
                                         void* workspace, size_t workspace_bytes, void* stream) {
    const bool some = activation != KDQ_ACT_NONE;
    if (!dy_bf16 || !transposed || !dx_bf16 || !m || !n || !k || !kept_bf16 == some ||
        !dpre_bf16 == some)
        return KDQ_ERR_ARGUMENT;
    if (const int rc = check_experts(offsets, experts))
        return rc;
    if (activation < KDQ_ACT_NONE || activation > KDQ_ACT_GELU)
        return KDQ_ERR_UNSUPPORTED;
    if (m > kMaxRows || n % 8 || !packs_transposed(n, k) || m * (n / 8) > UINT32_MAX - 255)
        return KDQ_ERR_SHAPE;
    if (const int rc = check_output(KDQ_BF16, dx_bf16, dx_stride, m, k))
        return rc;
    if (const int rc = check_input(dy_bf16, dy_stride, n))
        return rc;
    if (misaligned(transposed, 16) || misaligned(kept_bf16, 2) || misaligned(dpre_bf16, 16))
        return KDQ_ERR_ALIGNMENT;
    const Form f = transposed_form(n, k);
    const Range out[] = {{dpre_bf16, 2 * m * n},
                         {dx_bf16, extent(m, dx_stride, k, 2)},
                         {workspace, workspace_bytes}},
                in[] = {{dy_bf16, extent(m, dy_stride, n, 2)},
                        {kept_bf16, 2 * m * n},
                        {offsets, offset_bytes(offsets, experts)},
                        {transposed, bytes_of(f, experts)}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    Plan p{};
    ExpertsPlan e{};
    if (offsets) {
        e = plan_experts_backward(m, experts, n, k, false, compute_units());
        if (!launches(e))
            return KDQ_ERR_SHAPE;
        if (const int rc = check_workspace(partial_bytes(e), workspace, workspace_bytes))
            return rc;
    } else {
        p = plan_one_backward(m, n, k, compute_units());
        if (const int rc = check_workspace(partial_bytes(p, m), workspace, workspace_bytes))
            return rc;
    }
    const auto st = static_cast<hipStream_t>(stream);
    if (some) {
        hipLaunchKernelGGL(act_grad_kernel, dim3(unsigned(ceil_div(m * (n / 8), 256))), dim3(256),
                           0, st, dy_bf16, dy_stride, unsigned(m), unsigned(n), kept_bf16,
                           activation, dpre_bf16);
        KDQ_HIP(hipGetLastError());
    }
    const Target t{dx_bf16, dx_stride, unsigned(m), unsigned(k), nullptr, nullptr, nullptr};
    Gemm g = gemm_of(transposed, transposed, some ? dpre_bf16 : dy_bf16, some ? n : dy_stride, n,
                     f, t);
    if (!offsets)
        return run_gemm<kTransposed, kOutOneBackward>(g, p, workspace, st);
    g.stack = stack_of(offsets, experts, f);
    return run_experts_gemm<kTransposed, kOutExpertsOneBackward>(g, e, workspace, st);
}

extern "C" size_t kdq_mxfp4_experts_gated_workspace(size_t m, size_t experts, size_t n, size_t k,
                                                    int kept) {
    if (!m || !n || !k || !experts || experts > kMaxExperts || !sizes_ok(m, n, k) || n % 32)
        return 0;
    return partial_bytes(plan_experts(m, experts, n, k, true, kept != 0, compute_units()));
}

extern "C" size_t kdq_mxfp4_experts_gated_backward_workspace(size_t m, size_t experts, size_t n,
                                                             size_t k) {
    if (!m || !n || !k || !experts || experts > kMaxExperts || !backward_sizes_ok(m, n, k))
        return 0;
    return partial_bytes(plan_experts_backward(m, experts, n, k, true, compute_units()));
}

extern "C" int kdq_mxfp4_experts_gated(const uint16_t* x_bf16, size_t x_stride, size_t m,
                                       const int32_t* offsets, size_t experts,
                                       const uint8_t* gate_packed, const uint8_t* up_packed,
                                       size_t n, size_t k, const float* gate_bias,
                                       const float* up_bias, int activation, uint16_t* h_bf16,
                                       size_t h_stride, uint16_t* kept_bf16, int8_t* kept_q8,
                                       float* kept_scales, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    if (!x_bf16 || !offsets || !gate_packed || !up_packed || !h_bf16 || !m || !n || !k ||
        (kept_bf16 && kept_q8) || !kept_q8 != !kept_scales || !gate_bias != !up_bias)
        return KDQ_ERR_ARGUMENT;
    if (const int rc = check_experts(offsets, experts))
        return rc;
    if (!sizes_ok(m, n, k) || n % 32)
        return KDQ_ERR_SHAPE;
    if (activation != KDQ_ACT_SILU && activation != KDQ_ACT_CLAMPED)
        return KDQ_ERR_UNSUPPORTED;
    if (const int rc = check_output(KDQ_BF16, h_bf16, h_stride, m, n))
        return rc;
    if (const int rc = check_input(x_bf16, x_stride, k))
        return rc;
    if (misaligned(gate_packed, 16) || misaligned(up_packed, 16) || misaligned(gate_bias, 4) ||
        misaligned(up_bias, 4) || misaligned(kept_bf16, 16) || misaligned(kept_q8, 16) ||
        misaligned(kept_scales, 4))
        return KDQ_ERR_ALIGNMENT;
    const Form f = packed_form(n, k);
    const Range out[] = {{h_bf16, extent(m, h_stride, n, 2)},
                         {kept_bf16, 4 * m * n},
                         {kept_q8, 2 * m * n},
                         {kept_scales, m * n / 4},
                         {workspace, workspace_bytes}},
                in[] = {{x_bf16, extent(m, x_stride, k, 2)},
                        {offsets, offset_bytes(offsets, experts)},
                        {gate_bias, experts * n * 4},
                        {up_bias, experts * n * 4},
                        {gate_packed, bytes_of(f, experts)},
                        {up_packed, bytes_of(f, experts)}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    const ExpertsPlan p =
        plan_experts(m, experts, n, k, true, kept_bf16 || kept_q8, compute_units());
    if (!launches(p))
        return KDQ_ERR_SHAPE;
    if (const int rc = check_workspace(partial_bytes(p), workspace, workspace_bytes))
        return rc;
    const auto st = static_cast<hipStream_t>(stream);
    Target t{h_bf16, h_stride, unsigned(m), unsigned(n), kept_bf16, kept_q8, kept_scales};
    t.e = {gate_bias, up_bias, nullptr, 0, activation, false};
    Gemm g = gemm_of(gate_packed, up_packed, x_bf16, x_stride, k, f, t);
    g.stack = stack_of(offsets, experts, f);
    return p.decode ? run_experts_decode<true, kOutExpertsGated>(decode_of(g, k), p.shape, st)
                    : run_experts_gemm<kBf16, kOutExpertsGated>(g, p, workspace, st);
}

extern "C" int kdq_mxfp4_experts_gated_backward(
    const uint16_t* dh_bf16, size_t dh_stride, size_t m, const int32_t* offsets, size_t experts,
    const uint16_t* kept_bf16, const int8_t* kept_q8, const float* kept_scales, int activation,
    const uint8_t* gate_transposed, const uint8_t* up_transposed, size_t n, size_t k,
    uint16_t* dgu_bf16, uint16_t* dx_bf16, size_t dx_stride, void* workspace,
    size_t workspace_bytes, void* stream) {
    if (!dh_bf16 || !offsets || !gate_transposed || !up_transposed || !dgu_bf16 || !dx_bf16 ||
        !m || !n || !k || !kept_bf16 == !kept_q8 || !kept_q8 != !kept_scales)
        return KDQ_ERR_ARGUMENT;
    if (const int rc = check_experts(offsets, experts))
        return rc;
    if (!backward_sizes_ok(m, n, k) || m * (n / 8) > UINT32_MAX - 255)
        return KDQ_ERR_SHAPE;
    if (activation != KDQ_ACT_SILU && activation != KDQ_ACT_CLAMPED)
        return KDQ_ERR_UNSUPPORTED;
    if (const int rc = check_output(KDQ_BF16, dx_bf16, dx_stride, m, k))
        return rc;
    if (const int rc = check_input(dh_bf16, dh_stride, n))
        return rc;
    if (misaligned(gate_transposed, 16) || misaligned(up_transposed, 16) ||
        misaligned(kept_bf16, 16) || misaligned(kept_q8, 16) || misaligned(kept_scales, 4) ||
        misaligned(dgu_bf16, 16))
        return KDQ_ERR_ALIGNMENT;
    const Form f = transposed_form(n, k);
    const Range out[] = {{dgu_bf16, 4 * m * n},
                         {dx_bf16, extent(m, dx_stride, k, 2)},
                         {workspace, workspace_bytes}},
                in[] = {{dh_bf16, extent(m, dh_stride, n, 2)},
                        {offsets, offset_bytes(offsets, experts)},
                        {kept_bf16, 4 * m * n},
                        {kept_q8, 2 * m * n},
                        {kept_scales, m * n / 4},
                        {gate_transposed, bytes_of(f, experts)},
                        {up_transposed, bytes_of(f, experts)}};
    if (any_overlap(out, in))
        return KDQ_ERR_ALIAS;
    const ExpertsPlan p = plan_experts_backward(m, experts, n, k, true, compute_units());
    if (!launches(p))
        return KDQ_ERR_SHAPE;
    if (const int rc = check_workspace(partial_bytes(p), workspace, workspace_bytes))
        return rc;
    const auto st = static_cast<hipStream_t>(stream);
    const auto gradients = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(unsigned(ceil_div(m * (n / 8), 256))), dim3(256), 0, st,
                           dh_bf16, dh_stride, unsigned(m), unsigned(n), kept_bf16, kept_q8,
                           kept_scales, dgu_bf16);
    };
    if (activation == KDQ_ACT_CLAMPED)
        kept_q8 ? gradients(gate_grad_kernel<true, true>)
                : gradients(gate_grad_kernel<false, true>);
    else
        kept_q8 ? gradients(gate_grad_kernel<true, false>)
                : gradients(gate_grad_kernel<false, false>);
    KDQ_HIP(hipGetLastError());
    const Target t{dx_bf16, dx_stride, unsigned(m), unsigned(k), nullptr, nullptr, nullptr};
    Gemm g = gemm_of(gate_transposed, up_transposed, dgu_bf16, 2 * n, n, f, t);
    g.x_second = unsigned(n * 2);
    g.stack = stack_of(offsets, experts, f);
    return run_experts_gemm<kTransposed, kOutExpertsBackward>(g, p, workspace, st);
}
