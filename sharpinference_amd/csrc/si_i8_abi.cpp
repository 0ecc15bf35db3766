// C ABI of the 8-bit integer rows (si_i8.hip, si_i8_gemm.hip): argument
// checks, then the launch on the context stream.
#include "si_context.hpp"
#include "si_i8.hpp"
#include "si_internal.hpp"

#include <cmath>

using namespace si_abi;

namespace {

constexpr int64_t MAX_ROWS = 1 << 21, MAX_COLS = 1 << 20;

int check_ptr(si_hip_context* ctx, const char* op, const void* p, const char* name, uintptr_t align)
{
    if (!p || !aligned(p, align))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %s must be a non-null %u-byte aligned device pointer", op, name,
                    static_cast<unsigned>(align));
    return SI_HIP_OK;
}

int check_extent(si_hip_context* ctx, const char* op, const char* name, int64_t n, int64_t max)
{
    if (n < 1 || n > max)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %s %lld outside 1..%lld", op, name, static_cast<long long>(n),
                    static_cast<long long>(max));
    return SI_HIP_OK;
}

struct Span {
    const void* p;
    uint64_t n;
};

// Fails when a written span overlaps a read one or another written one
// (absent operands are spans of no bytes).
int check_disjoint(si_hip_context* ctx, const char* op, std::initializer_list<Span> writes,
                   std::initializer_list<Span> reads)
{
    for (auto w = writes.begin(); w != writes.end(); ++w) {
        for (const auto& r : reads)
            if (overlaps(w->p, w->n, r.p, r.n))
                return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: an output overlaps an input", op);
        for (auto v = w + 1; v != writes.end(); ++v)
            if (overlaps(w->p, w->n, v->p, v->n))
                return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: outputs overlap", op);
    }
    return SI_HIP_OK;
}

int launched(si_hip_context* ctx, hipError_t e, const char* op)
{
    return e == hipSuccess ? SI_HIP_OK : hip_fail(ctx, e, op);
}

}  // namespace

extern "C" {

int si_hip_residual_rms_norm_i8(si_hip_context* ctx, const float* hidden, const float* residual, const float* weight,
                                float* updated, int8_t* codes, float* scale, int64_t rows, int64_t n, float eps)
{
    const char* op = "residual_rms_norm_i8";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (check_extent(ctx, op, "rows", rows, MAX_ROWS) || check_extent(ctx, op, "width", n, MAX_COLS))
        return SI_HIP_ERR_ARGUMENT;
    if (!std::isfinite(eps) || eps < 0.0f)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: epsilon must be finite and non-negative", op);
    if ((residual == nullptr) != (updated == nullptr))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: residual and updated come together or not at all", op);
    if (check_ptr(ctx, op, hidden, "hidden", 4) || check_ptr(ctx, op, weight, "weight", 4) ||
        check_ptr(ctx, op, codes, "codes", 1) || check_ptr(ctx, op, scale, "scale", 4) ||
        (residual && (check_ptr(ctx, op, residual, "residual", 4) || check_ptr(ctx, op, updated, "updated", 4))))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t count = static_cast<uint64_t>(rows) * n;
    if (check_disjoint(ctx, op, {{updated, updated ? count * 4 : 0}, {codes, count}, {scale, static_cast<uint64_t>(rows) * 4}},
                       {{hidden, count * 4}, {residual, residual ? count * 4 : 0}, {weight, static_cast<uint64_t>(n) * 4}}))
        return SI_HIP_ERR_ARGUMENT;
    return launched(ctx, si::launch_rms_norm_i8(hidden, residual, weight, updated, codes, scale, rows, n, eps, ctx->stream),
                    op);
}

int si_hip_quantize_i8(si_hip_context* ctx, int format, const void* x, int8_t* codes, float* scale, int64_t rows,
                       int64_t n)
{
    const char* op = "quantize_i8";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (format != SI_HIP_F32 && format != SI_HIP_F16 && format != SI_HIP_BF16)
        return fail(ctx, SI_HIP_ERR_UNSUPPORTED, "%s: rows of %s (%d) are not F32, F16 or BF16", op, fmt_name(format),
                    format);
    const uintptr_t size = format == SI_HIP_F32 ? 4 : 2;
    if (check_extent(ctx, op, "rows", rows, MAX_ROWS) || check_extent(ctx, op, "width", n, MAX_COLS) ||
        check_ptr(ctx, op, x, "input", size) || check_ptr(ctx, op, codes, "codes", 1) ||
        check_ptr(ctx, op, scale, "scale", 4))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t count = static_cast<uint64_t>(rows) * n;
    if (check_disjoint(ctx, op, {{codes, count}, {scale, static_cast<uint64_t>(rows) * 4}}, {{x, count * size}}))
        return SI_HIP_ERR_ARGUMENT;
    return launched(ctx, si::launch_quantize_i8(format, x, codes, scale, rows, n, ctx->stream), op);
}

int si_hip_dequant_i8(si_hip_context* ctx, const int8_t* codes, const float* scale, float* output, int64_t rows,
                      int64_t n)
{
    const char* op = "dequant_i8";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (check_extent(ctx, op, "rows", rows, MAX_ROWS) || check_extent(ctx, op, "width", n, MAX_COLS) ||
        check_ptr(ctx, op, codes, "codes", 1) || check_ptr(ctx, op, scale, "scale", 4) ||
        check_ptr(ctx, op, output, "output", 4))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t count = static_cast<uint64_t>(rows) * n;
    if (check_disjoint(ctx, op, {{output, count * 4}}, {{codes, count}, {scale, static_cast<uint64_t>(rows) * 4}}))
        return SI_HIP_ERR_ARGUMENT;
    return launched(ctx, si::launch_dequant_i8(codes, scale, output, rows, n, ctx->stream), op);
}

int si_hip_gemm_i8(si_hip_context* ctx, const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale,
                   float* y, int64_t m, int64_t rows, int64_t cols, const float* residual)
{
    const char* op = "gemm_i8";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (check_extent(ctx, op, "token rows", m, MAX_ROWS) || check_extent(ctx, op, "rows", rows, MAX_ROWS))
        return SI_HIP_ERR_ARGUMENT;
    // (codes of any value, -128 among them, sum to less than 2^31)
    if (cols < 16 || cols > 65536 || cols % 16 != 0)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %lld columns is not a multiple of 16 in 16..65536", op,
                    static_cast<long long>(cols));
    const uint64_t x_b = static_cast<uint64_t>(m) * cols, w_b = static_cast<uint64_t>(rows) * cols,
                   y_b = static_cast<uint64_t>(m) * rows * 4;
    if (check_ptr(ctx, op, x, "x", 16) || check_ptr(ctx, op, w, "weight", 16) ||
        check_ptr(ctx, op, x_scale, "x scale", 4) || check_ptr(ctx, op, w_scale, "weight scale", 4) ||
        check_ptr(ctx, op, y, "y", 4) || (residual && check_ptr(ctx, op, residual, "residual", 4)))
        return SI_HIP_ERR_ARGUMENT;
    if (residual && residual != y && overlaps(y, y_b, residual, y_b))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: y overlaps the residual without being it", op);
    if (check_disjoint(ctx, op, {{y, y_b}},
                       {{x, x_b}, {w, w_b}, {x_scale, static_cast<uint64_t>(m) * 4}, {w_scale, static_cast<uint64_t>(rows) * 4}}))
        return SI_HIP_ERR_ARGUMENT;
    si::GemmI8Args a{x, x_scale, w, w_scale, residual, y, m, rows, cols};
    return launched(ctx, si::launch_gemm_i8(a, ctx->stream), op);
}

}  // extern "C"
