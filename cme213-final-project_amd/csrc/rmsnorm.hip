// Entry points of the RMS norm calls: their checks, the backward pass's workspace and the sum of
// its partial rows.  The kernels are in mi_rmsnorm_kernels.hpp.
#include "mi_rmsnorm.hpp"
#include "mi_rowtype.hpp"

namespace mi {

namespace {

constexpr int kMaxCols = 1 << 24;

int check_rows(const char* name, int rows, int cols, int type) {
    if (rows < 0 || cols < 1 || cols > kMaxCols)
        return set_error(MI_ERR_INVALID_ARG, "%s: invalid shape rows=%d cols=%d (cols is 1 to %d)",
                         name, rows, cols, kMaxCols);
    if (!row_type_ok(type)) return set_error(MI_ERR_INVALID_ARG, "%s: type=%d", name, type);
    return MI_OK;
}

template <bool RESID, bool Q8>
int rms_forward(const char* name, const rms::Forward& c, void* stream) {
    if (int rc = check_rows(name, c.rows, c.cols, c.type)) return rc;
    if (!(c.eps >= 0.0f && c.eps <= 3.0e38f))
        return set_error(MI_ERR_INVALID_ARG, "%s: eps=%g", name, static_cast<double>(c.eps));
    if (Q8 && c.format != MI_ROW8_INT8 && c.format != MI_ROW8_E4M3)
        return set_error(MI_ERR_INVALID_ARG, "%s: format=%d", name, c.format);
    if (Q8 && c.block != 0 && c.block != MI_ROW8_BLOCK)
        return set_error(MI_ERR_INVALID_ARG, "%s: block=%d (0 or %d)", name, c.block,
                         MI_ROW8_BLOCK);
    if (c.rows == 0) return MI_OK;
    if (!c.a || !c.gamma || (RESID && (!c.b || !c.residual_out)) ||
        (Q8 ? !c.q || !c.scales : !c.out))
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    with_row_type(c.type,
                  [&](auto t) { rms::forward<decltype(t)::value>(c, to_stream(stream)); });
    return check_launch(name);
}

int rms_backward(const char* name, rms::Backward c, float* dgamma, void* stream) {
    if (int rc = check_rows(name, c.rows, c.cols, c.type)) return rc;
    if (c.rows == 0) return MI_OK;
    if (!c.grad_out || !c.x || !c.inv_rms || !c.gamma || !c.dx || !dgamma)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    hipStream_t st = to_stream(stream);
    int err = MI_OK;
    char* ws = static_cast<char*>(
        workspace_get(mi_rmsnorm_backward_workspace(c.rows, c.cols, c.type), st, &err));
    if (!ws) return err;
    c.part = reinterpret_cast<float*>(ws + colsum_part_offset());
    with_row_type(c.type, [&](auto t) { rms::backward<decltype(t)::value>(c, st); });
    if (int rc = check_launch(name)) return rc;
    return launch_colsum_finalize(c.part, rms::backward_blocks(c.rows, c.cols, c.type), c.cols,
                                  dgamma, c.cols, nullptr, st);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

int mi_rmsnorm_forward(const void* x, const float* gamma, void* out, float* inv_rms, int rows,
                       int cols, float eps, int type, void* stream) {
    return rms_forward<false, false>(
        "mi_rmsnorm_forward",
        rms::Forward{x, nullptr, gamma, nullptr, out, inv_rms, nullptr, nullptr, rows, cols, eps, 0, 0,
                type},
        stream);
}

int mi_residual_rmsnorm_forward(const void* a, const void* b, const float* gamma,
                                void* residual_out, void* out, float* inv_rms, int rows, int cols,
                                float eps, int type, void* stream) {
    return rms_forward<true, false>(
        "mi_residual_rmsnorm_forward",
        rms::Forward{a, b, gamma, residual_out, out, inv_rms, nullptr, nullptr, rows, cols, eps, 0, 0,
                type},
        stream);
}

int mi_rmsnorm_forward_row8(const void* x, const float* gamma, void* q, float* scales, void* out,
                            float* inv_rms, int rows, int cols, float eps, int block, int format,
                            int type, void* stream) {
    return rms_forward<false, true>(
        "mi_rmsnorm_forward_row8",
        rms::Forward{x, nullptr, gamma, nullptr, out, inv_rms, q, scales, rows, cols, eps, block,
                format, type},
        stream);
}

int mi_residual_rmsnorm_forward_row8(const void* a, const void* b, const float* gamma,
                                     void* residual_out, void* q, float* scales, void* out,
                                     float* inv_rms, int rows, int cols, float eps, int block,
                                     int format, int type, void* stream) {
    return rms_forward<true, true>(
        "mi_residual_rmsnorm_forward_row8",
        rms::Forward{a, b, gamma, residual_out, out, inv_rms, q, scales, rows, cols, eps, block, format,
                type},
        stream);
}

int mi_rmsnorm_backward(const void* grad_out, const void* x, const float* inv_rms,
                        const float* gamma, void* grad_x, float* dgamma, int rows, int cols,
                        int type, void* stream) {
    return rms_backward("mi_rmsnorm_backward",
                        rms::Backward{grad_out, x, inv_rms, gamma, grad_x, false, rows, cols, type,
                                      nullptr},
                        dgamma, stream);
}

int mi_rmsnorm_backward_residual(const void* grad_out, const void* x, const float* inv_rms,
                                 const float* gamma, void* grad_residual, float* dgamma, int rows,
                                 int cols, int type, void* stream) {
    return rms_backward("mi_rmsnorm_backward_residual",
                        rms::Backward{grad_out, x, inv_rms, gamma, grad_residual, true, rows, cols,
                                      type, nullptr},
                        dgamma, stream);
}

size_t mi_rmsnorm_backward_workspace(int rows, int cols, int type) {
    if (rows <= 0 || cols <= 0 || !row_type_ok(type)) return 0;
    return colsum_bytes(rms::backward_blocks(rows, cols, type), cols);
}

}  // extern "C"
