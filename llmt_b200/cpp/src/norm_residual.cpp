// kernels::norm_residual_fwd / _bwd over the llmt_b200 C ABI.
#include "llmt/core/error.h"
#include "llmt/kernels/norm_residual.h"
#include "llmt_b200.h"

namespace llmt::kernels {

namespace {

const Tensor& rows_like(const char* who, const Tensor& t, const Tensor& like, const char* name) noexcept {
    if (!t.valid()) detail::fatal(who, "invalid tensor (null data)");
    if (t.shape != like.shape) detail::fatal(who, "%s must have the residual stream's shape", name);
    return t;
}

float* floats(const char* who, const Tensor* t, int64_t n, const char* name) noexcept {
    if (t == nullptr) return nullptr;
    if (!t->valid() || t->dtype != DType::FP32 || t->numel() != n) detail::fatal(who, "%s must be fp32 with %lld values", name, static_cast<long long>(n));
    return static_cast<float*>(t->data);
}

// What both directions fill in.  `res` is a tensor of the residual stream, `act` one of the block (null: there is none).
llmt_b200_norm_residual_desc describe(const char* who, const Tensor& res, const Tensor* act, const NormResidual& n) noexcept {
    llmt_b200_norm_residual_desc d{};
    if (!res.valid()) detail::fatal(who, "invalid tensor (null data)");
    d.cols = res.shape[res.shape.rank - 1];
    d.rows = d.cols > 0 ? res.numel() / d.cols : 0;
    d.groups = 1;
    if (n.gate != nullptr) {
        if (!n.gate->valid() || n.gate->dtype != DType::FP32 || n.gate->shape[n.gate->shape.rank - 1] != d.cols || n.gate->shape.rank > 2)
            detail::fatal(who, "gate must be fp32 [C] or [groups, C]");
        d.gate = static_cast<const float*>(n.gate->data);
        d.groups = n.gate->shape.rank == 2 ? n.gate->shape[0] : 1;
    }
    d.dtype_res = static_cast<int32_t>(res.dtype);
    d.dtype_act = static_cast<int32_t>(act != nullptr ? act->dtype : res.dtype);
    d.scale = n.scale; d.eps = n.eps;
    d.w_post = floats(who, n.w_post, d.cols, "w_post");
    d.w_pre = floats(who, n.w_pre, d.cols, "w_pre");
    d.rstd_post = floats(who, n.rstd_post, d.rows, "rstd_post");
    d.rstd_pre = floats(who, n.rstd_pre, d.rows, "rstd_pre");
    d.ld_x = d.ld_y = d.ld_out = d.ld_h = d.ld_dout = d.ld_dh = d.ld_dx = d.ld_dy = d.cols;
    return d;
}

void one_type(const char* who, const Tensor* a, const Tensor* b, const char* what) noexcept {
    if (a != nullptr && b != nullptr && a->dtype != b->dtype) detail::fatal(who, "%s must have one type", what);
}

void put_grads(const char* who, llmt_b200_norm_residual_desc& d, const NormResidualGrads& g) noexcept {
    d.dw_post = floats(who, g.dw_post, d.cols, "dw_post");
    d.dgate = floats(who, g.dgate, d.groups * d.cols, "dgate");
    d.dw_pre = floats(who, g.dw_pre, d.cols, "dw_pre");
    d.beta = g.beta;
}

}  // namespace

void norm_residual_fwd(const RunCtx& ctx, Tensor* out, Tensor* h, const Tensor& x, const Tensor* y, const NormResidual& n) noexcept {
    const char* who = "norm_residual_fwd";
    one_type(who, y, h, "y and h");
    llmt_b200_norm_residual_desc d = describe(who, x, y != nullptr ? y : h, n);
    d.x = x.data;
    if (y != nullptr) {
        d.y = rows_like(who, *y, x, "y").data;
        if (out == nullptr) detail::fatal(who, "invalid tensor (null data)");
        d.out = rows_like(who, *out, x, "out").data;
        one_type(who, &x, out, "x and out");
    }
    if (h != nullptr) d.h = rows_like(who, *h, x, "h").data;
    if (llmt_b200_norm_residual_fwd(&d, ctx.stream) != LLMT_B200_OK) detail::fatal(who, "%s", llmt_b200_last_error());
}

size_t norm_residual_workspace_bytes(const Tensor& dx, const Tensor* y, const NormResidual& n, const NormResidualGrads& grads) noexcept {
    const char* who = "norm_residual_bwd";
    llmt_b200_norm_residual_desc d = describe(who, dx, y, n);
    if (y != nullptr) d.y = y->data;
    put_grads(who, d, grads);
    return static_cast<size_t>(llmt_b200_norm_residual_workspace_bytes(&d));
}

void norm_residual_bwd(const RunCtx& ctx, Tensor& dx, Tensor* dy, const Tensor* dout, const Tensor* dh, const Tensor* out, const Tensor* y,
                       const NormResidual& n, const NormResidualGrads& grads) noexcept {
    const char* who = "norm_residual_bwd";
    one_type(who, y, dh, "y and dh");
    llmt_b200_norm_residual_desc d = describe(who, dx, y != nullptr ? y : dh, n);
    put_grads(who, d, grads);
    d.dx = dx.data;
    if (dout != nullptr) d.dout = rows_like(who, *dout, dx, "dout").data;
    one_type(who, &dx, dout, "dx and dout");
    if (dh != nullptr) {
        if (out == nullptr) detail::fatal(who, "invalid tensor (null data)");
        d.dh = rows_like(who, *dh, dx, "dh").data;
        d.out = rows_like(who, *out, dx, "out").data;
        one_type(who, &dx, out, "dx and out");
    }
    if (y != nullptr) {
        if (dy == nullptr) detail::fatal(who, "invalid tensor (null data)");
        d.y = rows_like(who, *y, dx, "y").data;
        d.dy = rows_like(who, *dy, dx, "dy").data;
        one_type(who, y, dy, "y and dy");
    }
    d.workspace = ctx.blas_workspace;
    d.workspace_bytes = ctx.blas_workspace_bytes;
    if (llmt_b200_norm_residual_bwd(&d, ctx.stream) != LLMT_B200_OK) detail::fatal(who, "%s", llmt_b200_last_error());
}

}  // namespace llmt::kernels
