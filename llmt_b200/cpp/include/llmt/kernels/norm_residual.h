// The norms after and before a block with the block's gate and the residual, in one pass over the rows (llmt
// include/llmt/kernels/rmsnorm.h and residual.h are a kernel each):
//   N(z; w) = z * rsqrt(mean(z^2) + eps) * w
//   out = x + scale * gate * N(y; w_post),   h = N(out; w_pre)
// x, out: the residual stream; y, h: the block's type ((fp32, fp32), (fp32, bf16) or (bf16, bf16)), all of one shape
// [..., C].  Weights, gate, statistics and their gradients are fp32: w [C], gate [C] or [groups, C], rstd one value per row.
// Tensors that a call does without are null.  out may be x, dx may be dout.
#pragma once

#include "llmt/core/run_ctx.h"
#include "llmt/core/types.h"

namespace llmt::kernels {

struct NormResidual {
    const Tensor* w_post = nullptr;
    const Tensor* gate = nullptr;
    const Tensor* w_pre = nullptr;
    Tensor* rstd_post = nullptr;  // written forward, read backward
    Tensor* rstd_pre = nullptr;
    float scale = 1.0f;
    float eps = 1e-5f;
};
struct NormResidualGrads {  // d = beta * d + sum over rows; null: not wanted
    Tensor* dw_post = nullptr;
    Tensor* dgate = nullptr;
    Tensor* dw_pre = nullptr;
    float beta = 1.0f;
};

// y null: out is not written, h = N(x; w_pre).  h null: no norm follows.
void norm_residual_fwd(const RunCtx& ctx, Tensor* out, Tensor* h, const Tensor& x, const Tensor* y, const NormResidual& n) noexcept;
// out: the forward call's (its x where y is null).  dout or dh may be null; dy goes with y.  ctx.blas_workspace must hold
// norm_residual_workspace_bytes(...) bytes.
void norm_residual_bwd(const RunCtx& ctx, Tensor& dx, Tensor* dy, const Tensor* dout, const Tensor* dh, const Tensor* out, const Tensor* y,
                       const NormResidual& n, const NormResidualGrads& grads) noexcept;
size_t norm_residual_workspace_bytes(const Tensor& dx, const Tensor* y, const NormResidual& n, const NormResidualGrads& grads) noexcept;

}  // namespace llmt::kernels
