// Rotary positions on the q and k heads of a packed projection, in place (llmt include/llmt/kernels/rope.h turns separate
// q and k tensors, rotate-half only).
//   qkv   [B, T, (H + 2 Hkv) * hd], per token Q | K | V, fp32 or bf16: the first H + Hkv heads are turned
//   freqs device, fp64 [rot_dim / 2], radians per token (llmt_b200_rope_frequencies fills a host array)
// inverse = true makes the gradient of the unturned projection out of that of the turned one.
#pragma once

#include "llmt/core/run_ctx.h"
#include "llmt/core/types.h"

namespace llmt::kernels {

struct RopeSpec {
    const double* freqs = nullptr;
    int64_t rot_dim = 0;                // values of a head that turn; the others stay
    const Tensor* positions = nullptr;  // I32 [B, T]; null: offset, offset + 1, ...
    int64_t offset = 0;
    bool interleaved = false;           // pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)
    float scale = 1.0f;
};

void rope_packed(const RunCtx& ctx, Tensor& qkv, int64_t n_head, int64_t n_kv_head, const RopeSpec& spec, bool inverse = false) noexcept;

}  // namespace llmt::kernels
