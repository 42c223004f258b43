// kernels::rope_packed over the llmt_b200 C ABI.
#include "llmt/core/error.h"
#include "llmt/kernels/rope.h"
#include "llmt_b200.h"

namespace llmt::kernels {

void rope_packed(const RunCtx& ctx, Tensor& qkv, int64_t n_head, int64_t n_kv_head, const RopeSpec& spec, bool inverse) noexcept {
    const char* who = "rope_packed";
    if (!qkv.valid()) detail::fatal(who, "invalid tensor (null data)");
    const int64_t parts = n_head + 2 * n_kv_head;
    if (qkv.shape.rank != 3 || n_head <= 0 || n_kv_head <= 0 || qkv.shape[2] % parts != 0) detail::fatal(who, "qkv must be [B, T, (H + 2 Hkv)·hd]");
    llmt_b200_rope_desc d{};
    d.batch = qkv.shape[0]; d.tokens = qkv.shape[1]; d.heads = n_head + n_kv_head; d.head_dim = qkv.shape[2] / parts;
    d.rot_dim = spec.rot_dim;
    d.x.data = qkv.data;
    d.x.stride_batch = d.tokens * qkv.shape[2]; d.x.stride_token = qkv.shape[2]; d.x.stride_head = d.head_dim;
    d.y = d.x;
    d.freqs = spec.freqs;
    if (spec.positions != nullptr) {
        if (!spec.positions->valid() || spec.positions->dtype != DType::I32 || spec.positions->shape != Shape{d.batch, d.tokens})
            detail::fatal(who, "positions must be I32 [B, T]");
        d.positions = static_cast<const int32_t*>(spec.positions->data);
    }
    d.offset = spec.offset;
    d.dtype = static_cast<int32_t>(qkv.dtype);
    d.interleaved = spec.interleaved; d.inverse = inverse;
    d.scale = spec.scale;
    if (llmt_b200_rope(&d, ctx.stream) != LLMT_B200_OK) detail::fatal(who, "%s", llmt_b200_last_error());
}

}  // namespace llmt::kernels
