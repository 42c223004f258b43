// Causal attention with a sliding window and sinks where there are no queries or no keys, a warp for each row: a forward pass
// over no keys (zeros and -inf), its gradient, and the keys' gradients without queries or query heads (zeros).  No tensor map
// describes a tensor without elements; everything else is in the tiled kernels.
#include "attention_rows.cuh"
#include "ptx_sm100.cuh"

namespace llmt_b200 {
namespace {

constexpr int kRowThreads = 128;

__global__ void __launch_bounds__(kRowThreads) attention_fwd_rows_kernel(AttentionParams p) {
    ptx::grid_dependency_wait();
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) >> 5;
    if (row >= static_cast<int64_t>(p.batch) * p.heads * p.tq) return;
    const int64_t i = row % p.tq, bh = row / p.tq;
    attn::forward_row(p, bh / p.heads, bh % p.heads, i, i + p.tk - p.tq);
}

__global__ void __launch_bounds__(kRowThreads) attention_dq_rows_kernel(AttentionParams p) {
    ptx::grid_dependency_wait();
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) >> 5;
    if (row >= static_cast<int64_t>(p.batch) * p.heads * p.tq) return;
    const int64_t i = row % p.tq, bh = row / p.tq, b = bh / p.heads, h = bh % p.heads;
    const float d = attn::dot_rows(attn::row_of(p.dout, b, i, h), attn::row_of(p.out, b, i, h), p.head_dim);
    if ((threadIdx.x & 31) == 0) p.dvec[row] = d;
    attn::dq_row(p, b, h, i, d);
}

__global__ void __launch_bounds__(kRowThreads) attention_dkdv_rows_kernel(AttentionParams p) {
    ptx::grid_dependency_wait();
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) >> 5;
    const int64_t hkv = p.kv_heads;
    if (row >= static_cast<int64_t>(p.batch) * hkv * p.tk) return;
    const int64_t j = row % p.tk, bh = row / p.tk;
    attn::dkdv_row(p, bh / hkv, bh % hkv, j);
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>((rows * 32 + kRowThreads - 1) / kRowThreads); }

}  // namespace

cudaError_t launch_attention_window_fwd(const AttentionParams& p, cudaStream_t stream) {
    return launch_dependent(attention_fwd_rows_kernel, row_blocks(static_cast<int64_t>(p.batch) * p.heads * p.tq), kRowThreads, stream, p);
}
cudaError_t launch_attention_window_bwd(AttentionParams p, void* workspace, cudaStream_t stream) {
    p.dvec = static_cast<float*>(workspace);
    if (p.tq > 0 && p.heads > 0) {
        const cudaError_t e = launch_dependent(attention_dq_rows_kernel, row_blocks(static_cast<int64_t>(p.batch) * p.heads * p.tq), kRowThreads, stream, p);
        if (e != cudaSuccess || p.tk == 0) return e;
    }
    return launch_dependent(attention_dkdv_rows_kernel, row_blocks(static_cast<int64_t>(p.batch) * p.kv_heads * p.tk), kRowThreads, stream, p);
}

}  // namespace llmt_b200
