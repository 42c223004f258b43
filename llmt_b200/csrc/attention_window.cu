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
    attn::Four().store(attn::row_to(p.out, bh / p.heads, i, bh % p.heads), 0.0f, p.head_dim);
    if ((threadIdx.x & 31) == 0 && p.lse != nullptr) p.lse[row] = -INFINITY;
}

__global__ void __launch_bounds__(kRowThreads) attention_dq_rows_kernel(AttentionParams p) {
    ptx::grid_dependency_wait();
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) >> 5;
    if (row >= static_cast<int64_t>(p.batch) * p.heads * p.tq) return;
    const int64_t i = row % p.tq, bh = row / p.tq;
    attn::Four().store(attn::row_to(p.dq, bh / p.heads, i, bh % p.heads), 0.0f, p.head_dim);
}

__global__ void __launch_bounds__(kRowThreads) attention_dkdv_rows_kernel(AttentionParams p) {
    ptx::grid_dependency_wait();
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) >> 5;
    if (row >= static_cast<int64_t>(p.batch) * p.kv_heads * p.tk) return;
    const int64_t j = row % p.tk, bh = row / p.tk;
    attn::Four().store(attn::row_to(p.dk, bh / p.kv_heads, j, bh % p.kv_heads), 0.0f, p.head_dim);
    attn::Four().store(attn::row_to(p.dv, bh / p.kv_heads, j, bh % p.kv_heads), 0.0f, p.head_dim);
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>((rows * 32 + kRowThreads - 1) / kRowThreads); }

}  // namespace

cudaError_t launch_attention_window_fwd(const AttentionParams& p, cudaStream_t stream) {
    return launch_dependent(attention_fwd_rows_kernel, row_blocks(static_cast<int64_t>(p.batch) * p.heads * p.tq), kRowThreads, stream, p);
}
cudaError_t launch_attention_window_bwd(const AttentionParams& p, cudaStream_t stream) {
    if (p.tq > 0 && p.heads > 0) {
        const cudaError_t e = launch_dependent(attention_dq_rows_kernel, row_blocks(static_cast<int64_t>(p.batch) * p.heads * p.tq), kRowThreads, stream, p);
        if (e != cudaSuccess || p.tk == 0) return e;
    }
    return launch_dependent(attention_dkdv_rows_kernel, row_blocks(static_cast<int64_t>(p.batch) * p.kv_heads * p.tk), kRowThreads, stream, p);
}

}  // namespace llmt_b200
