// The norms after and before a block with the block's gate and residual in one pass: see llmt_b200_norm_residual_fwd / _bwd in
// the public header.
//
// Mathematics, per row (N(z; w) = z rstd(z) w, rstd(z) = (mean z^2 + eps)^-1/2):
//   out = x + k N(y; w_post),  k = scale gate;   h = N(out; w_pre)
// Backward, with b = out rstd_pre, a = dh w_pre, c = y rstd_post, e = k w_post:
//   g  = dout + rstd_pre (a - b mean(a b))                      the gradient of x
//   dy = rstd_post (e g - c mean(e g c))
//   dw_pre += dh b,  dw_post += k g c,  dgate += scale g c w_post
// mean(e g c) is linear in mean(a b), so the three row sums  a b,  e c (dout + rstd_pre a)  and  e c b  are formed in one round.
//
// Bound: memory; every tensor is read and written once, all sums are fp32.  Forward: a row's values stay in the registers of
// the warps that own the row.  Backward: a block owns all columns (a cluster of blocks those of a wide row), takes rows one after
// the other with the next row's loads in flight, and keeps the three weight gradients of its columns in registers; each
// block leaves one row of sums, and a second launch adds those in a fixed order.
#include <cuda_bf16.h>

#include "common.h"
#include "ptx_sm100.cuh"

namespace llmt_b200 {
namespace {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// V values of a row that start on a multiple of V: one or two 16-byte accesses (V = 8) or one value (V = 1).
template <typename T, int V> struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Vec { T v[V]; };

template <int V> __device__ __forceinline__ void load_weights(float* w, const float* at, bool there, float otherwise) {
    if (there) {
        const Vec<float, V> x = *reinterpret_cast<const Vec<float, V>*>(at);
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = x.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = otherwise;
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ------------------------------------------------------------------------------------------------------------ forward

constexpr int kFwdRows = 4;   // rows of a block whose rows are one warp's each

// The sum over the warps of a row (all of the block's, or one).
__device__ __forceinline__ float row_sum(float v, float* part, int warps) {
    v = warp_sum(v);
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < warps; ++i) s += part[i];
    return s;
}

template <typename TR, typename TA, int V, int NV>
__global__ void __launch_bounds__(512) norm_residual_fwd_kernel(NormResidualParams p, int warps) {
    __shared__ float part[2][16];
    ptx::grid_dependency_wait();
    const int64_t row = warps == 1 ? static_cast<int64_t>(blockIdx.x) * kFwdRows + (threadIdx.x >> 5) : static_cast<int64_t>(blockIdx.x);
    if (row >= p.rows) return;
    const int across = warps * 32, me = warps == 1 ? threadIdx.x & 31 : threadIdx.x;
    const TR* x = static_cast<const TR*>(p.x) + row * p.ld_x;
    const TA* y = static_cast<const TA*>(p.y) + row * p.ld_y;
    const float* gate = p.gate != nullptr ? p.gate + row / p.rows_per_gate * p.cols : nullptr;
    const bool block = p.y != nullptr;
    Vec<TR, V> xs[NV];
    Vec<TA, V> ys[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int col = (me + n * across) * V;
        xs[n] = {};
        ys[n] = {};
        if (col < p.cols) {
            xs[n] = *reinterpret_cast<const Vec<TR, V>*>(x + col);
            if (block) ys[n] = *reinterpret_cast<const Vec<TA, V>*>(y + col);
        }
    }
    const float of = 1.0f / static_cast<float>(p.cols);
    float k = p.scale;
    if (block && p.w_post != nullptr) {
        float s = 0.0f;
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int i = 0; i < V; ++i) s = fmaf(to_float(ys[n].v[i]), to_float(ys[n].v[i]), s);
        const float r = 1.0f / sqrtf(row_sum(s, part[0], warps) * of + p.eps);
        if (me == 0 && p.rstd_post != nullptr) p.rstd_post[row] = r;
        k *= r;
    }
    float z[NV * V], s = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int col = (me + n * across) * V;
        if (col < p.cols) {
            if (block) {
                float w[V], g[V];
                load_weights<V>(w, p.w_post + col, p.w_post != nullptr, 1.0f);
                load_weights<V>(g, gate + col, gate != nullptr, 1.0f);
                Vec<TR, V> o;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    z[n * V + i] = fmaf(k * to_float(ys[n].v[i]), w[i] * g[i], to_float(xs[n].v[i]));
                    o.v[i] = rounded<TR>(z[n * V + i]);
                }
                *reinterpret_cast<Vec<TR, V>*>(static_cast<TR*>(p.out) + row * p.ld_out + col) = o;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) z[n * V + i] = to_float(xs[n].v[i]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) s = fmaf(z[n * V + i], z[n * V + i], s);
        }
    }
    if (p.h == nullptr) return;
    const float r = 1.0f / sqrtf(row_sum(s, part[1], warps) * of + p.eps);
    if (me == 0 && p.rstd_pre != nullptr) p.rstd_pre[row] = r;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int col = (me + n * across) * V;
        if (col < p.cols) {
            float w[V];
            load_weights<V>(w, p.w_pre + col, true, 1.0f);
            Vec<TA, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = rounded<TA>(z[n * V + i] * r * w[i]);
            *reinterpret_cast<Vec<TA, V>*>(static_cast<TA*>(p.h) + row * p.ld_h + col) = o;
        }
    }
}

// ----------------------------------------------------------------------------------------------------------- backward

constexpr int kBwdWarps = 16;                  // of a block at most
constexpr int kBwdCols = kBwdWarps * 32 * 8;   // columns that one block owns at most

// Eight columns of a thread: V = 8 neighbours, or (V = 1) eight that are the block's width apart.
template <typename T, int V> struct Eight {
    Vec<T, V> g[8 / V];
    __device__ __forceinline__ float at(int i) const { return to_float(g[i / V].v[i % V]); }
    __device__ __forceinline__ void put(int i, float x) { g[i / V].v[i % V] = rounded<T>(x); }
    __device__ __forceinline__ void load(const T* row, int first, int step, int cols, bool there) {
#pragma unroll
        for (int n = 0; n < 8 / V; ++n) {
            g[n] = {};
            if (there && first + n * step < cols) g[n] = *reinterpret_cast<const Vec<T, V>*>(row + first + n * step);
        }
    }
    __device__ __forceinline__ void store(T* row, int first, int step, int cols) const {
#pragma unroll
        for (int n = 0; n < 8 / V; ++n)
            if (first + n * step < cols) *reinterpret_cast<Vec<T, V>*>(row + first + n * step) = g[n];
    }
};
template <typename TR, typename TA, int V> struct BwdRow {
    Eight<TR, V> out, dout;
    Eight<TA, V> dh, y;
    float r_pre, r_post;
};

// `units` pieces of equal groups of rows (rows of one gate); block (cluster) b takes units b, b + grid, ...
template <typename TR, typename TA, int V, bool CLUSTER>
__global__ void __launch_bounds__(kBwdWarps * 32, 1) norm_residual_bwd_kernel(NormResidualParams p, int units, int per_group) {
    __shared__ float part[2][4 * kBwdWarps][3];   // of every warp of the cluster (up to four blocks)
    ptx::grid_dependency_wait();
    const int threads = blockDim.x, warps = threads >> 5;
    const int ranks = CLUSTER ? p.cluster : 1;
    const int rank = CLUSTER ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const int me = blockIdx.x / ranks, blocks = gridDim.x / ranks;
    const int first = V == 8 ? (rank * threads + static_cast<int>(threadIdx.x)) * 8 : rank * threads * 8 + static_cast<int>(threadIdx.x);
    const int step = V == 8 ? 0 : threads;
    const int cols = V == 8 ? p.cols : (p.cols < (rank + 1) * threads * 8 ? p.cols : (rank + 1) * threads * 8);
    const bool pre = p.dh != nullptr, block = p.y != nullptr, post = p.w_post != nullptr;
    const float of = 1.0f / static_cast<float>(p.cols);
    if (CLUSTER) ptx::cluster_sync_all();   // nobody writes into a block's shared memory before it runs

    Eight<float, V> weight;
    float w_pre[8], e_w[8], acc_pre[8], acc_post[8];
    weight.load(p.w_pre, first, step, cols, pre);
#pragma unroll
    for (int i = 0; i < 8; ++i) { w_pre[i] = weight.at(i); acc_pre[i] = acc_post[i] = 0.0f; }
    weight.load(p.w_post, first, step, cols, post);
#pragma unroll
    for (int i = 0; i < 8; ++i) e_w[i] = post ? weight.at(i) : 1.0f;

    BwdRow<TR, TA, V> next;
    auto load = [&](int64_t row) {
        next.out.load(static_cast<const TR*>(p.out) + row * p.ld_out, first, step, cols, pre);
        next.dout.load(static_cast<const TR*>(p.dout) + row * p.ld_dout, first, step, cols, p.dout != nullptr);
        next.dh.load(static_cast<const TA*>(p.dh) + row * p.ld_dh, first, step, cols, pre);
        next.y.load(static_cast<const TA*>(p.y) + row * p.ld_y, first, step, cols, block);
        next.r_pre = pre ? p.rstd_pre[row] : 0.0f;
        next.r_post = block && post ? p.rstd_post[row] : 1.0f;
    };
    int turn = 0;
    for (int u = me; u < units; u += blocks) {
        const int64_t group = u / per_group, part_of = u % per_group;
        const int64_t r0 = group * p.rows_per_gate + p.rows_per_gate * part_of / per_group;
        const int64_t r1 = group * p.rows_per_gate + p.rows_per_gate * (part_of + 1) / per_group;
        float gate[8], acc_gate[8];
        weight.load(p.gate + group * p.cols, first, step, cols, p.gate != nullptr);
#pragma unroll
        for (int i = 0; i < 8; ++i) { gate[i] = p.gate != nullptr ? weight.at(i) : 1.0f; acc_gate[i] = 0.0f; }
        if (r0 < r1) load(r0);
        for (int64_t row = r0; row < r1; ++row) {
            const BwdRow<TR, TA, V> now = next;
            if (row + 1 < r1) load(row + 1);
            float s_ab = 0.0f, s_eg = 0.0f, s_eb = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = now.dh.at(i) * w_pre[i], b = now.out.at(i) * now.r_pre;
                s_ab = fmaf(a, b, s_ab);
                const float ec = gate[i] * e_w[i] * now.y.at(i);
                s_eg = fmaf(ec, fmaf(now.r_pre, a, now.dout.at(i)), s_eg);
                s_eb = fmaf(ec, b, s_eb);
            }
            s_ab = warp_sum(s_ab);
            s_eg = warp_sum(s_eg);
            s_eb = warp_sum(s_eb);
            if (CLUSTER || warps > 1) {
                // two turns of sums: whoever writes a third has seen everybody read the first
                float (*mine)[3] = part[turn];
                turn ^= 1;
                const int lane = threadIdx.x & 31, w = rank * warps + (threadIdx.x >> 5);
                if (CLUSTER) {
                    if (lane < ranks) {
                        const uint32_t at = ptx::mapa_shared(ptx::smem_u32(&mine[w][0]), static_cast<uint32_t>(lane));
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(s_ab) : "memory");
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(s_eg) : "memory");
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(s_eb) : "memory");
                    }
                    __syncwarp();
                    ptx::cluster_sync_all();
                } else {
                    if (lane == 0) { mine[w][0] = s_ab; mine[w][1] = s_eg; mine[w][2] = s_eb; }
                    __syncthreads();
                }
                s_ab = s_eg = s_eb = 0.0f;
                for (int i = 0; i < ranks * warps; ++i) { s_ab += mine[i][0]; s_eg += mine[i][1]; s_eb += mine[i][2]; }
            }
            const float m_ab = s_ab * of;
            // mean(e g c), with the factors that a row shares (scale, rstd_post) outside
            const float m_eg = p.scale * now.r_post * of * fmaf(-now.r_pre * m_ab, s_eb, s_eg);
            Eight<TR, V> dx;
            Eight<TA, V> dy;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float dh = now.dh.at(i), b = now.out.at(i) * now.r_pre;
                const float g = fmaf(now.r_pre, fmaf(-b, m_ab, dh * w_pre[i]), now.dout.at(i));
                dx.put(i, g);
                acc_pre[i] = fmaf(dh, b, acc_pre[i]);
                const float c = now.y.at(i) * now.r_post, kg = p.scale * gate[i] * g;
                acc_post[i] = fmaf(kg, c, acc_post[i]);
                acc_gate[i] = fmaf(p.scale * g, c * e_w[i], acc_gate[i]);
                dy.put(i, post ? now.r_post * fmaf(-c, m_eg, kg * e_w[i]) : kg);
            }
            dx.store(static_cast<TR*>(p.dx) + row * p.ld_dx, first, step, cols);
            if (block) dy.store(static_cast<TA*>(p.dy) + row * p.ld_dy, first, step, cols);
        }
        if (p.part_gate != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) weight.put(i, acc_gate[i]);
            weight.store(p.part_gate + static_cast<int64_t>(u) * p.cols, first, step, cols);
        }
    }
    if (p.part_w != nullptr) {
        float* to = p.part_w + static_cast<int64_t>(me) * 2 * p.cols;
#pragma unroll
        for (int i = 0; i < 8; ++i) weight.put(i, acc_pre[i]);
        weight.store(to, first, step, cols);
#pragma unroll
        for (int i = 0; i < 8; ++i) weight.put(i, acc_post[i]);
        weight.store(to + p.cols, first, step, cols);
    }
}

// Sums of the blocks' rows in a fixed order: blockIdx.y 0 -> dw_pre, 1 -> dw_post, 2 + g -> dgate of group g.
constexpr int kSumCols = 32, kSumWays = 16;
__global__ void __launch_bounds__(kSumCols * kSumWays) norm_residual_sums_kernel(NormResidualParams p, int blocks, int64_t groups, int per_group, float beta) {
    __shared__ float part[kSumWays][kSumCols];
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x % kSumCols, way = threadIdx.x / kSumCols;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kSumCols + lane;
    for (int64_t what = blockIdx.y; what < 2 + groups; what += gridDim.y) {
        float* to = what == 0 ? p.dw_pre : what == 1 ? p.dw_post : p.dgate;
        if (to == nullptr) continue;
        const float* from = what < 2 ? p.part_w + what * p.cols : p.part_gate + (what - 2) * per_group * p.cols;
        const int64_t pitch = what < 2 ? 2 * static_cast<int64_t>(p.cols) : p.cols;
        const int n = what < 2 ? blocks : per_group;
        float s = 0.0f;
        if (col < p.cols)
            for (int i = way; i < n; i += kSumWays) s += from[i * pitch + col];
        part[way][lane] = s;
        __syncthreads();
        if (way == 0 && col < p.cols) {
#pragma unroll
            for (int i = 1; i < kSumWays; ++i) s += part[i][lane];
            to += what < 2 ? col : (what - 2) * p.cols + col;
            *to = beta == 0.0f ? s : fmaf(beta, *to, s);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------------------- launches

template <typename TR, typename TA, int V, int NV>
cudaError_t fwd_rows(const NormResidualParams& p, cudaStream_t stream) {
    const int warps = (p.cols + V * NV * 32 - 1) / (V * NV * 32);
    const int64_t blocks = warps == 1 ? (p.rows + kFwdRows - 1) / kFwdRows : p.rows;
    return launch_dependent(norm_residual_fwd_kernel<TR, TA, V, NV>, static_cast<unsigned>(blocks), 32u * (warps == 1 ? kFwdRows : warps), stream, p, warps);
}
template <typename TR, typename TA>
cudaError_t fwd_typed(const NormResidualParams& p, bool wide, cudaStream_t stream) {
    if (wide) return p.cols <= 256 ? fwd_rows<TR, TA, 8, 1>(p, stream) : p.cols <= 1024 ? fwd_rows<TR, TA, 8, 2>(p, stream) : fwd_rows<TR, TA, 8, 4>(p, stream);
    return p.cols <= 2048 ? fwd_rows<TR, TA, 1, 8>(p, stream) : fwd_rows<TR, TA, 1, 32>(p, stream);
}

template <typename TR, typename TA>
cudaError_t bwd_typed(const NormResidualParams& p, const NormResidualPlan& pl, bool wide, cudaStream_t stream) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(pl.cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(pl.blocks * pl.cluster));
    cfg.blockDim = dim3(32u * pl.warps);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = pl.cluster > 1 ? 2 : 1;
    auto kernel = pl.cluster > 1 ? (wide ? norm_residual_bwd_kernel<TR, TA, 8, true> : norm_residual_bwd_kernel<TR, TA, 1, true>)
                                 : (wide ? norm_residual_bwd_kernel<TR, TA, 8, false> : norm_residual_bwd_kernel<TR, TA, 1, false>);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, pl.units, pl.per_group);
    count_launch(1);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

int norm_residual_max_cols() { return 4 * kBwdCols; }

NormResidualPlan norm_residual_plan(int64_t rows, int64_t cols, int64_t groups, bool want_w, bool want_gate, int sms) {
    NormResidualPlan pl{};
    pl.cluster = static_cast<int>((cols + kBwdCols - 1) / kBwdCols);
    pl.warps = static_cast<int>((cols + pl.cluster * 256 - 1) / (pl.cluster * 256));
    // Blocks that share an SM hide each other's row sums; each of them leaves a row of sums behind, so none takes less
    // than eight rows while every SM has one.
    int64_t most = static_cast<int64_t>(sms) * (pl.warps <= 8 ? (16 / pl.warps > 8 ? 8 : 16 / pl.warps) : 1) / pl.cluster;
    if (most < 1) most = 1;
    const int64_t few = (rows + 7) / 8 > sms ? (rows + 7) / 8 : sms;
    if (most > few) most = few;
    if (most > rows) most = rows;
    const int64_t per_group_rows = rows / groups;
    int64_t per_group = most / groups > 0 ? most / groups : 1;
    if (per_group > per_group_rows) per_group = per_group_rows;
    pl.per_group = static_cast<int>(per_group);
    pl.units = static_cast<int>(groups * per_group);
    pl.blocks = static_cast<int>(pl.units < most ? pl.units : most);
    if (pl.blocks < 1) pl.blocks = 1;
    pl.floats_w = want_w ? 2 * cols * pl.blocks : 0;
    pl.floats_gate = want_gate ? cols * pl.units : 0;
    return pl;
}

cudaError_t launch_norm_residual_fwd(const NormResidualParams& p, int res_bf16, int act_bf16, bool wide, cudaStream_t stream) {
    if (res_bf16) return fwd_typed<__nv_bfloat16, __nv_bfloat16>(p, wide, stream);
    return act_bf16 ? fwd_typed<float, __nv_bfloat16>(p, wide, stream) : fwd_typed<float, float>(p, wide, stream);
}

cudaError_t launch_norm_residual_bwd(const NormResidualParams& p, const NormResidualPlan& pl, int res_bf16, int act_bf16, bool wide, float beta,
                                     cudaStream_t stream) {
    cudaError_t e = res_bf16   ? bwd_typed<__nv_bfloat16, __nv_bfloat16>(p, pl, wide, stream)
                    : act_bf16 ? bwd_typed<float, __nv_bfloat16>(p, pl, wide, stream)
                               : bwd_typed<float, float>(p, pl, wide, stream);
    if (e != cudaSuccess || (p.part_w == nullptr && p.part_gate == nullptr)) return e;
    const int64_t groups = p.part_gate != nullptr ? pl.units / pl.per_group : 0;
    const unsigned down = static_cast<unsigned>(2 + groups < 1024 ? 2 + groups : 1024);
    return launch_dependent(norm_residual_sums_kernel, dim3(static_cast<unsigned>((p.cols + kSumCols - 1) / kSumCols), down), kSumCols * kSumWays, stream,
                            p, pl.blocks, groups, pl.per_group, beta);
}

}  // namespace llmt_b200
