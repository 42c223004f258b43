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
// While the gate stays the same, dw_post and dgate are the same sum of g c, times scale gate and times scale w_post: one sum per
// block and piece of a gate's rows serves both.
//
// Bound: memory; every tensor is read and written once, all sums are fp32.  A block owns all columns, takes rows one after the
// other and keeps the weights of its columns in registers (read for every row they are more than the row).  A thread copies
// its own pieces of the rows to come into shared memory (cp.async, two or three rows ahead): what is under way takes no
// registers, and nobody else reads it, so nothing has to be waited for but the row sums.
// Measured at 8192 x 1600: forward (fp32 stream, bf16 block, both norms and the gate) 28.9 us, 157 MB at 5.4 TB/s; backward
// (bf16, a gate a sequence, all three weight gradients) 43.8 us, 157 MB with the sums' way through memory at 3.6 TB/s: its
// 420 instructions a row and warp keep the schedulers busy 60 % of the time, the row sums' exchange takes most of the rest (with
// 64 registers and four blocks an SM, which spill: 63 us; sums of three values in 6 exchanges for 15 and statistics loaded a row
// ahead: the same).  8 rows of 768: 6.9 us, launch and two row sums.
// Backward: a cluster of blocks owns a row of more than 4096 columns; the three weight gradients of a block's columns are in
// registers too, each block leaves one row of sums, and a second launch adds those in a fixed order.
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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Eight columns of a thread: V = 8 neighbours, or two groups of V = 4 neighbours or eight single ones (V = 1) that are the
// block's width apart.
template <typename T, int V> struct Eight {
    Vec<T, V> g[8 / V];
    __device__ __forceinline__ float at(int i) const { return to_float(g[i / V].v[i % V]); }
    __device__ __forceinline__ void put(int i, float x) { g[i / V].v[i % V] = rounded<T>(x); }
    // All eight; bf16 in pairs (a conversion of one value takes four times as long as that of two).
    __device__ __forceinline__ void put(const float (&x)[8]) {
        if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) put(i, x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(x[i], x[i + 1]);
                g[i / V].v[i % V] = reinterpret_cast<const T&>(two.x);
                g[(i + 1) / V].v[(i + 1) % V] = reinterpret_cast<const T&>(two.y);
            }
        }
    }
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

// A thread's eight columns of one tensor's row on their way through shared memory: `place` is where the thread's share begins in the
// tensor's part of a stage, [16-byte piece or value][thread].  Places whose columns are not there are never copied to: the
// kernels put zeros into all of them once.
template <typename T, int V> struct Staged {
    static constexpr int kUnit = V == 8 ? 16 : V * static_cast<int>(sizeof(T)), kUnits = 8 * static_cast<int>(sizeof(T)) / kUnit;
    static __device__ __forceinline__ void copy(uint8_t* to, const T* row, int first, int step, int cols) {
        const int threads = blockDim.x;
        if (V == 8) {
            if (first < cols) {
#pragma unroll
                for (int n = 0; n < kUnits; ++n)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(to + n * threads * kUnit)), "l"(row + first + n * (16 / sizeof(T))) : "memory");
            }
        } else if (kUnit == 16) {
#pragma unroll
            for (int n = 0; n < kUnits; ++n)
                if (first + n * step < cols)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(to + n * threads * kUnit)), "l"(row + first + n * step) : "memory");
        } else if (kUnit >= 4) {
#pragma unroll
            for (int n = 0; n < kUnits; ++n)
                if (first + n * step < cols)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(ptx::smem_u32(to + n * threads * kUnit)), "l"(row + first + n * step), "n"(kUnit < 4 ? 4 : kUnit) : "memory");
        } else {   // two bytes are no asynchronous copy
            T v[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) v[n] = first + n * step < cols ? row[first + n * step] : rounded<T>(0.0f);
#pragma unroll
            for (int n = 0; n < 8; ++n) *reinterpret_cast<T*>(to + n * threads * kUnit) = v[n];
        }
    }
    static __device__ __forceinline__ void get(Eight<T, V>& e, const uint8_t* from) {
        const int threads = blockDim.x;
        if (V == 8) {
            uint4 w[kUnits];
#pragma unroll
            for (int n = 0; n < kUnits; ++n) w[n] = *reinterpret_cast<const uint4*>(from + n * threads * kUnit);
            e = *reinterpret_cast<const Eight<T, V>*>(w);
        } else {
#pragma unroll
            for (int n = 0; n < kUnits; ++n) e.g[n] = *reinterpret_cast<const Vec<T, V>*>(from + n * threads * kUnit);
        }
    }
    static __device__ __forceinline__ uint8_t* place(uint8_t* part) { return part + threadIdx.x * kUnit; }
    static __device__ __forceinline__ void clear(uint8_t* to) {
        const int threads = blockDim.x;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
            if (kUnit == 16) *reinterpret_cast<uint4*>(to + n * threads * kUnit) = make_uint4(0, 0, 0, 0);
            else *reinterpret_cast<Vec<T, V>*>(to + n * threads * kUnit) = {};
        }
    }
};
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Of neighbours that a thread owns where alignment allows it: 16 bytes of a residual stream's row, so that what a warp accesses
// at once is contiguous (8192 x 1600 forward, an fp32 stream: 28.9 us, with eight neighbours in two accesses 37.4).
template <typename TR> constexpr int kWide = 16 / sizeof(TR);

constexpr int kMostWarps = 16;                  // of a block
constexpr int kMostCols = kMostWarps * 32 * 8;  // columns that a block owns eight a thread

// ------------------------------------------------------------------------------------------------------------ forward

// Rows in shared memory, the one at work among them: two (three were no faster), or what 200 KB hold of
// rows of more than 8192 columns.
template <typename TR, typename TA, int N> constexpr int fwd_depth() { return N < 4 ? 2 : sizeof(TR) + sizeof(TA) == 8 ? 1 : 2; }
// N: eights of columns of a thread, `threads` * 8 columns apart.
template <typename TR, typename TA, int V, int N>
__global__ void __launch_bounds__(kMostWarps * 32) norm_residual_fwd_kernel(NormResidualParams p) {
    extern __shared__ __align__(16) uint8_t stages[];
    __shared__ float4 part[2][2][kMostWarps / 4];
    constexpr int kDepth = fwd_depth<TR, TA, N>();
    ptx::grid_dependency_wait();
    const int threads = blockDim.x, warps = threads >> 5, lane = threadIdx.x & 31, me = threadIdx.x;
    const int first = me * V, step = threads * V;
    const bool block = p.y != nullptr, post = p.w_post != nullptr, pre = p.h != nullptr;
    const uint32_t of_x = threads * 8 * sizeof(TR), of_y = threads * 8 * sizeof(TA), stage_bytes = N * (of_x + of_y);
    auto cols_of = [&](int n) { return V == 8 ? p.cols - n * threads * 8 : min(p.cols - n * threads * 8, threads * 8); };   // of the n-th eight
    const float of = 1.0f / static_cast<float>(p.cols);
    const int64_t r0 = p.rows * blockIdx.x / gridDim.x, r1 = p.rows * (blockIdx.x + 1) / gridDim.x;

    if (me < kMostWarps) part[me / 8][me / 4 % 2][me % 4] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // warps that are not there
    __syncthreads();
    uint8_t* const mine_x = Staged<TR, V>::place(stages);
    uint8_t* const mine_y = Staged<TA, V>::place(stages + N * of_x);
    for (int s = 0; s < kDepth; ++s)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            Staged<TR, V>::clear(mine_x + s * stage_bytes + n * of_x);
            Staged<TA, V>::clear(mine_y + s * stage_bytes + n * of_y);
        }
    // the next row to copy, and the row at work
    const TR* next_x = static_cast<const TR*>(p.x) + r0 * p.ld_x;
    const TA* next_y = static_cast<const TA*>(p.y) + r0 * p.ld_y;
    TR* to_out = static_cast<TR*>(p.out) + r0 * p.ld_out;
    TA* to_h = static_cast<TA*>(p.h) + r0 * p.ld_h;
    auto copy = [&](bool there, int stage) {
        if (there) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                Staged<TR, V>::copy(mine_x + stage * stage_bytes + n * of_x, next_x + n * threads * 8, first, step, cols_of(n));
                if (block) Staged<TA, V>::copy(mine_y + stage * stage_bytes + n * of_y, next_y + n * threads * 8, first, step, cols_of(n));
            }
            next_x += p.ld_x;
            next_y += p.ld_y;
        }
        commit_copies();
    };
#pragma unroll
    for (int i = 0; i + 1 < kDepth; ++i) copy(r0 + i < r1, i);
    int stage = 0;
    // k = gate w_post, changed with the gate's row
    float k[N][8], w_pre[N][8];
    Eight<float, V> w;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        w.load(p.w_pre + n * threads * 8, first, step, cols_of(n), pre);
#pragma unroll
        for (int i = 0; i < 8; ++i) w_pre[n][i] = w.at(i);
    }
    auto load_k = [&](int64_t group) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            w.load(p.w_post + n * threads * 8, first, step, cols_of(n), post);
#pragma unroll
            for (int i = 0; i < 8; ++i) k[n][i] = post ? w.at(i) : 1.0f;
            if (p.gate != nullptr) {
                w.load(p.gate + group * p.cols + n * threads * 8, first, step, cols_of(n), true);
#pragma unroll
                for (int i = 0; i < 8; ++i) k[n][i] *= w.at(i);
            }
        }
    };
    // The sum over the block; two sets of places in turn, so that nobody writes one that is still read.
    int turn = 0;
    auto row_sum = [&](float s, int which) {
        s = warp_sum(s);
        if (warps == 1) return s;
        if (lane == 0) reinterpret_cast<float*>(part[turn][which])[me >> 5] = s;
        __syncthreads();
        s = 0.0f;
        for (int i = 0; i < warps; i += 4) {
            const float4 v = part[turn][which][i / 4];
            s += (v.x + v.y) + (v.z + v.w);
        }
        return s;
    };
    int64_t next_group = r0;   // first row of the next gate row
    for (int64_t row = r0; row < r1; ++row, to_out += p.ld_out, to_h += p.ld_h) {
        copy(row + kDepth - 1 < r1, stage == 0 ? kDepth - 1 : stage - 1);
        if (row == next_group) {
            const int64_t group = row / p.rows_per_gate;
            load_k(group);
            next_group = (group + 1) * p.rows_per_gate;
        }
        wait_copies<kDepth - 1>();
        Eight<TR, V> x[N];
        Eight<TA, V> y[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            Staged<TR, V>::get(x[n], mine_x + stage * stage_bytes + n * of_x);
            Staged<TA, V>::get(y[n], mine_y + stage * stage_bytes + n * of_y);
        }
        if (++stage == kDepth) stage = 0;
        float scale = p.scale, s = 0.0f;
        if (post) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(y[n].at(i), y[n].at(i), s);
            const float r = rsqrtf(fmaf(row_sum(s, 0), of, p.eps));
            if (me == 0 && p.rstd_post != nullptr) p.rstd_post[row] = r;
            scale *= r;
            s = 0.0f;
        }
        float z[N][8];
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[n][i] = block ? fmaf(scale * y[n].at(i), k[n][i], x[n].at(i)) : x[n].at(i);
                s = fmaf(z[n][i], z[n][i], s);
            }
            x[n].put(z[n]);
            if (block) x[n].store(to_out + n * threads * 8, first, step, cols_of(n));
        }
        if (pre) {
            const float r = rsqrtf(fmaf(row_sum(s, 1), of, p.eps));
            if (me == 0 && p.rstd_pre != nullptr) p.rstd_pre[row] = r;
#pragma unroll
            for (int n = 0; n < N; ++n) {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[n][i] *= r * w_pre[n][i];
                y[n].put(z[n]);
                y[n].store(to_h + n * threads * 8, first, step, cols_of(n));
            }
        }
        turn ^= 1;
    }
}

// ----------------------------------------------------------------------------------------------------------- backward

template <typename TR, typename TA> constexpr int bwd_depth() { return sizeof(TR) + sizeof(TA) == 8 ? 3 : 4; }

// `units` pieces of equal groups of rows (rows of one gate); block (cluster) b takes units b, b + grid, ...
// WARPS: of a block at most; of up to eight three blocks share an SM.
template <typename TR, typename TA, int V, bool CLUSTER, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 8 ? 3 : 1) norm_residual_bwd_kernel(NormResidualParams p, int units, int per_group) {
    extern __shared__ __align__(16) uint8_t stages[];
    __shared__ float4 part[2][4 * kMostWarps];   // of every warp of the cluster (up to four blocks)
    constexpr int kDepth = bwd_depth<TR, TA>();
    if (p.part_w != nullptr || p.part_gc != nullptr) ptx::grid_launch_dependents();   // the launch that adds the sums
    ptx::grid_dependency_wait();
    const int threads = blockDim.x, warps = threads >> 5;
    const int ranks = CLUSTER ? p.cluster : 1;
    const int rank = CLUSTER ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const int me = blockIdx.x / ranks, blocks = gridDim.x / ranks;
    const int first = rank * threads * 8 + static_cast<int>(threadIdx.x) * V, step = threads * V;
    const int cols = V == 8 ? p.cols : min(p.cols, (rank + 1) * threads * 8);
    const bool pre = p.dh != nullptr, block = p.y != nullptr, post = p.w_post != nullptr, more = p.dout != nullptr;
    const uint32_t of_r = threads * 8 * sizeof(TR), of_a = threads * 8 * sizeof(TA), stage_bytes = 2 * (of_r + of_a);
    const float of = 1.0f / static_cast<float>(p.cols);
    if (CLUSTER) ptx::cluster_sync_all();   // nobody writes into a block's shared memory before it runs

    Eight<float, V> weight;
    float w_pre[8], acc_pre[8];
    weight.load(p.w_pre, first, step, cols, pre);
#pragma unroll
    for (int i = 0; i < 8; ++i) { w_pre[i] = weight.at(i); acc_pre[i] = 0.0f; }

    uint8_t* const mine_r = Staged<TR, V>::place(stages);
    uint8_t* const mine_a = Staged<TA, V>::place(stages + 2 * of_r);
    for (int s = 0; s < kDepth; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            Staged<TR, V>::clear(mine_r + s * stage_bytes + n * of_r);
            Staged<TA, V>::clear(mine_a + s * stage_bytes + n * of_a);
        }

    int turn = 0;
    for (int u = me; u < units; u += blocks) {
        const int64_t group = u / per_group, part_of = u % per_group;
        const int64_t r0 = group * p.rows_per_gate + p.rows_per_gate * part_of / per_group;
        const int64_t r1 = group * p.rows_per_gate + p.rows_per_gate * (part_of + 1) / per_group;
        // the next row to copy, and the row at work
        const TR* next_out = static_cast<const TR*>(p.out) + r0 * p.ld_out;
        const TA* next_dh = static_cast<const TA*>(p.dh) + r0 * p.ld_dh;
        const TR* next_dout = static_cast<const TR*>(p.dout) + r0 * p.ld_dout;
        const TA* next_y = static_cast<const TA*>(p.y) + r0 * p.ld_y;
        TR* to_dx = static_cast<TR*>(p.dx) + r0 * p.ld_dx;
        TA* to_dy = static_cast<TA*>(p.dy) + r0 * p.ld_dy;
        auto copy = [&](bool there, int stage) {
            if (there) {
                uint8_t* const at = mine_r + stage * stage_bytes;
                uint8_t* const to = mine_a + stage * stage_bytes;
                if (pre) {
                    Staged<TR, V>::copy(at, next_out, first, step, cols);
                    Staged<TA, V>::copy(to, next_dh, first, step, cols);
                }
                if (more) Staged<TR, V>::copy(at + of_r, next_dout, first, step, cols);
                if (block) Staged<TA, V>::copy(to + of_a, next_y, first, step, cols);
                next_out += p.ld_out;
                next_dh += p.ld_dh;
                next_dout += p.ld_dout;
                next_y += p.ld_y;
            }
            commit_copies();
        };
        int stage = 0;
#pragma unroll
        for (int i = 0; i + 1 < kDepth; ++i) copy(r0 + i < r1, i);
        // k = scale gate w_post
        float k[8], sum_gc[8];
        Eight<float, V> gate;
        gate.load(p.gate + group * p.cols, first, step, cols, p.gate != nullptr);
        weight.load(p.w_post, first, step, cols, post);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k[i] = p.scale * (p.gate != nullptr ? gate.at(i) : 1.0f) * (post ? weight.at(i) : 1.0f);
            sum_gc[i] = 0.0f;
        }
        for (int64_t row = r0; row < r1; ++row, to_dx += p.ld_dx, to_dy += p.ld_dy) {
            copy(row + kDepth - 1 < r1, stage == 0 ? kDepth - 1 : stage - 1);
            const float r_pre = pre ? p.rstd_pre[row] : 0.0f, r_post = block && post ? p.rstd_post[row] : 1.0f;
            wait_copies<kDepth - 1>();
            const uint8_t* const at = mine_r + stage * stage_bytes;
            const uint8_t* const from = mine_a + stage * stage_bytes;
            if (++stage == kDepth) stage = 0;
            float b[8], c[8], q[8];   // q = dout + rstd_pre a
            float s_ab = 0.0f, s_eg = 0.0f, s_eb = 0.0f;
            {
                Eight<TR, V> o, d;
                Eight<TA, V> h, v;
                Staged<TR, V>::get(o, at);
                Staged<TR, V>::get(d, at + of_r);
                Staged<TA, V>::get(h, from);
                Staged<TA, V>::get(v, from + of_a);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // b and c are of ordinary size whatever the rows' is; products of rstd alone may leave the range
                    b[i] = o.at(i) * r_pre;
                    c[i] = v.at(i) * r_post;
                    const float a = h.at(i) * w_pre[i], ec = k[i] * c[i];
                    q[i] = fmaf(r_pre, a, d.at(i));
                    acc_pre[i] = fmaf(h.at(i), b[i], acc_pre[i]);
                    s_ab = fmaf(a, b[i], s_ab);
                    s_eg = fmaf(ec, q[i], s_eg);
                    s_eb = fmaf(ec, b[i], s_eb);
                }
            }
            s_ab = warp_sum(s_ab);
            if (block && post) {
                s_eg = warp_sum(s_eg);
                s_eb = warp_sum(s_eb);
            }
            if (CLUSTER || warps > 1) {
                // two turns of sums: whoever writes a third has seen everybody read the first
                float4* const mine = part[turn];
                turn ^= 1;
                const int lane = threadIdx.x & 31, w = rank * warps + (threadIdx.x >> 5);
                if (CLUSTER) {
                    if (lane < ranks) {
                        const uint32_t to = ptx::mapa_shared(ptx::smem_u32(&mine[w]), static_cast<uint32_t>(lane));
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(s_ab) : "memory");
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(s_eg) : "memory");
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(s_eb) : "memory");
                    }
                    __syncwarp();
                    ptx::cluster_sync_all();
                } else {
                    if (lane == 0) mine[w] = make_float4(s_ab, s_eg, s_eb, 0.0f);
                    __syncthreads();
                }
                s_ab = s_eg = s_eb = 0.0f;
                for (int i = 0; i < ranks * warps; ++i) {
                    const float4 v = mine[i];
                    s_ab += v.x;
                    s_eg += v.y;
                    s_eb += v.z;
                }
            }
            // g = q - b rstd_pre mean(a b);   dy = rstd_post (e g - c mean(e g c))
            const float m_ab = s_ab * of * r_pre;
            const float m_eg = post ? of * fmaf(-m_ab, s_eb, s_eg) : 0.0f;
            Eight<TR, V> dx;
            Eight<TA, V> dy;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[i] = fmaf(-b[i], m_ab, q[i]);
                sum_gc[i] = fmaf(q[i], c[i], sum_gc[i]);
                c[i] = post ? r_post * fmaf(-c[i], m_eg, k[i] * q[i]) : k[i] * q[i];   // without a norm y has no part in it, whatever it holds
            }
            dx.put(q);
            dy.put(c);
            dx.store(to_dx, first, step, cols);
            if (block) dy.store(to_dy, first, step, cols);
        }
        wait_copies<0>();   // the next unit's copies start anew
        if (p.part_gc != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) weight.put(i, sum_gc[i]);
            weight.store(p.part_gc + static_cast<int64_t>(u) * p.cols, first, step, cols);
        }
    }
    if (p.part_w != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) weight.put(i, acc_pre[i]);
        weight.store(p.part_w + static_cast<int64_t>(me) * p.cols, first, step, cols);
    }
}

// Sums of the blocks' rows in a fixed order: blockIdx.y 0 -> dw_pre, 1 -> dw_post, 2 + g -> dgate of group g.
constexpr int kSumCols = 16, kSumWays = 32;
__global__ void __launch_bounds__(kSumCols * kSumWays) norm_residual_sums_kernel(NormResidualParams p, int blocks, int units, int64_t groups, int per_group, float beta) {
    __shared__ float part[kSumWays][kSumCols];
    ptx::grid_dependency_wait();
    const int lane = threadIdx.x % kSumCols, way = threadIdx.x / kSumCols;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * kSumCols + lane;
    for (int64_t what = blockIdx.y; what < 2 + groups; what += gridDim.y) {
        float* to = what == 0 ? p.dw_pre : what == 1 ? p.dw_post : p.dgate;
        if (to == nullptr) continue;
        const float* from = what == 0 ? p.part_w : p.part_gc + (what == 1 ? 0 : (what - 2) * per_group * p.cols);
        const int n = what == 0 ? blocks : what == 1 ? units : per_group;
        float s = 0.0f;
        if (col < p.cols) {
            if (what == 1 && p.gate != nullptr) {
#pragma unroll 4
                for (int i = way; i < n; i += kSumWays) s = fmaf(p.gate[i / per_group * static_cast<int64_t>(p.cols) + col], from[i * static_cast<int64_t>(p.cols) + col], s);
            } else {
#pragma unroll 8
                for (int i = way; i < n; i += kSumWays) s += from[i * static_cast<int64_t>(p.cols) + col];
            }
        }
        part[way][lane] = s;
        __syncthreads();
        if (way == 0 && col < p.cols) {
#pragma unroll
            for (int i = 1; i < kSumWays; ++i) s += part[i][lane];
            if (what > 0) s *= p.scale;
            if (what > 1 && p.w_post != nullptr) s *= p.w_post[col];
            to += what < 2 ? col : (what - 2) * p.cols + col;
            *to = beta == 0.0f ? s : fmaf(beta, *to, s);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------------------- launches

// Blocks that share an SM, by its threads, shared memory and registers (`regs` a thread).
int blocks_per_sm(int warps, size_t smem, int regs) {
    const int by_threads = 64 / warps, by_smem = static_cast<int>((200u << 10) / (smem + 2048)), by_regs = 65536 / (warps * 32 * regs);
    int n = by_threads < by_smem ? by_threads : by_smem;
    n = n < by_regs ? n : by_regs;
    return n < 1 ? 1 : n > 16 ? 16 : n;
}

template <typename TR, typename TA, int V, int N>
cudaError_t fwd_rows(const NormResidualParams& p, int sms, cudaStream_t stream) {
    const int warps = (p.cols + N * 256 - 1) / (N * 256);
    const size_t smem = static_cast<size_t>(fwd_depth<TR, TA, N>()) * N * warps * 256 * (sizeof(TR) + sizeof(TA));
    auto kernel = norm_residual_fwd_kernel<TR, TA, V, N>;
    if (smem > 40 * 1024) {   // with what a block has beside it, 48 KB is the limit
        const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (set != cudaSuccess) return set;
    }
    const int64_t most = static_cast<int64_t>(sms) * blocks_per_sm(warps, smem, N == 1 ? 72 : 128);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows < most ? p.rows : most));
    cfg.blockDim = dim3(32u * warps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    count_launch(1);
    return e != cudaSuccess ? e : cudaGetLastError();
}
template <typename TR, typename TA>
cudaError_t fwd_typed(const NormResidualParams& p, bool wide, int sms, cudaStream_t stream) {
    if (wide) return p.cols <= kMostCols ? fwd_rows<TR, TA, kWide<TR>, 1>(p, sms, stream) : p.cols <= 2 * kMostCols ? fwd_rows<TR, TA, kWide<TR>, 2>(p, sms, stream) : fwd_rows<TR, TA, kWide<TR>, 4>(p, sms, stream);
    return p.cols <= kMostCols ? fwd_rows<TR, TA, 1, 1>(p, sms, stream) : p.cols <= 2 * kMostCols ? fwd_rows<TR, TA, 1, 2>(p, sms, stream) : fwd_rows<TR, TA, 1, 4>(p, sms, stream);
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
    cfg.dynamicSmemBytes = static_cast<size_t>(bwd_depth<TR, TA>()) * pl.warps * 512 * (sizeof(TR) + sizeof(TA));
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = pl.cluster > 1 ? 2 : 1;
    auto kernel = pl.cluster > 1 ? (wide ? norm_residual_bwd_kernel<TR, TA, kWide<TR>, true, 16> : norm_residual_bwd_kernel<TR, TA, 1, true, 16>)
                  : pl.warps > 8 ? (wide ? norm_residual_bwd_kernel<TR, TA, kWide<TR>, false, 16> : norm_residual_bwd_kernel<TR, TA, 1, false, 16>)
                                 : (wide ? norm_residual_bwd_kernel<TR, TA, kWide<TR>, false, 8> : norm_residual_bwd_kernel<TR, TA, 1, false, 8>);
    if (cfg.dynamicSmemBytes > 40 * 1024) {
        const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(cfg.dynamicSmemBytes));
        if (set != cudaSuccess) return set;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, pl.units, pl.per_group);
    count_launch(1);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

int norm_residual_max_cols() { return 4 * kMostCols; }

NormResidualPlan norm_residual_plan(int64_t rows, int64_t cols, int64_t groups, int row_bytes, bool want_pre, bool want_gc, int sms) {
    NormResidualPlan pl{};
    pl.cluster = static_cast<int>((cols + kMostCols - 1) / kMostCols);
    pl.warps = static_cast<int>((cols + pl.cluster * 256 - 1) / (pl.cluster * 256));
    // Blocks that share an SM hide each other's row sums; each of them leaves a row of sums behind, so none takes less
    // than two rows while every SM has one (1537 x 771 backward with sixteen rows or more each: 31 us, with two 17).
    int64_t most = static_cast<int64_t>(sms) * blocks_per_sm(pl.warps, static_cast<size_t>(row_bytes == 16 ? 3 : 4) * pl.warps * 256 * row_bytes, pl.warps > 8 ? 128 : 80) / pl.cluster;
    if (most < 1) most = 1;
    const int64_t few = (rows + 1) / 2 > sms ? (rows + 1) / 2 : sms;
    if (most > few) most = few;
    if (most > rows) most = rows;
    const int64_t per_group_rows = rows / groups;
    int64_t per_group = most / groups > 0 ? most / groups : 1;
    if (per_group > per_group_rows) per_group = per_group_rows;
    pl.per_group = static_cast<int>(per_group);
    pl.units = static_cast<int>(groups * per_group);
    pl.blocks = static_cast<int>(pl.units < most ? pl.units : most);
    if (pl.blocks < 1) pl.blocks = 1;
    pl.floats_w = want_pre ? cols * pl.blocks : 0;
    pl.floats_gc = want_gc ? cols * pl.units : 0;
    return pl;
}

cudaError_t launch_norm_residual_fwd(const NormResidualParams& p, int res_bf16, int act_bf16, bool wide, int sms, cudaStream_t stream) {
    if (res_bf16) return fwd_typed<__nv_bfloat16, __nv_bfloat16>(p, wide, sms, stream);
    return act_bf16 ? fwd_typed<float, __nv_bfloat16>(p, wide, sms, stream) : fwd_typed<float, float>(p, wide, sms, stream);
}

cudaError_t launch_norm_residual_bwd(const NormResidualParams& p, const NormResidualPlan& pl, int res_bf16, int act_bf16, bool wide, float beta,
                                     cudaStream_t stream) {
    cudaError_t e = res_bf16   ? bwd_typed<__nv_bfloat16, __nv_bfloat16>(p, pl, wide, stream)
                    : act_bf16 ? bwd_typed<float, __nv_bfloat16>(p, pl, wide, stream)
                               : bwd_typed<float, float>(p, pl, wide, stream);
    if (e != cudaSuccess || (p.part_w == nullptr && p.part_gc == nullptr)) return e;
    const int64_t groups = p.dgate != nullptr ? pl.units / pl.per_group : 0;
    const unsigned down = static_cast<unsigned>(2 + groups < 1024 ? 2 + groups : 1024);
    return launch_dependent(norm_residual_sums_kernel, dim3(static_cast<unsigned>((p.cols + kSumCols - 1) / kSumCols), down), kSumCols * kSumWays, stream,
                            p, pl.blocks, pl.units, groups, pl.per_group, beta);
}

}  // namespace llmt_b200
