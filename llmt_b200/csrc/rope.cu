// Rotary positions on the heads of a projection, forward and inverse (the gradient): see llmt_b200_rope in the public header.
//
// Mathematics.  A pair (u, w) of a head turns by the angle pos * f_i: (u cos - w sin, u sin + w cos), the inverse by minus it.
// fp32 has no angle for a far position (2^20 tokens in fp32 radians are off by 0.03), so the angle is kept as a fraction of
// a turn in 64-bit fixed point: F_i = f_i / 2 pi * 2^64, and pos * F_i modulo 2^64 is the angle without its whole turns, by
// one integer multiplication.  Its upper 32 bits, as a signed number, are the half-turns that sincospi takes.
//
// Bound: memory.  Every value is read and written once, in 16-byte accesses where the layout allows it; a sine and cosine
// serve all heads of their token through shared memory.
#include <cuda_bf16.h>

#include "common.h"
#include "ptx_sm100.cuh"

namespace llmt_b200 {
namespace {

constexpr int kRopeThreads = 256;

template <typename T, int V, int A> struct alignas(sizeof(T) * A) Pack { T v[V]; };   // V values that start on a multiple of A

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Turns per token of a frequency in radians, as a 64-bit fraction of a turn.
__device__ __forceinline__ uint64_t turns_u64(double radians) {
    const double t = radians * 0.15915494309189533577;   // 1 / 2 pi
    return __double2ull_rn((t - floor(t)) * 18446744073709551616.0);
}

// One block does `per_block` tokens: their sines and cosines first, then V values at a time of every head.  An item is
// a group of V values of the first of a pair and the group of their partners (half layout), a group of V values that holds
// V / 2 pairs (interleaved, V >= 2), or a group of V values behind the rotated ones that is copied.
template <typename T, int V, int A, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeParams p) {
    extern __shared__ float2 table[];   // [per_block][pairs] (cos, sin)
    ptx::grid_dependency_wait();
    const int pairs = p.rot / 2;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.per_block;
    const int count = static_cast<int>(p.total - first < p.per_block ? p.total - first : p.per_block);
    for (int i = threadIdx.x; i < count * pairs; i += kRopeThreads) {
        const int64_t t = first + i / pairs;
        const int64_t pos = p.positions != nullptr ? p.positions[t] : p.offset + t % p.tokens;
        const int64_t turn = static_cast<int64_t>(static_cast<uint64_t>(pos) * turns_u64(p.freqs[i % pairs]));
        float s, c;
        sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * (1.0f / 2147483648.0f), &s, &c);
        table[i] = make_float2(c * p.scale, p.inverse ? -s * p.scale : s * p.scale);
    }
    __syncthreads();
    using P = Pack<T, V, A>;
    const int turned = INTERLEAVED ? p.rot / V : pairs / V;
    constexpr int R = A == 1 ? 1 : V;   // what is copied may be odd in number where nothing is aligned
    using Rest = Pack<T, R, R>;
    const int items = turned + (p.copy_rest ? (p.head_dim - p.rot) / R : 0);
    const int per_token = items * p.heads;
    const int all = count * per_token;
    for (int i = threadIdx.x; i < all; i += kRopeThreads) {
        const int lt = i / per_token, rest = i % per_token, head = rest / items, it = rest % items;
        const int64_t t = first + lt, b = t / p.tokens, tok = t % p.tokens;
        const T* x = static_cast<const T*>(p.x) + b * p.x_batch + tok * p.x_token + head * p.x_head;
        T* y = static_cast<T*>(p.y) + b * p.y_batch + tok * p.y_token + head * p.y_head;
        const float2* cs = table + lt * pairs;
        if (it >= turned) {
            const int at = p.rot + (it - turned) * R;
            *reinterpret_cast<Rest*>(y + at) = *reinterpret_cast<const Rest*>(x + at);
        } else if (INTERLEAVED) {
            const int at = it * V;
            P u = *reinterpret_cast<const P*>(x + at);
#pragma unroll
            for (int k = 0; k + 1 < V; k += 2) {
                const float2 r = cs[(at + k) / 2];
                const float a = as_float(u.v[k]), w = as_float(u.v[k + 1]);
                u.v[k] = from_float<T>(a * r.x - w * r.y);
                u.v[k + 1] = from_float<T>(a * r.y + w * r.x);
            }
            *reinterpret_cast<P*>(y + at) = u;
        } else {
            const int at = it * V;
            P u = *reinterpret_cast<const P*>(x + at), w = *reinterpret_cast<const P*>(x + pairs + at);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float2 r = cs[at + k];
                const float a = as_float(u.v[k]), c = as_float(w.v[k]);
                u.v[k] = from_float<T>(a * r.x - c * r.y);
                w.v[k] = from_float<T>(a * r.y + c * r.x);
            }
            *reinterpret_cast<P*>(y + at) = u;
            *reinterpret_cast<P*>(y + pairs + at) = w;
        }
    }
}

// Whether every group of V values that the kernel touches starts on a multiple of V.
bool fits(const RopeParams& p, int v, int elem) {
    const int64_t part = p.interleaved ? p.rot : p.rot / 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y);
    return at % (static_cast<uintptr_t>(v) * elem) == 0 && (part | p.head_dim | p.x_batch | p.x_token | p.x_head | p.y_batch | p.y_token | p.y_head) % v == 0;
}

template <typename T, int V, int A, bool INTERLEAVED>
cudaError_t launch(RopeParams p, cudaStream_t stream) {
    const int64_t blocks = (p.total + p.per_block - 1) / p.per_block;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kRopeThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.per_block) * (p.rot / 2) * sizeof(float2);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, rope_kernel<T, V, A, INTERLEAVED>, p);
    count_launch(1);
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const RopeParams& p, cudaStream_t stream) {
    constexpr int kWide = 16 / sizeof(T);
    const bool wide = fits(p, kWide, sizeof(T));
    if (p.interleaved) return wide ? launch<T, kWide, kWide, true>(p, stream) : launch<T, 2, 1, true>(p, stream);
    return wide ? launch<T, kWide, kWide, false>(p, stream) : launch<T, 1, 1, false>(p, stream);
}

}  // namespace

cudaError_t launch_rope(RopeParams p, int is_bf16, cudaStream_t stream) {
    p.per_block = 8;
    return is_bf16 ? launch_typed<__nv_bfloat16>(p, stream) : launch_typed<float>(p, stream);
}

}  // namespace llmt_b200
