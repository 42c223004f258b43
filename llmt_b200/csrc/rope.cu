// Rotary positions on the heads of a projection, forward and inverse (the gradient): see llmt_b200_rope in the public header.
//
// Mathematics.  A pair (u, w) of a head turns by the angle pos * f_i: (u cos - w sin, u sin + w cos), the inverse by minus it.
// fp32 has no angle for a far position (2^20 tokens in fp32 radians are off by 0.03), so the angle is kept as a fraction of
// a turn in 64-bit fixed point: F_i = f_i / 2 pi * 2^64, and pos * F_i modulo 2^64 is the angle without its whole turns, by
// one integer multiplication.  Its upper 32 bits, as a signed number, are the half-turns that sincospi takes.
//
// Bound: memory.  Every value is read and written once, in 16-byte accesses where the layout allows it; a sine and cosine
// serve all heads of their token through shared memory.  Measured: 4.2 us for 8 tokens of 24 heads of 64 (a
// launch), 12.2 us at 4.1 TB/s for 8192 tokens of 24 heads of 64 in rows of 36 (50 MB), 137 us at 4.9 TB/s for 32768 tokens
// of 40 heads of 128, of which 64 values turn and 64 are copied (671 MB); a copy of as much takes 7.7 and 102 us.
#include <cuda_bf16.h>

#include "common.h"
#include "ptx_sm100.cuh"

namespace llmt_b200 {
namespace {

constexpr int kRopeThreads = 256;   // at most

template <typename T, int V, int A> struct alignas(sizeof(T) * A) Pack { T v[V]; };   // V values that start on a multiple of A

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
// Two values rounded (one bf16 conversion of two takes a quarter of the time of two of one).
__device__ __forceinline__ void from_floats(float& x, float& y, float a, float b) { x = a; y = b; }
__device__ __forceinline__ void from_floats(__nv_bfloat16& x, __nv_bfloat16& y, float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    x = v.x;
    y = v.y;
}

// Turns per token of a frequency in radians, as a 64-bit fraction of a turn.
__device__ __forceinline__ uint64_t turns_u64(double radians) {
    const double t = radians * 0.15915494309189533577;   // 1 / 2 pi
    return __double2ull_rn((t - floor(t)) * 18446744073709551616.0);
}

// One block does `per_block` tokens of a sequence: their sines and cosines, then V values at a time of every head.  An item is
// a group of V values of the first of a pair and the group of their partners (half layout), a group of V values that holds
// V / 2 pairs (interleaved, V >= 2), or a group of values behind the rotated ones that is copied.  A thread has one item of one
// head in several tokens, so that head and item are worked out once; kAhead tokens' loads are under way at a time, the first
// of them while the sines are formed.  What hides the memory's latency best is the number of blocks, not a thread's loads: the
// long case above takes 137 us with one, 166 with two (in half the blocks), 213 with four.
constexpr int kAhead = 1;
template <typename T, int V, int A, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads, 6) rope_kernel(RopeParams p) {
    extern __shared__ float4 raw[];
    float2* const table = reinterpret_cast<float2*>(raw);   // [per_block][pairs] (cos, sin)
    ptx::grid_dependency_wait();
    const int pairs = p.rot / 2;
    const int64_t b = blockIdx.x / p.blocks_per_sequence;
    const int first = static_cast<int>(blockIdx.x % p.blocks_per_sequence) * p.per_block;
    const int count = static_cast<int>(p.tokens - first < p.per_block ? p.tokens - first : p.per_block);
    using P = Pack<T, V, A>;
    constexpr int R = A == 1 ? 1 : V;   // what is copied may be odd in number where nothing is aligned
    using Rest = Pack<T, R, R>;
    const int turned = INTERLEAVED ? p.rot / V : pairs / V;
    const int items = turned + (p.copy_rest ? (p.head_dim - p.rot) / R : 0);
    const int per_token = items * p.heads;
    // `lanes` tokens side by side where a token has fewer items than the block threads
    const int lanes = per_token < static_cast<int>(blockDim.x) ? blockDim.x / per_token : 1;
    const int lane = lanes > 1 ? threadIdx.x / per_token : 0;
    int e = lanes > 1 ? threadIdx.x % per_token : threadIdx.x;
    if (lane >= lanes) e = per_token;   // helps with the sines only
    const int64_t hop_x = lanes * p.x_token, hop_y = lanes * p.y_token;
    const T* const x0 = static_cast<const T*>(p.x) + b * p.x_batch + (static_cast<int64_t>(first) + lane) * p.x_token;
    T* const y0 = static_cast<T*>(p.y) + b * p.y_batch + (static_cast<int64_t>(first) + lane) * p.y_token;
    P u[kAhead], w[kAhead];
    auto load = [&](const T* x, int t0, bool rest) {   // (w is the partner)
#pragma unroll
        for (int k = 0; k < kAhead; ++k, x += hop_x) {
            if (t0 + k * lanes >= count) break;
            if (rest) {
                reinterpret_cast<Rest&>(u[k]) = *reinterpret_cast<const Rest*>(x);
            } else {
                u[k] = *reinterpret_cast<const P*>(x);
                if (!INTERLEAVED) w[k] = *reinterpret_cast<const P*>(x + pairs);
            }
        }
    };
    auto place = [&](int item) { return item >= turned ? p.rot + (item - turned) * R : item * V; };
    if (e < per_token) load(x0 + e / items * p.x_head + place(e % items), lane, e % items >= turned);

    for (int i = threadIdx.x; i < count * pairs; i += blockDim.x) {
        const int64_t t = first + i / pairs;
        const int64_t pos = p.positions != nullptr ? p.positions[b * p.tokens + t] : p.offset + t;
        const int64_t turn = static_cast<int64_t>(static_cast<uint64_t>(pos) * turns_u64(p.freqs[i % pairs]));
        float s, c;
        sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * (1.0f / 2147483648.0f), &s, &c);
        table[i] = make_float2(c * p.scale, p.inverse ? -s * p.scale : s * p.scale);
    }
    __syncthreads();
    const int hop = lanes > 1 ? per_token : blockDim.x;
    for (bool loaded = true; e < per_token; e += hop) {
        const int head = e / items, it = e % items, at = place(it);
        const bool rest = it >= turned;
        const T* x = x0 + head * p.x_head + at;
        T* y = y0 + head * p.y_head + at;
        for (int t0 = lane; t0 < count; t0 += kAhead * lanes, x += kAhead * hop_x) {
            if (!loaded) load(x, t0, rest);
            loaded = false;
#pragma unroll
            for (int k = 0; k < kAhead; ++k, y += hop_y) {
                if (t0 + k * lanes >= count) break;
                if (rest) {
                    *reinterpret_cast<Rest*>(y) = reinterpret_cast<Rest&>(u[k]);
                    continue;
                }
                const float2* cs = table + (t0 + k * lanes) * pairs + (INTERLEAVED ? at / 2 : at);
                if (INTERLEAVED) {
#pragma unroll
                    for (int i = 0; i + 1 < V; i += 2) {
                        const float2 r = cs[i / 2];
                        const float a = as_float(u[k].v[i]), c = as_float(u[k].v[i + 1]);
                        from_floats(u[k].v[i], u[k].v[i + 1], a * r.x - c * r.y, a * r.y + c * r.x);
                    }
                    *reinterpret_cast<P*>(y) = u[k];
                } else {
#pragma unroll
                    for (int i = 0; i < V; i += 2) {   // two neighbours, so that they round together
                        constexpr int kNext = V > 1 ? 1 : 0;
                        const float2 r = cs[i], s = cs[i + kNext];
                        const float a = as_float(u[k].v[i]), c = as_float(w[k].v[i]), d = as_float(u[k].v[i + kNext]), f = as_float(w[k].v[i + kNext]);
                        if (V > 1) {
                            from_floats(u[k].v[i], u[k].v[i + kNext], a * r.x - c * r.y, d * s.x - f * s.y);
                            from_floats(w[k].v[i], w[k].v[i + kNext], a * r.y + c * r.x, d * s.y + f * s.x);
                        } else {
                            from_floats(u[k].v[i], w[k].v[i], a * r.x - c * r.y, a * r.y + c * r.x);
                        }
                    }
                    *reinterpret_cast<P*>(y) = u[k];
                    *reinterpret_cast<P*>(y + pairs) = w[k];
                }
            }
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
    // Threads: whole tokens' items where they fit, else a share of one's that leaves few idle.
    const int rest = p.copy_rest ? (p.head_dim - p.rot) / (A == 1 ? 1 : V) : 0;
    const int64_t per_token = static_cast<int64_t>((INTERLEAVED ? p.rot / V : p.rot / 2 / V) + rest) * p.heads;
    const int64_t passes = (per_token + kRopeThreads - 1) / kRopeThreads;
    const int64_t want = passes <= 1 ? per_token * (kRopeThreads / per_token) : (per_token + passes - 1) / passes;
    const int threads = static_cast<int>((want + 31) / 32 * 32);
    const int64_t blocks = p.batch * p.blocks_per_sequence;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
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

cudaError_t launch_rope(RopeParams p, int is_bf16, int sms, cudaStream_t stream) {
    // Eight tokens a block, fewer where the blocks would not reach every SM four times.
    p.per_block = 8;
    while (p.per_block > 1 && p.batch * ((p.tokens + p.per_block - 1) / p.per_block) < 4 * sms) p.per_block /= 2;
    p.blocks_per_sequence = (p.tokens + p.per_block - 1) / p.per_block;
    return is_bf16 ? launch_typed<__nv_bfloat16>(p, stream) : launch_typed<float>(p, stream);
}

}  // namespace llmt_b200
