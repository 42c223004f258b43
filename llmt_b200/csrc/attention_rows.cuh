// Causal attention with a sliding window and sinks, one row by one warp with plain loads and FMAs.
//
// A query at position p = i + tk - tq sees key j when j <= p and (j > p - window or j < sinks).  The functions here touch
// visible pairs only, so nothing that a hidden key or query holds reaches a result.
#pragma once

#include <cuda_bf16.h>

#include "common.h"

namespace llmt_b200 {
namespace attn {

__device__ __forceinline__ const __nv_bfloat16* row_of(const HeadView& v, int64_t b, int64_t t, int64_t h) {
    return static_cast<const __nv_bfloat16*>(v.data) + b * v.stride_batch + t * v.stride_token + h * v.stride_head;
}
__device__ __forceinline__ __nv_bfloat16* row_to(const HeadView& v, int64_t b, int64_t t, int64_t h) {
    return static_cast<__nv_bfloat16*>(v.data) + b * v.stride_batch + t * v.stride_token + h * v.stride_head;
}

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Product of two rows of n values (a multiple of 8), 16 bytes at a time.
__device__ __forceinline__ float dot_rows(const __nv_bfloat16* a, const __nv_bfloat16* b, int n) {
    float s = 0.0f;
    for (int d = 0; d < n; d += 8) {
        const uint4 x = *reinterpret_cast<const uint4*>(a + d), y = *reinterpret_cast<const uint4*>(b + d);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fmaf(hi_f(xs[i]), hi_f(ys[i]), fmaf(lo_f(xs[i]), lo_f(ys[i]), s));
    }
    return s;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Four neighbouring values of a row for each lane (columns 4 lane ..): added with a weight, and stored.
struct Four {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    __device__ __forceinline__ void add(const __nv_bfloat16* row, float w, int hd) {
        const int c = 4 * (threadIdx.x & 31);
        if (c >= hd) return;
        const uint2 x = *reinterpret_cast<const uint2*>(row + c);
        v[0] = fmaf(w, lo_f(x.x), v[0]);
        v[1] = fmaf(w, hi_f(x.x), v[1]);
        v[2] = fmaf(w, lo_f(x.y), v[2]);
        v[3] = fmaf(w, hi_f(x.y), v[3]);
    }
    __device__ __forceinline__ void store(__nv_bfloat16* row, float w, int hd) const {
        const int c = 4 * (threadIdx.x & 31);
        if (c >= hd) return;
        __nv_bfloat162 a = __floats2bfloat162_rn(v[0] * w, v[1] * w), b = __floats2bfloat162_rn(v[2] * w, v[3] * w);
        *reinterpret_cast<uint2*>(row + c) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    }
};

// The keys that the query at position `pos` sees (pos < 0: none): `sinks` first ones, then [low, pos].
struct Keys {
    int64_t sinks, low, count;
    __device__ __forceinline__ Keys(const AttentionParams& p, int64_t pos) {
        low = pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
        sinks = p.sinks < low ? p.sinks : low;
        count = pos < 0 ? 0 : sinks + pos - low + 1;
    }
    __device__ __forceinline__ int64_t at(int64_t n) const { return n < sinks ? n : low + n - sinks; }
};

// One row of the output and its log-sum-exp, for the query at position `pos`.
static __device__ __noinline__ void forward_row(const AttentionParams& p, int64_t b, int64_t h, int64_t i, int64_t pos) {
    const int lane = threadIdx.x & 31, hd = p.head_dim;
    const int64_t hk = h / p.group;
    const __nv_bfloat16* q = row_of(p.q, b, i, h);
    const Keys keys(p, pos);
    float m = -INFINITY, l = 0.0f;
    Four o;
    for (int64_t n0 = 0; n0 < keys.count; n0 += 32) {
        const int64_t n = n0 + lane;
        const float s = n < keys.count ? p.scale * dot_rows(q, row_of(p.k, b, keys.at(n), hk), hd) : -INFINITY;
        const float m_new = fmaxf(m, warp_max(s)), from = m_new == -INFINITY ? 0.0f : m_new;
        const float e = expf(s - from), shrink = expf(m - from);
        l = l * shrink + warp_add(e);
#pragma unroll
        for (float& x : o.v) x *= shrink;
        m = m_new;
        const int here = static_cast<int>(keys.count - n0 < 32 ? keys.count - n0 : 32);
        for (int k = 0; k < here; ++k) o.add(row_of(p.v, b, keys.at(n0 + k), hk), __shfl_sync(0xffffffffu, e, k), hd);
    }
    o.store(row_to(p.out, b, i, h), l == 0.0f ? 0.0f : 1.0f / l, hd);
    if (lane == 0 && p.lse != nullptr) p.lse[(b * p.heads + h) * p.tq + i] = l == 0.0f ? -INFINITY : m + logf(l);
}

// One row of dQ.
static __device__ __noinline__ void dq_row(const AttentionParams& p, int64_t b, int64_t h, int64_t i, float d) {
    const int lane = threadIdx.x & 31, hd = p.head_dim;
    const int64_t hk = h / p.group;
    const __nv_bfloat16 *q = row_of(p.q, b, i, h), *dout = row_of(p.dout, b, i, h);
    const float lse = p.lse[(b * p.heads + h) * p.tq + i];
    const Keys keys(p, i + p.tk - p.tq);
    Four dq;
    for (int64_t n0 = 0; n0 < keys.count; n0 += 32) {
        const int64_t n = n0 + lane;
        float ds = 0.0f;
        if (n < keys.count) {
            const int64_t j = keys.at(n);
            const float e = lse == -INFINITY ? 0.0f : expf(p.scale * dot_rows(q, row_of(p.k, b, j, hk), hd) - lse);
            ds = e * (dot_rows(dout, row_of(p.v, b, j, hk), hd) - d);
        }
        const int here = static_cast<int>(keys.count - n0 < 32 ? keys.count - n0 : 32);
        for (int k = 0; k < here; ++k) dq.add(row_of(p.k, b, keys.at(n0 + k), hk), __shfl_sync(0xffffffffu, ds, k), hd);
    }
    dq.store(row_to(p.dq, b, i, h), p.scale, hd);
}

// One row of dK and dV: the sums over the group's heads and the queries that see key j.
static __device__ __noinline__ void dkdv_row(const AttentionParams& p, int64_t b, int64_t hk, int64_t j) {
    const int lane = threadIdx.x & 31, hd = p.head_dim;
    const __nv_bfloat16 *k = row_of(p.k, b, j, hk), *v = row_of(p.v, b, j, hk);
    const int64_t off = static_cast<int64_t>(p.tk) - p.tq;
    const int64_t first = j - off > 0 ? j - off : 0;
    const int64_t last = j < p.sinks || j + p.window >= p.tk ? p.tq : j + p.window - off;   // one past the last query
    Four dk, dv;
    for (int64_t h = hk * p.group; h < (hk + 1) * p.group && h < p.heads; ++h)
        for (int64_t i0 = first; i0 < last; i0 += 32) {
            const int64_t i = i0 + lane;
            float e = 0.0f, ds = 0.0f;
            if (i < last) {
                const int64_t at = (b * p.heads + h) * p.tq + i;
                const float lse = p.lse[at];
                e = lse == -INFINITY ? 0.0f : expf(p.scale * dot_rows(row_of(p.q, b, i, h), k, hd) - lse);
                ds = e * (dot_rows(row_of(p.dout, b, i, h), v, hd) - p.dvec[at]);
            }
            const int here = static_cast<int>(last - i0 < 32 ? last - i0 : 32);
            for (int n = 0; n < here; ++n) {
                dv.add(row_of(p.dout, b, i0 + n, h), __shfl_sync(0xffffffffu, e, n), hd);
                dk.add(row_of(p.q, b, i0 + n, h), __shfl_sync(0xffffffffu, ds, n), hd);
            }
        }
    dk.store(row_to(p.dk, b, j, hk), p.scale, hd);
    dv.store(row_to(p.dv, b, j, hk), 1.0f, hd);
}

}  // namespace attn
}  // namespace llmt_b200
