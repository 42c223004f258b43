// Causal attention with a sliding window and sinks, one row by one warp with plain loads and FMAs: for rows that came out of the
// tiles with values that are not finite.
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

// Neighbouring tokens' rows of one head.
struct Rows {
    const __nv_bfloat16* at;
    int64_t stride;
    __device__ __forceinline__ Rows(const HeadView& v, int64_t b, int64_t t, int64_t h) : at(row_of(v, b, t, h)), stride(v.stride_token) {}
    __device__ __forceinline__ const __nv_bfloat16* operator[](int n) const { return at + n * stride; }
};

// The product of one row with each of n <= 32 others, lane l has that with the l-th.  Half a warp takes a row, 16 bytes a lane, so
// that loads are in flight together; the sums over the lanes are exchanged so that each lane ends with one.
__device__ __forceinline__ float dots_with(const __nv_bfloat16* a, int n, int hd, const Rows& rows) {
    const int lane = threadIdx.x & 31, half = lane & 16, c = 8 * (lane & 15);
    const bool there = c < hd;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (there) x = *reinterpret_cast<const uint4*>(a + c);
    const __nv_bfloat16* from = rows[half] + c;
    float s[16];
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k0 = 0; k0 < 16; k0 += 8) {
        uint4 y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k, from += rows.stride) {
            y[k] = make_uint4(0, 0, 0, 0);
            if (there && half + k0 + k < n) y[k] = *reinterpret_cast<const uint4*>(from);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t ys[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
            s[k0 + k] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[k0 + k] = fmaf(hi_f(xs[i]), hi_f(ys[i]), fmaf(lo_f(xs[i]), lo_f(ys[i]), s[k0 + k]));
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < o; ++k) {
            const float mine = lane & o ? s[k + o] : s[k], other = lane & o ? s[k] : s[k + o];
            s[k] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
    return s[0];
}

// Four neighbouring values of a row for each lane (columns 4 lane ..): added with a weight, and stored.
struct Four {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    // The first n <= 32 rows with the lanes' weights (0 in lanes from n on).
    __device__ __forceinline__ void add(float w, int n, int hd, const Rows& rows) {
        const int c = 4 * (threadIdx.x & 31);
        const __nv_bfloat16* from = rows.at + c;
        for (int k = 0; k < n; k += 8) {
            uint2 x[8];
#pragma unroll
            for (int y = 0; y < 8; ++y, from += rows.stride) {
                x[y] = make_uint2(0, 0);
                if (c < hd && k + y < n) x[y] = *reinterpret_cast<const uint2*>(from);
            }
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                const float f = __shfl_sync(0xffffffffu, w, k + y);
                v[0] = fmaf(f, lo_f(x[y].x), v[0]);
                v[1] = fmaf(f, hi_f(x[y].x), v[1]);
                v[2] = fmaf(f, lo_f(x[y].y), v[2]);
                v[3] = fmaf(f, hi_f(x[y].y), v[3]);
            }
        }
    }
    __device__ __forceinline__ void store(__nv_bfloat16* row, float w, int hd) const {
        const int c = 4 * (threadIdx.x & 31);
        if (c >= hd) return;
        __nv_bfloat162 a = __floats2bfloat162_rn(v[0] * w, v[1] * w), b = __floats2bfloat162_rn(v[2] * w, v[3] * w);
        *reinterpret_cast<uint2*>(row + c) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
    }
};

// The keys that the query at position `pos` sees (pos < 0: none): `sinks` first ones, then [low, pos].  As two ranges: the first
// key of either, and one past its last.
struct Keys {
    int64_t sinks, low, count;
    __device__ __forceinline__ Keys(const AttentionParams& p, int64_t pos) {
        low = pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
        sinks = p.sinks < low ? p.sinks : low;
        count = pos < 0 ? 0 : sinks + pos - low + 1;
    }
    __device__ __forceinline__ int64_t at(int64_t n) const { return n < sinks ? n : low + n - sinks; }
    __device__ __forceinline__ int64_t begin(int range) const { return range == 0 ? 0 : low; }
    __device__ __forceinline__ int64_t end(int range) const { return count == 0 ? 0 : range == 0 ? sinks : low + count - sinks; }
};

// A row that came out of the tiles with values that are not finite.  A column is a sum of its own, so a finite one is right; of
// the others some hold what a visible operand holds, and some only 0 times a hidden value.  Which is which is read off the
// visible operand rows first, one value a column each (hundreds of times less work than scores); what is left, columns whose
// visible operands are finite, is summed again from visible places.  A training step whose values have become NaN so takes
// about as long as another.  4 heads on 2 x 2048 of 128, forward and backward (clean: 34 + 73 us): NaN everywhere 34 + 77, a
// column of v 52 + 93 (with all such rows summed again 2743 + 5892 and 2781 + 5935); one query NaN 34 + 765, since the keys
// behind it in its tile are summed again, up to 128 rows a head.
//
// Bit i stands for column 4 lane + i.
__device__ __forceinline__ uint32_t not_finite(const __nv_bfloat16* row, int hd) {
    const int c = 4 * (threadIdx.x & 31);
    if (c >= hd) return 0;
    const uint2 x = __ldcg(reinterpret_cast<const uint2*>(row + c));   // written by a copy out of shared memory a moment ago
    auto bit = [](float f, int i) { return fabsf(f) < INFINITY ? 0u : 1u << i; };
    return bit(lo_f(x.x), 0) | bit(hi_f(x.x), 1) | bit(lo_f(x.y), 2) | bit(hi_f(x.y), 3);
}

// What the operand rows of a sum hold, by columns.  ANY_IS_NAN: the factors of an infinite operand are 0 or NaN (it is part of a
// score, which it made infinite), else they are positive.
template <bool ANY_IS_NAN> struct Seen {
    // the bits of the largest and least values, two columns a word, as signed numbers: an infinity is 0x7F80 or, where the
    // negative ones are turned round, -0x7F81; beyond them are NaNs
    uint2 top = make_uint2(0, 0), least = make_uint2(0, 0);
    __device__ __forceinline__ uint32_t columns(bool at_infinity, bool upper) const {   // beyond an infinity, or from it on
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = upper ? (i < 2 ? top.x : top.y) : ~(i < 2 ? least.x : least.y);
            const int v = static_cast<int16_t>(i & 1 ? w >> 16 : w & 0xFFFFu);
            if (v >= (at_infinity ? 0x7F80 : 0x7F81)) r |= 1u << i;
        }
        return r;
    }
    __device__ __forceinline__ uint32_t is_nan() const {
        const uint32_t above = columns(true, true), below = columns(true, false);
        return columns(false, true) | columns(false, false) | (ANY_IS_NAN ? above | below : above & below);
    }
    __device__ __forceinline__ uint32_t any() const { return columns(true, true) | columns(true, false); }
    __device__ __forceinline__ void look(uint2 x) {
        const auto ordered = [](uint32_t w) { return w ^ ((w >> 15 & 0x10001u) * 0x7FFFu); };   // as sign and magnitude -> as a signed number
        top = make_uint2(__vmaxs2(top.x, ordered(x.x)), __vmaxs2(top.y, ordered(x.y)));
        least = make_uint2(__vmins2(least.x, ordered(x.x)), __vmins2(least.y, ordered(x.y)));
    }
    // n rows, until every column of `bad` in the warp is known to be NaN.
    __device__ __forceinline__ void scan(uint32_t bad, int64_t n, int hd, const Rows& rows) {
        const int c = 4 * (threadIdx.x & 31);
        const __nv_bfloat16* from = rows.at + c;
        for (int64_t k = 0; k < n && __any_sync(0xffffffffu, (bad & ~is_nan()) != 0); k += 16) {
            uint2 x[16];
#pragma unroll
            for (int y = 0; y < 16; ++y, from += rows.stride) {
                x[y] = make_uint2(0, 0);
                if (c < hd && k + y < n) x[y] = *reinterpret_cast<const uint2*>(from);
            }
#pragma unroll
            for (int y = 0; y < 16; ++y) look(x[y]);
        }
    }
    // Writes the columns of `bad` that this explains, and returns the others.
    __device__ __forceinline__ uint32_t settle(uint32_t bad, __nv_bfloat16* row) const {
        const uint32_t known = bad & any(), not_a_number = is_nan(), above = columns(true, true);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (known >> i & 1u) row[4 * (threadIdx.x & 31) + i] = __ushort_as_bfloat16(not_a_number >> i & 1u ? 0x7FFF : above >> i & 1u ? 0x7F80 : 0xFF80);
        return bad & ~known;
    }
};

// Columns `which` of a sum.
__device__ __forceinline__ void store_columns(const Four& s, uint32_t which, float w, __nv_bfloat16* row) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (which >> i & 1u) row[4 * (threadIdx.x & 31) + i] = __float2bfloat16_rn(s.v[i] * w);
}

// The output of the query at position `pos`.  Its log-sum-exp is finite (or -inf): no visible score is NaN.
static __device__ __noinline__ void forward_row(const AttentionParams& p, int64_t b, int64_t h, int64_t i, int64_t pos) {
    const int lane = threadIdx.x & 31, hd = p.head_dim;
    const int64_t hk = h / p.group;
    const __nv_bfloat16* q = row_of(p.q, b, i, h);
    __nv_bfloat16* const to = row_to(p.out, b, i, h);
    const Keys keys(p, pos);
    uint32_t bad = not_finite(to, hd);
    Seen<false> seen;
    for (int range = 0; range < 2; ++range) seen.scan(bad, keys.end(range) - keys.begin(range), hd, Rows(p.v, b, keys.begin(range), hk));
    bad = seen.settle(bad, to);
    if (!__any_sync(0xffffffffu, bad != 0)) return;
    float m = -INFINITY, l = 0.0f;
    Four o;
    for (int range = 0; range < 2; ++range)
        for (int64_t j0 = keys.begin(range); j0 < keys.end(range); j0 += 32) {
            const int here = static_cast<int>(keys.end(range) - j0 < 32 ? keys.end(range) - j0 : 32);
            float s = p.scale * dots_with(q, here, hd, Rows(p.k, b, j0, hk));
            if (lane >= here) s = -INFINITY;
            const float m_new = fmaxf(m, warp_max(s)), from = m_new == -INFINITY ? 0.0f : m_new;
            const float e = expf(s - from), shrink = expf(m - from);
            l = l * shrink + warp_add(e);
#pragma unroll
            for (float& x : o.v) x *= shrink;
            m = m_new;
            o.add(e, here, hd, Rows(p.v, b, j0, hk));
        }
    store_columns(o, bad, l == 0.0f ? 0.0f : 1.0f / l, to);
}

// A row of dQ, of which no visible dS is NaN.
static __device__ __noinline__ void dq_row(const AttentionParams& p, int64_t b, int64_t h, int64_t i, float d) {
    const int lane = threadIdx.x & 31, hd = p.head_dim;
    const int64_t hk = h / p.group;
    const __nv_bfloat16 *q = row_of(p.q, b, i, h), *dout = row_of(p.dout, b, i, h);
    __nv_bfloat16* const to = row_to(p.dq, b, i, h);
    const Keys keys(p, i + p.tk - p.tq);
    uint32_t bad = not_finite(to, hd);
    Seen<true> seen;
    for (int range = 0; range < 2; ++range) seen.scan(bad, keys.end(range) - keys.begin(range), hd, Rows(p.k, b, keys.begin(range), hk));
    bad = seen.settle(bad, to);
    if (!__any_sync(0xffffffffu, bad != 0)) return;
    const float lse = p.lse[(b * p.heads + h) * p.tq + i];
    Four dq;
    for (int range = 0; range < 2; ++range)
        for (int64_t j0 = keys.begin(range); j0 < keys.end(range); j0 += 32) {
            const int here = static_cast<int>(keys.end(range) - j0 < 32 ? keys.end(range) - j0 : 32);
            const float s = p.scale * dots_with(q, here, hd, Rows(p.k, b, j0, hk)), dp = dots_with(dout, here, hd, Rows(p.v, b, j0, hk));
            const float ds = lane < here ? (lse == -INFINITY ? 0.0f : expf(s - lse)) * (dp - d) : 0.0f;
            dq.add(ds, here, hd, Rows(p.k, b, j0, hk));
        }
    store_columns(dq, bad, p.scale, to);
}

// A row of dK and dV: the sums over the group's heads and the queries that see key j.
static __device__ __noinline__ void dkdv_row(const AttentionParams& p, int64_t b, int64_t hk, int64_t j) {
    const int lane = threadIdx.x & 31, hd = p.head_dim;
    const __nv_bfloat16 *k = row_of(p.k, b, j, hk), *v = row_of(p.v, b, j, hk);
    __nv_bfloat16 *const to_k = row_to(p.dk, b, j, hk), *const to_v = row_to(p.dv, b, j, hk);
    const int64_t off = static_cast<int64_t>(p.tk) - p.tq;
    const int64_t first = j - off > 0 ? j - off : 0;
    const int64_t last = j < p.sinks || j + p.window >= p.tk ? p.tq : j + p.window - off;   // one past the last query
    uint32_t bad_k = not_finite(to_k, hd), bad_v = not_finite(to_v, hd);
    // A query whose log-sum-exp is NaN makes NaN of P and dS, one whose D is, of dS: all columns of the products are NaN then.
    bool nan_p = false, nan_ds = false;
    for (int64_t h = hk * p.group; h < (hk + 1) * p.group && !nan_p; ++h)
        for (int64_t i0 = first; i0 < last && !nan_p; i0 += 128) {
            bool x = false, y = false;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int64_t i = i0 + n * 32 + lane, at = (b * p.heads + h) * p.tq + i;
                if (i >= last) continue;
                const float lse = p.lse[at], d = p.dvec[at];
                x = x || lse != lse;
                y = y || d != d;
            }
            nan_p = __any_sync(0xffffffffu, x);
            nan_ds = nan_ds || __any_sync(0xffffffffu, y);
        }
    if (nan_p) return;
    if (nan_ds) bad_k = 0;
    Seen<true> seen_k;
    Seen<false> seen_v;
    for (int64_t h = hk * p.group; h < (hk + 1) * p.group; ++h) {
        seen_k.scan(bad_k, last - first, hd, Rows(p.q, b, first, h));
        seen_v.scan(bad_v, last - first, hd, Rows(p.dout, b, first, h));
    }
    bad_k = seen_k.settle(bad_k, to_k);
    bad_v = seen_v.settle(bad_v, to_v);
    if (!__any_sync(0xffffffffu, (bad_k | bad_v) != 0)) return;
    Four dk, dv;
    for (int64_t h = hk * p.group; h < (hk + 1) * p.group; ++h)
        for (int64_t i0 = first; i0 < last; i0 += 32) {
            const int here = static_cast<int>(last - i0 < 32 ? last - i0 : 32);
            const int64_t at = (b * p.heads + h) * p.tq + i0 + lane;
            const float lse = lane < here ? p.lse[at] : -INFINITY, d = lane < here ? p.dvec[at] : 0.0f;
            const float s = p.scale * dots_with(k, here, hd, Rows(p.q, b, i0, h)), dp = dots_with(v, here, hd, Rows(p.dout, b, i0, h));
            const float e = lse == -INFINITY ? 0.0f : expf(s - lse), ds = e * (dp - d);
            dv.add(e, here, hd, Rows(p.dout, b, i0, h));
            dk.add(ds, here, hd, Rows(p.q, b, i0, h));
        }
    store_columns(dk, bad_k, p.scale, to_k);
    store_columns(dv, bad_v, 1.0f, to_v);
}

}  // namespace attn
}  // namespace llmt_b200
