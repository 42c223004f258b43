// Causal attention with a sliding window and sinks on the tensor cores: see llmt_b200_attention_window_fwd in the public header.
//
// Mathematics.  One pass over the visible keys with a running maximum m and sum l per query:
//   S = Q K^T;  P = 2^(c S - c m) on visible places, else 0;  O = O 2^(c m_old - c m) + P V;  out = O / l,
// c = scale log2 e.  O is only rescaled where m grows by more than 2^8: until then P is up to 2^8 too large, which the
// same factor in l takes out again, and bf16 keeps its relative precision.
#include <cuda_bf16.h>

#include "attention_rows.cuh"
#include "common.h"
#include "ptx_sm100.cuh"
#include "waits_sm100.cuh"

namespace llmt_b200 {
namespace {

using namespace ptx;

constexpr int kRows = 128;                      // queries of a softmax warpgroup, keys of a tile
constexpr uint32_t kHalfTile = kRows * 128;     // 128 rows of 64 bf16 values, 128-byte swizzle
constexpr float kLog2e = 1.4426950408889634f;

struct alignas(64) AttentionMaps {
    CUtensorMap q, k, v, out, dout, dq, dk, dv;
};

// The high word of a shared-memory descriptor: 8-row groups of 1024 bytes, version 1, 128-byte swizzle.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t smem_desc(uint32_t at, uint32_t lbo) {
    return (static_cast<uint64_t>(kDescHi) << 32) | ((lbo >> 4) << 16) | (at >> 4);
}

// Bits [lo, hi) of a word that stands for places [base, base + 32).
__device__ __forceinline__ uint32_t bits_between(int lo, int hi, int base) {
    lo = max(lo - base, 0);
    hi = min(hi - base, 32);
    if (hi <= lo) return 0;
    return (0xFFFFFFFFu >> (32 - (hi - lo))) << lo;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// What a block of queries [r0, r0 + 128) of one head sees, in tiles of keys.
struct QueryBlock {
    int head, r0;
    int p0, p1;                // positions of the first and the last query
    int low, high, sinks;      // tiles [0, sinks) and [low, high]
    bool any;
    __device__ __forceinline__ QueryBlock(const AttentionParams& p, int head_, int r0_) {
        head = head_;
        r0 = r0_;
        p0 = r0 + p.tk - p.tq;
        p1 = min(r0 + kRows, p.tq) - 1 + p.tk - p.tq;
        any = r0 < p.tq && p1 >= 0;
        const int first = max(0, p0 - p.window + 1);
        low = first / kRows;
        high = p1 / kRows;
        sinks = min((min(p.sinks, first) + kRows - 1) / kRows, low);
    }
    __device__ __forceinline__ bool sees(int tile) const { return any && tile <= high && (tile >= low || tile < sinks); }
    // Every query sees every key of [j0, j0 + n).
    __device__ __forceinline__ bool sees_all(const AttentionParams& p, int j0, int n) const {
        return j0 + n - 1 <= p0 && (j0 > p1 - p.window || j0 + n <= p.sinks);
    }
};

// ------------------------------------------------------------------------------------------------------------ forward

// A block of threads does two query blocks, each with a warpgroup of its own (a query per thread), against the same keys:
// two heads that share a key head, or two neighbouring blocks of one head.  While one warpgroup takes its exponentials the
// tensor core works for the other.
constexpr int kFwdThreads = 320;   // two warpgroups, a TMA warp, an MMA warp
constexpr int kFwdSlots = 4;       // tiles of K and V in flight

struct FwdControl {
    uint64_t q_full[2], full[kFwdSlots], empty[kFwdSlots], s_full[2], p_ready[2], o_full[2];
    uint32_t tmem;
    int abort;
};

template <int HALVES> constexpr size_t fwd_smem() { return 2048 + static_cast<size_t>(2 + kFwdSlots) * HALVES * kHalfTile; }

template <int HALVES>
__global__ void __launch_bounds__(kFwdThreads, 1)
attention_fwd_kernel(const __grid_constant__ AttentionMaps maps, const __grid_constant__ AttentionParams p, int pair_heads, int blocks_q, DeviceStatus* status,
                     uint64_t wait_ns) {
    extern __shared__ uint8_t raw[];
    uint8_t* const base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    FwdControl* const ctl = reinterpret_cast<FwdControl*>(base);
    const uint32_t tiles = smem_u32(base + 1024);
    constexpr uint32_t kTile = HALVES * kHalfTile;
    constexpr int kHd = 64 * HALVES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* const abort_flag = &ctl->abort;

    // later queries see more keys: they go first
    const int units = p.batch * p.heads / (pair_heads ? 2 : 1);
    const int unit = blockIdx.x % units, tile_q = blocks_q - 1 - static_cast<int>(blockIdx.x / units);
    const int per_batch = units / p.batch, b = unit / per_batch, h0 = unit % per_batch * (pair_heads ? 2 : 1);
    const QueryBlock blk0(p, h0, tile_q * (pair_heads ? kRows : 2 * kRows));
    const QueryBlock blk1(p, pair_heads ? h0 + 1 : h0, pair_heads ? blk0.r0 : blk0.r0 + kRows);
    const int head_k = h0 / p.group;
    // the tiles that either sees: sinks, then a range
    const int low = blk0.any ? blk0.low : blk1.low;
    const int high = blk1.any ? blk1.high : blk0.high;
    const int sink_tiles = min(max(blk0.any ? blk0.sinks : 0, blk1.any ? blk1.sinks : 0), low);
    const int n_tiles = blk0.any || blk1.any ? sink_tiles + high - low + 1 : 0;
    auto tile_of = [&](int it) { return it < sink_tiles ? it : low + it - sink_tiles; };

    if (threadIdx.x == 0) {
        for (int w = 0; w < 2; ++w) {
            mbar_init(smem_u32(&ctl->q_full[w]), 1);
            mbar_init(smem_u32(&ctl->s_full[w]), 1);
            mbar_init(smem_u32(&ctl->p_ready[w]), 4);
            mbar_init(smem_u32(&ctl->o_full[w]), 1);
        }
        for (int s = 0; s < kFwdSlots; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        ctl->abort = 0;
        fence_barrier_init();
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(&ctl->tmem), 512);
        tmem_relinquish_alloc_permit();
    }
    if (warp == 8 && lane < 4) prefetch_tensormap(lane == 0 ? &maps.q : lane == 1 ? &maps.k : lane == 2 ? &maps.v : &maps.out);
    tc_fence_before_thread_sync();
    __syncthreads();
    tc_fence_after_thread_sync();
    const uint32_t tmem = ctl->tmem;
    grid_dependency_wait();

    const uint32_t q_at = tiles, ring = tiles + 2 * kTile;
    // TMEM: scores (and in their place the probabilities) of either block, then the outputs
    auto tmem_s = [&](int w) { return tmem + static_cast<uint32_t>(w) * kRows; };
    auto tmem_o = [&](int w) { return tmem + 2u * kRows + static_cast<uint32_t>(w) * kHd; };
    const int steps_d = (p.head_dim + 15) / 16;   // 16-deep steps of S, and 16-wide columns of O

    if (warp == 8) {
        // ---------------------------------------------------------------- loads
        const bool lead = elect_one();
        if (lead) {
            for (int w = 0; w < 2; ++w) {
                const QueryBlock& blk = w == 0 ? blk0 : blk1;
                if (!blk.any) continue;
                mbar_arrive_expect_tx(smem_u32(&ctl->q_full[w]), kTile);
                for (int x = 0; x < HALVES; ++x)
                    tma_load_4d(q_at + w * kTile + x * kHalfTile, &maps.q, smem_u32(&ctl->q_full[w]), x * 64, blk.r0, blk.head, b);
            }
        }
        __syncwarp();
        int slot = 0;
        uint32_t phase = 0;
        for (int i = 0; i < 2 * n_tiles; ++i) {
            if (!bounded_wait_warp(smem_u32(&ctl->empty[slot]), phase ^ 1u, abort_flag, status, kDevWaitSmemEmpty, slot, wait_ns)) break;
            if (elect_one()) {
                const uint32_t bar = smem_u32(&ctl->full[slot]), at = ring + slot * kTile;
                mbar_arrive_expect_tx(bar, kTile);
                for (int x = 0; x < HALVES; ++x)
                    tma_load_4d(at + x * kHalfTile, i & 1 ? &maps.v : &maps.k, bar, x * 64, tile_of(i >> 1) * kRows, head_k, b);
            }
            __syncwarp();
            if (++slot == kFwdSlots) { slot = 0; phase ^= 1u; }
        }
    } else if (warp == 9) {
        // ---------------------------------------------------------------- products
        const uint32_t idesc_s = make_idesc_bf16(kRows, kRows, 0, 0), idesc_o = make_idesc_bf16(kRows, steps_d * 16, 0, 1);
        int slot = 0;
        uint32_t phase = 0, p_phase[2] = {0, 0};
        int last[2] = {-1, -1};
        for (int it = 0; it < n_tiles; ++it) {
            if (blk0.sees(tile_of(it))) last[0] = it;
            if (blk1.sees(tile_of(it))) last[1] = it;
        }
        bool begun[2] = {false, false}, ok = true;
        for (int w = 0; w < 2 && ok; ++w)
            if ((w == 0 ? blk0 : blk1).any) ok = bounded_wait_warp(smem_u32(&ctl->q_full[w]), 0, abort_flag, status, kDevWaitSmemFull, 100 + w, wait_ns);
        // the ring holds K(0), V(0), K(1), ...; round `it` takes V(it) and K(it + 1)
        for (int it = -1; it < n_tiles && ok; ++it) {
            int v_slot = -1, k_slot = -1;
            if (it >= 0) {
                v_slot = slot;
                ok = bounded_wait_warp(smem_u32(&ctl->full[slot]), phase, abort_flag, status, kDevWaitSmemFull, slot, wait_ns);
                if (++slot == kFwdSlots) { slot = 0; phase ^= 1u; }
            }
            if (ok && it + 1 < n_tiles) {
                k_slot = slot;
                ok = bounded_wait_warp(smem_u32(&ctl->full[slot]), phase, abort_flag, status, kDevWaitSmemFull, slot, wait_ns);
                if (++slot == kFwdSlots) { slot = 0; phase ^= 1u; }
            }
            if (!ok) break;
            for (int w = 0; w < 2; ++w) {
                const QueryBlock& blk = w == 0 ? blk0 : blk1;
                if (it >= 0 && blk.sees(tile_of(it))) {
                    ok = bounded_wait_warp(smem_u32(&ctl->p_ready[w]), p_phase[w], abort_flag, status, kDevWaitTmemEmpty, w, wait_ns);
                    if (!ok) break;
                    p_phase[w] ^= 1u;
                    tc_fence_after_thread_sync();
                    if (elect_one()) {
                        const uint32_t v_at = ring + v_slot * kTile;
#pragma unroll
                        for (int k = 0; k < kRows / 16; ++k)
                            umma_bf16_ts(tmem_o(w), tmem_s(w) + k * 8, smem_desc(v_at + k * 2048, kHalfTile), idesc_o, begun[w] || k > 0 ? 1u : 0u);
                        if (it == last[w]) umma_commit(smem_u32(&ctl->o_full[w]));
                    }
                    __syncwarp();
                    begun[w] = true;
                }
                if (it + 1 < n_tiles && blk.sees(tile_of(it + 1))) {
                    tc_fence_after_thread_sync();
                    if (elect_one()) {
                        const uint32_t k_at = ring + k_slot * kTile;
                        for (int k = 0; k < steps_d; ++k) {
                            const uint32_t off = (k >> 2) * kHalfTile + (k & 3) * 32;
                            umma_bf16_cg<1>(tmem_s(w), smem_desc(q_at + w * kTile + off, 16), smem_desc(k_at + off, 16), idesc_s, k > 0 ? 1u : 0u);
                        }
                        umma_commit(smem_u32(&ctl->s_full[w]));
                    }
                    __syncwarp();
                }
            }
            if (elect_one()) {
                if (v_slot >= 0) umma_commit(smem_u32(&ctl->empty[v_slot]));
                if (k_slot >= 0) umma_commit(smem_u32(&ctl->empty[k_slot]));
            }
            __syncwarp();
        }
    } else {
        // ---------------------------------------------------------------- softmax: a query per thread
        const int w = warp >> 2, quarter = warp & 3;
        const QueryBlock& blk = w == 0 ? blk0 : blk1;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t ts = tmem_s(w) + lanes, to = tmem_o(w) + lanes;
        const int row = quarter * 32 + lane, i = blk.r0 + row, pos = i + p.tk - p.tq;
        const float c = p.scale * kLog2e;
        float m = -INFINITY, l = 0.0f;
        uint32_t phase = 0;
        bool ok = true, begun = false;
        for (int it = 0; it < n_tiles && ok; ++it) {
            const int tile = tile_of(it), j0 = tile * kRows;
            if (!blk.sees(tile)) continue;
            ok = bounded_wait_warp(smem_u32(&ctl->s_full[w]), phase, abort_flag, status, kDevWaitTmemFull, w, wait_ns);
            if (!ok) break;
            phase ^= 1u;
            tc_fence_after_thread_sync();
            uint32_t s[kRows];
#pragma unroll
            for (int x = 0; x < 4; ++x) tmem_ld_32x32(ts + x * 32, s + x * 32);
            tmem_ld_wait();
            if (!blk.sees_all(p, j0, kRows)) {
                const int from = pos - p.window + 1 - j0, to_ = pos + 1 - j0, first = min(p.sinks, pos + 1) - j0;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t seen = bits_between(from, to_, x * 32) | bits_between(0, first, x * 32);
#pragma unroll
                    for (int y = 0; y < 32; ++y)
                        if (!(seen >> y & 1u)) s[x * 32 + y] = 0xFF800000u;   // -inf
                }
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int y = 0; y < kRows; ++y) top[y & 3] = fmaxf(top[y & 3], __uint_as_float(s[y]));
            const float m_new = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), m);
            const bool grow = (m_new - m) * c > 8.0f;
            if (__any_sync(0xffffffffu, grow)) {
                // The product that wrote O last is complete: the scores of this tile were made after it.
                const float shrink = grow ? ex2_approx((m - m_new) * c) : 1.0f;
                if (grow) m = m_new;
                l *= shrink;
                if (begun) {
                    for (int x = 0; x < steps_d; ++x) {
                        uint32_t o[16];
                        tmem_ld_32x16(to + x * 16, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * shrink);
                        tmem_st_32x16(to + x * 16, o);
                    }
                }
            }
            begun = true;
            const float off = m == -INFINITY ? 0.0f : -m * c;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t e[32];
#pragma unroll
                for (int y = 0; y < 32; ++y) {
                    const float a = ex2_approx(fmaf(__uint_as_float(s[x * 64 + 2 * y]), c, off));
                    const float d = ex2_approx(fmaf(__uint_as_float(s[x * 64 + 2 * y + 1]), c, off));
                    sum[(2 * y) & 3] += a;
                    sum[(2 * y + 1) & 3] += d;
                    e[y] = pack_bf16(a, d);
                }
                tmem_st_32x32(ts + x * 32, e);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st_wait();
            tc_fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->p_ready[w]));
        }
        // ---------------------------------------------------------------- out, through the block's place in the Q tiles
        if (ok && begun) {
            ok = bounded_wait_warp(smem_u32(&ctl->o_full[w]), 0, abort_flag, status, kDevWaitTmemFull, 2 + w, wait_ns);
            tc_fence_after_thread_sync();
        }
        bool bad = false;
        if (blk.r0 < p.tq) {
            uint8_t* const mine = base + 1024 + w * kTile + row * 128;
            const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;   // l NaN: so is the row
            for (int x = 0; x < 4 * HALVES; ++x) {
                uint32_t o[16];
#pragma unroll
                for (int y = 0; y < 16; ++y) o[y] = 0;
                if (ok && begun && x < steps_d) {
                    tmem_ld_32x16(to + x * 16, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                    const float f = l == 0.0f ? 0.0f : __uint_as_float(o[y]) * inv;
                    bad = bad || !(fabsf(f) < INFINITY);
                    o[y] = __float_as_uint(f);
                }
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    uint4 v;
                    v.x = pack_bf16(__uint_as_float(o[8 * y]), __uint_as_float(o[8 * y + 1]));
                    v.y = pack_bf16(__uint_as_float(o[8 * y + 2]), __uint_as_float(o[8 * y + 3]));
                    v.z = pack_bf16(__uint_as_float(o[8 * y + 4]), __uint_as_float(o[8 * y + 5]));
                    v.w = pack_bf16(__uint_as_float(o[8 * y + 6]), __uint_as_float(o[8 * y + 7]));
                    const int chunk = ((x & 3) * 2 + y) ^ (row & 7);
                    *reinterpret_cast<uint4*>(mine + (x >> 2) * kHalfTile + chunk * 16) = v;
                }
            }
            if (i < p.tq && p.lse != nullptr)
                p.lse[(static_cast<int64_t>(b) * p.heads + blk.head) * p.tq + i] = l == 0.0f ? -INFINITY : fmaf(m, p.scale, log2f(l) * (1.0f / kLog2e));
            fence_proxy_async_smem();
            named_barrier_sync(1 + w, 128);
            if (row == 0) {
                for (int x = 0; x < HALVES; ++x) tma_store_4d(&maps.out, q_at + w * kTile + x * kHalfTile, x * 64, blk.r0, blk.head, b);
                bulk_commit_group();
                bulk_wait_group0();
            }
            named_barrier_sync(1 + w, 128);
            // A product with a hidden value that is not finite (0 * inf) has spoilt the row, or it sees such a value: it is
            // formed again from the keys it sees.
            uint32_t again = __ballot_sync(0xffffffffu, bad && ok && i < p.tq);
            while (again != 0) {
                const int r = __ffs(again) - 1;
                again &= again - 1;
                const int64_t at = blk.r0 + quarter * 32 + r;
                attn::forward_row(p, b, blk.head, at, at + p.tk - p.tq);
            }
        }
    }
    // -------------------------------------------------------------------- teardown
    if (*abort_flag) __nanosleep(200000);   // copies in flight land before the shared memory is given back
    tc_fence_before_thread_sync();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after_thread_sync();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------------------------------------------------- launches

template <typename K, typename... A>
cudaError_t launch_sm(K kernel, int64_t blocks, int threads, size_t smem, cudaStream_t stream, A... args) {
    const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (set != cudaSuccess) return set;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    count_launch(1);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_attention_fwd_sm100(const AttentionParams& p, const CUtensorMap* m, DeviceStatus* status, uint64_t wait_ns, cudaStream_t stream) {
    AttentionMaps maps{};
    maps.q = m[0]; maps.k = m[1]; maps.v = m[2]; maps.out = m[3];
    const int pair_heads = p.group % 2 == 0;
    const int per = pair_heads ? kRows : 2 * kRows, blocks_q = (p.tq + per - 1) / per;
    const int64_t blocks = static_cast<int64_t>(p.batch) * p.heads / (pair_heads ? 2 : 1) * blocks_q;
    return p.head_dim <= 64 ? launch_sm(attention_fwd_kernel<1>, blocks, kFwdThreads, fwd_smem<1>(), stream, maps, p, pair_heads, blocks_q, status, wait_ns)
                            : launch_sm(attention_fwd_kernel<2>, blocks, kFwdThreads, fwd_smem<2>(), stream, maps, p, pair_heads, blocks_q, status, wait_ns);
}

}  // namespace llmt_b200
