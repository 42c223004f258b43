// Causal attention with a sliding window and sinks on the tensor cores: see llmt_b200_attention_window_fwd in the public header.
//
// Mathematics.  One pass over the visible keys with a running maximum m and sum l per query:
//   S = Q K^T;  P = 2^(c S - c m) on visible places, else 0;  O = O 2^(c m_old - c m) + P V;  out = O / l,
// c = scale log2 e.  O is only rescaled where m grows by more than 2^8: until then P is up to 2^8 too large, which the
// same factor in l takes out again, and bf16 keeps its relative precision.
// Backward:  P = 2^(c S - lse log2 e);  dS = P (dP - D), dP = dO V^T;  dV = P^T dO, dK = scale dS^T Q, dQ = scale dS K.
// P and dS are rounded to bf16 as operands of the second products: each rounding is independent of the others, so a sum of
// many keeps a relative error of the size of one, about what the rounding of the result itself adds (2.4e-3 against 1.7e-3 of
// the norm); all else is fp32.
//
// Bound: neither memory nor the tensor core alone, but the way between them.  A thread has a row of scores; its exponentials
// (8 cycles a warp for each), maxima and conversions take as long as the products they stand between, and a tile is a chain
// scores -> probabilities -> product.  What helps is whatever runs beside that chain: a second block on the SM, a second
// warpgroup, scores made before they are wanted.
// Measured: 4 x 12 x 333 queries of 64, window 128: 9.6 us (a launch and three tiles); 8 x 12 x 1024 of 64, window 256,
// forward and backward: 31 + 86 us; 8192 queries, 16 heads on 4 of 128, window 2048: forward 131 us (921 TFLOP/s of visible
// pairs), backward 520 us (580).
#include <cuda_bf16.h>

#include <type_traits>

#include "attention_rows.cuh"
#include "common.h"
#include "ptx_sm100.cuh"
#include "waits_sm100.cuh"

namespace llmt_b200 {
namespace {

using namespace ptx;

constexpr int kRows = 128, kCols = 64;          // of a tile of scores (forward: 128 columns)
constexpr uint32_t kHalfTile = kRows * 128;     // 128 rows of 64 bf16 values, 128-byte swizzle
constexpr uint32_t kHalfCols = kCols * 128;     // 64 of them
constexpr float kLog2e = 1.4426950408889634f;

struct alignas(64) AttentionMaps {
    CUtensorMap q, k, v, out, dout, dq, dk, dv;
};

// The high word of a shared-memory descriptor: 8-row groups of 1024 bytes, version 1, 128-byte swizzle.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// Its low word for a tile at `at`; further steps of the product add to it in units of 16 bytes.
__device__ __forceinline__ uint32_t desc_lo(uint32_t at, uint32_t lbo) { return ((lbo >> 4) << 16) | (at >> 4); }
__device__ __forceinline__ uint64_t desc(uint32_t lo) { return (static_cast<uint64_t>(kDescHi) << 32) | static_cast<uint64_t>(lo); }

// Products of a tile, issued by one lane of a converged warp from warp-uniform operands and in unrolled loops: with
// descriptors in ordinary registers and loops that are not, an instruction takes 80 cycles to issue, longer than the tensor
// core takes for it.
//   D[128 x N] = A B^T over HALVES * 64 values: A 128 rows, B N rows of a tile of `half_a`, `half_b` bytes a half
template <int HALVES> __device__ __forceinline__ void product_ss(uint32_t d, uint32_t a_lo, uint32_t half_a, uint32_t b_lo, uint32_t half_b, uint32_t idesc, int steps) {
#pragma unroll
    for (int k = 0; k < 4 * HALVES; ++k)
        if (k < steps)
            umma_bf16_cg<1>(d, desc(a_lo + ((k >> 2) * half_a + (k & 3) * 32) / 16), desc(b_lo + ((k >> 2) * half_b + (k & 3) * 32) / 16), idesc, k > 0 ? 1u : 0u);
}
//   D[128 x N] (+)= A[tmem, 128 x 16 STEPS] B: B 16 STEPS rows, its columns the result's
//   (PART: the columns of A from each PART-th step on sit 2 * 8 * PART columns behind the last ones)
template <int STEPS, int PART = STEPS> __device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, bool accumulate) {
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
        umma_bf16_ts(d, a + (k / PART) * 16 * PART + (k % PART) * 8, desc(b_lo + k * (2048 / 16)), idesc, accumulate || k > 0 ? 1u : 0u);
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

// Two fp32 values as the packed instructions take them.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t two(uint32_t lo, uint32_t hi) { return two(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The larger of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// What a block of queries [r0, r0 + 128) of one head sees, in tiles of 128 keys.
struct QueryBlock {
    int head, r0;
    int low, high, sinks;      // tiles [0, sinks) and [low, high]
    bool any;
    __device__ __forceinline__ QueryBlock(const AttentionParams& p, int head_, int r0_) {
        head = head_;
        r0 = r0_;
        const int p0 = r0 + p.tk - p.tq, p1 = min(r0 + kRows, p.tq) - 1 + p.tk - p.tq;   // positions of the first and the last
        any = r0 < p.tq && p1 >= 0;
        const int first = max(0, p0 - p.window + 1);
        low = first / kRows;
        high = p1 / kRows;
        sinks = min((min(p.sinks, first) + kRows - 1) / kRows, low);
    }
    // of the tiles [from, to)
    __device__ __forceinline__ int count(int from, int to) const {
        return any ? max(0, min(to, sinks) - from) + max(0, min(to, high + 1) - max(from, low)) : 0;
    }
    __device__ __forceinline__ bool sees(int tile) const { return any && tile <= high && (tile >= low || tile < sinks); }
};

// What the 32 queries from position p0 on see of the 32 keys from j0 on: nothing, everything, or a part.
__device__ __forceinline__ bool sees_none(const AttentionParams& p, int p0, int j0) {
    return j0 > p0 + 31 || (j0 + 31 <= p0 - p.window && j0 >= p.sinks);
}
__device__ __forceinline__ bool sees_all(const AttentionParams& p, int p0, int j0) {
    return j0 + 31 <= p0 && (j0 > p0 + 31 - p.window || j0 + 32 <= p.sinks);
}
// The keys of [j0, j0 + 32) that the query at position pos sees.
__device__ __forceinline__ uint32_t seen_keys(const AttentionParams& p, int pos, int j0) {
    return bits_between(pos - p.window + 1 - j0, pos + 1 - j0, 0) | bits_between(0, min(p.sinks, pos + 1) - j0, 0);
}

// 16 fp32 values of a row as bf16 into a 128-row swizzled tile: columns 16 x .. of the row.
__device__ __forceinline__ void put_row16(uint8_t* tile, int row, int x, const uint32_t* o) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        uint4 v;
        v.x = pack_bf16(__uint_as_float(o[8 * y]), __uint_as_float(o[8 * y + 1]));
        v.y = pack_bf16(__uint_as_float(o[8 * y + 2]), __uint_as_float(o[8 * y + 3]));
        v.z = pack_bf16(__uint_as_float(o[8 * y + 4]), __uint_as_float(o[8 * y + 5]));
        v.w = pack_bf16(__uint_as_float(o[8 * y + 6]), __uint_as_float(o[8 * y + 7]));
        *reinterpret_cast<uint4*>(tile + (x >> 2) * kHalfTile + row * 128 + ((((x & 3) * 2 + y) ^ (row & 7)) * 16)) = v;
    }
}

// The end of a copy-out by `threads` threads that meet at barrier `id`: `mine` rows of this warp's 32 hold values that are
// not finite and may owe them to a hidden place.  store() issues the copies (by the thread that `first` names); the rows go to
// again(row) once the copies are complete, in turn to the warps.
template <typename Store, typename Again>
__device__ __forceinline__ void copy_out(uint32_t* bad, int id, int threads, bool first, int quarter, uint32_t mine, Store store, Again again) {
    if ((threadIdx.x & 31) == 0 && mine != 0) atomicOr(&bad[quarter], mine);
    fence_proxy_async_smem();
    named_barrier_sync(id, threads);
    const bool any = (bad[0] | bad[1] | bad[2] | bad[3]) != 0;
    if (first) {
        store();
        bulk_commit_group();
        if (any) bulk_wait_group0();
        else bulk_wait_group_read0();   // the tiles are given back, the copies end by themselves
    }
    if (!any) return;
    named_barrier_sync(id, threads);
    const int warps = threads / 32, me = static_cast<int>(threadIdx.x >> 5) % warps;
    int n = 0;
    for (int x = 0; x < 4; ++x)
        for (uint32_t m = bad[x]; m != 0; m &= m - 1, ++n)
            if (n % warps == me) again(x * 32 + __ffs(m) - 1);
}

// ------------------------------------------------------------------------------------------------------------ forward

// A warpgroup has a query block, a query per thread, and a tile of 128 keys at a time: with 64 the products of scores are
// bound by their reads of Q from shared memory (8192 tokens, window 2048, head_dim 128: 158 us against 133).
// head_dim <= 64: a block of threads has one warpgroup and 256 columns of tensor memory, and two blocks share an SM, so that
// one works while the other begins or ends.  The probabilities have a place beside the scores: as soon as a warpgroup has
// taken its scores out, the tensor core makes the next.
// head_dim <= 128: two warpgroups against the same keys: two heads that share a key head, or two neighbouring query blocks of
// one head.  Scores and outputs fill tensor memory, the probabilities take their scores' place, and while one warpgroup takes
// its exponentials the tensor core works for the other.
// Where there are few query blocks, several blocks of threads share the keys of each, leave their part's output and log-sum-exp
// in a workspace, and a second launch joins them.
template <int WGS> struct FwdControl {
    static constexpr int kSlots = 4;   // tiles of K and V in flight
    uint64_t q_full[WGS], full[kSlots], empty[kSlots], s_full[WGS], s_taken[WGS], p_ready[WGS], o_done[WGS], o_full[WGS];
    uint32_t tmem;
    int abort;
    uint32_t bad[WGS][4];
};

template <int HALVES, int WGS> constexpr size_t fwd_smem() { return 2048 + static_cast<size_t>(WGS + FwdControl<WGS>::kSlots) * HALVES * kHalfTile; }

template <int HALVES, int WGS, bool PARTS>
__global__ void __launch_bounds__(128 * WGS + 64, 3 - WGS)
attention_fwd_kernel(const __grid_constant__ AttentionMaps maps, const __grid_constant__ AttentionParams p, int pair_heads, int blocks_q, int n_parts,
                     DeviceStatus* status, uint64_t wait_ns) {
    const int parts = PARTS ? n_parts : 1;   // (known to be one: 131 us instead of 136 for 8192 queries, window 2048, head_dim 128)
    using Control = FwdControl<WGS>;
    constexpr int kSlots = Control::kSlots, kLoadWarp = 4 * WGS, kProductWarp = 4 * WGS + 1, kHd = 64 * HALVES;
    constexpr bool kApart = HALVES == 1;   // the probabilities have a place of their own
    constexpr uint32_t kTile = HALVES * kHalfTile, kScores = kRows + (kApart ? kRows / 2 : 0), kTmem = WGS * (kScores + kHd);
    static_assert(kTmem == 256 || kTmem == 512, "allocations are powers of two");
    extern __shared__ uint8_t raw[];
    uint8_t* const base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    Control* const ctl = reinterpret_cast<Control*>(base);
    const uint32_t tiles = smem_u32(base + 1024);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* const abort_flag = &ctl->abort;

    // later queries see more keys: they go first
    const int units = p.batch * p.heads / (pair_heads ? 2 : 1);
    const int unit = blockIdx.x % units, item = static_cast<int>(blockIdx.x / units), part = item % parts, tile_q = blocks_q - 1 - item / parts;
    const int per_batch = units / p.batch, b = unit / per_batch, h0 = unit % per_batch * (pair_heads ? 2 : 1);
    const QueryBlock blk0(p, h0, tile_q * (pair_heads ? kRows : WGS * kRows));
    const QueryBlock blk1(p, pair_heads ? h0 + 1 : h0, WGS == 1 ? p.tq : pair_heads ? blk0.r0 : blk0.r0 + kRows);
    auto block = [&](int w) -> const QueryBlock& { return WGS == 1 || w == 0 ? blk0 : blk1; };
    const int head_k = h0 / p.group;
    // the tiles that either sees: sinks, then a range
    const int low = blk0.any ? blk0.low : blk1.low;
    const int high = blk1.any ? blk1.high : blk0.high;
    const int sink_tiles = min(max(blk0.any ? blk0.sinks : 0, blk1.any ? blk1.sinks : 0), low);
    const int n_tiles = blk0.any || blk1.any ? sink_tiles + high - low + 1 : 0;
    auto tile_of = [&](int it) { return it < sink_tiles ? it : low + it - sink_tiles; };
    // this block's part of them
    const int first = static_cast<int>(static_cast<int64_t>(n_tiles) * part / parts), end = static_cast<int>(static_cast<int64_t>(n_tiles) * (part + 1) / parts);
    auto tiles_of = [&](int w) {
        return block(w).count(min(first, sink_tiles), min(end, sink_tiles)) + block(w).count(low + max(first - sink_tiles, 0), low + max(end - sink_tiles, 0));
    };

    if (threadIdx.x == 0) {
        for (int w = 0; w < WGS; ++w) {
            mbar_init(smem_u32(&ctl->q_full[w]), 1);
            mbar_init(smem_u32(&ctl->o_done[w]), 1);
            mbar_init(smem_u32(&ctl->o_full[w]), 1);
            mbar_init(smem_u32(&ctl->s_full[w]), 1);
            mbar_init(smem_u32(&ctl->s_taken[w]), 4);
            mbar_init(smem_u32(&ctl->p_ready[w]), 4);
            for (uint32_t& x : ctl->bad[w]) x = 0;
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        ctl->abort = 0;
        fence_barrier_init();
    }
    if (warp == kProductWarp) {
        tmem_alloc(smem_u32(&ctl->tmem), kTmem);
        tmem_relinquish_alloc_permit();
    }
    if (warp == kLoadWarp && lane < 4) prefetch_tensormap(lane == 0 ? &maps.q : lane == 1 ? &maps.k : lane == 2 ? &maps.v : &maps.out);
    tc_fence_before_thread_sync();
    __syncthreads();
    tc_fence_after_thread_sync();
    const uint32_t tmem = uniform(ctl->tmem);
    if (parts > 1) grid_launch_dependents();   // the launch that joins them
    grid_dependency_wait();

    const uint32_t q_at = tiles, ring = tiles + WGS * kTile;
    // TMEM of a block: scores (in their place or behind them the probabilities), then the output
    auto tmem_s = [&](int w) { return tmem + static_cast<uint32_t>(w) * kScores; };
    auto tmem_p = [&](int w) { return tmem_s(w) + (kApart ? kRows : 0); };
    auto tmem_o = [&](int w) { return tmem + WGS * kScores + static_cast<uint32_t>(w) * kHd; };
    const int steps_d = (p.head_dim + 15) / 16;   // 16-deep steps of S, and 16-wide columns of O

    // Round `it` takes K(it + 1) and V(it): the ring holds K(0), then K(1), V(0), K(2), V(1), ...
    if (warp == kLoadWarp) {
        // ---------------------------------------------------------------- loads
        if (elect_one()) {
            for (int w = 0; w < WGS; ++w) {
                if (!block(w).any) continue;
                mbar_arrive_expect_tx(smem_u32(&ctl->q_full[w]), kTile);
                for (int x = 0; x < HALVES; ++x)
                    tma_load_4d(q_at + w * kTile + x * kHalfTile, &maps.q, smem_u32(&ctl->q_full[w]), x * 64, block(w).r0, block(w).head, b);
            }
        }
        __syncwarp();
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        auto load = [&](const CUtensorMap* map, int tile) {
            ok = bounded_wait_warp(smem_u32(&ctl->empty[slot]), phase ^ 1u, abort_flag, status, kDevWaitSmemEmpty, slot, wait_ns);
            if (!ok) return;
            if (elect_one()) {
                const uint32_t bar = smem_u32(&ctl->full[slot]), at = ring + slot * kTile;
                mbar_arrive_expect_tx(bar, kTile);
                for (int x = 0; x < HALVES; ++x) tma_load_4d(at + x * kHalfTile, map, bar, x * 64, tile * kRows, head_k, b);
            }
            __syncwarp();
            if (++slot == kSlots) { slot = 0; phase ^= 1u; }
        };
        for (int it = first - 1; it < end && ok; ++it) {
            if (it + 1 < end) load(&maps.k, tile_of(it + 1));
            if (ok && it >= first) load(&maps.v, tile_of(it));
        }
    } else if (warp == kProductWarp) {
        // ---------------------------------------------------------------- products
        const uint32_t idesc_s = make_idesc_bf16(kRows, kRows, 0, 0), idesc_o = make_idesc_bf16(kRows, steps_d * 16, 0, 1);
        const uint32_t q_lo = uniform(desc_lo(q_at, 16)), ring_k = uniform(desc_lo(ring, 16)), ring_v = uniform(desc_lo(ring, kHalfTile));
        int slot = 0;
        uint32_t phase = 0;
        int scores[2] = {0, 0}, values[2] = {0, 0};   // products made for either block
        const int most[2] = {tiles_of(0), WGS == 1 ? 0 : tiles_of(1)};
        bool ok = true;
        for (int w = 0; w < WGS && ok; ++w)
            if (block(w).any) ok = bounded_wait_warp(smem_u32(&ctl->q_full[w]), 0, abort_flag, status, kDevWaitSmemFull, 100 + w, wait_ns);
        auto next = [&]() {
            const int s = slot;
            ok = bounded_wait_warp(smem_u32(&ctl->full[slot]), phase, abort_flag, status, kDevWaitSmemFull, slot, wait_ns);
            if (++slot == kSlots) { slot = 0; phase ^= 1u; }
            return s;
        };
        auto make_scores = [&](int w, int k_slot) {
            // their place is free: the last ones are taken out (or, as probabilities, the operand of a product made before)
            if (kApart && scores[w] > 0) {
                ok = bounded_wait_warp(smem_u32(&ctl->s_taken[w]), static_cast<uint32_t>(scores[w] - 1) & 1u, abort_flag, status, kDevWaitTmemEmpty, 10 + w, wait_ns);
                if (!ok) return;
            }
            tc_fence_after_thread_sync();
            if (elect_one()) {
                product_ss<HALVES>(tmem_s(w), q_lo + w * (kTile / 16), kHalfTile, ring_k + k_slot * (kTile / 16), kHalfTile, idesc_s, steps_d);
                umma_commit(smem_u32(&ctl->s_full[w]));
            }
            __syncwarp();
            ++scores[w];
        };
        auto make_values = [&](int w, int v_slot) {
            ok = bounded_wait_warp(smem_u32(&ctl->p_ready[w]), static_cast<uint32_t>(values[w]) & 1u, abort_flag, status, kDevWaitTmemEmpty, w, wait_ns);
            if (!ok) return;
            tc_fence_after_thread_sync();
            if (elect_one()) {
                product_ts<kRows / 16>(tmem_o(w), tmem_p(w), ring_v + v_slot * (kTile / 16), idesc_o, values[w] > 0);
                umma_commit(smem_u32(values[w] + 1 < most[w] ? &ctl->o_done[w] : &ctl->o_full[w]));
            }
            __syncwarp();
            ++values[w];
        };
        for (int it = first - 1; it < end && ok; ++it) {
            int v_slot = -1, k_slot = -1;
            if (it + 1 < end) k_slot = next();
            if (kApart) {   // scores first: their operands are there long before the probabilities
                if (ok && k_slot >= 0) {
#pragma unroll
                    for (int w = 0; w < WGS; ++w)
                        if (ok && block(w).sees(tile_of(it + 1))) make_scores(w, k_slot);
                    if (elect_one()) umma_commit(smem_u32(&ctl->empty[k_slot]));
                    __syncwarp();
                }
                if (ok && it >= first) v_slot = next();
                if (ok && v_slot >= 0) {
#pragma unroll
                    for (int w = 0; w < WGS; ++w)
                        if (ok && block(w).sees(tile_of(it))) make_values(w, v_slot);
                    if (elect_one()) umma_commit(smem_u32(&ctl->empty[v_slot]));
                    __syncwarp();
                }
            } else {
                if (ok && it >= first) v_slot = next();
#pragma unroll
                for (int w = 0; w < WGS; ++w) {
                    if (ok && v_slot >= 0 && block(w).sees(tile_of(it))) make_values(w, v_slot);
                    if (ok && k_slot >= 0 && block(w).sees(tile_of(it + 1))) make_scores(w, k_slot);
                }
                if (elect_one()) {
                    if (v_slot >= 0) umma_commit(smem_u32(&ctl->empty[v_slot]));
                    if (k_slot >= 0) umma_commit(smem_u32(&ctl->empty[k_slot]));
                }
                __syncwarp();
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax: a query per thread
        const int w = WGS == 1 ? 0 : warp >> 2, quarter = warp & 3;
        const QueryBlock& blk = block(w);
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t ts = tmem_s(w) + lanes, tp = tmem_p(w) + lanes, to = tmem_o(w) + lanes;
        const int row = quarter * 32 + lane, i = blk.r0 + row, pos = i + p.tk - p.tq, pw = blk.r0 + quarter * 32 + p.tk - p.tq;
        const float c = p.scale * kLog2e;
        float m = -INFINITY;
        uint64_t l2 = 0;
        int done = 0;   // tiles of this block
        bool ok = true;
        // The product of the tile before `done` has written O and read its probabilities; the one before that is known to have, so
        // the barrier is in one of two phases.
        auto wait_o = [&]() {
            ok = bounded_wait_warp(smem_u32(&ctl->o_done[w]), static_cast<uint32_t>(done - 1) & 1u, abort_flag, status, kDevWaitTmemFull, 2 + w, wait_ns);
            tc_fence_after_thread_sync();
        };
        for (int it = first; it < end && ok; ++it) {
            const int j0 = tile_of(it) * kRows;
            if (!blk.sees(tile_of(it))) continue;
            ok = bounded_wait_warp(smem_u32(&ctl->s_full[w]), static_cast<uint32_t>(done) & 1u, abort_flag, status, kDevWaitTmemFull, w, wait_ns);
            if (!ok) break;
            tc_fence_after_thread_sync();
            uint32_t s[kRows];
#pragma unroll
            for (int x = 0; x < 4; ++x) tmem_ld_32x32(ts + x * 32, s + x * 32);
            tmem_ld_wait();
            if (kApart) {
                tc_fence_before_thread_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->s_taken[w]));
            }
            if (!(j0 + kRows - 1 <= pw && (j0 > pw + 31 - p.window || j0 + kRows <= p.sinks))) {   // hidden places for one of the warp's queries
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t seen = seen_keys(p, pos, j0 + x * 32);
#pragma unroll
                    for (int y = 0; y < 32; ++y)
                        if (!(seen >> y & 1u)) s[x * 32 + y] = 0xFF800000u;   // -inf
                }
            }
            float top[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int y = 0; y < kRows; y += 2) top[y / 2 & 3] = max3(top[y / 2 & 3], __uint_as_float(s[y]), __uint_as_float(s[y + 1]));
            const float m_new = fmaxf(max3(top[0], top[1], top[2]), top[3]);
            const bool grow = (m_new - m) * c > 8.0f;
            if (kApart && done > 0) {   // the last tile's probabilities have been read, and O holds its product
                wait_o();
                if (!ok) break;
            }
            if (__any_sync(0xffffffffu, grow)) {
                const float shrink = grow ? ex2_approx((m - m_new) * c) : 1.0f;
                if (grow) m = m_new;
                l2 = mul2(l2, two(shrink, shrink));
                for (int x = 0; x < (done > 0 ? steps_d : 0); ++x) {
                    uint32_t o[16];
                    tmem_ld_32x16(to + x * 16, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * shrink);
                    tmem_st_32x16(to + x * 16, o);
                }
            }
            const float off = m == -INFINITY ? 0.0f : -m * c;
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int y = 0; y < 32; ++y) {
                    const float2 a = make_float2(fmaf(__uint_as_float(s[x * 64 + 2 * y]), c, off), fmaf(__uint_as_float(s[x * 64 + 2 * y + 1]), c, off));
                    const float e0 = ex2_approx(a.x), e1 = ex2_approx(a.y);
                    sum[y & 1] = add2(sum[y & 1], two(e0, e1));
                    s[x * 64 + y] = pack_bf16(e0, e1);
                }
                tmem_st_32x32(tp + x * 32, s + x * 64);
            }
            l2 = add2(l2, add2(sum[0], sum[1]));
            tmem_st_wait();
            tc_fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->p_ready[w]));
            ++done;
        }
        // ---------------------------------------------------------------- out, through the block's place in the Q tiles
        if (ok && done > 0) ok = bounded_wait_warp(smem_u32(&ctl->o_full[w]), 0, abort_flag, status, kDevWaitTmemFull, 4 + w, wait_ns);
        tc_fence_after_thread_sync();
        if (blk.r0 < p.tq) {
            const float l = both(l2).x + both(l2).y;
            const float inv = l > 0.0f ? 1.0f / l : l;   // l NaN: so is the row
            bool bad = false;
            const int64_t line = (static_cast<int64_t>(b) * p.heads + blk.head) * p.tq + i;
            // of a block's part in the workspace: 16-byte pieces of rows, [piece][row], so that a warp's stores are contiguous
            const int64_t place = ((static_cast<int64_t>(b) * p.heads + blk.head) * ((p.tq + kRows - 1) / kRows) + blk.r0 / kRows) * parts + part;
            for (int x = 0; x < 4 * HALVES; ++x) {
                uint32_t o[16];
#pragma unroll
                for (int y = 0; y < 16; ++y) o[y] = 0;
                if (ok && done > 0 && x < steps_d) {
                    tmem_ld_32x16(to + x * 16, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                    const float f = l == 0.0f ? 0.0f : __uint_as_float(o[y]) * inv;
                    bad = bad || !(fabsf(f) < INFINITY);
                    o[y] = __float_as_uint(f);
                }
                if (parts == 1) {
                    put_row16(base + 1024 + w * kTile, row, x, o);
                } else if (i < p.tq && x < steps_d) {
                    uint4* const to_part = reinterpret_cast<uint4*>(p.partial) + (place * (kHd / 4) + x * 4) * kRows + row;
#pragma unroll
                    for (int y = 0; y < 4; ++y) to_part[y * kRows] = make_uint4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
                }
            }
            if (parts > 1) {
                if (i < p.tq) p.part_stats[place * kRows + row] = l == 0.0f ? -INFINITY : fmaf(m, c, log2f(l));
            } else {
                if (i < p.tq && p.lse != nullptr) p.lse[line] = l == 0.0f ? -INFINITY : fmaf(m, p.scale, log2f(l) * (1.0f / kLog2e));
                // A product with a hidden value that is not finite (0 * inf) may have spoilt columns of the row.  A sum that is NaN
                // is of visible scores only: so is the whole row then.
                copy_out(ctl->bad[w], 1 + w, 128, row == 0, quarter, __ballot_sync(0xffffffffu, bad && l == l && ok && i < p.tq), [&] {
                    for (int x = 0; x < HALVES; ++x) tma_store_4d(&maps.out, q_at + w * kTile + x * kHalfTile, x * 64, blk.r0, blk.head, b);
                }, [&](int r) {
                    const int64_t at = blk.r0 + r;
                    attn::forward_row(p, b, blk.head, at, at + p.tk - p.tq);
                });
            }
        }
    }
    // -------------------------------------------------------------------- teardown
    if (*abort_flag) __nanosleep(200000);   // copies in flight land before the shared memory is given back
    tc_fence_before_thread_sync();
    __syncthreads();
    if (warp == kProductWarp) {
        tc_fence_after_thread_sync();
        tmem_dealloc(tmem, kTmem);
    }
}

// Joins the parts of 32 rows that were done in parts.  Forward: out = sum of 2^(s_part - max) out_part over the sum of the
// 2^(s_part - max), s_part = log2 sum exp of a part's scores.  Backward: dQ and D are the parts' sums.  A lane has a row, a warp
// PIECES of the row's 16-byte pieces; the results cross shared memory, so that reads and writes are contiguous.
constexpr int kJoinWarps = 8, kMostParts = 32;
// (Blocks an SM: as many as the join alone would have; rows that are formed again may not cost it registers.)
template <int PIECES, bool FORWARD>
__global__ void __launch_bounds__(kJoinWarps * 32, FORWARD ? 3 : 2) attention_join_kernel(const __grid_constant__ AttentionParams p, int parts) {
    constexpr int kPieces = PIECES * kJoinWarps;
    __shared__ uint2 tile[32][kPieces + 1];
    __shared__ uint32_t bad[kJoinWarps];
    if (!FORWARD) grid_launch_dependents();   // the launch for dK and dV
    grid_dependency_wait();
    const int blocks_q = (p.tq + kRows - 1) / kRows, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t block = blockIdx.x / 4, bh = block / blocks_q, b = bh / p.heads, h = bh % p.heads;
    const int in_block = static_cast<int>(blockIdx.x % 4) * 32 + lane;
    const int64_t r0 = block % blocks_q * kRows + blockIdx.x % 4 * 32, i = r0 + lane;
    if (r0 >= p.tq) return;
    const float* const stat = p.part_stats + block * parts * kRows + in_block;
    const float4* const from = reinterpret_cast<const float4*>(p.partial) + (block * parts * kPieces + warp * PIECES) * kRows + in_block;
    float top = -INFINITY, total = 0.0f, o[PIECES][4] = {};
    if (i < p.tq) {
        for (int part = 0; FORWARD && part < parts; ++part) top = fmaxf(top, stat[part * kRows]);
#pragma unroll 2
        for (int part = 0; part < parts; ++part) {
            const float s = stat[part * kRows], w = !FORWARD ? 1.0f : s == -INFINITY ? 0.0f : exp2f(s - top);   // NaN in a part: in all
            total += FORWARD ? w : s;
#pragma unroll
            for (int n = 0; n < PIECES; ++n) {
                if ((warp * PIECES + n) * 4 >= p.head_dim || w == 0.0f) continue;
                const float4 v = from[(static_cast<int64_t>(part) * kPieces + n) * kRows];
                o[n][0] = fmaf(w, v.x, o[n][0]); o[n][1] = fmaf(w, v.y, o[n][1]); o[n][2] = fmaf(w, v.z, o[n][2]); o[n][3] = fmaf(w, v.w, o[n][3]);
            }
        }
    }
    const float inv = !FORWARD ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
    // a sum that is NaN is of visible places only (or a D without any): so is the whole row
    const bool known = total != total && i + p.tk - p.tq >= 0;
    bool off = false;
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
#pragma unroll
        for (float& x : o[n]) {
            x *= inv;
            off = off || (!known && !(fabsf(x) < INFINITY));
        }
        tile[lane][warp * PIECES + n] = make_uint2(pack_bf16(o[n][0], o[n][1]), pack_bf16(o[n][2], o[n][3]));
    }
    const uint32_t mine = __ballot_sync(0xffffffffu, off);
    if (lane == 0) bad[warp] = mine;
    if (warp == 0 && i < p.tq) {
        if (FORWARD && p.lse != nullptr) p.lse[bh * p.tq + i] = total == 0.0f ? -INFINITY : (top + log2f(total)) * (1.0f / kLog2e);
        if (!FORWARD)
            p.dvec[bh * p.tq + i] = fabsf(total) < INFINITY ? total : attn::dot_rows(attn::row_of(p.dout, b, i, h), attn::row_of(p.out, b, i, h), p.head_dim);
    }
    __syncthreads();
    uint32_t again = 0;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) again |= bad[w];
    for (int r = warp; r < 32 && r0 + r < p.tq; r += kJoinWarps)
        if (lane * 4 < p.head_dim) *reinterpret_cast<uint2*>(attn::row_to(FORWARD ? p.out : p.dq, b, r0 + r, h) + lane * 4) = tile[r][lane];
    for (int r = warp; again != 0 && r < 32 && r0 + r < p.tq; r += kJoinWarps) {   // as after one pass
        if (!(again >> r & 1u)) continue;
        if (FORWARD) attn::forward_row(p, b, h, r0 + r, r0 + r + p.tk - p.tq);
        else attn::dq_row(p, b, h, r0 + r, attn::dot_rows(attn::row_of(p.dout, b, r0 + r, h), attn::row_of(p.out, b, r0 + r, h), p.head_dim));
    }
}

// ----------------------------------------------------------------------------------------------------------- backward

// The tiles of 64 queries that see a key of [j0, j0 + 128).
struct QueryTiles {
    int first, count;
    __host__ __device__ QueryTiles(const AttentionParams& p, int j0) {
        const int64_t off = static_cast<int64_t>(p.tk) - p.tq, j1 = j0 + kRows - 1;
        const int64_t begin = j0 - off > 0 ? j0 - off : 0;
        int64_t end = j0 < p.sinks ? p.tq : j1 + p.window - off;   // one past the last
        if (end > p.tq) end = p.tq;
        first = static_cast<int>(begin / 64);
        count = end > begin ? static_cast<int>((end - 1) / 64) - first + 1 : 0;
    }
};

// How the key tiles are shared out: those with keys that stay visible in `sink_parts` parts, the others in `parts`.
struct DkdvPlan {
    int tiles, sink_tiles, sink_parts, parts;
    __host__ __device__ int64_t items() const { return static_cast<int64_t>(sink_tiles) * sink_parts + static_cast<int64_t>(tiles - sink_tiles) * parts; }
    // Places in the workspace: [unit][item] of either class, where it is done in more than one part.
    __host__ __device__ int64_t kept_slots(int64_t units) const { return sink_parts > 1 ? units * sink_tiles * sink_parts : 0; }
    __host__ __device__ int64_t slots(int64_t units) const { return kept_slots(units) + (parts > 1 ? units * (tiles - sink_tiles) * parts : 0); }
    __device__ int64_t slot(bool kept, int unit, int item, int units) const {
        return kept ? static_cast<int64_t>(unit) * sink_tiles * sink_parts + item
                    : kept_slots(units) + static_cast<int64_t>(unit) * (tiles - sink_tiles) * parts + item;
    }
};

// dQ and dK, dV are two kernels, each of which forms P and dS again for itself: neither has to add to memory that another
// block adds to, so the order of every sum is fixed.  Both walk tiles of 64 columns, which as many warpgroups take in turn as
// tensor memory has places for scores: two or three.  A warpgroup's turn is a chain of 900 cycles of its own work and 900 of
// waiting for its products; with two of them both the tensor core and the exponentials stood still for a third of the time
// (two warpgroups on the halves of one tile, three places: no better, they want the special-function unit at the same time).
constexpr int kBwdSlots = 4;

constexpr int kMaxBuffers = 3;

struct BwdControl {
    uint64_t fixed, full[kBwdSlots], empty[kBwdSlots], scores[kMaxBuffers], ready[kMaxBuffers], taken, done;
    uint32_t tmem;
    int abort;
    uint32_t bad[4];
    float d[kRows];               // dQ: D of the block's queries
    float sums[kMaxBuffers][kRows];   // dQ: row sums of dS by each warpgroup
    alignas(16) float4 stats[4 * kMaxBuffers][kCols / 2];   // dK, dV: of each warp, for two queries of a tile each: - lse log2 e of both, - D of both
};
static_assert(sizeof(BwdControl) <= 9 * 1024, "the control block sits below the tiles");
constexpr uint32_t kBwdControl = 9 * 1024;
template <int HALVES> constexpr size_t bwd_smem() { return 1024 + kBwdControl + 2 * HALVES * kHalfTile + static_cast<size_t>(kBwdSlots) * 2 * HALVES * kHalfCols; }

// What both kernels have around their loops: barriers, tensor memory, and the pipeline over BUFFERS places for scores, each
// with a warpgroup of its own (warps 0 .. 4 BUFFERS - 1; then a warp for the loads and one for the products)
//   scores(0), .., scores(BUFFERS - 1), then for each tile: its second products when its P / dS are there, scores BUFFERS on.
template <int BUFFERS, int TMEM> struct BwdRoles {
    static constexpr int kTmem = TMEM <= 256 ? 256 : 512;
    static_assert(TMEM <= 512, "tensor memory has 512 columns");
    static constexpr int kSoftmax = 128 * BUFFERS, kThreads = kSoftmax + 64, kLoadWarp = 4 * BUFFERS, kProductWarp = 4 * BUFFERS + 1;
    BwdControl* ctl;
    volatile int* abort_flag;
    DeviceStatus* status;
    uint64_t wait_ns;
    int n;

    __device__ __forceinline__ void set_up(int warp) {
        if (threadIdx.x == 0) {
            mbar_init(smem_u32(&ctl->fixed), 1);
            mbar_init(smem_u32(&ctl->done), 1);
            mbar_init(smem_u32(&ctl->taken), 4);
            for (int w = 0; w < BUFFERS; ++w) {
                mbar_init(smem_u32(&ctl->scores[w]), 1);
                mbar_init(smem_u32(&ctl->ready[w]), 4);
            }
            for (int s = 0; s < kBwdSlots; ++s) {
                mbar_init(smem_u32(&ctl->full[s]), 1);
                mbar_init(smem_u32(&ctl->empty[s]), 1);
            }
            ctl->abort = 0;
            for (uint32_t& x : ctl->bad) x = 0;
            fence_barrier_init();
        }
        if (warp == kProductWarp) {
            tmem_alloc(smem_u32(&ctl->tmem), kTmem);
            tmem_relinquish_alloc_permit();
        }
        tc_fence_before_thread_sync();
        __syncthreads();
        tc_fence_after_thread_sync();
    }
    // load(tile, slot, barrier): the tile's copies, issued by one lane.
    template <typename Load> __device__ __forceinline__ void loads(uint32_t bytes, Load load) const {
        int slot = 0;
        uint32_t phase = 0;
        for (int it = 0; it < n; ++it) {
            if (!bounded_wait_warp(smem_u32(&ctl->empty[slot]), phase ^ 1u, abort_flag, status, kDevWaitSmemEmpty, slot, wait_ns)) break;
            if (elect_one()) {
                mbar_arrive_expect_tx(smem_u32(&ctl->full[slot]), bytes);
                load(it, slot, smem_u32(&ctl->full[slot]));
            }
            __syncwarp();
            if (++slot == kBwdSlots) { slot = 0; phase ^= 1u; }
        }
    }
    // first(slot, buffer), second(slot, buffer, accumulate): the products, issued by one lane.  EARLY (one buffer): dS has a
    // place of its own, and the next scores are made as soon as the warpgroup has taken the last ones out.
    template <bool EARLY, typename First, typename Second> __device__ __forceinline__ void products(First first, Second second) const {
        static_assert(!EARLY || BUFFERS == 1, "one place for scores");
        bool ok = n == 0 || bounded_wait_warp(smem_u32(&ctl->fixed), 0, abort_flag, status, kDevWaitSmemFull, 100, wait_ns);
        int slot = 0, buffer = 0, slot_2 = 0, buffer_2 = 0;   // of the next first products, and of the next second ones
        uint32_t phase = 0, phase_2 = 0;
        auto make_second = [&](int it) {
            ok = bounded_wait_warp(smem_u32(&ctl->ready[buffer_2]), phase_2, abort_flag, status, kDevWaitTmemEmpty, buffer_2, wait_ns);
            if (!ok) return;
            tc_fence_after_thread_sync();
            if (elect_one()) {
                second(slot_2, buffer_2, it > 0);
                umma_commit(smem_u32(&ctl->empty[slot_2]));
                if (it + 1 == n) umma_commit(smem_u32(&ctl->done));
            }
            __syncwarp();
            if (++slot_2 == kBwdSlots) slot_2 = 0;
            if (++buffer_2 == BUFFERS) { buffer_2 = 0; phase_2 ^= 1u; }
        };
        for (int it = -BUFFERS; it < n && ok; ++it) {
            if (!EARLY && it >= 0) make_second(it);
            if (ok && it + BUFFERS < n) {
                ok = bounded_wait_warp(smem_u32(&ctl->full[slot]), phase, abort_flag, status, kDevWaitSmemFull, slot, wait_ns);
                if (ok && EARLY && it >= 0)
                    ok = bounded_wait_warp(smem_u32(&ctl->taken), static_cast<uint32_t>(it) & 1u, abort_flag, status, kDevWaitTmemEmpty, 50, wait_ns);
                if (!ok) break;
                tc_fence_after_thread_sync();
                if (elect_one()) {
                    first(slot, buffer);
                    umma_commit(smem_u32(&ctl->scores[buffer]));
                }
                __syncwarp();
                if (++slot == kBwdSlots) { slot = 0; phase ^= 1u; }
                if (++buffer == BUFFERS) buffer = 0;
            }
            if (EARLY && ok && it >= 0) make_second(it);
        }
    }
    // The second products of a tile are complete.
    __device__ __forceinline__ bool wait_second(int it) const {
        const bool ok = bounded_wait_warp(smem_u32(&ctl->empty[it % kBwdSlots]), static_cast<uint32_t>(it / kBwdSlots) & 1u, abort_flag, status, kDevWaitTmemFull, 60, wait_ns);
        tc_fence_after_thread_sync();
        return ok;
    }
    __device__ __forceinline__ void post_taken() const {
        tc_fence_before_thread_sync();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl->taken));
    }
    // work(it): what warpgroup `w` does with a tile's scores once they are there; before(it) ahead of the wait; last() when the
    // warpgroup has no more tiles, before the products of all are waited for.
    template <typename Before, typename Work, typename Last> __device__ __forceinline__ bool tiles(int w, Before before, Work work, Last last) const {
        uint32_t phase = 0;
        for (int it = w; it < n; it += BUFFERS) {
            before(it);
            if (!bounded_wait_warp(smem_u32(&ctl->scores[w]), phase, abort_flag, status, kDevWaitTmemFull, w, wait_ns)) return false;
            tc_fence_after_thread_sync();
            work(it);
            tmem_st_wait();
            tc_fence_before_thread_sync();
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl->ready[w]));
            phase ^= 1u;
        }
        last();
        if (n == 0) return true;
        const bool ok = bounded_wait_warp(smem_u32(&ctl->done), 0, abort_flag, status, kDevWaitTmemFull, 100, wait_ns);
        tc_fence_after_thread_sync();
        return ok;
    }
    __device__ __forceinline__ void tear_down(int warp, uint32_t tmem) {
        if (*abort_flag) __nanosleep(200000);
        tc_fence_before_thread_sync();
        __syncthreads();
        if (warp == kProductWarp) {
            tc_fence_after_thread_sync();
            tmem_dealloc(tmem, kTmem);
        }
    }
};

// D of 128 queries into shared memory by the first WARPS warps: 8 HALVES lanes for a row, a row's 16 bytes
// each, so that the loads of all of a warp's rows are in flight at once (a thread a row took 6000 to 12000 cycles).
template <int HALVES, int WARPS>
__device__ __forceinline__ void row_products(const AttentionParams& p, int b, int h, int r0, float* d, int warp) {
    constexpr int kLanes = 8 * HALVES, kAtOnce = 32 / kLanes, kEach = kRows / WARPS, kTurns = kEach / kAtOnce;
    if (warp >= WARPS) return;
    const int lane = threadIdx.x & 31, col = lane % kLanes * 8, first = warp * kEach + lane / kLanes;
    uint4 x[kTurns], y[kTurns];
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
        const int i = r0 + first + n * kAtOnce;
        x[n] = y[n] = make_uint4(0, 0, 0, 0);
        if (i < p.tq && col < p.head_dim) {
            x[n] = *reinterpret_cast<const uint4*>(attn::row_of(p.dout, b, i, h) + col);
            y[n] = *reinterpret_cast<const uint4*>(attn::row_of(p.out, b, i, h) + col);
        }
    }
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
        const uint32_t xs[4] = {x[n].x, x[n].y, x[n].z, x[n].w}, ys[4] = {y[n].x, y[n].y, y[n].z, y[n].w};
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) s = fmaf(attn::hi_f(xs[k]), attn::hi_f(ys[k]), fmaf(attn::lo_f(xs[k]), attn::lo_f(ys[k]), s));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane % kLanes == 0) d[first + n * kAtOnce] = s;
    }
}

// dQ of 128 queries: S = Q K^T and dP = dO V^T of 64 keys, dS = P (dP - D), dQ += dS K.
// D = rowsum(dO out) carries the rounding of out.  Over many keys that is lost beside the roundings of dS; over few it is not
// (normal operands, error of dQ's norm against the result's own rounding of 1.7e-3: 4.4e-3 for 2 keys, 2.9e-3 for 8, 2.5e-3 for
// 128, where an exact D gives 2.4e-3 for any number).  `exact`, for calls in which no query sees more than 128 keys: the tiles are
// gone through twice, the first time for D as the sum of P dP, with zeros for dS.  The first queries of other calls, which see
// few keys too, keep the rounded D, as the public header says.  (Three kinds of the kernel, since the ordinary one gains 3 % from not having the others.)
// head_dim <= 64: one warpgroup a block and two blocks an SM, so that one works while the other begins or ends; dS has a place
// of its own, and the next scores are made while the warpgroup works on the last ones.  (BUFFERS = 3 there: 8 x 12 x 1024,
// window 256: dQ, dK, dV 100 us against 90; 2 x 16 x 4096: 368 against 344.)  Few query blocks are done in parts, as in the
// forward pass.
template <int HALVES, int BUFFERS> using DqRoles = BwdRoles<BUFFERS, BUFFERS * 2 * kCols + (BUFFERS == 1 ? kCols / 2 : 0) + 64 * HALVES>;
enum class Dq { kWhole, kParts, kExact };
template <int HALVES, int BUFFERS, Dq KIND>
__global__ void __launch_bounds__(128 * BUFFERS + 64, BUFFERS == 1 ? 2 : 1)
attention_dq_kernel(const __grid_constant__ AttentionMaps maps, const __grid_constant__ AttentionParams p, int blocks_q, int n_parts, DeviceStatus* status,
                    uint64_t wait_ns) {
    const int parts = KIND == Dq::kParts ? n_parts : 1;
    constexpr bool exact = KIND == Dq::kExact;
    extern __shared__ uint8_t raw[];
    uint8_t* const base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* const tiles_ptr = base + kBwdControl;
    const uint32_t tiles = smem_u32(tiles_ptr);
    constexpr int kBuffers = BUFFERS;
    constexpr bool kEarly = BUFFERS == 1;
    constexpr uint32_t kFixed = HALVES * kHalfTile, kStream = HALVES * kHalfCols;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int units = p.batch * p.heads, unit = blockIdx.x % units;
    const int b = unit / p.heads, h = unit % p.heads, hk = h / p.group;
    const int item = static_cast<int>(blockIdx.x / units), part = item % parts, r0 = (blocks_q - 1 - item / parts) * kRows;
    const int p0 = r0 + p.tk - p.tq, p1 = min(r0 + kRows, p.tq) - 1 + p.tk - p.tq;
    const int first = max(0, p0 - p.window + 1);
    const int low = first / kCols, sink_tiles = min((min(p.sinks, first) + kCols - 1) / kCols, low);
    // this block's part of the tiles
    const int n_tiles = p1 >= 0 ? sink_tiles + p1 / kCols - low + 1 : 0;
    const int begin = static_cast<int>(static_cast<int64_t>(n_tiles) * part / parts), end = static_cast<int>(static_cast<int64_t>(n_tiles) * (part + 1) / parts);
    const int once = end - begin;
    DqRoles<HALVES, BUFFERS> roles{reinterpret_cast<BwdControl*>(base), nullptr, status, wait_ns, exact ? 2 * once : once};
    roles.abort_flag = &roles.ctl->abort;
    auto tile_of = [&](int it) {
        const int n = begin + (it < once ? it : it - once);
        return n < sink_tiles ? n : low + n - sink_tiles;
    };
    roles.set_up(warp);
    const uint32_t tmem = uniform(roles.ctl->tmem);
    grid_launch_dependents();   // the launch that joins the parts, or the one for dK and dV
    grid_dependency_wait();
    const int steps_d = (p.head_dim + 15) / 16;
    const uint32_t ring = tiles + 2 * kFixed;
    const uint32_t tmem_ds = tmem + 2u * kCols, tmem_dq = tmem + kBuffers * 2u * kCols + (kEarly ? kCols / 2 : 0);   // behind the places of S and dP

    if (warp == roles.kLoadWarp) {
        if (roles.n > 0 && elect_one()) {
            mbar_arrive_expect_tx(smem_u32(&roles.ctl->fixed), 2 * kFixed);
            for (int x = 0; x < HALVES; ++x) {
                tma_load_4d(tiles + x * kHalfTile, &maps.q, smem_u32(&roles.ctl->fixed), x * 64, r0, h, b);
                tma_load_4d(tiles + kFixed + x * kHalfTile, &maps.dout, smem_u32(&roles.ctl->fixed), x * 64, r0, h, b);
            }
        }
        __syncwarp();
        roles.loads(2 * kStream, [&](int it, int slot, uint32_t bar) {
            const uint32_t at = ring + slot * 2 * kStream;
            for (int x = 0; x < HALVES; ++x) {
                tma_load_4d(at + x * kHalfCols, &maps.k, bar, x * 64, tile_of(it) * kCols, hk, b);
                tma_load_4d(at + kStream + x * kHalfCols, &maps.v, bar, x * 64, tile_of(it) * kCols, hk, b);
            }
        });
    } else if (warp == roles.kProductWarp) {
        const uint32_t idesc_s = make_idesc_bf16(kRows, kCols, 0, 0), idesc_d = make_idesc_bf16(kRows, steps_d * 16, 0, 1);
        const uint32_t fixed_lo = uniform(desc_lo(tiles, 16)), ring_lo = uniform(desc_lo(ring, 16)), ring_mn = uniform(desc_lo(ring, kHalfCols));
        roles.template products<kEarly>(
            [&](int slot, int buffer) {
                const uint32_t at = ring_lo + slot * (2 * kStream / 16), to = tmem + buffer * 2 * kCols;
                product_ss<HALVES>(to, fixed_lo, kHalfTile, at, kHalfCols, idesc_s, steps_d);
                product_ss<HALVES>(to + kCols, fixed_lo + kFixed / 16, kHalfTile, at + kStream / 16, kHalfCols, idesc_s, steps_d);
            },
            [&](int slot, int buffer, bool more) {
                if (kEarly) product_ts<kCols / 16>(tmem_dq, tmem_ds, ring_mn + slot * (2 * kStream / 16), idesc_d, more);
                else product_ts<kCols / 16, 2>(tmem_dq, tmem + buffer * 2 * kCols, ring_mn + slot * (2 * kStream / 16), idesc_d, more);
            });
    } else {
        const int w = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane, i = r0 + row, pos = i + p.tk - p.tq;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const float c = p.scale * kLog2e;
        const int64_t at = (static_cast<int64_t>(b) * p.heads + h) * p.tq + i;
        float d = 0.0f;
        if (!exact) {
            row_products<HALVES, BUFFERS == 1 ? 4 : 8>(p, b, h, r0, roles.ctl->d, warp);
            named_barrier_sync(1, roles.kSoftmax);
            d = roles.ctl->d[row];
        }
        float lse2 = INFINITY;   // P = 0 for a query that is not there or sees nothing
        if (i < p.tq) {
            const float lse = p.lse[at];
            if (lse != -INFINITY) lse2 = lse * kLog2e;
        }
        const int pw = r0 + quarter * 32 + p.tk - p.tq;   // position of the warp's first query
        uint64_t sum = 0;
        const uint64_t c2 = two(c, c), less2 = two(-lse2, -lse2);
        uint64_t lessd = two(-d, -d);
        bool first_time = exact;   // D is still being summed
        auto have_d = [&]() {
            roles.ctl->sums[w][row] = both(sum).x + both(sum).y;
            named_barrier_sync(1, roles.kSoftmax);
#pragma unroll
            for (int x = 0; x < kBuffers; ++x) d += roles.ctl->sums[x][row];
            named_barrier_sync(1, roles.kSoftmax);   // they are written once more
            lessd = two(-d, -d);
            sum = 0;
            first_time = false;
        };
        const bool ok = roles.tiles(w, [&](int it) {
            if (first_time && it >= once) have_d();
        }, [&](int it) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {   // 32 keys at a time
                const uint32_t ts = tmem + w * 2 * kCols + x * 32 + lanes;
                const int j0 = tile_of(it) * kCols + x * 32;
                const bool none = sees_none(p, pw, j0);
                uint32_t s[32], dp[32];
                if (!none) {
                    tmem_ld_32x32(ts, s);
                    tmem_ld_32x32(ts + kCols, dp);
                    tmem_ld_wait();
                }
                if (kEarly && x == 1) roles.post_taken();
                if (none) {
#pragma unroll
                    for (int y = 0; y < 16; ++y) s[y] = 0;
                } else {
                    uint64_t f[16];
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        const float2 a = both(fma2(two(s[2 * y], s[2 * y + 1]), c2, less2));
                        f[y] = mul2(two(ex2_approx(a.x), ex2_approx(a.y)), add2(two(dp[2 * y], dp[2 * y + 1]), lessd));
                    }
                    if (!sees_all(p, pw, j0)) {
                        const uint32_t seen = seen_keys(p, pos, j0);
#pragma unroll
                        for (int y = 0; y < 16; ++y) {
                            const float2 a = both(f[y]);
                            f[y] = two(seen >> 2 * y & 1u ? a.x : 0.0f, seen >> 2 * y & 2u ? a.y : 0.0f);
                        }
                    }
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        sum = add2(sum, f[y]);
                        s[y] = first_time ? 0 : pack_bf16(both(f[y]).x, both(f[y]).y);
                    }
                }
                if (kEarly && x == 0 && it > 0) roles.wait_second(it - 1);   // they have read the last dS (a wait that runs out ends the next one too)
                tmem_st_32x16(kEarly ? tmem_ds + x * 16 + lanes : ts, s);
            }
        }, [&] {
            if (first_time) have_d();   // before the last products are waited for: they wait for the other warpgroups' tiles
        });
        if (first_time) have_d();   // a wait has run out: the other warpgroups are not left at the barrier
        // A row of dS adds up to nothing but for what the rounding of `out` has put into D: dK's kernel gets D without it.
        roles.ctl->sums[w][row] = both(sum).x + both(sum).y;
        if (exact && w == 0) roles.ctl->d[row] = d;   // for a row that is formed again
        named_barrier_sync(1, roles.kSoftmax);
        float of_row = 0.0f;
#pragma unroll
        for (int x = 0; x < kBuffers; ++x) of_row += roles.ctl->sums[x][row];
        const int64_t place = (static_cast<int64_t>(unit) * blocks_q + r0 / kRows) * parts + part;   // of this part in the workspace, as in the forward pass
        if (w == 0 && i < p.tq) {
            const float more = (part == 0 ? d : 0.0f) + of_row;
            if (parts > 1) p.part_stats[place * kRows + row] = more;
            else p.dvec[at] = fabsf(more) < INFINITY ? more : d;
        }
        bool bad = false;
        for (int x = w; x < 4 * HALVES; x += kBuffers) {   // the warpgroups share the columns
            uint32_t o[16];
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] = 0;
            if (ok && roles.n > 0 && x < steps_d) {
                tmem_ld_32x16(tmem_dq + lanes + x * 16, o);
                tmem_ld_wait();
            }
#pragma unroll
            for (int y = 0; y < 16; ++y) {
                const float f = __uint_as_float(o[y]) * p.scale;
                bad = bad || !(fabsf(f) < INFINITY);
                o[y] = __float_as_uint(f);
            }
            if (parts == 1) {
                put_row16(tiles_ptr, row, x, o);
            } else if (i < p.tq && x < steps_d) {
                uint4* const to_part = reinterpret_cast<uint4*>(p.partial) + (place * (16 * HALVES) + x * 4) * kRows + row;
#pragma unroll
                for (int y = 0; y < 4; ++y) to_part[y * kRows] = make_uint4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
            }
        }
        if (parts == 1) {
            // as in the forward kernel: a hidden key that is not finite may have spoilt the row, unless its dS is NaN
            copy_out(roles.ctl->bad, 1, roles.kSoftmax, threadIdx.x == 0, quarter, __ballot_sync(0xffffffffu, bad && of_row == of_row && ok && i < p.tq), [&] {
                for (int x = 0; x < HALVES; ++x) tma_store_4d(&maps.dq, tiles + x * kHalfTile, x * 64, r0, h, b);
            }, [&](int r) { attn::dq_row(p, b, h, r0 + r, roles.ctl->d[r]); });
        }
    }
    roles.tear_down(warp, tmem);
}

// dK and dV of 128 keys: S^T = K Q^T and dP^T = V dO^T of 64 queries, dV += P^T dO, dK += dS^T Q.  The queries are those of all
// heads of the group, one head after the other.  A block may do a part of them only: its sums then go to the workspace in
// fp32, and attention_dkdv_sum_kernel adds the parts in order.
template <int HALVES, int BUFFERS> using DkdvRoles = BwdRoles<BUFFERS, BUFFERS * 2 * kCols + 128 * HALVES>;
template <int HALVES, int BUFFERS>
__global__ void __launch_bounds__(128 * BUFFERS + 64, 1)
attention_dkdv_kernel(const __grid_constant__ AttentionMaps maps, const __grid_constant__ AttentionParams p, const DkdvPlan plan, DeviceStatus* status,
                      uint64_t wait_ns) {
    extern __shared__ uint8_t raw[];
    uint8_t* const base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* const tiles_ptr = base + kBwdControl;
    const uint32_t tiles = smem_u32(tiles_ptr);
    constexpr uint32_t kFixed = HALVES * kHalfTile, kStream = HALVES * kHalfCols;
    constexpr int kHd = 64 * HALVES;
    constexpr int kBuffers = BUFFERS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads_k = p.heads / p.group, units = p.batch * heads_k, unit = blockIdx.x % units;
    const int b = unit / heads_k, hk = unit % heads_k;
    // tiles whose keys stay visible come first, in their parts, then the others in theirs
    const int item = static_cast<int>(blockIdx.x / units);
    const bool keep = item < plan.sink_tiles * plan.sink_parts;
    const int parts = keep ? plan.sink_parts : plan.parts;
    const int at_item = keep ? item : item - plan.sink_tiles * plan.sink_parts;
    const int tile = (keep ? 0 : plan.sink_tiles) + at_item / parts, part = at_item % parts;
    const int j0 = tile * kRows, off = p.tk - p.tq;
    const QueryTiles q(p, j0);
    const int all = q.count * p.group, it0 = static_cast<int>(static_cast<int64_t>(all) * part / parts);
    DkdvRoles<HALVES, BUFFERS> roles{reinterpret_cast<BwdControl*>(base), nullptr, status, wait_ns, static_cast<int>(static_cast<int64_t>(all) * (part + 1) / parts) - it0};
    roles.abort_flag = &roles.ctl->abort;
    auto head_of = [&](int it) { return hk * p.group + (it0 + it) / q.count; };
    auto query_of = [&](int it) { return (q.first + (it0 + it) % q.count) * kCols; };
    roles.set_up(warp);
    const uint32_t tmem = uniform(roles.ctl->tmem);
    if (plan.parts > 1 || plan.sink_parts > 1) grid_launch_dependents();   // the launch that adds the parts
    grid_dependency_wait();
    const int steps_d = (p.head_dim + 15) / 16;
    const uint32_t ring = tiles + 2 * kFixed;
    auto tmem_acc = [&](int w) { return tmem + kBuffers * 2u * kCols + static_cast<uint32_t>(w) * kHd; };   // dV, dK

    if (warp == roles.kLoadWarp) {
        if (roles.n > 0 && elect_one()) {
            mbar_arrive_expect_tx(smem_u32(&roles.ctl->fixed), 2 * kFixed);
            for (int x = 0; x < HALVES; ++x) {
                tma_load_4d(tiles + x * kHalfTile, &maps.k, smem_u32(&roles.ctl->fixed), x * 64, j0, hk, b);
                tma_load_4d(tiles + kFixed + x * kHalfTile, &maps.v, smem_u32(&roles.ctl->fixed), x * 64, j0, hk, b);
            }
        }
        __syncwarp();
        roles.loads(2 * kStream, [&](int it, int slot, uint32_t bar) {
            const uint32_t at = ring + slot * 2 * kStream;
            for (int x = 0; x < HALVES; ++x) {
                tma_load_4d(at + x * kHalfCols, &maps.q, bar, x * 64, query_of(it), head_of(it), b);
                tma_load_4d(at + kStream + x * kHalfCols, &maps.dout, bar, x * 64, query_of(it), head_of(it), b);
            }
        });
    } else if (warp == roles.kProductWarp) {
        const uint32_t idesc_s = make_idesc_bf16(kRows, kCols, 0, 0), idesc_d = make_idesc_bf16(kRows, steps_d * 16, 0, 1);
        const uint32_t fixed_lo = uniform(desc_lo(tiles, 16)), ring_lo = uniform(desc_lo(ring, 16)), ring_mn = uniform(desc_lo(ring, kHalfCols));
        roles.template products<false>(
            [&](int slot, int buffer) {
                const uint32_t at = ring_lo + slot * (2 * kStream / 16), to = tmem + buffer * 2 * kCols;
                product_ss<HALVES>(to, fixed_lo, kHalfTile, at, kHalfCols, idesc_s, steps_d);
                product_ss<HALVES>(to + kCols, fixed_lo + kFixed / 16, kHalfTile, at + kStream / 16, kHalfCols, idesc_s, steps_d);
            },
            [&](int slot, int buffer, bool more) {
                const uint32_t at = ring_mn + slot * (2 * kStream / 16), from = tmem + buffer * 2 * kCols;
                product_ts<kCols / 16, 2>(tmem_acc(0), from, at + kStream / 16, idesc_d, more);        // dV += P^T dO
                product_ts<kCols / 16, 2>(tmem_acc(1), from + kCols, at, idesc_d, more);               // dK += dS^T Q
            });
    } else {
        const int w = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane, j = j0 + row;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const float c = p.scale * kLog2e;
        float4* const stats = roles.ctl->stats[warp];
        const uint64_t c2 = two(c, c);
        const int jw = j0 + quarter * 32;   // the warp's first key
        const bool ok = roles.tiles(w, [&](int it) {
            const int i0 = query_of(it);
            const int64_t at = (static_cast<int64_t>(b) * p.heads + head_of(it)) * p.tq + i0;
            // lane l has queries 2 l and 2 l + 1; P = 0 for a query that is not there or sees nothing
            float lse[2], d[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const bool there = i0 + 2 * lane + x < p.tq;
                lse[x] = there ? p.lse[at + 2 * lane + x] : -INFINITY;
                d[x] = there ? p.dvec[at + 2 * lane + x] : 0.0f;
                lse[x] = lse[x] == -INFINITY ? INFINITY : lse[x] * kLog2e;
            }
            __syncwarp();
            stats[lane] = make_float4(-lse[0], -lse[1], -d[0], -d[1]);
            __syncwarp();
        }, [&](int it) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {   // 32 queries at a time
                const uint32_t ts = tmem + w * 2 * kCols + x * 32 + lanes;
                const int p0 = query_of(it) + x * 32 + off;   // position of the first of them
                uint32_t s[32], dp[32];
                if (sees_none(p, p0, jw)) {
#pragma unroll
                    for (int y = 0; y < 16; ++y) s[y] = dp[y] = 0;
                } else {
                    tmem_ld_32x32(ts, s);
                    tmem_ld_32x32(ts + kCols, dp);
                    tmem_ld_wait();
                    if (sees_all(p, p0, jw)) {
#pragma unroll
                        for (int y = 0; y < 16; ++y) {
                            const ulonglong2 st = *reinterpret_cast<const ulonglong2*>(&stats[x * 16 + y]);
                            const float2 a = both(fma2(two(s[2 * y], s[2 * y + 1]), c2, st.x));
                            const float e0 = ex2_approx(a.x), e1 = ex2_approx(a.y);
                            const float2 f = both(mul2(two(e0, e1), add2(two(dp[2 * y], dp[2 * y + 1]), st.y)));
                            s[y] = pack_bf16(e0, e1);
                            dp[y] = pack_bf16(f.x, f.y);
                        }
                    } else {
                        const int from = j - p0;
                        const uint32_t seen = bits_between(from, j < p.sinks || from > 32 - p.window ? 32 : from + p.window, 0);
#pragma unroll
                        for (int y = 0; y < 16; ++y) {
                            const ulonglong2 st = *reinterpret_cast<const ulonglong2*>(&stats[x * 16 + y]);
                            const float2 a = both(fma2(two(s[2 * y], s[2 * y + 1]), c2, st.x));
                            float e0 = ex2_approx(a.x), e1 = ex2_approx(a.y);
                            float2 f = both(mul2(two(e0, e1), add2(two(dp[2 * y], dp[2 * y + 1]), st.y)));
                            if (!(seen >> 2 * y & 1u)) e0 = f.x = 0.0f;
                            if (!(seen >> 2 * y & 2u)) e1 = f.y = 0.0f;
                            s[y] = pack_bf16(e0, e1);
                            dp[y] = pack_bf16(f.x, f.y);
                        }
                    }
                }
                tmem_st_32x16(ts, s);
                tmem_st_32x16(ts + kCols, dp);
            }
        }, [] {});
        // the warpgroups share the 16-column pieces of dV and dK
        bool bad = false;
        for (int x = w; x < 8 * HALVES; x += kBuffers) {
            const int which = x / (4 * HALVES), piece = x % (4 * HALVES);
            const float factor = which == 0 ? 1.0f : p.scale;
            uint32_t o[16];
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] = 0;
            if (ok && roles.n > 0 && piece < steps_d) {
                tmem_ld_32x16(tmem_acc(which) + lanes + piece * 16, o);
                tmem_ld_wait();
            }
#pragma unroll
            for (int y = 0; y < 16; ++y) {
                const float f = __uint_as_float(o[y]) * factor;
                bad = bad || !(fabsf(f) < INFINITY);
                o[y] = __float_as_uint(f);
            }
            if (parts > 1) {
                float* const sums = p.partial + ((plan.slot(keep, unit, at_item, units) * 2 + which) * kRows + row) * kHd + piece * 16;
#pragma unroll
                for (int y = 0; y < 16; y += 4) *reinterpret_cast<uint4*>(sums + y) = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
            } else {
                put_row16(tiles_ptr + which * kFixed, row, piece, o);
            }
        }
        if (parts == 1)
            copy_out(roles.ctl->bad, 1, roles.kSoftmax, threadIdx.x == 0, quarter, __ballot_sync(0xffffffffu, bad && ok && j < p.tk), [&] {
                for (int x = 0; x < HALVES; ++x) {
                    tma_store_4d(&maps.dv, tiles + x * kHalfTile, x * 64, j0, hk, b);
                    tma_store_4d(&maps.dk, tiles + kFixed + x * kHalfTile, x * 64, j0, hk, b);
                }
            }, [&](int r) { attn::dkdv_row(p, b, hk, j0 + r); });
    }
    roles.tear_down(warp, tmem);
}

// Adds the parts of the tiles that were done in parts, a row of dV and dK per warp.
constexpr int kSumThreads = 256;
__global__ void __launch_bounds__(kSumThreads, 2) attention_dkdv_sum_kernel(const __grid_constant__ AttentionParams p, DkdvPlan plan, int kept, int pitch) {
    grid_dependency_wait();
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * kSumThreads + threadIdx.x) >> 5;
    const int units = p.batch * (p.heads / p.group), n_tiles = kept ? plan.sink_tiles : plan.tiles - plan.sink_tiles, parts = kept ? plan.sink_parts : plan.parts;
    if (at >= static_cast<int64_t>(units) * n_tiles * kRows) return;
    const int row = static_cast<int>(at % kRows), tile = static_cast<int>(at / kRows % n_tiles), unit = static_cast<int>(at / kRows / n_tiles);
    const int64_t j = static_cast<int64_t>(tile + (kept ? 0 : plan.sink_tiles)) * kRows + row;
    if (j >= p.tk) return;
    const int b = unit / (p.heads / p.group), hk = unit % (p.heads / p.group), c = 4 * (threadIdx.x & 31);
    bool bad = false;
    for (int what = 0; what < 2; ++what) {
        attn::Four s;
        if (c < p.head_dim)
            for (int part = 0; part < parts; ++part) {
                const float4 v = *reinterpret_cast<const float4*>(p.partial + ((plan.slot(kept != 0, unit, tile * parts + part, units) * 2 + what) * kRows + row) * pitch + c);
                s.v[0] += v.x; s.v[1] += v.y; s.v[2] += v.z; s.v[3] += v.w;
            }
        for (const float x : s.v) bad = bad || !(fabsf(x) < INFINITY);
        s.store(attn::row_to(what == 0 ? p.dv : p.dk, b, j, hk), 1.0f, p.head_dim);
    }
    if (__any_sync(0xffffffffu, bad)) {
        __syncwarp();
        attn::dkdv_row(p, b, hk, j);
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

DkdvPlan dkdv_plan(const AttentionParams& p, int sms) {
    DkdvPlan pl{};
    pl.tiles = (p.tk + kRows - 1) / kRows;
    // keys that queries far behind their window see: only worth a class of their own where such queries are
    const int last_far = (p.sinks < p.tk - p.window ? p.sinks : p.tk - p.window) - 1;   // the last sink that is one beyond its window
    pl.sink_tiles = last_far < 0 ? 0 : last_far / kRows + 1;
    pl.sink_parts = pl.parts = 1;
    if (p.tq == 0) return pl;
    // Microseconds of a tile and of a block's beginning and end, measured (8192 tokens, 16 heads on 4 of 128; 4096 tokens of 64).
    const float per_tile = p.head_dim <= 64 ? 0.75f : 1.05f, per_block = 5.0f;
    const int64_t units = static_cast<int64_t>(p.batch) * (p.heads / p.group), others = units * (pl.tiles - pl.sink_tiles);
    const int step = pl.tiles / 512 + 1;
    int64_t total = 0, most = 0, most_kept = 0;
    for (int t = 0; t < pl.tiles; t += step) {
        const int64_t n = static_cast<int64_t>(QueryTiles(p, t * kRows).count) * p.group;
        total += n * step * units;
        int64_t& m = t < pl.sink_tiles ? most_kept : most;
        m = n > m ? n : m;
    }
    // Time of a list of blocks, longest first: an even share of all, and a part of the longest that comes last.  Parts cost
    // their sums' way through memory and the launch that adds them.
    float best = 0.0f;
    for (int parts : {1, 2, 3, 4, 6, 8, 12, 16}) {
        if (parts > 1 && parts * 4 > most) break;
        const float all = static_cast<float>(total) * per_tile + static_cast<float>(others * parts) * per_block;
        const float longest = per_block + static_cast<float>((most + parts - 1) / parts) * per_tile;
        const float share = all / static_cast<float>(sms);
        const float cost = (share > longest ? share : longest) + 0.5f * longest +
                           (parts > 1 ? 4.0f + static_cast<float>(others * parts) * (p.head_dim <= 64 ? 0.044f : 0.087f) : 0.0f);
        if (parts == 1 || cost < best) {
            best = cost;
            pl.parts = parts;
        }
    }
    // Tiles that all later queries see: parts no longer than the other tiles' blocks.
    const int64_t longest = (most + pl.parts - 1) / pl.parts > 16 ? (most + pl.parts - 1) / pl.parts : 16;
    if (most_kept > longest) pl.sink_parts = static_cast<int>((most_kept + longest - 1) / longest < 64 ? (most_kept + longest - 1) / longest : 64);
    return pl;
}

size_t dkdv_partial_floats(const AttentionParams& p, const DkdvPlan& pl) {
    const int64_t units = static_cast<int64_t>(p.batch) * (p.heads / p.group);
    return static_cast<size_t>(pl.slots(units)) * 2 * kRows * (p.head_dim <= 64 ? 64 : 128);
}

size_t dvec_bytes(const AttentionParams& p) { return (static_cast<size_t>(p.batch) * p.heads * p.tq * sizeof(float) + 255) / 256 * 256; }

}  // namespace

// In how many parts the keys of a query block are done: more than one where the blocks alone leave SMs without work.
namespace {
// Microseconds of a tile (where blocks share an SM's time, and where they do not), of a block's beginning and end.
struct PartCosts {
    float alone, shared, per_block;
};
int query_parts(const AttentionParams& p, int sms, int per, int64_t units, int blocks_per_sm, int cols, PartCosts cost_of) {
    const int64_t blocks_q = (p.tq + per - 1) / per, blocks = units * blocks_q, slots = static_cast<int64_t>(sms) * blocks_per_sm;
    if (blocks >= 2 * slots) return 1;
    int64_t total = 0, most = 0;   // tiles of all blocks, of the longest
    for (int64_t q = 0; q < blocks_q; ++q) {
        const int64_t p0 = q * per + p.tk - p.tq, p1 = (p.tq < (q + 1) * per ? p.tq : (q + 1) * per) - 1 + p.tk - p.tq;
        if (p1 < 0) continue;
        const int64_t begin = p0 - p.window + 1 > 0 ? p0 - p.window + 1 : 0, low = begin / cols;
        const int64_t kept = ((p.sinks < begin ? p.sinks : begin) + cols - 1) / cols;
        const int64_t n = (kept < low ? kept : low) + p1 / cols - low + 1;
        total += n;
        most = n > most ? n : most;
    }
    const int64_t row_blocks = static_cast<int64_t>(p.batch) * p.heads * ((p.tq + kRows - 1) / kRows);
    float best = 0.0f;
    int chosen = 1;
    for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, kMostParts}) {
        if (parts > 1 && parts * 2 * kRows > most * cols) break;
        const float longest = cost_of.per_block + static_cast<float>((most + parts - 1) / parts) * (blocks * parts > sms ? cost_of.shared : cost_of.alone);
        const float share = (static_cast<float>(total * units) * cost_of.shared + static_cast<float>(blocks * parts) * cost_of.per_block) / static_cast<float>(slots);
        const float cost = (blocks * parts <= slots ? longest : (share > longest ? share : longest) + 0.25f * longest) +
                           (parts > 1 ? 4.0f + static_cast<float>(row_blocks * parts) * (p.head_dim <= 64 ? 32768.0f : 65536.0f) / 3.5e6f : 0.0f);   // the join
        if (parts == 1 || cost < best) {
            best = cost;
            chosen = parts;
        }
    }
    return chosen;
}
// Costs fitted to 1 .. 32 parts of seventeen shapes.  Forward: 64 queries on 8192 keys, 16 heads on 4 of 128: 125 us whole, 22 in 16
// parts; 2 x 8192 of 128: 127 and 56 (4 parts); 4 x 4096 of 64: 49 and 37 (4); 12 x 1024 of 64: 16.4 and 20 (2: not taken).
// Backward (with dK and dV): the first 124 and 46 (8 parts of dQ); 1 x 8192 of 64: 165 and 82 (8), of 128: 173 and 105 (4); 4 heads
// on 1, 8192 of 128: 296 and 313 (2: not taken).
int fwd_parts(const AttentionParams& p, int sms) {
    const bool narrow = p.head_dim <= 64, pair_heads = !narrow && p.group % 2 == 0;
    return query_parts(p, sms, narrow || pair_heads ? kRows : 2 * kRows, static_cast<int64_t>(p.batch) * p.heads / (pair_heads ? 2 : 1), narrow ? 2 : 1, kRows,
                       narrow ? PartCosts{1.3f, 1.7f, 6.0f} : PartCosts{1.85f, 1.85f, 6.0f});
}
int dq_parts(const AttentionParams& p, int sms) {
    const bool narrow = p.head_dim <= 64;
    return query_parts(p, sms, kRows, static_cast<int64_t>(p.batch) * p.heads, narrow ? 2 : 1, kCols, narrow ? PartCosts{0.75f, 1.2f, 6.0f} : PartCosts{0.9f, 0.9f, 8.0f});
}
// What parts of query blocks take in a workspace: 16-byte pieces of fp32 rows, and a float a row.
int64_t query_part_floats(const AttentionParams& p, int parts) {
    return parts == 1 ? 0 : static_cast<int64_t>(p.batch) * p.heads * ((p.tq + kRows - 1) / kRows) * kRows * parts * ((p.head_dim <= 64 ? 64 : 128) + 1);
}
void put_query_parts(AttentionParams& p, int parts) {
    p.part_stats = parts == 1 ? nullptr : p.partial + static_cast<int64_t>(p.batch) * p.heads * ((p.tq + kRows - 1) / kRows) * kRows * parts * (p.head_dim <= 64 ? 64 : 128);
}
template <bool FORWARD> cudaError_t launch_join(const AttentionParams& p, int parts, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(static_cast<int64_t>(p.batch) * p.heads * ((p.tq + kRows - 1) / kRows) * 4);
    return p.head_dim <= 64 ? launch_dependent(attention_join_kernel<2, FORWARD>, blocks, kJoinWarps * 32, stream, p, parts)
                            : launch_dependent(attention_join_kernel<4, FORWARD>, blocks, kJoinWarps * 32, stream, p, parts);
}
}  // namespace

size_t attention_bwd_sm100_workspace(const AttentionParams& p, int sms) {
    // the parts of dQ are joined before those of dK and dV come
    const int64_t of_dq = p.tq > 0 && p.tk > 0 && p.batch > 0 && p.heads > 0 ? query_part_floats(p, dq_parts(p, sms)) : 0, of_dkdv = dkdv_partial_floats(p, dkdv_plan(p, sms));
    return dvec_bytes(p) + (of_dq > of_dkdv ? of_dq : of_dkdv) * sizeof(float);
}

cudaError_t launch_attention_bwd_sm100(AttentionParams p, const CUtensorMap* m, void* workspace, int sms, DeviceStatus* status, uint64_t wait_ns,
                                       cudaStream_t stream) {
    p.dvec = static_cast<float*>(workspace);
    p.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + dvec_bytes(p));
    AttentionMaps maps{};
    // dQ: blocks of 128 queries, tiles of 64 keys; dK, dV: blocks of 128 keys, tiles of 64 queries
    maps.q = m[0]; maps.dout = m[1]; maps.k = m[2]; maps.v = m[3]; maps.dq = m[4];
    const int blocks_q = (p.tq + kRows - 1) / kRows;
    const bool narrow = p.head_dim <= 64;
    const int parts = dq_parts(p, sms);
    put_query_parts(p, parts);
    // A query sees 128 keys or fewer: six tiles, twice, are never done in parts.
    const int64_t seen = static_cast<int64_t>(p.window) + p.sinks;
    const bool exact = (seen < p.tk ? seen : p.tk) <= 128;
    int64_t blocks = static_cast<int64_t>(p.batch) * p.heads * blocks_q * parts;
    auto dq = [&](auto kernel, int threads, size_t smem) { return launch_sm(kernel, blocks, threads, smem, stream, maps, p, blocks_q, parts, status, wait_ns); };
    cudaError_t e = narrow ? dq(parts > 1 ? attention_dq_kernel<1, 1, Dq::kParts> : exact ? attention_dq_kernel<1, 1, Dq::kExact> : attention_dq_kernel<1, 1, Dq::kWhole>,
                                DqRoles<1, 1>::kThreads, bwd_smem<1>())
                           : dq(parts > 1 ? attention_dq_kernel<2, 3, Dq::kParts> : exact ? attention_dq_kernel<2, 3, Dq::kExact> : attention_dq_kernel<2, 3, Dq::kWhole>,
                                DqRoles<2, 3>::kThreads, bwd_smem<2>());
    if (e == cudaSuccess && parts > 1) e = launch_join<false>(p, parts, stream);
    if (e != cudaSuccess) return e;
    maps.q = m[5]; maps.dout = m[6]; maps.k = m[7]; maps.v = m[8]; maps.dk = m[9]; maps.dv = m[10];
    const DkdvPlan pl = dkdv_plan(p, sms);
    const int64_t units = static_cast<int64_t>(p.batch) * (p.heads / p.group);
    blocks = units * pl.items();
    e = narrow ? launch_sm(attention_dkdv_kernel<1, 3>, blocks, DkdvRoles<1, 3>::kThreads, bwd_smem<1>(), stream, maps, p, pl, status, wait_ns)
               : launch_sm(attention_dkdv_kernel<2, 2>, blocks, DkdvRoles<2, 2>::kThreads, bwd_smem<2>(), stream, maps, p, pl, status, wait_ns);
    for (int kept = 1; kept >= 0 && e == cudaSuccess; --kept) {
        const int n_tiles = kept ? pl.sink_tiles : pl.tiles - pl.sink_tiles;
        if (n_tiles == 0 || (kept ? pl.sink_parts : pl.parts) == 1) continue;
        const int64_t rows = units * n_tiles * kRows;
        e = launch_dependent(attention_dkdv_sum_kernel, static_cast<unsigned>((rows * 32 + kSumThreads - 1) / kSumThreads), kSumThreads, stream, p, pl, kept,
                             narrow ? 64 : 128);
    }
    return e;
}

size_t attention_fwd_sm100_workspace(const AttentionParams& p, int sms) {
    if (p.tq == 0 || p.tk == 0 || p.batch == 0 || p.heads == 0) return 0;
    return static_cast<size_t>(query_part_floats(p, fwd_parts(p, sms))) * sizeof(float);
}

cudaError_t launch_attention_fwd_sm100(AttentionParams p, const CUtensorMap* m, void* workspace, int sms, DeviceStatus* status, uint64_t wait_ns,
                                       cudaStream_t stream) {
    AttentionMaps maps{};
    maps.q = m[0]; maps.k = m[1]; maps.v = m[2]; maps.out = m[3];
    const bool narrow = p.head_dim <= 64;
    const int parts = workspace != nullptr ? fwd_parts(p, sms) : 1;
    const int64_t heads = static_cast<int64_t>(p.batch) * p.heads;
    p.partial = static_cast<float*>(workspace);
    put_query_parts(p, parts);
    cudaError_t e;
    if (narrow) {
        const int blocks_q = (p.tq + kRows - 1) / kRows;
        e = launch_sm(parts > 1 ? attention_fwd_kernel<1, 1, true> : attention_fwd_kernel<1, 1, false>, heads * blocks_q * parts, 192, fwd_smem<1, 1>(), stream, maps, p, 0, blocks_q, parts, status, wait_ns);
    } else {
        const int pair_heads = p.group % 2 == 0, per = pair_heads ? kRows : 2 * kRows, blocks_q = (p.tq + per - 1) / per;
        e = launch_sm(parts > 1 ? attention_fwd_kernel<2, 2, true> : attention_fwd_kernel<2, 2, false>, heads / (pair_heads ? 2 : 1) * blocks_q * parts, 320, fwd_smem<2, 2>(), stream, maps, p, pair_heads, blocks_q,
                      parts, status, wait_ns);
    }
    return e != cudaSuccess || parts == 1 ? e : launch_join<true>(p, parts, stream);
}

}  // namespace llmt_b200
