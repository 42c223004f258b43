// Attention of one new token per sequence over a cache: see llmt_b200_attention_window_decode in the public header.
//
// Bound: memory; each visible row of K and V is read once for all query heads that share it.  A warp takes 16 keys at a time:
// S = Q K^T and O += P V by 16 x 8 x 16 matrix instructions whose 16 rows are the heads.  The order of a product's inner index
// is free as long as both operands have the same, and so is the order of the result's columns: a thread's operand values are
// the 16 bytes that it loads (eight neighbouring values of its key for S, of two keys for P V), and nothing passes through
// shared memory from one thread to another.  It does wait there: each thread copies its own 16-byte pieces of the steps to
// come into shared memory (cp.async, kStages - 1 steps ahead), which keeps 128 KB an SM under way where registers held 64.
// The warps of a block share a chunk of a sequence's keys and join their running maxima, sums and outputs at the end; where a
// sequence has several chunks, a second launch joins those.  Chunks have one length for all sequences, so a long one of a
// ragged batch is many blocks (shares of every sequence, in clusters that join through distributed shared memory: 4 sequences
// of 8 to 65536 places, 32 heads on 8 of 128, 177 us against 147).
// Measured: those 4 sequences 153 us with both launches, 721 MB at 4.7 TB/s; 32 sequences of up to 1024 places, 12 heads of 64,
// window 256: 8.7 us for 25 MB, a launch and one chunk's latency.
#include "attention_rows.cuh"
#include "ptx_sm100.cuh"

namespace llmt_b200 {
namespace {

constexpr int kDecodeWarps = 4, kStages = 2;
constexpr float kLog2e = 1.4426950408889634f;

// D += A B, 16 x 8 x 16; lane 4 g + t has A[g][.], A[g + 8][.] (inner values 2t, 2t + 1 and 2t + 8, 2t + 9 of either),
// B[.][g] (the same inner values) and D[g][2t, 2t + 1], D[g + 8][2t, 2t + 1].
__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The steps under way, [step][piece][thread]; afterwards the maxima, sums and outputs of the warps.
template <int ROWS, int CHUNKS> union DecodeShared {
    uint4 pieces[kStages][8 * CHUNKS][kDecodeWarps * 32];
    struct {
        float part_o[kDecodeWarps][ROWS][64 * CHUNKS];
        float part_m[kDecodeWarps][ROWS], part_l[kDecodeWarps][ROWS];
    } join;
};

// How a sequence's keys are shared out, and where the chunks' results go (where there are several).
struct DecodePlan {
    int chunks, steps;   // at most; of 16 keys each
    float* o;            // [batch][heads][chunks][64 CHUNKS]
    float2* ml;          // [batch][heads][chunks]
};

// 16 bytes into shared memory, zeros where there is nothing to copy.
__device__ __forceinline__ void copy16(uint4* to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// The place of a sequence's newest key: never past the cache, -1 for an empty one.
__device__ __forceinline__ int64_t last_place(const AttentionParams& p, int b) {
    const int64_t n = p.lengths != nullptr ? p.lengths[b] : p.tk;
    return (n < p.tk ? n : p.tk) - 1;
}
// One value of a head's output from the maximum score, the sum of exponentials and the sum of values.
__device__ __forceinline__ void finish(const AttentionParams& p, int b, int h, int col, float top, float sum, float total) {
    if (col < p.head_dim) attn::row_to(p.out, b, 0, h)[col] = __float2bfloat16_rn(total == 0.0f ? 0.0f : sum / total);
    if (col == 0 && p.lse != nullptr)
        p.lse[static_cast<int64_t>(b) * p.heads + h] = total == 0.0f ? -INFINITY : fmaf(top, p.scale, log2f(total) * (1.0f / kLog2e));
}

// CHUNKS: head_dim in steps of 64; ROWS: heads of a block, 8 or 16 (a group of more heads is several blocks).
template <int CHUNKS, int ROWS>
__global__ void __launch_bounds__(kDecodeWarps * 32, 2) attention_decode_kernel(AttentionParams p, int head_blocks, DecodePlan plan) {
    constexpr int kHd = 64 * CHUNKS, kRows = ROWS / 8;
    extern __shared__ float4 raw[];
    auto& sh = *reinterpret_cast<DecodeShared<ROWS, CHUNKS>*>(raw);
    auto& part_o = sh.join.part_o;
    auto& part_m = sh.join.part_m;
    auto& part_l = sh.join.part_l;
    ptx::grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // neighbouring blocks do the same places of neighbouring heads, whose rows are neighbours in memory where a token's are
    const int heads_k = p.heads / p.group;
    const int hb = blockIdx.x % head_blocks, hk = blockIdx.x / head_blocks % heads_k;
    const int chunk = blockIdx.x / (head_blocks * heads_k) % plan.chunks, b = blockIdx.x / (head_blocks * heads_k) / plan.chunks;
    const int h0 = hk * p.group + hb * ROWS, heads = min(ROWS, p.group - hb * ROWS);
    const attn::Keys keys(p, last_place(p, b));
    const int64_t steps = (keys.count + 15) / 16, step0 = static_cast<int64_t>(chunk) * plan.steps;
    const int64_t step1 = step0 + plan.steps < steps ? step0 + plan.steps : steps;
    if (chunk > 0 && step0 >= steps) return;   // the sequence has no such chunk (its first one is there even if it has no keys)
    const float c = p.scale * kLog2e;

    // Q's rows g (and g + 8): of each run of 32 values the eight from 8 t on
    uint4 q[kRows][2 * CHUNKS];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int x = 0; x < 2 * CHUNKS; ++x) {
            const int at = 32 * x + 8 * t;
            q[r][x] = make_uint4(0, 0, 0, 0);
            if (g + 8 * r < heads && at < p.head_dim) q[r][x] = *reinterpret_cast<const uint4*>(attn::row_of(p.q, b, 0, h0 + g + 8 * r) + at);
        }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[8 * CHUNKS][4];
#pragma unroll
    for (int x = 0; x < 8 * CHUNKS; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[x][y] = 0.0f;
    const __nv_bfloat16 *const k0 = attn::row_of(p.k, b, 0, hk), *const v0 = attn::row_of(p.v, b, 0, hk);

    // One group of copies a step, empty past the last, so that the wait below always counts the same.  Most steps are whole
    // and behind the sinks: their rows are kDecodeWarps * 16 places behind the warp's last ones.
    const int64_t hop_k = p.k.stride_token * (16 * kDecodeWarps), hop_v = p.v.stride_token * (16 * kDecodeWarps);
    const int64_t shift = keys.low - keys.sinks, begin = (step0 + warp) * 16 + shift;
    const __nv_bfloat16* kp[2] = {k0 + (begin + g) * p.k.stride_token + 8 * t, k0 + (begin + 8 + g) * p.k.stride_token + 8 * t};
    const __nv_bfloat16* vp[2] = {v0 + (begin + 2 * t) * p.v.stride_token + 8 * g, v0 + (begin + 8 + 2 * t) * p.v.stride_token + 8 * g};
    bool in_k[2 * CHUNKS], in_v[CHUNKS];
#pragma unroll
    for (int x = 0; x < 2 * CHUNKS; ++x) in_k[x] = 32 * x + 8 * t < p.head_dim;
#pragma unroll
    for (int x = 0; x < CHUNKS; ++x) in_v[x] = 64 * x + 8 * g < p.head_dim;
    auto load = [&](int64_t step, int stage) {
        if (step < step1) {
            const int64_t n0 = step * 16;
            uint4* to = &sh.pieces[stage][0][threadIdx.x];
            const bool plain = n0 >= keys.sinks && n0 + 16 <= keys.count;
#pragma unroll
            for (int y = 0; y < 2; ++y) {   // keys g and 8 + g of the sixteen
                const int64_t at = n0 + 8 * y + g;
                const bool there = plain || at < keys.count;
                const __nv_bfloat16* row = plain ? kp[y] : k0 + (there ? keys.at(at) : 0) * p.k.stride_token + 8 * t;
#pragma unroll
                for (int x = 0; x < 2 * CHUNKS; ++x, to += kDecodeWarps * 32) copy16(to, in_k[x] ? row + 32 * x : k0, there && in_k[x]);
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {   // keys 2t, 2t + 1, 8 + 2t, 9 + 2t
                const int64_t at = n0 + 8 * (y >> 1) + 2 * t + (y & 1);
                const bool there = plain || at < keys.count;
                const __nv_bfloat16* row = plain ? vp[y >> 1] + (y & 1) * p.v.stride_token : v0 + (there ? keys.at(at) : 0) * p.v.stride_token + 8 * g;
#pragma unroll
                for (int x = 0; x < CHUNKS; ++x, to += kDecodeWarps * 32) copy16(to, in_v[x] ? row + 64 * x : v0, there && in_v[x]);
            }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            kp[y] += hop_k;
            vp[y] += hop_v;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int stage = 0;
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) load(step0 + warp + i * kDecodeWarps, i);

    for (int64_t step = step0 + warp; step < step1; step += kDecodeWarps) {
        const int64_t n0 = step * 16;
        const int free = stage == 0 ? kStages - 1 : stage - 1;   // what the last round has read
        load(step + (kStages - 1) * kDecodeWarps, free);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        uint4 kx[2][2 * CHUNKS], vx[4][CHUNKS];
        const uint4* from = &sh.pieces[stage][0][threadIdx.x];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 2 * CHUNKS; ++x, from += kDecodeWarps * 32) kx[y][x] = *from;
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int x = 0; x < CHUNKS; ++x, from += kDecodeWarps * 32) vx[y][x] = *from;
        if (++stage == kStages) stage = 0;
        float s[2][4];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int z = 0; z < 4; ++z) s[y][z] = 0.0f;
#pragma unroll
            for (int x = 0; x < 2 * CHUNKS; ++x) {
                const uint4 q1 = kRows == 2 ? q[kRows - 1][x] : make_uint4(0, 0, 0, 0);
                mma_bf16(s[y], q[0][x].x, q1.x, q[0][x].y, q1.y, kx[y][x].x, kx[y][x].y);
                mma_bf16(s[y], q[0][x].z, q1.z, q[0][x].w, q1.w, kx[y][x].z, kx[y][x].w);
            }
            if (n0 + 16 > keys.count) {   // this thread has the scores of keys 2t and 2t + 1 of the eight
                if (n0 + 8 * y + 2 * t >= keys.count) s[y][0] = s[y][2] = -INFINITY;
                if (n0 + 8 * y + 2 * t + 1 >= keys.count) s[y][1] = s[y][3] = -INFINITY;
            }
        }
        uint32_t pr[2][2] = {{0, 0}, {0, 0}};   // [row][half of the keys]
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m_new = fmaxf(m[r], top), from = m_new == -INFINITY ? 0.0f : m_new * c;
            if (__any_sync(0xffffffffu, m_new > m[r])) {
                const float shrink = ex2_approx(m[r] * c - from);   // 0 for the first keys
                l[r] *= shrink;
#pragma unroll
                for (int x = 0; x < 8 * CHUNKS; ++x) {
                    o[x][2 * r] *= shrink;
                    o[x][2 * r + 1] *= shrink;
                }
                m[r] = m_new;
            }
            float e[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) e[z] = ex2_approx(fmaf(s[z >> 1][2 * r + (z & 1)], c, -from));
            l[r] += (e[0] + e[1]) + (e[2] + e[3]);
            pr[r][0] = pack2(e[0], e[1]);
            pr[r][1] = pack2(e[2], e[3]);
        }
#pragma unroll
        for (int x = 0; x < CHUNKS; ++x) {
            const uint32_t a[4] = {vx[0][x].x, vx[0][x].y, vx[0][x].z, vx[0][x].w}, bb[4] = {vx[1][x].x, vx[1][x].y, vx[1][x].z, vx[1][x].w};
            const uint32_t cc[4] = {vx[2][x].x, vx[2][x].y, vx[2][x].z, vx[2][x].w}, d[4] = {vx[3][x].x, vx[3][x].y, vx[3][x].z, vx[3][x].w};
#pragma unroll
            for (int y = 0; y < 8; ++y) {   // column g of result y is value 64 x + 8 g + y
                const uint32_t pick = y & 1 ? 0x7632u : 0x5410u;
                mma_bf16(o[8 * x + y], pr[0][0], pr[1][0], pr[0][1], pr[1][1], __byte_perm(a[y >> 1], bb[y >> 1], pick), __byte_perm(cc[y >> 1], d[y >> 1], pick));
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();   // the steps' place is free
    // ---- the warps' parts: thread (g, t) has rows g, g + 8 and of each result the columns 2t, 2t + 1, i.e. values 64 x + 16 t + y and + 8
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (t == 0) {
            part_m[warp][g + 8 * r] = m[r];
            part_l[warp][g + 8 * r] = l[r];
        }
#pragma unroll
        for (int x = 0; x < CHUNKS; ++x)
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                part_o[warp][g + 8 * r][64 * x + 16 * t + y] = o[8 * x + y][2 * r];
                part_o[warp][g + 8 * r][64 * x + 16 * t + 8 + y] = o[8 * x + y][2 * r + 1];
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * kHd; i += kDecodeWarps * 32) {
        const int row = i / kHd, col = i % kHd;
        float top = -INFINITY, sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int x = 0; x < kDecodeWarps; ++x) top = fmaxf(top, part_m[x][row]);
        const float from = top == -INFINITY ? 0.0f : top * c;
#pragma unroll
        for (int x = 0; x < kDecodeWarps; ++x) {
            const float w = ex2_approx(part_m[x][row] * c - from);
            sum = fmaf(w, part_o[x][row][col], sum);
            total = fmaf(w, part_l[x][row], total);
        }
        if (row >= heads) continue;
        if (plan.chunks == 1) {
            finish(p, b, h0 + row, col, top, sum, total);
        } else {
            const int64_t at = (static_cast<int64_t>(b) * p.heads + h0 + row) * plan.chunks + chunk;
            plan.o[at * kHd + col] = sum;
            if (col == 0) plan.ml[at] = make_float2(top, total);
        }
    }
}

// Joins the chunks of one head's sequence.  A thread has four neighbouring values of every 16th chunk (head_dim 128; of every
// 32nd for 64), eight of them under way: with one after the other 148 chunks took 40 us, with a value and every fourth chunk a
// thread one sequence of 65536 places (4 heads on 1, 256 chunks) 27 us with both launches, so 15.
constexpr int kJoinThreads = 512;
__global__ void __launch_bounds__(kJoinThreads) attention_decode_join_kernel(AttentionParams p, DecodePlan plan, int pitch) {
    __shared__ float weight[kJoinThreads], red[32];
    __shared__ float4 part[kJoinThreads];
    ptx::grid_dependency_wait();
    const int b = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
    const int fours = pitch / 4, groups = kJoinThreads / fours, group = threadIdx.x / fours;
    const attn::Keys keys(p, last_place(p, b));
    const int64_t steps = (keys.count + 15) / 16;
    const int chunks = steps > plan.steps ? static_cast<int>((steps + plan.steps - 1) / plan.steps) : 1;
    const float2* ml = plan.ml + static_cast<int64_t>(blockIdx.x) * plan.chunks;
    const float4* o = reinterpret_cast<const float4*>(plan.o) + static_cast<int64_t>(blockIdx.x) * plan.chunks * fours + threadIdx.x % fours;
    auto block = [&](float v, bool max) {   // of all threads, in one order
        v = max ? attn::warp_max(v) : attn::warp_add(v);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        float r = red[0];
        for (int i = 1; i < kJoinThreads / 32; ++i) r = max ? fmaxf(r, red[i]) : r + red[i];
        return r;
    };
    float top = -INFINITY, total = 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int x = threadIdx.x; x < chunks; x += kJoinThreads) top = fmaxf(top, ml[x].x);
    top = block(top, true);
    const float c = p.scale * kLog2e, from = top == -INFINITY ? 0.0f : top * c;
    for (int x0 = 0; x0 < chunks; x0 += kJoinThreads) {
        const int n = chunks - x0 < kJoinThreads ? chunks - x0 : kJoinThreads;
        float w = 0.0f;
        if (static_cast<int>(threadIdx.x) < n) {
            const float2 v = ml[x0 + threadIdx.x];
            w = ex2_approx(v.x * c - from);
            total = fmaf(w, v.y, total);
        }
        __syncthreads();
        weight[threadIdx.x] = w;
        __syncthreads();
#pragma unroll 8
        for (int x = group; x < n; x += groups) {
            const float4 v = o[static_cast<int64_t>(x0 + x) * fours];
            const float w = weight[x];
            sum.x = fmaf(w, v.x, sum.x); sum.y = fmaf(w, v.y, sum.y); sum.z = fmaf(w, v.z, sum.z); sum.w = fmaf(w, v.w, sum.w);
        }
    }
    part[threadIdx.x] = sum;
    total = block(total, false);
    const int col = threadIdx.x;
    if (col >= p.head_dim) return;
    float s = 0.0f;
    for (int i = 0; i < groups; ++i) s += reinterpret_cast<const float*>(part)[i * pitch + col];
    finish(p, b, h, col, top, s, total);
}

template <int CHUNKS, int ROWS>
cudaError_t launch_decode(const AttentionParams& p, const DecodePlan& plan, cudaStream_t stream) {
    const int head_blocks = (p.group + ROWS - 1) / ROWS;
    const int64_t units = static_cast<int64_t>(p.batch) * (p.heads / p.group) * head_blocks;
    constexpr size_t kShared = sizeof(DecodeShared<ROWS, CHUNKS>);
    const cudaError_t set = cudaFuncSetAttribute(attention_decode_kernel<CHUNKS, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kShared));
    if (set != cudaSuccess) return set;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(units * plan.chunks));
    cfg.blockDim = dim3(kDecodeWarps * 32);
    cfg.dynamicSmemBytes = kShared;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, attention_decode_kernel<CHUNKS, ROWS>, p, head_blocks, plan);
    count_launch(1);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess || plan.chunks == 1) return e;
    return launch_dependent(attention_decode_join_kernel, static_cast<unsigned>(p.batch * p.heads), kJoinThreads, stream, p, plan, 64 * CHUNKS);
}

// Chunks: none shorter than 256 keys; of short sequences as many as give each SM two blocks, of long ones eight, so that
// blocks that begin later even out the lengths.
DecodePlan decode_plan(const AttentionParams& p, int sms) {
    const int rows = p.group <= 8 ? 8 : 16;
    const int64_t units = static_cast<int64_t>(p.batch) * (p.heads / p.group) * ((p.group + rows - 1) / rows);
    const int64_t longest = static_cast<int64_t>(p.window) + p.sinks < p.tk ? static_cast<int64_t>(p.window) + p.sinks : p.tk;
    int64_t chunks = ((longest >= 4096 ? 8 : 2) * static_cast<int64_t>(sms) + units - 1) / units;
    if (chunks > longest / 256) chunks = longest / 256;
    if (chunks < 1) chunks = 1;
    DecodePlan plan{};
    plan.steps = static_cast<int>(((longest + 15) / 16 + chunks - 1) / chunks);
    if (plan.steps < 1) plan.steps = 1;
    plan.chunks = static_cast<int>(((longest + 15) / 16 + plan.steps - 1) / plan.steps);
    if (plan.chunks < 1) plan.chunks = 1;
    return plan;
}

}  // namespace

// Of each chunk of each head: fp32 outputs, and a maximum and a sum.
size_t attention_decode_workspace(const AttentionParams& p, int sms) {
    if (p.batch == 0 || p.heads == 0) return 0;
    const DecodePlan plan = decode_plan(p, sms);
    return plan.chunks == 1 ? 0 : static_cast<size_t>(p.batch) * p.heads * plan.chunks * ((p.head_dim <= 64 ? 64 : 128) + 2) * sizeof(float);
}

cudaError_t launch_attention_window_decode(const AttentionParams& p, int sms, void* workspace, cudaStream_t stream) {
    DecodePlan plan = decode_plan(p, sms);
    plan.o = static_cast<float*>(workspace);
    plan.ml = reinterpret_cast<float2*>(plan.o + static_cast<int64_t>(p.batch) * p.heads * plan.chunks * (p.head_dim <= 64 ? 64 : 128));
    if (p.head_dim <= 64) return p.group <= 8 ? launch_decode<1, 8>(p, plan, stream) : launch_decode<1, 16>(p, plan, stream);
    return p.group <= 8 ? launch_decode<2, 8>(p, plan, stream) : launch_decode<2, 16>(p, plan, stream);
}

}  // namespace llmt_b200
