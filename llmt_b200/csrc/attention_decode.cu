// Attention of one new token per sequence over a cache: see llmt_b200_attention_window_decode in the public header.
//
// Bound: memory; each visible row of K and V is read once for all query heads that share it.  A warp takes 16 keys at a time:
// S = Q K^T and O += P V by 16 x 8 x 16 matrix instructions whose 16 rows are the heads.  The order of a product's inner index
// is free as long as both operands have the same, and so is the order of the result's columns: a thread's operand values are
// the 16 bytes that it loads (eight neighbouring values of its key for S, of two keys for P V), and nothing passes through
// shared memory on the way.  The warps of a block, and the blocks of a cluster, share a sequence's keys and join their
// running maxima, sums and outputs at the end.
#include <cooperative_groups.h>

#include "attention_rows.cuh"
#include "ptx_sm100.cuh"

namespace llmt_b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kDecodeWarps = 8;
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

// Maxima, sums and outputs of the warps, and of the block.
template <int ROWS, int HD> struct DecodeShared {
    float part_o[kDecodeWarps][ROWS][HD], own_o[ROWS][HD];
    float part_m[kDecodeWarps][ROWS], part_l[kDecodeWarps][ROWS], own_m[ROWS], own_l[ROWS];
};

// CHUNKS: head_dim in steps of 64; ROWS: heads of a block, 8 or 16 (a group of more heads is several blocks).
template <int CHUNKS, int ROWS>
__global__ void __launch_bounds__(kDecodeWarps * 32) attention_decode_kernel(AttentionParams p, int head_blocks, int splits) {
    constexpr int kHd = 64 * CHUNKS, kRows = ROWS / 8;
    using Shared = DecodeShared<ROWS, kHd>;
    extern __shared__ float4 raw[];
    Shared& sh = *reinterpret_cast<Shared*>(raw);
    auto& part_o = sh.part_o;
    auto& part_m = sh.part_m;
    auto& part_l = sh.part_l;
    auto& own_o = sh.own_o;
    auto& own_m = sh.own_m;
    auto& own_l = sh.own_l;
    ptx::grid_dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % splits, unit = blockIdx.x / splits;
    const int heads_k = p.heads / p.group;
    const int hb = unit % head_blocks, hk = unit / head_blocks % heads_k, b = unit / head_blocks / heads_k;
    const int h0 = hk * p.group + hb * ROWS, heads = min(ROWS, p.group - hb * ROWS);
    int64_t n = p.lengths != nullptr ? p.lengths[b] : p.tk;
    n = n < p.tk ? n : p.tk;   // never past the cache
    const attn::Keys keys(p, n - 1);
    const int64_t steps = (keys.count + 15) / 16;
    const int64_t step0 = steps * rank / splits, step1 = steps * (rank + 1) / splits;
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

    for (int64_t step = step0 + warp; step < step1; step += kDecodeWarps) {
        const int64_t n0 = step * 16;
        uint4 kx[2][2 * CHUNKS], vx[4][CHUNKS];
#pragma unroll
        for (int y = 0; y < 2; ++y) {   // keys g and 8 + g of the sixteen
            const int64_t at = n0 + 8 * y + g;
            const __nv_bfloat16* row = k0 + keys.at(at) * p.k.stride_token;
#pragma unroll
            for (int x = 0; x < 2 * CHUNKS; ++x) {
                kx[y][x] = make_uint4(0, 0, 0, 0);
                if (at < keys.count && 32 * x + 8 * t < p.head_dim) kx[y][x] = *reinterpret_cast<const uint4*>(row + 32 * x + 8 * t);
            }
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {   // keys 2t, 2t + 1, 8 + 2t, 9 + 2t
            const int64_t at = n0 + 8 * (y >> 1) + 2 * t + (y & 1);
            const __nv_bfloat16* row = v0 + keys.at(at) * p.v.stride_token;
#pragma unroll
            for (int x = 0; x < CHUNKS; ++x) {
                vx[y][x] = make_uint4(0, 0, 0, 0);
                if (at < keys.count && 64 * x + 8 * g < p.head_dim) vx[y][x] = *reinterpret_cast<const uint4*>(row + 64 * x + 8 * g);
            }
        }
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
            // this thread has the scores of keys 2t and 2t + 1 of the eight
            if (n0 + 8 * y + 2 * t >= keys.count) s[y][0] = s[y][2] = -INFINITY;
            if (n0 + 8 * y + 2 * t + 1 >= keys.count) s[y][1] = s[y][3] = -INFINITY;
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
        own_o[row][col] = sum;
        if (col == 0) { own_m[row] = top; own_l[row] = total; }
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    // ---- the blocks' parts: each block joins a share of the values
    for (int i = rank * kDecodeWarps * 32 + threadIdx.x; i < heads * kHd; i += splits * kDecodeWarps * 32) {
        const int row = i / kHd, col = i % kHd;
        float top = -INFINITY, sum = 0.0f, total = 0.0f;
        for (int x = 0; x < splits; ++x) top = fmaxf(top, *cluster.map_shared_rank(&own_m[row], x));
        const float from = top == -INFINITY ? 0.0f : top * c;
        for (int x = 0; x < splits; ++x) {
            const float w = ex2_approx(*cluster.map_shared_rank(&own_m[row], x) * c - from);
            sum = fmaf(w, *cluster.map_shared_rank(&own_o[row][col], x), sum);
            total = fmaf(w, *cluster.map_shared_rank(&own_l[row], x), total);
        }
        if (col < p.head_dim) attn::row_to(p.out, b, 0, h0 + row)[col] = __float2bfloat16_rn(total == 0.0f ? 0.0f : sum / total);
        if (col == 0 && p.lse != nullptr)
            p.lse[static_cast<int64_t>(b) * p.heads + h0 + row] = total == 0.0f ? -INFINITY : fmaf(top, p.scale, log2f(total) * (1.0f / kLog2e));
    }
    cluster.sync();   // no block leaves while another reads its part
}

template <int CHUNKS, int ROWS>
cudaError_t launch_decode(const AttentionParams& p, int sms, cudaStream_t stream) {
    const int head_blocks = (p.group + ROWS - 1) / ROWS;
    const int64_t units = static_cast<int64_t>(p.batch) * (p.heads / p.group) * head_blocks;
    // Blocks enough for the machine, none with less than two steps for each of its warps.
    const int64_t longest = p.window + static_cast<int64_t>(p.sinks) < p.tk ? p.window + p.sinks : p.tk;
    int splits = 1;
    while (splits < 8 && units * splits < 2 * sms && longest > splits * 2 * kDecodeWarps * 32) splits *= 2;
    constexpr size_t kShared = sizeof(DecodeShared<ROWS, 64 * CHUNKS>);
    if (kShared > 48 * 1024) {
        const cudaError_t set = cudaFuncSetAttribute(attention_decode_kernel<CHUNKS, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kShared));
        if (set != cudaSuccess) return set;
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(units * splits));
    cfg.blockDim = dim3(kDecodeWarps * 32);
    cfg.dynamicSmemBytes = kShared;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, attention_decode_kernel<CHUNKS, ROWS>, p, head_blocks, splits);
    count_launch(1);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_attention_window_decode(const AttentionParams& p, int sms, cudaStream_t stream) {
    if (p.head_dim <= 64) return p.group <= 8 ? launch_decode<1, 8>(p, sms, stream) : launch_decode<1, 16>(p, sms, stream);
    return p.group <= 8 ? launch_decode<2, 8>(p, sms, stream) : launch_decode<2, 16>(p, sms, stream);
}

}  // namespace llmt_b200
